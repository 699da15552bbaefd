// matrix.hpp -- tiles of matrix products in the matrix cores, for the units that need them
// (linear_ce.hip).
//
// A workgroup forms BM x BN elements of A B^T, a step of k at a time: 64 bytes, 32 elements of 16
// bits or 16 of float.  An operand's rows run along k, or (ALONG) its memory's rows are steps of k
// and run along the rows of the product: no transposed copy is made of either.  Operands go from
// memory to LDS without passing through registers, three steps ahead of their use, into STAGES buffers.
#pragma once
#include "learn.hpp"

namespace mat {

using learn::bf16;
using learn::f16;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 64;    // bytes of a row that one step takes
constexpr int STAGES = 4;

// acc += the products of one 16-byte piece of 32 rows of either operand: lane l holds row l % 32,
// piece 2 s + l / 32 of step half s.
template <typename T> struct Mma;
template <> struct Mma<bf16> {
    static __device__ __forceinline__ void add(f32x16 &acc, u32x4 a, u32x4 b)
    {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                      __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    }
};
template <> struct Mma<f16> {
    static __device__ __forceinline__ void add(f32x16 &acc, u32x4 a, u32x4 b)
    {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                     __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    }
};
template <> struct Mma<float> {
    // (the two halves of a wave hold different k: any pairing will do, as it is the same in both)
    static __device__ __forceinline__ void add(f32x16 &acc, u32x4 a, u32x4 b)
    {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[k], y[k], acc, 0, 0, 0);
    }
};

// Element (row of A, row of B) of register r of a 32 x 32 accumulator in lane l.
__device__ __forceinline__ int acc_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }
__device__ __forceinline__ int acc_col(int lane) { return lane & 31; }

// An operand of a tile: rows [0, rows) of `base`, `pitch` bytes apart (a multiple of 16, as `base`).
// Rows past the last one read as the last one, and 16-byte pieces of a row past `k` bytes as the last
// of it.  ALONG k: `base` has `k` steps, those past the last read as the last, and `rows` elements in
// each, up to a multiple of 16 bytes.  (What is read twice meets zeros in the other operand.)
struct Operand {
    const char *base;
    int64_t pitch;
    int rows, k;
};

template <typename T, int TM_, int TN_, int WM_, int WN_> struct Tile {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int GROUPS = (BM + BN) / 16;           // of 1 KiB: one load of a wave
    // every wave loads alike (the last ones bring B's last part again, behind it)
    static constexpr int EACH = (GROUPS + WAVES - 1) / WAVES;
    static constexpr int BYTES = EACH * WAVES * 1024;       // of a stage
    static constexpr int LDS = STAGES * BYTES;
    static constexpr int KE = STEP / sizeof(T);             // elements of a step
    static_assert(LDS <= 160 * 1024, "stages fit the LDS");

    f32x16 acc[TM][TN];

    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

    static __device__ __forceinline__ const char *uniform(const char *p)
    {
        const uint64_t x = (uint64_t)p;
        return (const char *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 |
                              (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
    }

    // 1 KiB to LDS, 16 bytes a lane, in the order of the lanes.
    static __device__ __forceinline__ void fetch(uint32_t lds, uint32_t offset, const char *base)
    {
        asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
    }

    // How pieces lie in LDS: where a wave's reads want several at once they are on different banks.
    // Rows along k: 64 bytes of a row, its 16-byte pieces exchanged by the row.
    static __device__ __forceinline__ int mix_row(int row) { return row >> 1 & 3; }
    // Steps of k: W * sizeof(T) bytes of one, its 32-byte units exchanged by the step.
    template <int W> static __device__ __forceinline__ int mix_step(int k)
    {
        const int x = sizeof(T) == 2 ? (k & 3) | (k >> 1 & 4) : k & 4;
        return x & (W * (int)sizeof(T) / 32 - 1);
    }

    // Where lane l of a load finds what belongs at place g of an operand's part of a stage; steps of k
    // (pieces of it, where rows run along k) past `most` read as that one.
    template <int W, bool ALONG>
    static __device__ __forceinline__ uint32_t source(const Operand &o, int g, int lane, int most)
    {
        if constexpr (!ALONG) {
            const int r = g * 16 + (lane >> 2), row = r < o.rows ? r : o.rows - 1;
            const int piece = (lane & 3) ^ mix_row(r);
            return (uint32_t)(row * o.pitch) + ((piece < most ? piece : most) << 4);
        } else {
            constexpr int PIECES = W * sizeof(T) / 16;      // of a step
            const int at = g * 64 + lane, k = at / PIECES, slot = at % PIECES;
            const int from = k < most ? k : most;
            int piece = (((slot >> 1) ^ mix_step<W>(k)) << 1) | (slot & 1);
            const int last = (o.rows * (int)sizeof(T) + 15) / 16 - 1;
            piece = piece < last ? piece : last;
            return (uint32_t)(from * (int)o.pitch) + (piece << 4);
        }
    }

    // The part of a 32-row tile that starts at row m0 of an operand, half s of a step.
    template <int W, bool ALONG> static __device__ __forceinline__ u32x4 part(const char *x, int m0, int s, int lane)
    {
        const int half = lane >> 5;
        if constexpr (!ALONG) {
            const int r = m0 + (lane & 31);
            return *(const u32x4 *)(x + r * STEP + (((2 * s + half) ^ mix_row(r)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            // the transposing read: 16 lanes bring four steps of 16 rows, lane i keeps row i of them
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 *Ptr;
            const int k = 16 * s + 8 * half + (lane >> 2 & 3), unit = (m0 >> 4) + (lane >> 4 & 1);
            const char *const y = x + k * (W * 2) + ((unit ^ mix_step<W>(k)) << 5) + ((lane & 3) << 3);
            const uint64_t lo = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(uintptr_t)y));
            const uint64_t hi = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(uintptr_t)(y + 4 * (W * 2))));
            return (u32x4){(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
        } else {
            const int k = 4 * (2 * s + half), m = m0 + (lane & 31);
            const char *const y = x + k * (W * 4) + (((m >> 3) ^ mix_step<W>(k)) << 5) + ((m & 7) << 2);
            return (u32x4){*(const uint32_t *)y, *(const uint32_t *)(y + W * 4), *(const uint32_t *)(y + W * 8),
                           *(const uint32_t *)(y + W * 12)};
        }
    }

    template <bool AK, bool BK>
    static __device__ __forceinline__ uint32_t offset(const Operand &a, const Operand &b, int at, int lane, int most)
    {
        const int g = at < GROUPS ? at : GROUPS - 1;         // (A's places, then B's)
        return g >= BM / 16 ? source<BN, BK>(b, g - BM / 16, lane, most) : source<BM, AK>(a, g, lane, most);
    }

    // acc += A[., k] B[., k] for steps [first, last).
    template <bool AK = false, bool BK = false>
    __device__ __forceinline__ void run(char *lds, const Operand &a, const Operand &b, int first, int last)
    {
        if (first >= last) return;
        const int lane = threadIdx.x & 63, w = wave();
        constexpr int GA = BM / 16;
        uint32_t off[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            off[e] = offset<AK, BK>(a, b, w * EACH + e, lane, KE);
        }
        const int64_t step_a = AK ? KE * a.pitch : STEP, step_b = BK ? KE * b.pitch : STEP;
        const char *pa = uniform(a.base + first * step_a), *pb = uniform(b.base + first * step_b);
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
        const int n = __builtin_amdgcn_readfirstlane(last - first);
        int at = __builtin_amdgcn_readfirstlane(first), ahead = 0;
        auto load = [&](int stage) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const bool isb = w * EACH + e >= GA;
                uint32_t o = off[e];
                const int most_a = AK ? a.k - 1 - at * KE : (a.k >> 4) - 1 - at * (STEP / 16);
                const int most_b = BK ? b.k - 1 - at * KE : (b.k >> 4) - 1 - at * (STEP / 16);
                if ((isb ? most_b : most_a) < (isb ? (BK ? KE : STEP / 16) : (AK ? KE : STEP / 16)) - 1)
                    o = offset<AK, BK>(a, b, w * EACH + e, lane, isb ? most_b : most_a);
                fetch(__builtin_amdgcn_readfirstlane(lds0 + stage * BYTES + (w * EACH + e) * 1024), o, isb ? pb : pa);
            }
            // (past the end the last step is brought again, into a buffer that nothing reads)
            if (++ahead < n) {
                pa += step_a;
                pb += step_b;
                ++at;
            }
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) load(s);
        const int wm = w / WN, wn = w % WN;
        int stage = 0;
        for (int k = 0; k < n; ++k) {
            // this wave's part of step k has come; then everybody's has, and nobody reads step k - 1
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(EACH * (STAGES - 2)) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            // Both halves' parts are asked for before the first product: left to itself the compiler keeps
            // one part at a time and waits for each.
            const char *const x = lds + stage * BYTES;
            u32x4 fa[2][TM], fb[2][TN];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[s][j] = part<BN, BK>(x + BM * STEP, (wn * TN + j) * 32, s, lane);
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[s][i] = part<BM, AK>(x, (wm * TM + i) * 32, s, lane);
                __builtin_amdgcn_sched_barrier(0);
            }
            load(stage == 0 ? STAGES - 1 : stage - 1);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) Mma<T>::add(acc[i][j], fa[s][i], fb[s][j]);
            __builtin_amdgcn_s_setprio(0);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        // nothing is in flight to the LDS, and nobody reads it, when this returns
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
    }

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    }
};

// Which tile a workgroup takes: workgroups go round the eight dies (each with an L2 of its own) one
// by one, so each die is given a stretch of the tiles, in groups of eight rows of tiles that share
// their B operand while it is in L2.
__device__ __forceinline__ void tile_of(int block, int blocks, int nm, int nn, int &m, int &n)
{
    const int die = block & 7, each = blocks >> 3, more = blocks & 7;
    int t = die * each + (die < more ? die : more) + (block >> 3);
    const int per = 8 * nn, group = t / per;
    const int first = group * 8, size = nm - first < 8 ? nm - first : 8;
    t -= group * per;
    m = first + t % size;
    n = t / size;
}

}  // namespace mat
