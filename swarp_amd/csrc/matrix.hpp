// matrix.hpp -- tiles of matrix products in the matrix cores, for the units that need them
// (linear_ce.hip).
//
// A workgroup forms BM x BN elements of A B^T from operands whose rows run along k (in bytes:
// 64 of a row and operand a step, 32 elements of 16 bits or 16 of float).  Operands go from memory
// to LDS without passing through registers, three steps ahead of their use, into STAGES buffers.
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
// Rows past the last one read as the last one.
struct Operand {
    const char *base;
    int64_t pitch;
    int rows;
};

template <typename T, int TM_, int TN_, int WM_, int WN_> struct Tile {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int GROUPS = (BM + BN) / 16;           // of 16 rows: one load of a wave
    // every wave loads alike (the last ones bring B's last rows again, behind them)
    static constexpr int EACH = (GROUPS + WAVES - 1) / WAVES;
    static constexpr int BYTES = EACH * WAVES * 16 * STEP;  // of a stage
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

    // 16 rows of 64 bytes to LDS: lane l brings row l / 4, piece (l % 4) ^ (row / 2 % 4), which puts
    // the pieces that a wave's reads want at once (8 rows, one piece) on different banks.
    static __device__ __forceinline__ void fetch(uint32_t lds, uint32_t offset, const char *base)
    {
        asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
    }

    // acc += A[., k] B[., k] for steps [first, last).
    __device__ __forceinline__ void run(char *lds, const Operand &a, const Operand &b, int first, int last)
    {
        if (first >= last) return;
        const int lane = threadIdx.x & 63, w = wave();
        uint32_t off[EACH];
        const char *pa = uniform(a.base + (int64_t)first * STEP), *pb = uniform(b.base + (int64_t)first * STEP);
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int at = w * EACH + e, g = at < GROUPS ? at : GROUPS - 1;  // (A's groups, then B's)
            const bool isb = g >= BM / 16;
            const Operand &o = isb ? b : a;
            const int r = (isb ? g - BM / 16 : g) * 16 + (lane >> 2);
            const int row = r < o.rows ? r : o.rows - 1;
            off[e] = (uint32_t)(row * o.pitch) + (((lane & 3) ^ (r >> 1 & 3)) << 4);
        }
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
        const int n = __builtin_amdgcn_readfirstlane(last - first);
        int ahead = 0;
        auto load = [&](int stage) {
#pragma unroll
            for (int e = 0; e < EACH; ++e)
                fetch(__builtin_amdgcn_readfirstlane(lds0 + stage * BYTES + (w * EACH + e) * 1024), off[e],
                      w * EACH + e >= BM / 16 ? pb : pa);
            // (past the end the last step is brought again, into a buffer that nothing reads)
            if (++ahead < n) {
                pa += STEP;
                pb += STEP;
            }
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) load(s);
        const int wm = w / WN, wn = w % WN;
        const int ra = wm * TM * 32 + (lane & 31), rb = BM + wn * TN * 32 + (lane & 31);
        int stage = 0;
        for (int k = 0; k < n; ++k) {
            // this wave's part of step k has come; then everybody's has, and nobody reads step k - 1
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(EACH * (STAGES - 2)) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            load(stage == 0 ? STAGES - 1 : stage - 1);
            const char *const x = lds + stage * BYTES;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 fa[TM], fb[TN];
                const int piece = 2 * s + (lane >> 5);
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    fa[i] = *(const u32x4 *)(x + (ra + 32 * i) * STEP + ((piece ^ (ra >> 1 & 3)) << 4));
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    fb[j] = *(const u32x4 *)(x + (rb + 32 * j) * STEP + ((piece ^ (rb >> 1 & 3)) << 4));
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) Mma<T>::add(acc[i][j], fa[i], fb[j]);
            }
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
