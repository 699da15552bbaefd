// decay.hip -- linear attention with a decay for each head, along a rollout (swarp_decay_fwd,
// swarp_decay_bwd, swarp_decay_step).
//
// Per batch entry and head, with the state S [dk, dv] and lambda = exp(log_decay):
//   S_t = (starts_t ? 0 : lambda S_{t-1}) + k_t v_t^T,   o_t = scale q_t S_t.
// Over a chunk of 32 steps that S enters (0 <= t, i < 32, both of one episode where they meet):
//   o_t = scale (sum_{i <= t} lambda^(t-i) (q_t k_i) v_i + lambda^(t+1) q_t S),
//   S' = lambda^32 S + sum_i lambda^(31-i) k_i v_i^T:
// four small matrix products, all powers at most 1.
//
// The gradients are scans of the same kind with the parts exchanged:
//   dq_t = scale sum_{i <= t} lambda^(t-i) (do_t v_i) k_i + ...     forwards,  (do, v, k), state S^T
//   dk_i = scale sum_{t >= i} lambda^(t-i) (v_i do_t) q_t + ...     backwards, (v, do, q), state dS^T
//   dv_i = scale sum_{t >= i} lambda^(t-i) (k_i q_t) do_t + ...     backwards, (k, q, do), state dS
// so that one kernel does all four; below, q, k and v are a scan's own parts.
//
// Where there are fewer heads than SIMDs the steps are cut into segments: one kernel finds the state that each
// would end with if none entered, a second joins them, a third does the segments, each from its state.
#include <math.h>

#include "parts.hpp"

namespace {

using namespace learn;
using namespace part;

constexpr int BLOCK = 256, WAVES = BLOCK / 64;
constexpr int CHUNK = 32;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int MOST_DIM = 128, MOST_HEADS = 1 << 22;

// One of a call's scans.
struct Scan {
    const void *q, *k, *v;
    void *out;
    int64_t qs[3], ks[3], vs[3], os[3];  // elements: step, batch, head
    int dk, dv;                          // of this scan
    int back;                            // from the last step to the first
    int slices, first;                   // of 32 columns of v; where they lie among those of all scans
    int64_t spans;                       // k_together: a workgroup takes every spans-th four heads
    float score, grow, carry;            // factors of the scores, of k v^T in the state, of q S in the output
    const float *state;                  // before the first step, or NULL; element (i, j) at i si + j sj of a head's
    float *state_out;                    // after the last, or NULL
    int si, sj;
    float *between;                      // [segments][batch heads][area]: states that segments end with (ENDS)
    int32_t *cut;                        // or start with (k_between); [segments][batch heads]: no state gets through
};

struct Call {
    Scan scan[3];
    int scans, slices;     // slices of all scans
    int64_t spans;         // k_alone: a wave takes every spans-th batch entry: those at work at once are neighbours
    int segments, chunks;  // of the steps, and chunks of a segment
    int64_t units;         // batch * heads * segments * slices: what one state goes through
    int64_t steps, batch, group;
    int heads, area;       // area: dk dv of a state
    const float *log_decay;
    const uint8_t *starts;
    uint8_t *wrong;        // [units]: something was not finite
};

// What a wave does: the outputs of a segment, or (ENDS) the state that it ends with if none enters.
enum { OUTPUTS, ENDS };

// What a wave keeps of a head from chunk to chunk: the state's columns -- element
// (32 t + 16 (r / 8) + 8 half + r % 8, j) in register r of tile t --, whether it is still zero, and a number
// that is 0 as long as its outputs and the state that it leaves are finite.  A product with 0 is not 0 where a
// part, a score or the state (of finite parts, past the largest float) is not finite; that always shows
// in an output of the chunk or in the leaving state, and the head is done again by k_exact.
template <int KT> struct Kept {
    f32x16 S[KT];
    bool none;
    float odd;
};
// Powers of a head's decay: between the steps of a lane's scores, from the state to a lane's step, from a
// step to the leaving state, and over the chunk.
struct Powers {
    float D[16], w0, u[16], whole;
    int width;  // of the chunk that u and whole are for

    __device__ __forceinline__ void set(const Scan &s, float a2, int col, int half)
    {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = 16 * (r >> 3) + 8 * half + (r & 7);
            D[r] = col >= i ? s.score * __builtin_amdgcn_exp2f(a2 * (float)(col - i)) : 0.0f;
        }
        w0 = s.carry * __builtin_amdgcn_exp2f(a2 * (float)(col + (s.back ? 0 : 1)));
        width = 0;
    }
    __device__ __forceinline__ void over(const Scan &s, float a2, int half, int L)
    {
        if (L == width) return;
        width = L;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = 16 * (r >> 3) + 8 * half + (r & 7);
            u[r] = i < L ? s.grow * __builtin_amdgcn_exp2f(a2 * (float)(L - 1 - i + (s.back ? 1 : 0))) : 0.0f;
        }
        whole = __builtin_amdgcn_exp2f(a2 * (float)L);
    }
};
__device__ __forceinline__ float decay_of(const Call &c, int h)
{
    const float a2 = c.log_decay[h] * LOG2E;
    return a2 < -1e30f ? -1e30f : a2;  // (-inf times 0 steps is no decay)
}

// The state that enters a segment; and the one that leaves it, if it is wanted.
template <int KT, int WHAT, int FIT>
__device__ __forceinline__ void enter(const Call &c, const Scan &s, int64_t bh, int segment, bool at_work, int half, int j, Kept<KT> &w)
{
    const float *from = WHAT == ENDS || !at_work ? nullptr
                        : segment                ? s.between + ((int64_t)segment * c.batch * c.heads + bh) * c.area
                        : s.state                ? s.state + bh * c.area
                                                 : nullptr;
    int rest = s.dk - 8 * half;  // (worked out at the place, not kept in registers throughout)
    asm volatile("" : "+v"(rest));
    if (from) from += (int64_t)(8 * half) * s.si + (int64_t)j * s.sj;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = 32 * t + 16 * (r >> 3) + (r & 7);
            w.S[t][r] = from && (FIT == FULL || (i < rest && j < s.dv)) ? from[i * s.si] : 0.0f;
        }
    w.none = !from;
    w.odd = 0.0f;
}
// odd + 0 times what a tile holds: not 0 where some of it is not finite.
__device__ __forceinline__ float odd_of(const f32x16 &x, float odd)
{
#pragma unroll
    for (int r = 0; r < 16; ++r) odd = __builtin_fmaf(x[r], 0.0f, odd);
    return odd;
}
template <int KT, int WHAT, int FIT>
__device__ __forceinline__ void leave(const Call &c, const Scan &s, int64_t bh, int segment, bool ends, int lane, int j, int slice,
                                      Kept<KT> &w, bool any)
{
    const int half = lane >> 5;
    float *to = WHAT == ENDS        ? s.between + ((int64_t)segment * c.batch * c.heads + bh) * c.area
                : ends && s.state_out ? s.state_out + bh * c.area
                                      : nullptr;
    if (to) {
        int rest = s.dk - 8 * half;
        asm volatile("" : "+v"(rest));
        to += (int64_t)(8 * half) * s.si + (int64_t)j * s.sj;
        // (backwards: what an episode that starts with the first step leaves of the state before it)
        const bool clear = WHAT == OUTPUTS && s.back && c.starts && c.steps > 0 &&
                           c.starts[(uint32_t)bh / (uint32_t)c.heads / (uint32_t)c.group];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = 32 * t + 16 * (r >> 3) + (r & 7);
                if (FIT == FULL || (i < rest && j < s.dv)) to[i * s.si] = clear ? 0.0f : w.S[t][r];
            }
    }
    if (WHAT == OUTPUTS) {
        if (to) {
#pragma unroll
            for (int t = 0; t < KT; ++t) w.odd = odd_of(w.S[t], w.odd);
        }
        const bool wrong = __ballot(!(w.odd == 0.0f)) != 0;
        if (lane == 0) c.wrong[(bh * c.segments + segment) * c.slices + s.first + slice] = wrong;
    } else if (lane == 0) s.cut[(int64_t)segment * c.batch * c.heads + bh] = any;
}

// A chunk of a head: from its scores p, q's parts and the rows of k and v in LDS, the outputs o of 32
// columns from j0 on (lane: step; register: column, as the state's rows) and the state after it.
template <typename T, int KT, int WHAT>
__device__ __forceinline__ void chunk(Kept<KT> &w, const Powers &f, const Part<T> (&qf)[2 * KT], f32x16 p, const T *kx, int kp,
                                      const T *vx, int vp, int j0, uint32_t cut, bool goes_on, int lane, f32x16 &o)
{
    const int half = lane >> 5, col = lane & 31;
    f32x16(&S)[KT] = w.S;
    bool &none = w.none;
    Part<T> vf[2];
    vf[0] = column_of<T>(vx, vp, 0, j0, lane);
    vf[1] = column_of<T>(vx, vp, 16, j0, lane);
    Part<T> pf[2], pl[2];
    if (WHAT == OUTPUTS) {
        const uint32_t upto = cut & (0xffffffffu >> (31 - col));
        const int since = upto ? 31 - __clz(upto) : 0;  // first step that enters step `col`
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= f.D[r];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float y[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) y[r] = p[8 * x + r];
            if (cut) {
#pragma unroll
                for (int r = 0; r < 8; ++r) y[r] = 16 * x + 8 * half + r >= since ? y[r] : 0.0f;
            }
            pf[x] = term_of<T>(y, true);
            if (Part<T>::TERMS) pl[x] = term_of<T>(y, false);
        }
    }
    if (WHAT == OUTPUTS) {
        o = {};
        if (!none) {
#pragma unroll
            for (int x = 0; x < 2 * KT; ++x) {
                float y[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) y[r] = S[x >> 1][8 * (x & 1) + r];
                mma<T>(o, term_of<T>(y, true), qf[x]);
                if (Part<T>::TERMS) mma<T>(o, term_of<T>(y, false), qf[x]);
            }
            const float g = cut & (0xffffffffu >> (31 - col)) ? 0.0f : f.w0;
#pragma unroll
            for (int r = 0; r < 16; ++r) o[r] *= g;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            mma<T>(o, vf[x], pf[x]);
            if (Part<T>::TERMS) mma<T>(o, vf[x], pl[x]);
        }
        w.odd = odd_of(o, w.odd);
    }
    if (goes_on) {
        const int kept = cut ? 31 - __clz(cut) : 0;  // first step that enters the leaving state
        if (!none) {
            const float g = cut ? 0.0f : f.whole;
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[t][r] *= g;
        }
        none = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float y[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) y[r] = element(vf[x], r) * f.u[8 * x + r];
            if (cut) {
#pragma unroll
                for (int r = 0; r < 8; ++r) y[r] = 16 * x + 8 * half + r >= kept ? y[r] : 0.0f;
            }
            Part<T> z[3];
            z[0] = term_of<T>(y, true);
            if (Part<T>::TERMS) {
                z[1] = term_of<T>(y, true);
                z[2] = term_of<T>(y, false);
            }
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const Part<T> kc = column_of<T>(kx, kp, 16 * x, 32 * t, lane);
                mma<T>(S[t], kc, z[0]);
                if (Part<T>::TERMS) {
                    mma<T>(S[t], kc, z[1]);
                    mma<T>(S[t], kc, z[2]);
                }
            }
        }
    }
}

// One wave: one head, 32 columns of v, the steps of a segment, for some batch entries in turn.  The
// state's columns stay in its registers; KT: 32s of dk.  A wave works alone: its part of the LDS
// holds the chunk's rows of k and v, to be read as columns.  The next chunk's rows (the next entry's
// first ones) are on their way meanwhile.
// What bounds it is one wave's chain through a chunk (rows to LDS, scores, output, state: some 40 products of
// 32 x 32 x 16 behind one another, two waves a SIMD): 4095 steps of 384 heads of 64, bfloat16, forward and
// backward 1.22 ms, 0.4 of it bytes; 1023 steps of 256 heads of 40 x 72, float32, 0.77 ms, 0.13 of it bytes.
template <typename T, int KT, int WHAT, int FIT>
__global__ __launch_bounds__(BLOCK, (KT + (WHAT == OUTPUTS)) * sizeof(T) < 10 ? 2 : 1) void k_alone(const Call c)
{
    constexpr int KP = 32 * KT + 16 / (int)sizeof(T), VP = 32 + 16 / (int)sizeof(T);
    __shared__ __align__(16) T room[WAVES][32 * (KP + VP)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    T *const kx = room[wave], *const vx = kx + 32 * KP;
    // (neighbouring waves have neighbouring columns, then segments, then heads)
    const uint32_t kinds = (uint32_t)(c.slices * c.heads * c.segments);
    const int64_t number = (int64_t)blockIdx.x * WAVES + wave, span = number / kinds;
    const uint32_t kind = (uint32_t)(number - span * kinds), lines = kind / (uint32_t)c.slices;
    const int h = (int)(lines / (uint32_t)c.segments), segment = (int)(lines % (uint32_t)c.segments);
    int64_t b = span;
    if (b >= c.spans) return;
    int slice = (int)(kind % (uint32_t)c.slices), which = 0;
    while (slice >= c.scan[which].slices) slice -= c.scan[which++].slices;
    const Scan &s = c.scan[which];
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, perm = swapped(col);
    const bool back = s.back;
    const int64_t steps = c.steps, origin = back ? steps - 1 : 0, way = back ? -1 : 1;
    const int64_t qt = way * s.qs[0], kt = way * s.ks[0], vt = way * s.vs[0], ot = way * s.os[0];
    const int64_t begin = (int64_t)segment * c.chunks * CHUNK;
    const int64_t end = begin + (int64_t)c.chunks * CHUNK < steps ? begin + (int64_t)c.chunks * CHUNK : steps;
    const int dk = s.dk, dv = s.dv, j0 = 32 * slice, j = j0 + perm;
    const uint32_t group = (uint32_t)c.group;
    const int64_t groups = c.batch / c.group;
    const bool ends = end == steps;  // the last segment

    const float a2 = decay_of(c, h);
    Powers f;
    f.set(s, a2, col, half);

    // Rows as they lie in memory: q by lane, k by swapped lane, v by quarters of rows; and whether
    // anything enters a lane's step.  Where a row or a step is past the end the last one is read
    // again: only q has to be zero past dk, what else it brings meets a zero (of q, of D, of u) or is
    // not written.
    Raw<T> qr[2 * KT], kr[2 * KT], vr[2];
    uint8_t sr = 0;
    const T *qb = (const T *)s.q + h * s.qs[2] + origin * s.qs[0] + b * s.qs[1] + (begin + col) * qt;
    const T *kb = (const T *)s.k + h * s.ks[2] + origin * s.ks[0] + b * s.ks[1] + (begin + perm) * kt;
    const T *vb = (const T *)s.v + h * s.vs[2] + origin * s.vs[0] + b * s.vs[1] + (begin + (lane >> 2)) * vt;
    T *ob = (T *)s.out + h * s.os[2] + origin * s.os[0] + b * s.os[1] + (begin + col) * ot + j0 + 8 * half;
    const T *qp = qb, *kp = kb, *vp = vb;
    auto starts_of = [&](int64_t b) {
        return c.starts + (uint32_t)b / group + (back ? steps - (begin + col) : begin + col) * groups;
    };
    const uint8_t *sp = c.starts ? starts_of(b) : nullptr;
    auto load = [&](int64_t c0) {
        const int L = (int)(end - c0 < CHUNK ? end - c0 : CHUNK);
        const T *x = qp, *y = kp, *z[2] = {vp, vp + 16 * vt};
        if (L < CHUNK) {
            x -= (col < L ? 0 : col - (L - 1)) * qt;
            y -= (perm < L ? 0 : perm - (L - 1)) * kt;
#pragma unroll
            for (int t = 0; t < 2; ++t) z[t] -= (16 * t + (lane >> 2) < L ? 0 : 16 * t + (lane >> 2) - (L - 1)) * vt;
        }
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
            if (WHAT == OUTPUTS) qr[t] = row_of<T, FIT>(x, 16 * t + 8 * half, dk, 16 * t + 16 > dk);
            kr[t] = row_of<T, FIT>(y, 16 * t + 8 * half, dk, false);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) vr[t] = row_of<T, FIT>(z[t], j0 + 8 * (lane & 3), dv, false);
        if (sp) {
            sr = 0;
            if (col < L && (!back || c0 + col > 0)) sr = *sp;
        }
    };
    if (begin < end) load(begin);
    for (; b < c.batch; b += c.spans) {
        const int64_t bh = b * c.heads + h;
        Kept<KT> w;
        enter<KT, WHAT, FIT>(c, s, bh, segment, true, half, j, w);
        uint32_t any = 0;
        T *op = ob;
        for (int64_t c0 = begin; c0 < end; c0 += CHUNK) {
            const int L = (int)(end - c0 < CHUNK ? end - c0 : CHUNK);
            const bool more = c0 + CHUNK < end;
            f.over(s, a2, half, L);
            // steps that nothing before them enters
            const uint32_t cut = (uint32_t)__ballot(sr);
            any |= cut;
            // the rows of k and v into LDS
#pragma unroll
            for (int t = 0; t < 2 * KT; ++t) *(Raw<T> *)(kx + perm * KP + 16 * t + 8 * half) = kr[t];
#pragma unroll
            for (int t = 0; t < 2; ++t) *(Raw<T> *)(vx + (16 * t + (lane >> 2)) * VP + 8 * (lane & 3)) = vr[t];
            Part<T> qf[2 * KT];
            f32x16 p = {};
            if (WHAT == OUTPUTS) {
#pragma unroll
                for (int t = 0; t < 2 * KT; ++t) {
                    qf[t] = part_of(qr[t]);
                    mma<T>(p, part_of(kr[t]), qf[t]);
                }
            }
            if (more) {
                qp += CHUNK * qt;
                kp += CHUNK * kt;
                vp += CHUNK * vt;
                if (sp) sp += CHUNK * way * groups;
            } else {
                qp = qb += c.spans * s.qs[1];
                kp = kb += c.spans * s.ks[1];
                vp = vb += c.spans * s.vs[1];
                if (sp) sp = starts_of(b + c.spans);
            }
            if (more || b + c.spans < c.batch) load(more ? c0 + CHUNK : begin);
            f32x16 o;
            chunk<T, KT, WHAT>(w, f, qf, p, kx, KP, vx, VP, 0, cut, WHAT == ENDS || more || (ends && s.state_out), lane, o);
            if (WHAT == OUTPUTS && col < L) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int n = dv - j0 - 8 * half - 16 * x;
                    Span<T, 8> e;
#pragma unroll
                    for (int r = 0; r < 8; ++r) e.e[r] = (T)o[8 * x + r];
                    if (FIT == FULL || (FIT == EIGHTS ? n > 0 : n >= 8)) *(Span<T, 8> *)(op + 16 * x) = e;
                    else if constexpr (FIT <= ANY) {
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (r < n) op[16 * x + r] = e.e[r];
                    }
                }
            }
            op += CHUNK * ot;
        }
        ob += c.spans * s.os[1];
        leave<KT, WHAT, FIT>(c, s, bh, segment, ends, lane, j, slice, w, any != 0);
    }
}

// The same for heads up to 32 wide: a workgroup brings the rows of its four heads into LDS together.
// Heads and batch entries next to each other lie next to each other in memory, so that a load takes
// few rows of many bytes.  (A rollout's steps are far apart: 32
// rows a load are 32 pages, and translations then cost more than the bytes.)  Its outputs leave the
// same way.  The next chunk's rows, or the next heads' first ones, are on their way meanwhile.
// 32 steps of 512000 heads of 32, bfloat16: 6.3 GB in 1.5 ms, 4.2 TB/s.
template <typename T, int WHAT, int FIT>
__global__ __launch_bounds__(BLOCK, 2) void k_together(const Call c)
{
    constexpr int PAD = 16 / (int)sizeof(T), P = 32 + PAD, ROOM = WAVES * 32 * P;
    constexpr int EACH = 2;  // pieces of q, k or v that a thread brings
    __shared__ __align__(16) T room[(WHAT == OUTPUTS ? 4 : 2) * ROOM];
    T *const kx = room, *const vx = kx + ROOM, *const qx = vx + ROOM, *const ox = qx + ROOM;
    const uint32_t index = blockIdx.x / (uint32_t)c.scans;
    const Scan &s = c.scan[blockIdx.x % (uint32_t)c.scans];
    const int segment = (int)(index % (uint32_t)c.segments);
    int64_t group = index / (uint32_t)c.segments;     // of four heads
    if (group >= s.spans) return;
    const int mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t lines = c.batch * c.heads, groups = (lines + WAVES - 1) / WAVES;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, perm = swapped(col);
    const bool back = s.back;
    const int64_t steps = c.steps, origin = back ? steps - 1 : 0, way = back ? -1 : 1;
    const int64_t begin = (int64_t)segment * c.chunks * CHUNK;
    const int64_t end = begin + (int64_t)c.chunks * CHUNK < steps ? begin + (int64_t)c.chunks * CHUNK : steps;
    const int dk = s.dk, dv = s.dv;
    const bool ends = end == steps;  // the last segment
    // (a workgroup's next heads are a whole number of batch entries on: a wave's h is always the same)
    const uint32_t line0 = (uint32_t)(group * WAVES + mine);
    const int h = (int)(line0 % (uint32_t)c.heads);
    const int64_t far = s.spans * WAVES / c.heads;

    const float a2 = decay_of(c, h);
    Powers f;
    f.set(s, a2, col, half);

    // A thread's pieces, of eight elements, in the order row, head, place.  Where a step is past the end
    // the last one is read again: q is zero past dk, and what else that brings meets a zero (of q, of
    // D, of u) or is not written.
    struct Piece {
        int row, head, at;
    };
    auto piece = [](int n) {
        const int x = n * BLOCK + (int)threadIdx.x;
        return Piece{x >> 4, x >> 2 & 3, 8 * (x & 3)};
    };
    auto entry = [&](const int64_t (&st)[3], const Piece &y) {  // (elements to a piece's first step)
        const uint32_t line = (uint32_t)(group * WAVES + y.head);
        const uint32_t b = line / (uint32_t)c.heads;
        return (int64_t)b * st[1] + (int64_t)(line - b * (uint32_t)c.heads) * st[2] + (origin + way * (begin + y.row)) * st[0];
    };
    const T *qb[EACH], *kb[EACH], *vb[EACH];
    T *ob[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
        if (WHAT == OUTPUTS) {
            qb[n] = (const T *)s.q + entry(s.qs, piece(n));
            ob[n] = (T *)s.out + entry(s.os, piece(n)) + piece(n).at;
        }
        kb[n] = (const T *)s.k + entry(s.ks, piece(n));
        vb[n] = (const T *)s.v + entry(s.vs, piece(n));
    }
    Raw<T> qr[EACH], kr[EACH], vr[EACH];
    uint8_t sr = 0;  // whether nothing before it enters a lane's step
    auto load = [&](int64_t c0, int64_t group, int64_t skip) {
        const int L = (int)(end - c0 < CHUNK ? end - c0 : CHUNK);
        const int64_t t = way * (c0 - begin);
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const Piece y = piece(n);
            const int64_t yt = t - way * (y.row < L ? 0 : y.row - (L - 1));
            if (group * WAVES + y.head < lines) {
                if (WHAT == OUTPUTS) qr[n] = row_of<T, FIT>(qb[n] + skip * s.qs[1] + yt * s.qs[0], y.at, dk, true);
                kr[n] = row_of<T, FIT>(kb[n] + skip * s.ks[1] + yt * s.ks[0], y.at, dk, false);
                vr[n] = row_of<T, FIT>(vb[n] + skip * s.vs[1] + yt * s.vs[0], y.at, dv, false);
            }
        }
        if (c.starts) {
            sr = 0;
            const int64_t line = group * WAVES + mine, x = c0 + col;
            if (col < L && (!back || x > 0) && line < lines)
                sr = c.starts[(back ? steps - x : x) * (c.batch / c.group) + (uint32_t)((uint32_t)line / (uint32_t)c.heads) / (uint32_t)c.group];
        }
    };
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
        qr[n] = {};
        kr[n] = {};
        vr[n] = {};
    }
    if (begin < end) load(begin, group, 0);
    for (; group < groups; group += s.spans) {
        const int64_t bh = group * WAVES + mine;
        const bool at_work = bh < lines;  // (the same for a wave)
        Kept<1> w;
        enter<1, WHAT, FIT>(c, s, bh, segment, at_work, half, perm, w);
        uint32_t any = 0;
        for (int64_t c0 = begin; c0 < end; c0 += CHUNK) {
            const int L = (int)(end - c0 < CHUNK ? end - c0 : CHUNK);
            const bool more = c0 + CHUNK < end;
            f.over(s, a2, half, L);
            // steps that nothing before them enters
            const uint32_t cut = (uint32_t)__ballot(sr);
            any |= cut;
            // rows into LDS
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                const Piece y = piece(n);
                const int at = (y.head * 32 + y.row) * P + y.at;
                if (WHAT == OUTPUTS) *(Raw<T> *)(qx + at) = qr[n];
                *(Raw<T> *)(kx + at) = kr[n];
                *(Raw<T> *)(vx + at) = vr[n];
            }
            __syncthreads();
            if (more) load(c0 + CHUNK, group, 0);
            else if (group + s.spans < groups) load(begin, group + s.spans, far);
            if (at_work) {
                const T *const kw = kx + mine * 32 * P, *const vw = vx + mine * 32 * P;
                Part<T> qf[2];
                f32x16 p = {}, o;
                if (WHAT == OUTPUTS) {
                    const T *const qw = qx + (mine * 32 + col) * P + 8 * half, *const kr = kw + perm * P + 8 * half;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        qf[t] = part_of(*(const Raw<T> *)(qw + 16 * t));
                        mma<T>(p, part_of(*(const Raw<T> *)(kr + 16 * t)), qf[t]);
                    }
                }
                chunk<T, 1, WHAT>(w, f, qf, p, kw, P, vw, P, 0, cut, WHAT == ENDS || more || (ends && s.state_out), lane, o);
                if (WHAT == OUTPUTS) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        Span<T, 8> e;
#pragma unroll
                        for (int r = 0; r < 8; ++r) e.e[r] = (T)o[8 * x + r];
                        *(Raw<T> *)(ox + (mine * 32 + col) * P + 16 * x + 8 * half) = __builtin_bit_cast(Raw<T>, e);
                    }
                }
            }
            __syncthreads();
            if (WHAT == OUTPUTS) {
#pragma unroll
                for (int n = 0; n < EACH; ++n) {
                    const Piece z = piece(n);
                    if (z.row >= L || group * WAVES + z.head >= lines) continue;
                    const Span<T, 8> e = __builtin_bit_cast(Span<T, 8>, *(const Raw<T> *)(ox + (z.head * 32 + z.row) * P + z.at));
                    T *const to = ob[n] + way * (c0 - begin) * s.os[0];
                    const int left = dv - z.at;
                    if (FIT == FULL || (FIT == EIGHTS ? left > 0 : left >= 8)) *(Span<T, 8> *)to = e;
                    else if constexpr (FIT <= ANY) {
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (r < left) to[r] = e.e[r];
                    }
                }
            }
        }
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            if (WHAT == OUTPUTS) {
                qb[n] += far * s.qs[1];
                ob[n] += far * s.os[1];
            }
            kb[n] += far * s.ks[1];
            vb[n] += far * s.vs[1];
        }
        if (at_work) leave<1, WHAT, FIT>(c, s, bh, segment, ends, lane, perm, 0, w, any != 0);
    }
}

// All gradients of heads up to 32 wide over at most 32 steps, where one chunk is all: q, k, v and do are
// read once.  As k_together a workgroup has four heads, whose rows it brings and writes together; a
// wave then works on its head alone.  With the powers w_ti (0 across an end of an episode),
//   dP_ti = w_ti (do_t v_i), P_ti = w_ti (q_t k_i):  dq = dP k,  dk = dP^T q,  dv = P^T do,
// and with the state S0 before the first step and the gradient Z of the one after the last
//   dq_t += lambda^(t+1) S0 do_t,  dk_i += lambda^(T-1-i) Z v_i,  dv_i += lambda^(T-1-i) Z^T k_i,
//   d S0 = lambda^T Z + sum_t lambda^(t+1) q_t do_t^T.
// dP is formed twice, with a lane's step that of dq and that of dk: either way it is the next product's
// operand as it lies.
// 32 steps of 512000 heads of 32, bfloat16: 1.74 ms for 7.3 GB; as three scans it was 3.1 ms for twice the bytes.
// Bounds: the bytes, then what two waves a SIMD leave uncovered of the way from LDS to the products.
template <typename T, int FIT> __global__ __launch_bounds__(BLOCK, 2) void k_short(const Call c, const Scan sq, const Scan sk, const Scan sv)
{
    constexpr int PAD = 16 / (int)sizeof(T), P = 32 + PAD, ROOM = WAVES * 32 * P, EACH = 2;
    __shared__ __align__(16) T room[4 * ROOM];
    const int mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t lines = c.batch * c.heads, groups = (lines + WAVES - 1) / WAVES;
    int64_t group = blockIdx.x;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, perm = swapped(col);
    const int L = (int)c.steps, dk = sq.dv, dv = sq.dk;
    const int h = (int)((uint32_t)(group * WAVES + mine) % (uint32_t)c.heads);
    const float a2 = decay_of(c, h);
    // powers from step i = register to step t = lane (D), from step i = lane to step t = register (E)
    float D[16], E[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = 16 * (r >> 3) + 8 * half + (r & 7);
        D[r] = col >= i ? sq.score * __builtin_amdgcn_exp2f(a2 * (float)(col - i)) : 0.0f;
        E[r] = i >= col && i < L ? sq.score * __builtin_amdgcn_exp2f(a2 * (float)(i - col)) : 0.0f;
    }
    const float first = sq.carry * __builtin_amdgcn_exp2f(a2 * (float)(col + 1)), last = __builtin_amdgcn_exp2f(a2 * (float)(L - 1 - col));

    // pieces as in k_together: q, k, v, do in, dq, dk, dv out
    struct Array {
        const void *p;
        const int64_t *st;
        int n;
    };
    const Array in[4] = {{sk.v, sk.vs, dk}, {sq.v, sq.vs, dk}, {sq.k, sq.ks, dv}, {sq.q, sq.qs, dv}};
    const Array to[3] = {{sv.out, sv.os, dv}, {sk.out, sk.os, dk}, {sq.out, sq.os, dk}};  // where q, k, v were
    Raw<T> raw[4][EACH];
    uint8_t sr = 0;
    auto load = [&](int64_t group) {
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            int x = n * BLOCK + (int)threadIdx.x;
            asm volatile("" : "+v"(x));
            const int row = (x >> 4) < L ? x >> 4 : L - 1, at = 8 * (x & 3);
            const uint32_t line = (uint32_t)(group * WAVES + (x >> 2 & 3)), b = line / (uint32_t)c.heads;
            if (line >= lines) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const T *const y = (const T *)in[k].p + row * in[k].st[0] + b * in[k].st[1] + (line - b * (uint32_t)c.heads) * in[k].st[2];
                // (q and do are zero past their ends: what k, v and columns bring there meets them)
                raw[k][n] = row_of<T, FIT>(y, at, in[k].n, true);
            }
        }
        const int64_t line = group * WAVES + mine;
        sr = 0;
        if (c.starts && col < L && line < lines)
            sr = c.starts[col * (c.batch / c.group) + (uint32_t)line / (uint32_t)c.heads / (uint32_t)c.group];
    };
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int n = 0; n < EACH; ++n) raw[k][n] = {};
    load(group);
    for (; group < groups; group += sq.spans) {
        const int64_t bh = group * WAVES + mine;
        // an episode starts with these steps: step t is entered from `since` on, step i enters up to `until`
        const uint32_t cut = (uint32_t)__ballot(sr);
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int x = n * BLOCK + (int)threadIdx.x, row = x >> 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // (steps past the last are zeros)
#pragma unroll
                for (int w = 0; w < (int)(2 * sizeof(T)); ++w) raw[k][n].w[w] = row < L ? raw[k][n].w[w] : 0;
                *(Raw<T> *)(room + k * ROOM + ((x >> 2 & 3) * 32 + row) * P + 8 * (x & 3)) = raw[k][n];
            }
        }
        __syncthreads();
        if (group + sq.spans < groups) load(group + sq.spans);
        if (bh < lines) {
            // (what follows from the lane is worked out here, and not kept in registers from head to head)
            int lane = threadIdx.x & 63;
            asm volatile("" : "+v"(lane));
            const int half = lane >> 5, col = lane & 31, perm = swapped(col);
            T *const qx = room + mine * 32 * P, *const kx = qx + ROOM, *const vx = kx + ROOM, *const ox = vx + ROOM;
            auto rows = [&](const T *x, int row, Part<T> (&y)[2]) {
                y[0] = part_of(*(const Raw<T> *)(x + row * P + 8 * half));
                y[1] = part_of(*(const Raw<T> *)(x + row * P + 8 * half + 16));
            };
            const uint32_t upto = cut & (0xffffffffu >> (31 - col)), after = col < 31 ? cut >> (col + 1) << (col + 1) : 0;
            const int since = upto ? 31 - __clz(upto) : 0, until = after ? __ffs((int)after) - 1 : 32;
            Part<T> a[2], b[2], hi[2], lo[2];
            f32x16 p;
            // scores of `a` (rows by swapped lane) and `b` (by lane), times their powers, as operands
            auto scores = [&](const float (&w)[16], int from, int below) {
                p = {};
                mma<T>(p, a[0], b[0]);
                mma<T>(p, a[1], b[1]);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float y[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const int i = 16 * x + 8 * half + r;
                        y[r] = p[8 * x + r] * w[8 * x + r];
                        if (cut) y[r] = i >= from && i < below ? y[r] : 0.0f;
                    }
                    hi[x] = term_of<T>(y, true);
                    if (Part<T>::TERMS) lo[x] = term_of<T>(y, false);
                }
            };
            auto times = [&](f32x16 &o, const T *x) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const Part<T> z = column_of<T>(x, P, 16 * y, 0, lane);
                    mma<T>(o, z, hi[y]);
                    if (Part<T>::TERMS) mma<T>(o, z, lo[y]);
                }
            };
            // o += M y for a state M: eight of its elements a lane, `step` apart, beside y's parts
            auto state = [&](f32x16 &o, const float *m, int64_t lane_step, int64_t step, int across, int along, const Part<T> (&y)[2]) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float z[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const int i = 16 * x + 8 * half + r;
                        z[r] = perm < across && i < along ? m[perm * lane_step + i * step] : 0.0f;
                    }
                    mma<T>(o, term_of<T>(z, true), y[x]);
                    if (Part<T>::TERMS) mma<T>(o, term_of<T>(z, false), y[x]);
                }
            };
            auto put = [&](T *x, const f32x16 &o) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    Span<T, 8> e;
#pragma unroll
                    for (int r = 0; r < 8; ++r) e.e[r] = (T)o[8 * n + r];
                    *(Raw<T> *)(x + col * P + 16 * n + 8 * half) = __builtin_bit_cast(Raw<T>, e);
                }
            };
            f32x16 dq = {}, dk_ = {}, dv_ = {};
            if (sq.state) {  // dq: S0 [dk][dv] do
                rows(ox, col, b);
                state(dq, sq.state + bh * c.area, dv, 1, dk, dv, b);
                const float f = upto ? 0.0f : first;
#pragma unroll
                for (int r = 0; r < 16; ++r) dq[r] *= f;
            }
            if (sk.state) {
                const float *const z = sk.state + bh * c.area;
                const float f = after ? 0.0f : last;
                rows(vx, col, b);
                state(dk_, z, dv, 1, dk, dv, b);
                rows(kx, col, b);
                state(dv_, z, 1, dv, dv, dk, b);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    dk_[r] *= f;
                    dv_[r] *= f;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            rows(vx, perm, a);
            rows(ox, col, b);
            scores(D, since, 32);
            times(dq, kx);
            float odd = odd_of(dq, 0.0f);  // (as in chunk())
            __builtin_amdgcn_sched_barrier(0);
            rows(ox, perm, a);
            rows(vx, col, b);
            scores(E, 0, until);
            times(dk_, qx);
            odd = odd_of(dk_, odd);
            __builtin_amdgcn_sched_barrier(0);
            put(vx, dq);  // (a wave has read what it needs of v: gradients take the rows' place)
            rows(qx, perm, a);
            rows(kx, col, b);
            scores(E, 0, until);
            times(dv_, ox);
            odd = odd_of(dv_, odd);
            __builtin_amdgcn_sched_barrier(0);
            if (sv.state_out) {  // d S0: columns of q, and of do times their powers
                f32x16 z = {};
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const Part<T> qc = column_of<T>(qx, P, 16 * x, 0, lane), oc = column_of<T>(ox, P, 16 * x, 0, lane);
                    float y[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const int t = 16 * x + 8 * half + r;
                        const float w = cut & (0xffffffffu >> (31 - t)) ? 0.0f : sq.score * __builtin_amdgcn_exp2f(a2 * (float)(t + 1));
                        y[r] = element(oc, r) * w;
                    }
#pragma unroll
                    for (int n = 0; n < (Part<T>::TERMS ? 3 : 1); ++n) mma<T>(z, qc, term_of<T>(y, n < 2));
                }
                const float f = cut ? 0.0f : __builtin_amdgcn_exp2f(a2 * (float)L);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = 16 * (r >> 3) + 8 * half + (r & 7);
                    const int64_t at = bh * c.area + i * dv + perm;
                    if (i < dk && perm < dv) {
                        const float y = z[r] + (sk.state && !cut ? f * sk.state[at] : 0.0f);
                        odd = __builtin_fmaf(y, 0.0f, odd);
                        sv.state_out[at] = y;
                    }
                }
            }
            const bool wrong = __ballot(!(odd == 0.0f)) != 0;
            if (lane < 3) c.wrong[bh * 3 + lane] = wrong;
            put(kx, dk_);
            put(qx, dv_);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            int x = n * BLOCK + (int)threadIdx.x;
            asm volatile("" : "+v"(x));
            const int row = x >> 4, at = 8 * (x & 3);
            const uint32_t line = (uint32_t)(group * WAVES + (x >> 2 & 3)), b = line / (uint32_t)c.heads;
            if (row >= L || line >= lines) continue;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const Span<T, 8> e = __builtin_bit_cast(Span<T, 8>, *(const Raw<T> *)(room + k * ROOM + ((x >> 2 & 3) * 32 + row) * P + at));
                T *const y = (T *)to[k].p + row * to[k].st[0] + b * to[k].st[1] + (line - b * (uint32_t)c.heads) * to[k].st[2] + at;
                const int left = to[k].n - at;
                if (FIT == FULL || (FIT == EIGHTS ? left > 0 : left >= 8)) *(Span<T, 8> *)y = e;
                else if constexpr (FIT <= ANY) {
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < left) y[r] = e.e[r];
                }
            }
        }
        __syncthreads();
    }
}

// The heads (and columns) where something was not finite, step by step, as the definition has it: what
// a start or the order of the steps keeps from an output does not reach it as a product with 0.
// A wave takes every `waves`-th unit, since those of one padded sequence are neighbours; lane l looks at the l-th of
// them.  It does a unit with a column a lane, half of the state's rows in either half of the wave, from 16 steps'
// rows in LDS; the next 16 are on their way meanwhile.  What bounds it is that chain: 4 operations for every row
// of the half, 0.65 us a step of 64 rows.  4095 steps of 384 heads of 64, bfloat16, padded with NaN: 3.0 ms, of one sequence
// of 96 the same (0.35 with nothing to do again; 64 units behind one another in a wave, as neighbours: 991 and 105).
template <typename T, int KT> __global__ __launch_bounds__(BLOCK, KT <= 2 ? 2 : 1) void k_exact(const Call c, int64_t n)
{
    constexpr int STEPS = 16, HALF = 16 * KT, WIDE = 2 * HALF, EACH = STEPS * WIDE / 64;
    struct __align__(16) F4 { float e[4]; };
    __shared__ F4 room[WAVES][STEPS * (2 * WIDE + 32) / 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    float *const kx = (float *)room[wave], *const qx = kx + STEPS * WIDE, *const vx = qx + STEPS * WIDE;
    const int64_t waves = (int64_t)gridDim.x * WAVES;
    for (int64_t first = (int64_t)blockIdx.x * WAVES + wave; first < n; first += 64 * waves) {
        uint64_t wrong = 0;
        const int64_t own = first + lane * waves;
        if (own < n) {
            const int64_t bh = own / c.slices, at = bh * c.segments * c.slices + (own - bh * c.slices);
            for (int i = 0; i < c.segments; ++i) wrong |= c.wrong[at + (int64_t)i * c.slices];
        }
        wrong = __ballot(wrong != 0);
        for (; wrong; wrong &= wrong - 1) {
            const int64_t unit = first + (__ffsll((unsigned long long)wrong) - 1) * waves;
            const int64_t bh = unit / c.slices, b = bh / c.heads;
            const int h = (int)(bh - b * c.heads);
            int slice = (int)(unit - bh * c.slices), which = 0;
            while (slice >= c.scan[which].slices) slice -= c.scan[which++].slices;
            const Scan &s = c.scan[which];
            const int j = 32 * slice + col, dk = s.dk, upper = (dk + 1) / 2, lower = dk - upper;  // rows of the halves
            const int count = half ? lower : upper, row0 = half ? upper : 0;
            const bool back = s.back, mine = j < s.dv;
            const int64_t steps = c.steps, groups = c.batch / c.group;
            const T *const q = (const T *)s.q + b * s.qs[1] + h * s.qs[2], *const k = (const T *)s.k + b * s.ks[1] + h * s.ks[2];
            const T *const v = (const T *)s.v + b * s.vs[1] + h * s.vs[2] + 32 * slice;
            T *const out = (T *)s.out + b * s.os[1] + h * s.os[2] + j;
            const uint8_t *const starts = c.starts ? c.starts + b / c.group : nullptr;
            const int64_t at = bh * c.area + (int64_t)row0 * s.si + (int64_t)j * s.sj;
            float S[HALF];
#pragma unroll
            for (int r = 0; r < HALF; ++r) S[r] = s.state && r < count && mine ? s.state[at + (int64_t)r * s.si] : 0.0f;
            const float lambda = __builtin_amdgcn_exp2f(c.log_decay[h] * LOG2E), pre = back ? 1.0f : lambda, post = back ? lambda : 1.0f;
            T kr[EACH], qr[EACH], vr[STEPS / 2];
            uint8_t sr = 0;
            auto time = [&](int64_t x) { return back ? steps - 1 - x : x; };
            // (past the end of a row, or of the steps, the last element, or the last row: read, and not used)
            const int j0 = mine ? col : s.dv - 1 - 32 * slice;
            auto load = [&](int64_t x0) {
#pragma unroll
                for (int m = 0; m < EACH; ++m) {
                    const int e = m * 64 + lane, i = e % WIDE < dk ? e % WIDE : dk - 1;
                    const int64_t t = time(x0 + e / WIDE < steps ? x0 + e / WIDE : steps - 1);
                    kr[m] = k[t * s.ks[0] + i];
                    qr[m] = q[t * s.qs[0] + i];
                }
#pragma unroll
                for (int m = 0; m < STEPS / 2; ++m) {
                    const int64_t x = x0 + 2 * m + half;
                    vr[m] = v[time(x < steps ? x : steps - 1) * s.vs[0] + j0];
                }
                const int64_t x = x0 + lane;
                sr = starts && lane < STEPS && x < steps && (!back || x > 0) ? starts[(back ? steps - x : x) * groups] : 0;
            };
            if (steps > 0) load(0);
            for (int64_t x0 = 0; x0 < steps; x0 += STEPS) {
#pragma unroll
                for (int m = 0; m < EACH; ++m) {
                    const int e = m * 64 + lane, i = e % WIDE;
                    if (i >= dk) continue;
                    const int to = e / WIDE * WIDE + (i < upper ? i : HALF + i - upper);
                    kx[to] = (float)kr[m];
                    qx[to] = (float)qr[m];
                }
#pragma unroll
                for (int m = 0; m < STEPS / 2; ++m) vx[m * 64 + lane] = (float)vr[m] * s.grow;
                const uint32_t fresh = (uint32_t)__ballot(sr);
                __builtin_amdgcn_wave_barrier();
                if (x0 + STEPS < steps) load(x0 + STEPS);
                const int L = steps - x0 < STEPS ? (int)(steps - x0) : STEPS;
#pragma unroll 1
                for (int x = 0; x < L; ++x) {
                    // (all asked for together; what lies behind the half's rows is not used)
                    const F4 *const kk = (const F4 *)(kx + x * WIDE + half * HALF), *const qq = (const F4 *)(qx + x * WIDE + half * HALF);
                    F4 k4[HALF / 4], q4[HALF / 4];
#pragma unroll
                    for (int r = 0; r < HALF / 4; ++r) {
                        k4[r] = kk[r];
                        q4[r] = qq[r];
                    }
                    const float vj = vx[x * 32 + col];
                    __builtin_amdgcn_sched_barrier(0);
                    if (fresh >> x & 1) {
#pragma unroll
                        for (int r = 0; r < HALF; ++r) S[r] = 0.0f;
                    }
                    float o[4] = {};
#pragma unroll
                    for (int r0 = 0; r0 < HALF; r0 += 4) {
                        // (the same for all lanes, but for the lower half's last row)
                        if (r0 + 4 <= lower) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float y = __builtin_fmaf(pre, S[r0 + r], k4[r0 / 4].e[r] * vj);
                                o[r] = __builtin_fmaf(q4[r0 / 4].e[r], y, o[r]);
                                S[r0 + r] = post * y;
                            }
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                if (r0 + r >= upper) continue;
                                const float y = __builtin_fmaf(pre, S[r0 + r], k4[r0 / 4].e[r] * vj), z = __builtin_fmaf(q4[r0 / 4].e[r], y, o[r]);
                                o[r] = r0 + r < lower || half == 0 ? z : o[r];
                                S[r0 + r] = post * y;
                            }
                        }
                    }
                    float sum = (o[0] + o[1]) + (o[2] + o[3]);
                    sum += __shfl_xor(sum, 32, 64);
                    if (half == 0 && mine) out[time(x0 + x) * s.os[0]] = (T)(sum * s.carry);
                }
                __builtin_amdgcn_wave_barrier();
            }
            if (s.state_out && mine) {
                const bool clear = back && starts && steps > 0 && starts[0];
#pragma unroll
                for (int r = 0; r < HALF; ++r)
                    if (r < count) s.state_out[at + (int64_t)r * s.si] = clear ? 0.0f : S[r];
            }
        }
    }
}

// The states that segments end with if none enters become those that they start with.
__global__ __launch_bounds__(BLOCK) void k_between(const Call c, int64_t n)
{
    const Scan &s = c.scan[blockIdx.y];
    const int64_t heads = c.batch * c.heads;
    for (int64_t x = (int64_t)blockIdx.x * BLOCK + threadIdx.x; x < n; x += (int64_t)gridDim.x * BLOCK) {
        const int64_t bh = x / c.area;
        float a2 = c.log_decay[bh % c.heads] * LOG2E;
        a2 = a2 < -1e30f ? -1e30f : a2;
        const float f = __builtin_amdgcn_exp2f(a2 * (float)((int64_t)c.chunks * CHUNK));
        float now = s.state ? s.state[x] : 0.0f;
        for (int i = 0; i < c.segments; ++i) {
            float *const y = s.between + i * n + x;
            const float end = *y;
            *y = now;
            now = s.cut[i * heads + bh] ? end : __builtin_fmaf(f, now, end);
        }
    }
}

// One step: the state is read and written once, which is all that counts.  A wave a head; a lane has
// four columns of every (64 / LANES)-th row, LANES of them a row.  512000 heads of 32, bfloat16: 4.3 GB in
// 0.81 ms, 5.4 TB/s (half of it written: above the rate of a copy).  Few heads: 4.5 us, a launch.
template <typename T, int LANES> __global__ __launch_bounds__(BLOCK) void k_step(const swarp_decay_t a, int64_t heads)
{
    constexpr int ROWS = 64 / LANES, AHEAD = 4;  // rows of a wave at once, and how many times that are under way
    struct __attribute__((packed, aligned(4))) Four { float e[4]; };
    const int lane = threadIdx.x & 63, i0 = lane / LANES, j4 = lane % LANES * 4;
    const int dk = a.dk, dv = a.dv;
    const bool mine = j4 < dv;
    // (the last four columns overlap those before them: a wave has read all of a row before it writes it, and
    // writes the same there twice)
    const int j = j4 < dv - 4 ? j4 : dv - 4;
    const int64_t step = (int64_t)gridDim.x * WAVES;
    for (int64_t bh = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); bh < heads; bh += step) {
        const int64_t b = (uint32_t)bh / (uint32_t)a.heads;  // (at most 2^31 heads)
        const int h = (int)(bh - b * a.heads);
        const T *const q = (const T *)a.q + b * a.q_stride[1] + h * a.q_stride[2];
        const T *const k = (const T *)a.k + b * a.k_stride[1] + h * a.k_stride[2];
        const T *const v = (const T *)a.v + b * a.v_stride[1] + h * a.v_stride[2];
        // (lane l brings elements l and l + 64 of q and k)
        const int l0 = lane < dk ? lane : dk - 1, l1 = lane + 64 < dk ? lane + 64 : dk - 1;
        const float q0 = (float)q[l0], q1 = (float)q[l1], k0 = (float)k[l0], k1 = (float)k[l1];
        float vj[4], o[4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) vj[c] = mine ? (float)v[j + c] : 0.0f;
        const bool fresh = !a.state || (a.starts && a.starts[(uint32_t)b / (uint32_t)a.group]);
        const float lambda = __builtin_amdgcn_exp2f(a.log_decay[h] * LOG2E);
        const float *const from = a.state + bh * dk * dv + j;
        float *const to = a.state_out + bh * dk * dv + j;
#pragma unroll 1
        for (int r0 = 0; r0 < dk; r0 += ROWS * AHEAD) {
            Four s[AHEAD];
#pragma unroll
            for (int x = 0; x < AHEAD; ++x) {
                const int i = r0 + x * ROWS + i0;
                s[x] = {};
                if (mine && i < dk && !fresh) s[x] = *(const Four *)(from + i * dv);
            }
#pragma unroll
            for (int x = 0; x < AHEAD; ++x) {
                const int i = r0 + x * ROWS + i0;
                float ki = __shfl(k0, i & 63, 64), qi = __shfl(q0, i & 63, 64);
                if (dk > 64) {  // (the same for all lanes)
                    const float k2 = __shfl(k1, i & 63, 64), q2 = __shfl(q1, i & 63, 64);
                    ki = i < 64 ? ki : k2;
                    qi = i < 64 ? qi : q2;
                }
                if (mine && i < dk) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float kv = ki * vj[c];
                        s[x].e[c] = fresh ? kv : __builtin_fmaf(lambda, s[x].e[c], kv);
                        o[c] = __builtin_fmaf(qi, s[x].e[c], o[c]);
                    }
                    *(Four *)(to + i * dv) = s[x];
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int d = LANES; d < 64; d <<= 1) o[c] += __shfl_xor(o[c], d, 64);
        if (i0 == 0 && mine) {
            T *const y = (T *)a.out + bh * dv + j;
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = (T)(o[c] * (float)a.scale);
        }
    }
}

// The same for 1, 2, 3 or 5 columns of v: a thread one of them, all of dk in turn.
template <typename T> __global__ __launch_bounds__(BLOCK) void k_step_any(const swarp_decay_t a, int64_t n)
{
    for (int64_t x = (int64_t)blockIdx.x * BLOCK + threadIdx.x; x < n; x += (int64_t)gridDim.x * BLOCK) {
        const int64_t bh = x / a.dv, b = bh / a.heads;
        const int j = (int)(x - bh * a.dv), h = (int)(bh - b * a.heads);
        const T *const q = (const T *)a.q + b * a.q_stride[1] + h * a.q_stride[2];
        const T *const k = (const T *)a.k + b * a.k_stride[1] + h * a.k_stride[2];
        const float v = (float)((const T *)a.v)[b * a.v_stride[1] + h * a.v_stride[2] + j];
        const bool fresh = !a.state || (a.starts && a.starts[b / a.group]);
        const float lambda = __builtin_amdgcn_exp2f(a.log_decay[h] * LOG2E);
        const int64_t at = bh * a.dk * a.dv + j;
        float o = 0.0f;
        for (int i = 0; i < a.dk; ++i) {
            const int64_t e = at + (int64_t)i * a.dv;
            const float kv = (float)k[i] * v;
            const float s = fresh ? kv : __builtin_fmaf(lambda, a.state[e], kv);
            a.state_out[e] = s;
            o = __builtin_fmaf((float)q[i], s, o);
        }
        ((T *)a.out)[x] = (T)(o * (float)a.scale);
    }
}

int check(const swarp_decay_t *a)
{
    swarp::set_error("");
    if (!a) return fail("arguments must be set");
    if (a->dtype != SWARP_F32 && a->dtype != SWARP_BF16 && a->dtype != SWARP_F16) return fail("unknown dtype");
    if (a->steps < 0 || a->batch < 0 || a->heads < 1 || a->dk < 1 || a->dk > MOST_DIM || a->dv < 1 ||
        a->dv > MOST_DIM || a->group < 1 || a->batch % a->group)
        return fail("bad sizes");
    // (a launch has fewer than 2^32 threads: a wave, or a share of a workgroup, for every head, slice and scan)
    if (a->heads > MOST_HEADS || a->batch * a->heads > 1ll << 31 || a->steps > 1ll << 40) return fail("bad sizes");
    return 0;
}

void strides(int64_t (&to)[3], const swarp_decay_t *a, int d)
{
    to[0] = a->batch * a->heads * d;
    to[1] = (int64_t)a->heads * d;
    to[2] = d;
}
void copy(int64_t (&to)[3], const int64_t *from)
{
    for (int i = 0; i < 3; ++i) to[i] = from[i];
}

// How the steps are cut: only as far as gives every SIMD a wave.  A segment's start costs some ten
// chunks (the state, the powers, the first rows' way), its end a second reading of k and v: 4095 steps of
// 384 heads of 64, 768 waves forward and 2304 backward, take 1250 us uncut, 1460 with segments for 2048
// waves; 32769 steps of 16 heads of 128 take 360 us in 16 segments, 375 in 32.
constexpr int WANTED = 1024, LEAST_CHUNKS = 4, MOST_SEGMENTS = 256;
constexpr int64_t MOST_WAVES = 8192;  // of a launch, about: beyond it one takes several heads in turn

struct Cuts {
    int segments, chunks;
};
Cuts cuts_of(const swarp_decay_t *a, int slices)
{
    const int64_t waves = a->batch * a->heads * slices, chunks = (a->steps + CHUNK - 1) / CHUNK;
    int64_t n = waves > 0 ? WANTED / waves : 1;
    if (n > chunks / LEAST_CHUNKS) n = chunks / LEAST_CHUNKS;
    if (n > MOST_SEGMENTS) n = MOST_SEGMENTS;
    if (n < 2) return {1, (int)(chunks < 1 << 30 ? (chunks < 1 ? 1 : chunks) : 1 << 30)};
    const int64_t each = (chunks + n - 1) / n;
    return {(int)((chunks + each - 1) / each), (int)each};
}
int slices_of(const swarp_decay_t *a, bool back)
{
    const int k = (a->dk + 31) / 32, v = (a->dv + 31) / 32;
    return back ? 2 * k + v : v;
}
uint64_t work_of(const swarp_decay_t *a, bool back)
{
    const int slices = slices_of(a, back);
    const Cuts n = cuts_of(a, slices);
    const uint64_t heads = (uint64_t)(a->batch * a->heads), scans = n.segments < 2 ? 0 : back ? 2 : 1;
    return n.segments * heads * (scans * (4ull * a->dk * a->dv + 4) + slices) + 256;
}

template <typename T, int KT, int WHAT> void alone(Call &c, int fit, hipStream_t st)
{
    const int64_t kinds = (int64_t)c.heads * c.segments * c.slices, spans = MOST_WAVES / kinds;
    c.spans = spans < 1 ? 1 : spans < c.batch ? spans : c.batch;
    const dim3 grid((unsigned)((c.spans * kinds + WAVES - 1) / WAVES));
    if (fit == FULL) hipLaunchKernelGGL((k_alone<T, KT, WHAT, FULL>), grid, dim3(BLOCK), 0, st, c);
    else if (fit == EIGHTS) hipLaunchKernelGGL((k_alone<T, KT, WHAT, EIGHTS>), grid, dim3(BLOCK), 0, st, c);
    else if (fit == ANY) hipLaunchKernelGGL((k_alone<T, KT, WHAT, ANY>), grid, dim3(BLOCK), 0, st, c);
    else hipLaunchKernelGGL((k_alone<T, KT, WHAT, SHORT>), grid, dim3(BLOCK), 0, st, c);
}

// Workgroups of four heads each, of which each has the same h in every wave throughout: four times
// their number is a multiple of the call's heads, as far as there is more than one group for each.
int64_t spans_of(const Call &c, int64_t want)
{
    const int64_t groups = (c.batch * c.heads + WAVES - 1) / WAVES;
    const int64_t whole = c.heads % 4 == 0 ? c.heads / 4 : c.heads % 2 == 0 ? c.heads / 2 : c.heads;
    const int64_t n = want < whole ? whole : want / whole * whole;
    return n < groups ? n : groups;
}

template <typename T, int WHAT> void together(Call &c, int fit, hipStream_t st)
{
    for (int i = 0; i < c.scans; ++i) c.scan[i].spans = spans_of(c, MOST_WAVES / WAVES / (c.segments * c.scans));
    const dim3 grid((unsigned)(c.scan[0].spans * c.segments * c.scans));
    if (fit == FULL) hipLaunchKernelGGL((k_together<T, WHAT, FULL>), grid, dim3(BLOCK), 0, st, c);
    else if (fit == EIGHTS) hipLaunchKernelGGL((k_together<T, WHAT, EIGHTS>), grid, dim3(BLOCK), 0, st, c);
    else if (fit == ANY) hipLaunchKernelGGL((k_together<T, WHAT, ANY>), grid, dim3(BLOCK), 0, st, c);
    else hipLaunchKernelGGL((k_together<T, WHAT, SHORT>), grid, dim3(BLOCK), 0, st, c);
}

template <typename T, int KT, int WHAT> void scan(Call &c, int fit, hipStream_t st)
{
    // Heads up to 32 wide go together: their rows are short (32 x 256000 x 2 heads of 32, forward and
    // backward: 1.52 and 3.07 ms, alone 1.88 and 3.44); wider ones alone (4095 x 96 x 4 heads of 64: 0.28 and
    // 0.88, together 0.29 and 1.11: barriers between waves that have much to do).
    if (KT == 1 && c.scans == 3 && c.slices == 3 && c.steps >= 1 && c.steps <= CHUNK) {
        // One chunk, backward: all three at once.
        c.scan[0].spans = spans_of(c, MOST_WAVES / WAVES);
        const dim3 grid((unsigned)c.scan[0].spans);
        if (fit == FULL) hipLaunchKernelGGL((k_short<T, FULL>), grid, dim3(BLOCK), 0, st, c, c.scan[0], c.scan[1], c.scan[2]);
        else if (fit == EIGHTS) hipLaunchKernelGGL((k_short<T, EIGHTS>), grid, dim3(BLOCK), 0, st, c, c.scan[0], c.scan[1], c.scan[2]);
        else if (fit == ANY) hipLaunchKernelGGL((k_short<T, ANY>), grid, dim3(BLOCK), 0, st, c, c.scan[0], c.scan[1], c.scan[2]);
        else hipLaunchKernelGGL((k_short<T, SHORT>), grid, dim3(BLOCK), 0, st, c, c.scan[0], c.scan[1], c.scan[2]);
    } else if (KT == 1 && c.slices == c.scans) together<T, WHAT>(c, fit, st);
    else alone<T, KT, WHAT>(c, fit, st);
    if (WHAT == OUTPUTS) {
        const int64_t n = c.units / c.segments;
        const int64_t blocks = (n + WAVES - 1) / WAVES, most = MOST_WAVES / WAVES;  // (of up to 2^34 units)
        hipLaunchKernelGGL((k_exact<T, KT>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(BLOCK), 0, st, c, n);
    }
}

template <typename T, int WHAT> void scan(Call &c, hipStream_t st)
{
    int kt = 0;
    c.slices = 0;
    for (int i = 0; i < c.scans; ++i) {
        c.scan[i].slices = (c.scan[i].dv + 31) / 32;
        c.scan[i].first = c.slices;
        c.slices += c.scan[i].slices;
        if ((c.scan[i].dk + 31) / 32 > kt) kt = (c.scan[i].dk + 31) / 32;
    }
    int fit = FULL;
    for (int i = 0; i < c.scans; ++i) {
        if (c.scan[i].dk != 32 * kt || c.scan[i].dv % 32) fit = fit < EIGHTS ? fit : EIGHTS;
        if (c.scan[i].dk % 8 || c.scan[i].dv % 8) fit = fit < ANY ? fit : ANY;
        if (c.scan[i].dk < 8 || c.scan[i].dv < 8) fit = SHORT;
    }
    c.units = c.batch * c.heads * c.segments * c.slices;
    if (kt == 1) scan<T, 1, WHAT>(c, fit, st);
    else if (kt == 2) scan<T, 2, WHAT>(c, fit, st);
    else if (kt == 3) scan<T, 3, WHAT>(c, fit, st);
    else scan<T, 4, WHAT>(c, fit, st);
}

// `ends`: the scans whose states between segments are to be found first; the others have theirs.
template <typename T> void launch(Call &c, const Call &ends, hipStream_t st)
{
    if (c.segments > 1) {
        Call e = ends;
        scan<T, ENDS>(e, st);
        const int64_t n = c.batch * c.heads * c.area, blocks = (n + BLOCK - 1) / BLOCK;
        hipLaunchKernelGGL(k_between, dim3((unsigned)(blocks < 4096 ? blocks : 4096), e.scans), dim3(BLOCK), 0, st, e, n);
    }
    scan<T, OUTPUTS>(c, st);
}

int launch(const swarp_decay_t *a, Call &c, const Call &ends, hipStream_t st)
{
    switch (a->dtype) {
    case SWARP_F32: launch<float>(c, ends, st); break;
    case SWARP_BF16: launch<bf16>(c, ends, st); break;
    default: launch<f16>(c, ends, st); break;
    }
    return launched();
}

int work(const swarp_decay_t *a, bool back)
{
    if (!a->work || a->work_bytes < work_of(a, back)) return fail("work must be set, swarp_decay_work_bytes() long");
    if ((uintptr_t)a->work & 255u) return fail("work must be 256-byte aligned");
    return 0;
}

// Room for the states between a scan's segments, the n-th of the call.
void between(const swarp_decay_t *a, const Call &c, Scan &s, int n, int scans)
{
    const int64_t heads = c.segments * a->batch * a->heads;
    s.between = (float *)a->work + n * heads * c.area;
    s.cut = (int32_t *)((float *)a->work + scans * heads * c.area) + n * heads;
}

Call call_of(const swarp_decay_t *a, bool back)
{
    Call c = {};
    const Cuts n = cuts_of(a, slices_of(a, back));
    c.segments = n.segments;
    c.chunks = n.chunks;
    c.wrong = (uint8_t *)a->work + work_of(a, back) - n.segments * a->batch * a->heads * slices_of(a, back);
    c.steps = a->steps;
    c.batch = a->batch;
    c.group = a->group;
    c.heads = a->heads;
    c.area = a->dk * a->dv;
    c.log_decay = a->log_decay;
    c.starts = a->starts;
    return c;
}

template <typename T> void step(const swarp_decay_t *a, hipStream_t st)
{
    const int64_t heads = a->batch * a->heads, n = heads * a->dv;
    auto blocks = [](int64_t n, int64_t each) { return dim3((unsigned)((n + each - 1) / each < 16384 ? (n + each - 1) / each : 16384)); };
    const dim3 grid = blocks(heads, WAVES), block(BLOCK);
    // (25068 heads of 112 x 86, bfloat16: 402 us, a thread a column 901; 100000 of 16 x 5, float32: 51 and 43)
    if (a->dv < 6 && a->dv != 4) hipLaunchKernelGGL((k_step_any<T>), blocks(n, BLOCK), block, 0, st, *a, n);
    else if (a->dv <= 4) hipLaunchKernelGGL((k_step<T, 1>), grid, block, 0, st, *a, heads);
    else if (a->dv <= 8) hipLaunchKernelGGL((k_step<T, 2>), grid, block, 0, st, *a, heads);
    else if (a->dv <= 16) hipLaunchKernelGGL((k_step<T, 4>), grid, block, 0, st, *a, heads);
    else if (a->dv <= 32) hipLaunchKernelGGL((k_step<T, 8>), grid, block, 0, st, *a, heads);
    else if (a->dv <= 64) hipLaunchKernelGGL((k_step<T, 16>), grid, block, 0, st, *a, heads);
    else hipLaunchKernelGGL((k_step<T, 32>), grid, block, 0, st, *a, heads);
}
void step_of(const swarp_decay_t *a, hipStream_t st)
{
    switch (a->dtype) {
    case SWARP_F32: return step<float>(a, st);
    case SWARP_BF16: return step<bf16>(a, st);
    default: return step<f16>(a, st);
    }
}

}  // namespace

extern "C" {

uint64_t swarp_decay_work_bytes(const swarp_decay_t *a)
{
    if (check(a)) return 0;
    const uint64_t f = work_of(a, false), b = work_of(a, true);
    return f > b ? f : b;
}

int swarp_decay_fwd(const swarp_decay_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->batch) return 0;
    if (!a->log_decay || (a->steps && (!a->q || !a->k || !a->v || !a->out))) return fail("pointer arguments must be set");
    // (a head that is done again starts from it once more)
    if (a->state && a->state == a->state_out) return fail("state_out must not be state");
    if (work(a, false)) return -1;
    // One step is mostly its states: 13487 x 4 heads of 32, float32, 81 us, and 282 as a chunk of one step; 3000
    // heads of 128, bfloat16, 79 and 132; 200000 of 4, float32, 82 and 1023.
    if (a->steps == 1 && a->state_out && a->dv >= 4) {
        step_of(a, (hipStream_t)stream);
        return launched();
    }
    Call c = call_of(a, false);
    Scan &s = c.scan[0];
    s.q = a->q;
    s.k = a->k;
    s.v = a->v;
    s.out = a->out;
    copy(s.qs, a->q_stride);
    copy(s.ks, a->k_stride);
    copy(s.vs, a->v_stride);
    strides(s.os, a, a->dv);
    s.dk = a->dk;
    s.dv = a->dv;
    s.score = s.carry = (float)a->scale;
    s.grow = 1.0f;
    s.state = a->state;
    s.state_out = a->state_out;
    s.si = a->dv;
    s.sj = 1;
    c.scans = 1;
    if (c.segments > 1) between(a, c, s, 0, 1);
    return launch(a, c, c, (hipStream_t)stream);
}

int swarp_decay_bwd(const swarp_decay_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->batch) return 0;
    if (!a->log_decay || (a->steps && (!a->q || !a->k || !a->v || !a->adj_out)))
        return fail("pointer arguments must be set");
    if (a->steps && (!a->d_q || !a->d_k || !a->d_v)) return fail("d_q, d_k and d_v must be set, all three together");
    // (the scans of k and of v both start from it)
    if (a->adj_state && a->adj_state == a->d_state) return fail("d_state must not be adj_state");
    if (work(a, true)) return -1;
    Call c = call_of(a, true);
    const float scale = (float)a->scale;
    Scan q = {}, k = {}, v = {};
    q.q = k.k = v.v = a->adj_out;
    strides(q.qs, a, a->dv);
    strides(k.ks, a, a->dv);
    strides(v.vs, a, a->dv);
    q.k = k.q = a->v;
    copy(q.ks, a->v_stride);
    copy(k.qs, a->v_stride);
    q.v = v.q = a->k;
    copy(q.vs, a->k_stride);
    copy(v.qs, a->k_stride);
    k.v = v.k = a->q;
    copy(k.vs, a->q_stride);
    copy(v.ks, a->q_stride);
    q.out = a->d_q;
    k.out = a->d_k;
    v.out = a->d_v;
    strides(q.os, a, a->dk);
    strides(k.os, a, a->dk);
    strides(v.os, a, a->dv);
    q.dk = k.dk = v.dv = a->dv;
    q.dv = k.dv = v.dk = a->dk;
    q.score = k.score = v.score = scale;
    q.carry = k.grow = v.grow = scale;
    q.grow = k.carry = v.carry = 1.0f;
    k.back = v.back = 1;
    q.state = a->state;
    k.state = v.state = a->adj_state;
    v.state_out = a->d_state;
    q.si = k.si = v.sj = 1;
    q.sj = k.sj = v.si = a->dv;
    Call ends = c;
    if (c.segments > 1) {
        // (the states of the k and the v scan are one matrix and its transpose)
        between(a, c, q, 0, 2);
        between(a, c, v, 1, 2);
        k.between = v.between;
        ends.scan[0] = q;
        ends.scan[1] = v;
        ends.scans = 2;
    }
    c.scan[0] = q;
    c.scan[1] = k;
    c.scan[2] = v;
    c.scans = 3;
    return launch(a, c, ends, (hipStream_t)stream);
}

int swarp_decay_step(const swarp_decay_t *a, void *stream)
{
    if (check(a)) return -1;
    if (!a->batch) return 0;
    if (a->steps != 1) return fail("a step is one step");
    if (!a->log_decay || !a->q || !a->k || !a->v || !a->out || !a->state_out)
        return fail("pointer arguments must be set");
    // (the state is changed while others still read what the step is made of)
    const uintptr_t size = a->dtype == SWARP_F32 ? 4 : 2, from = (uintptr_t)a->state_out;
    const uintptr_t to = from + (uintptr_t)a->batch * a->heads * a->dk * a->dv * 4;
    auto apart = [&](const void *x, const int64_t *stride, int d) {
        const uintptr_t n = (uintptr_t)((a->batch - 1) * stride[1] + (a->heads - 1) * stride[2] + d) * size;
        return (uintptr_t)x >= to || (uintptr_t)x + n <= from;
    };
    if (!apart(a->q, a->q_stride, a->dk) || !apart(a->k, a->k_stride, a->dk) || !apart(a->v, a->v_stride, a->dv))
        return fail("q, k and v must not lie in the state");
    const uintptr_t decay = (uintptr_t)a->log_decay, starts = (uintptr_t)a->starts;
    if ((decay < to && decay + 4 * (uintptr_t)a->heads > from) || (starts && starts < to && starts + a->batch / a->group > from))
        return fail("log_decay and starts must not lie in the state");
    step_of(a, (hipStream_t)stream);
    return launched();
}

}  // extern "C"
