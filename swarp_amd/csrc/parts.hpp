// parts.hpp -- small products in a wave's own registers, for the units whose kernels work a chunk of 32
// rows at a time (decay.hip, narrow_ce.hip).
#pragma once
#include "learn.hpp"

namespace part {

using learn::bf16;
using learn::f16;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Span {
    T e[N];
};

// What a lane gives to a product of 32 x 32 over 16 k: row (or column) l % 32, the eight k from
// 8 (l / 32) on.  bfloat16 goes into the matrix cores as it is, what is in float as a sum of
// bfloat16 terms; the others are multiplied in float (float16 has not the range for the states).
template <typename T> struct Part {
    float x[8];
    static constexpr bool TERMS = false;
};
template <> struct Part<bf16> {
    u32x4 w;
    static constexpr bool TERMS = true;
};

template <typename T> __device__ __forceinline__ void mma(f32x16 &acc, const Part<T> &a, const Part<T> &b)
{
    if constexpr (Part<T>::TERMS) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w),
                                                      acc, 0, 0, 0);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[k], b.x[k], acc, 0, 0, 0);
    }
}

// Eight elements as they came from memory.
template <typename T> struct Raw {
    uint32_t w[2 * sizeof(T)];
};
template <typename T> __device__ __forceinline__ float element(const Raw<T> &r, int k)
{
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, r.w[k]);
    else if constexpr (Part<T>::TERMS) return __builtin_bit_cast(float, k & 1 ? r.w[k >> 1] & 0xffff0000u : r.w[k >> 1] << 16);
    else return (float)__builtin_bit_cast(f16, (uint16_t)(r.w[k >> 1] >> 16 * (k & 1)));
}
template <typename T> __device__ __forceinline__ Part<T> part_of(const Raw<T> &r)
{
    Part<T> p;
    if constexpr (Part<T>::TERMS) p.w = __builtin_bit_cast(u32x4, r);
    else {
#pragma unroll
        for (int k = 0; k < 8; ++k) p.x[k] = element(r, k);
    }
    return p;
}
// The next term of x, which is left with what remains of it.
template <typename T> __device__ __forceinline__ Part<T> term_of(float (&x)[8], bool more)
{
    Part<T> p;
    if constexpr (!Part<T>::TERMS) {
#pragma unroll
        for (int k = 0; k < 8; ++k) p.x[k] = x[k];
    } else {
        Raw<T> r;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            r.w[k] = __builtin_bit_cast(uint32_t, Span<bf16, 2>{{(bf16)x[2 * k], (bf16)x[2 * k + 1]}});
        if (more) {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] -= element(r, k);
        }
        p = part_of(r);
    }
    return p;
}
// How the heads' widths fit the tiles: FULL, dk the tiles' and dv a multiple of 32; EIGHTS, both
// multiples of 8; ANY, both at least 8; SHORT.
enum { SHORT, ANY, EIGHTS, FULL };

// Elements at .. at + 7 of a row of n; past its end its last ones, or with `zero` (and ANY) zeros.
template <typename T, int FIT> __device__ __forceinline__ Raw<T> row_of(const T *x, int at, int n, bool zero)
{
    Raw<T> r;
    if constexpr (FIT == FULL) r = __builtin_bit_cast(Raw<T>, *(const Span<T, 8> *)(x + at));
    else if constexpr (FIT == EIGHTS) {
        r = __builtin_bit_cast(Raw<T>, *(const Span<T, 8> *)(x + (at < n ? at : n - 8)));
        if (zero) {
#pragma unroll
            for (int k = 0; k < (int)(2 * sizeof(T)); ++k) r.w[k] = at < n ? r.w[k] : 0;
        }
    } else if constexpr (FIT == ANY) {
        // the row's last eight, moved down to where its end belongs; zeros behind it (72 steps of 9412 heads of
        // 58 x 23, bfloat16, forward and backward: 0.89 ms; element by element, as SHORT rows are, 1.98)
        const int over = at + 8 - n;
        r = __builtin_bit_cast(Raw<T>, *(const Span<T, 8> *)(x + (over > 0 ? n - 8 : at)));
        if (over > 0) {
            constexpr int WORDS = 2 * sizeof(T), EACH = 4 / sizeof(T);  // elements of a word
#pragma unroll
            for (int far = WORDS / 2; far > 0; far >>= 1)
#pragma unroll
                for (int k = 0; k < WORDS; ++k)
                    r.w[k] = over / EACH & far ? (k + far < WORDS ? r.w[k + far] : 0u) : r.w[k];
            if constexpr (EACH == 2) {
#pragma unroll
                for (int k = 0; k < WORDS; ++k) r.w[k] = over & 1 ? r.w[k] >> 16 | (k + 1 < WORDS ? r.w[k + 1] << 16 : 0u) : r.w[k];
            }
#pragma unroll
            for (int k = 0; k < WORDS; ++k) r.w[k] = over < 8 ? r.w[k] : 0u;
        }
    } else {
        Span<T, 8> e;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const T y = x[at + k < n ? at + k : n - 1];
            e.e[k] = zero && at + k >= n ? (T)0.0f : y;
        }
        r = __builtin_bit_cast(Raw<T>, e);
    }
    return r;
}

// Row m of a 32 x 32 accumulator is what operand row m was; swapping two bits of the operand's
// rows makes a lane's registers 8 s .. 8 s + 7 stand for the rows 16 s + 8 (l / 32) + 0 .. 7, which is
// how it holds an operand: accumulators go into the next product as they are.
__device__ __forceinline__ int swapped(int m) { return (m & 0x13) | (m & 4) << 1 | (m & 8) >> 1; }

// Rows of a chunk in LDS, `pitch` elements apart, read as columns: lane l has column
// col + swapped(l % 32), rows row + 8 (l / 32) + 0 .. 7.  16-bit elements come by the transposing read:
// 16 lanes bring four rows of 16 elements, lane i keeps column i of them.
template <typename T> __device__ __forceinline__ Part<T> column_of(const T *x, int pitch, int row, int col, int lane)
{
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 *Ptr;
        const int four = lane & 3, at = (lane & 16) + 4 * ((four & 1) << 1 | four >> 1);
        const T *const y = x + (row + 8 * half + ((lane & 15) >> 2)) * pitch + col + at;
        Raw<T> r;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(uintptr_t)(y));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(uintptr_t)(y + 4 * pitch));
        const uint64_t lo = __builtin_bit_cast(uint64_t, a), hi = __builtin_bit_cast(uint64_t, b);
        r.w[0] = (uint32_t)lo;
        r.w[1] = (uint32_t)(lo >> 32);
        r.w[2] = (uint32_t)hi;
        r.w[3] = (uint32_t)(hi >> 32);
        return part_of(r);
    } else {
        const T *const y = x + (row + 8 * half) * pitch + col + swapped(lane & 31);
        Part<T> p;
#pragma unroll
        for (int k = 0; k < 8; ++k) p.x[k] = y[k * pitch];
        return p;
    }
}
template <typename T> __device__ __forceinline__ float element(const Part<T> &p, int k)
{
    if constexpr (Part<T>::TERMS) return element(__builtin_bit_cast(Raw<T>, p.w), k);
    else return p.x[k];
}

}  // namespace part
