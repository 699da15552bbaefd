// learn.hpp -- scalar types, reductions and launch helpers shared by the units of the policy
// update (gae.hip, policy.hip, adamw.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "swarp_hip.h"

namespace swarp {
int set_error(const char *msg);  // swarp_hip.hip: the message swarp_last_error() returns
}

namespace learn {

inline int fail(const char *msg) { return swarp::set_error(msg); }

// Result of the launches of one entry point.
inline int launched()
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail(hipGetErrorString(e));
}

// Storage types of heads, parameters and gradients.  Arithmetic is in Acc<T>::type.
typedef __bf16 bf16;
typedef _Float16 f16;
template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };

template <typename T> __device__ __forceinline__ typename Acc<T>::type up(T x)
{
    return (typename Acc<T>::type)x;
}

// Sum over the lanes of a wave; every lane has it.
template <typename A> __device__ __forceinline__ A wave_sum(A v)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
template <typename A> __device__ __forceinline__ A wave_max(A v)
{
    for (int d = 32; d > 0; d >>= 1) {
        const A y = __shfl_xor(v, d, 64);
        v = y > v ? y : v;
    }
    return v;
}

}  // namespace learn
