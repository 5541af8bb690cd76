// ung_elements.h -- device helpers shared by the score operators' translation units
// (ung_fp8.hip, ung_scores.hip): element types, 16-byte vectors of them, reductions over a
// wave and a block, and the host's launch checks.  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "ung_hip.h"
#include "ung_internal.h"

namespace ung {

using bf16_t = __bf16;
using fp16_t = _Float16;

template <class T>
__device__ inline float to_float(T v)
{
    return (float)v;
}

// Round to nearest even; one rounding, from 32 bits to the element type.
template <class T>
__device__ inline T from_float(float v)
{
    return (T)v;
}

// A 16-byte vector of elements.
template <class T>
struct alignas(16) Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

// exp(x) for x <= 0 (weights relative to a maximum): 2^(x log2 e) on the hardware's exp2.
// Its relative error is that of the rounded product, |x| 2^-24, so the terms that carry a
// sum (x near 0) are as exact as the library's.
__device__ inline float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

template <class F>
__device__ inline float wave_reduce(float v, F f)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v = f(v, __shfl_xor(v, o));
    return v;
}

// Maximum that keeps a NaN (fmaxf drops it).
__device__ inline float max_nan(float a, float b) { return (a > b || a != a) ? a : b; }
__device__ inline float add(float a, float b) { return a + b; }

// f over one value of every thread of a block of NT threads; `red`: NT / 64 floats of LDS,
// free again after the block's next barrier.
template <int NT, class F>
__device__ inline float block_reduce(float v, float *red, F f)
{
    v = wave_reduce(v, f);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0)
            red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w)
            v = f(v, red[w]);
    }
    return v;
}

inline bool known_type(int t) { return t == UNG_HIP_F32 || t == UNG_HIP_F16 || t == UNG_HIP_BF16; }
inline uint64_t type_size(int t) { return t == UNG_HIP_F32 ? 4 : 2; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// The launch's own error, as a return code.
inline int launched(const char *what)
{
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess)
        return UNG_HIP_OK;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return UNG_HIP_EDEVICE;
}

// Calls f with a value of the element type `t` (checked by known_type before).
template <class F>
int with_type(int t, F f)
{
    if (t == UNG_HIP_F32)
        return f(float{});
    if (t == UNG_HIP_F16)
        return f(fp16_t{});
    return f(bf16_t{});
}

} // namespace ung
