// ung_elements.h -- device helpers shared by the score operators' translation units
// (ung_fp8.hip, ung_scores.hip): element types, 16-byte vectors of them, reductions over a
// wave and a block, and the host's launch checks.  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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

// A 16-byte vector of elements, as the four registers that hold it.
template <class T>
struct alignas(16) Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    static constexpr uint32_t NEG_INF_BITS =
        sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, bf16_t> ? 0xFF80FF80u : 0xFC00FC00u;
    uint32_t w[4];

    __device__ float get(int e) const
    {
        if constexpr (sizeof(T) == 4)
            return __builtin_bit_cast(float, w[e]);
        else if constexpr (std::is_same_v<T, bf16_t>)
            return __builtin_bit_cast(float, e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
        else
            return (float)__builtin_bit_cast(fp16_t, (uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2]));
    }
    __device__ T element(int e) const
    {
        if constexpr (sizeof(T) == 4)
            return __builtin_bit_cast(T, w[e]);
        else
            return __builtin_bit_cast(T, (uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2]));
    }
    __device__ void set(int e, T x)
    {
        if constexpr (sizeof(T) == 4)
            w[e] = __builtin_bit_cast(uint32_t, x);
        else if (e & 1)
            w[e / 2] = (w[e / 2] & 0xFFFFu) | (uint32_t)__builtin_bit_cast(uint16_t, x) << 16;
        else
            w[e / 2] = (w[e / 2] & 0xFFFF0000u) | __builtin_bit_cast(uint16_t, x);
    }
    __device__ void fill_neg_inf()
    {
        w[0] = w[1] = w[2] = w[3] = NEG_INF_BITS;
    }
    // Elements e and e + 1 (e even) from 32 bits.
    __device__ void put2(int e, float a, float b)
    {
        if constexpr (sizeof(T) == 4) {
            w[e] = __builtin_bit_cast(uint32_t, a);
            w[e + 1] = __builtin_bit_cast(uint32_t, b);
        } else {
            using Two = T __attribute__((ext_vector_type(2)));
            const Two two = {from_float<T>(a), from_float<T>(b)};
            w[e / 2] = __builtin_bit_cast(uint32_t, two);
        }
    }
};

// exp((s - top) / T) by the hardware's 2^x, c = log2(e) / T.  The difference is taken first:
// it is exact where s is near top, so the terms that carry a sum are as exact as the library's
// (the others are off by |exponent| 2^-24 of themselves), and rows of any size are served,
// rows masked by the type's lowest value among them.
__device__ inline float weight_of(float s, float top, float c) { return __builtin_amdgcn_exp2f((s - top) * c); }

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

// A launch's threads are counted in 32 bits along each axis.
inline uint64_t most_blocks(uint32_t threads) { return UINT32_MAX / threads; }

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
