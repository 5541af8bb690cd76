// ung_elements.h -- device helpers shared by the score operators' translation units
// (ung_fp8.hip, ung_scores.hip, ung_int8.hip, ung_table_loss.hip, ung_gradients.hip): element
// types, 16-byte vectors of them, reductions over a wave and a block, loads past the registers,
// the order of tiles, and the host's launch checks.  Not part of the public ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
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

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

// 16 bytes from an address that is aligned to its elements alone; global memory takes such
// loads whole (300000 x 203 bf16 44 us, by elements 67).
template <class T>
__device__ inline Vec<T> load_loose(const T *p)
{
    Vec<T> v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}

template <class T>
__device__ inline void store_loose(T *p, const Vec<T> &v)
{
    __builtin_memcpy(p, &v, sizeof v);
}

// N consecutive elements of a row from column c; those at or past `cols` are 0.
template <class T>
__device__ inline Vec<T> load_row(const T *row, uint64_t c, uint64_t cols)
{
    Vec<T> v;
    if (c + Vec<T>::N <= cols)
        return load_loose(row + c);
    v.w[0] = v.w[1] = v.w[2] = v.w[3] = 0;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e)
        if (c + e < cols)
            v.set(e, row[c + e]);
    return v;
}

// Largest magnitude as the bits of its absolute value: whole numbers order like the
// magnitudes, and a NaN is above every one of them, so it reaches the scale.
__device__ inline uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// x / s rounded as the division rounds, with r = 1 / s from one division a block: the
// product's remainder, exact in a fused multiply-add, corrects it (Markstein's step; r is
// itself correctly rounded, s is a normal number).  A block with an infinity has s = inf,
// r = 0, where the step would make a NaN of every value: with s = 0 there it adds nothing.
struct alignas(8) Divisor {
    float s, r;
    Divisor() = default;
    __device__ explicit Divisor(float scale) : s(scale), r(1.0f / scale)
    {
        if (r == 0.0f)
            s = 0.0f;
    }
};
__device__ inline float quotient(float x, Divisor d)
{
    const float q = x * d.r;
    return __builtin_fmaf(__builtin_fmaf(-d.s, q, x), d.r, q);
}

// What lanes of a wave wrote to LDS is read by others after this, and the other way round (a
// wave's LDS operations are done in order).
__device__ inline void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 16 (or 4) bytes a lane from global memory straight into LDS, at `lds` + 16 (4) * lane.
using lds_ptr = __attribute__((address_space(3))) void *;
__device__ inline void to_lds16(__amdgpu_buffer_rsrc_t from, uint32_t offset, uint32_t advance, void *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)lds, 16, offset, advance, 0, 0);
}
__device__ inline void to_lds4(__amdgpu_buffer_rsrc_t from, uint32_t offset, uint32_t advance, void *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)lds, 4, offset, advance, 0, 0);
}

__device__ inline __amdgpu_buffer_rsrc_t buffer_of(const void *p, uint32_t bytes = 0xFFFFFFFFu)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00020000);
}

template <int N>
__device__ inline void await_loads()
{
    // at most N of the wave's memory operations are still under way; loads into LDS count
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Blocks go to the eight XCDs in turn; with this each XCD takes a contiguous run of `total`.
__device__ inline uint32_t xcd_run(uint32_t id, uint32_t total)
{
    const uint32_t xcd = id & 7, each = total >> 3, extra = total & 7;
    return xcd * each + (xcd < extra ? xcd : extra) + (id >> 3);
}

// Tile t of m_tiles x n_tiles, in bands of `band` tiles of m.
__device__ inline void tile_of(uint32_t t, uint32_t band, uint32_t m_tiles, uint32_t n_tiles, uint32_t &tm,
                               uint32_t &tn)
{
    const uint32_t b = t / (band * n_tiles), in = t - b * band * n_tiles;
    const uint32_t high = m_tiles - b * band < band ? m_tiles - b * band : band;
    tm = b * band + in % high;
    tn = in / high;
}

// Divisions leave a block's numbers in vector registers.
__device__ inline uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// CUs of the current device, asked for once.
inline uint32_t cu_count()
{
    static std::atomic<uint32_t> known[64];
    int device = 0, n = 0;
    if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) {
        (void)hipGetLastError();
        return 256;
    }
    uint32_t got = known[device].load(std::memory_order_relaxed);
    if (!got) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 8) {
            (void)hipGetLastError();
            n = 256;
        }
        known[device].store(got = (uint32_t)n, std::memory_order_relaxed);
    }
    return got;
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
