// ung_fp8.hip -- 8-bit operands with a scale for each block of 128, and their product, on
// gfx950: the kernels and the entry points ung_hip_fp8_* of include/ung_hip.h.
//
// An operand holds rows of e4m3 bytes, padded with zeros to a whole number of 128-byte
// blocks, so a block of a row is one 128-byte run: one line of memory, and the inner length
// of one v_mfma_f32_16x16x128_f8f6f4.  The value of a byte is its e4m3 value times its
// block's scale, s = max(largest magnitude, 2^-64) * (1 / 448), rounded to 32 bits.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ung_elements.h"
#include "ung_hip.h"
#include "ung_internal.h"

using namespace ung;

namespace {

constexpr int KB = UNG_HIP_FP8_BLOCK; // inner length of a block: 128
constexpr float LARGEST = 448.0f;     // largest finite e4m3 value
constexpr float SMALLEST = 0x1p-64f;  // a block's largest magnitude counts as this at least

// ---- quantisation --------------------------------------------------------------------

// Largest magnitude as the bits of its absolute value: whole numbers order like the
// magnitudes, and a NaN is above every one of them, so it reaches the scale.
__device__ inline uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ inline float scale_of(uint32_t most)
{
    const uint32_t least = __float_as_uint(SMALLEST);
    return __uint_as_float(most > least ? most : least) * (1.0f / LARGEST);
}

// x / s rounded as the division rounds, with r = 1 / s from one division a block: the
// product's remainder, exact in a fused multiply-add, corrects it (Markstein's step; r is
// itself correctly rounded, s is a normal number).  A block with an infinity has s = inf,
// r = 0, where the step would make a NaN of every value: there the product alone is right.
__device__ inline float quotient(float x, float s, float r)
{
    const float q = x * r;
    return r == 0.0f ? q : __builtin_fmaf(__builtin_fmaf(-s, q, x), r, q);
}

__device__ inline uint2 pack8(const float *y)
{
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Eight consecutive elements of a row from column c; those at or past `cols` are 0.  ALIGNED:
// rows start at 16-byte boundaries and their distance is a multiple of 16 bytes.
template <class T, bool ALIGNED>
__device__ inline void load8(const T *row, uint64_t c, uint64_t cols, float *x)
{
    if (ALIGNED && c + 8 <= cols) {
#pragma unroll
        for (int h = 0; h < 8 / Vec<T>::N; ++h) {
            const Vec<T> v = *reinterpret_cast<const Vec<T> *>(row + c + h * Vec<T>::N);
#pragma unroll
            for (int i = 0; i < Vec<T>::N; ++i)
                x[h * Vec<T>::N + i] = v.get(i);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = c + i < cols ? to_float(row[c + i]) : 0.0f;
}

// Rows to 8 bits, a scale for each 128 columns of a row: 16 lanes hold a block, 8 elements a
// lane, and agree on its largest magnitude by four exchanges.  One read and one write of the
// data, bound by memory.
template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void ung_fp8_rows_kernel(const T *x, uint64_t rows, uint64_t cols, uint64_t stride,
                                                           uint32_t blocks, uint8_t *q, float *scale)
{
    const uint64_t total = rows * blocks;
    const uint32_t lane = threadIdx.x & 15;
    for (uint64_t b = blockIdx.x * 16ull + (threadIdx.x >> 4); b < total; b += gridDim.x * 16ull) {
        const uint64_t r = b / blocks;
        const uint32_t kb = (uint32_t)(b - r * blocks);
        float v[8], y[8];
        load8<T, ALIGNED>(x + r * stride, (uint64_t)kb * KB + lane * 8, cols, v);
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            most = max(most, magnitude(v[i]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
            most = max(most, (uint32_t)__shfl_xor((int)most, o));
        const float s = scale_of(most), inv = 1.0f / s;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = quotient(v[i], s, inv);
        *reinterpret_cast<uint2 *>(q + b * KB + lane * 8) = pack8(y);
        if (lane == 0)
            scale[b] = s;
    }
}

// A 128 x 128 tile to 8 bits, both ways round: q with scales of its rows' blocks or of the
// whole square, and (qt) the transposed rows with scales of theirs.  A thread holds an 8 x 8
// patch, so a transposed row's eight bytes are packed in registers; they cross the block
// through LDS and leave as whole 128-byte runs.
template <class T, bool ALIGNED, bool SQUARE>
__global__ __launch_bounds__(256) void ung_fp8_tile_kernel(const T *x, uint64_t rows, uint64_t cols, uint64_t stride,
                                                           uint32_t col_blocks, uint32_t row_blocks, uint8_t *q,
                                                           float *scale, uint8_t *qt, float *scale_t)
{
    __shared__ uint32_t most_of[4][KB];
    __shared__ alignas(16) uint8_t turned[KB][KB + 16];
    const uint32_t cb = blockIdx.x % col_blocks, rb = blockIdx.x / col_blocks;
    const uint32_t tr = threadIdx.x >> 4, tc = threadIdx.x & 15;
    const uint64_t r0 = (uint64_t)rb * KB + tr * 8, c0 = (uint64_t)cb * KB + tc * 8;
    float v[8][8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (r0 + i < rows)
            load8<T, ALIGNED>(x + (r0 + i) * stride, c0, cols, v[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[i][j] = 0.0f;
    }
    float s_all = 0.0f, inv_all = 0.0f;
    if (SQUARE) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                most = max(most, magnitude(v[i][j]));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            most = max(most, (uint32_t)__shfl_xor((int)most, o));
        if ((threadIdx.x & 63) == 0)
            most_of[0][threadIdx.x >> 6] = most;
        __syncthreads();
        most = max(max(most_of[0][0], most_of[0][1]), max(most_of[0][2], most_of[0][3]));
        s_all = scale_of(most);
        inv_all = 1.0f / s_all;
        if (threadIdx.x == 0) {
            scale[(uint64_t)rb * col_blocks + cb] = s_all;
            if (qt)
                scale_t[(uint64_t)cb * row_blocks + rb] = s_all;
        }
    }
    if (q) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float s = s_all, inv = inv_all;
            if (!SQUARE) {
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    most = max(most, magnitude(v[i][j]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
                    most = max(most, (uint32_t)__shfl_xor((int)most, o));
                s = scale_of(most);
                inv = 1.0f / s;
            }
            if (r0 + i < rows) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    y[j] = quotient(v[i][j], s, inv);
                *reinterpret_cast<uint2 *>(q + ((r0 + i) * col_blocks + cb) * KB + tc * 8) = pack8(y);
                if (!SQUARE && tc == 0)
                    scale[(r0 + i) * col_blocks + cb] = s;
            }
        }
    }
    if (!qt)
        return;
    float s_col[8], inv_col[8];
    if (!SQUARE) {
        uint32_t most[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            most[j] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                most[j] = max(most[j], magnitude(v[i][j]));
            most[j] = max(most[j], (uint32_t)__shfl_xor((int)most[j], 16));
            most[j] = max(most[j], (uint32_t)__shfl_xor((int)most[j], 32));
            if ((threadIdx.x & 63) < 16)
                most_of[threadIdx.x >> 6][tc * 8 + j] = most[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t c = tc * 8 + j;
            s_col[j] = scale_of(max(max(most_of[0][c], most_of[1][c]), max(most_of[2][c], most_of[3][c])));
            inv_col[j] = 1.0f / s_col[j];
            if (tr == 0 && c0 + j < cols)
                scale_t[(c0 + j) * row_blocks + rb] = s_col[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float s = SQUARE ? s_all : s_col[j], inv = SQUARE ? inv_all : inv_col[j];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = quotient(v[i][j], s, inv);
        *reinterpret_cast<uint2 *>(&turned[tc * 8 + j][tr * 8]) = pack8(y);
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const uint32_t c = p * 32 + (threadIdx.x >> 3), at = (threadIdx.x & 7) * 16;
        if ((uint64_t)cb * KB + c < cols)
            *reinterpret_cast<uint4 *>(qt + (((uint64_t)cb * KB + c) * row_blocks + rb) * KB + at) =
                *reinterpret_cast<const uint4 *>(&turned[c][at]);
    }
}

// ---- product -------------------------------------------------------------------------

using i32x8 = __attribute__((ext_vector_type(8))) int;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;

// A lane's part of 16 rows of one block: row lane % 16, 32 of its 128 bytes by lane / 16.
union Frag {
    i32x8 v;
    uint4 h[2];
    uint32_t w[8];
};

// The same as bf16, which holds every e4m3 value exactly: 32 values in four groups of eight.
union Wide {
    bf16x8 q[4];
    bf16x2 p[16];
};

__device__ inline Wide widen(const Frag &f)
{
    Wide o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        o.p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.w[i], 1.0f, false);
        o.p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f.w[i], 1.0f, true);
    }
    return o;
}

// One block's 16 x 16 products: sums of 128 products from zero.  The result's lane holds
// column lane % 16 (rows of y) and rows lane / 16 * 4 + i (rows of x).
//
// The 8-bit matrix instruction aligns each group of eight products (eight neighbouring bytes)
// to the group's largest and keeps 13 bits below it; groups are summed in 24 bits.  On values
// of normal distribution that is an error of 1.4e-5 of the result's norm, a hundredth of what
// rounding to bf16 leaves and a fifteenth of fp16's, so it makes the 16-bit results.
__device__ inline f32x4 block_product(const Frag &x, const Frag &y)
{
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.v, y.v, zero, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
}

// 32-bit results are made by bf16 matrix instructions (half the rate), which sum the same
// products in 32 bits: an error of 1e-8.
__device__ inline f32x4 block_product(const Wide &x, const Wide &y)
{
    f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.q[i], y.q[i], p, 0, 0, 0);
    return p;
}

// 16 bytes a lane from global memory straight into LDS, at `lds` + 16 * lane.
__device__ inline void to_lds(const uint8_t *src, uint8_t *lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)src,
                                     (__attribute__((address_space(3))) uint32_t *)lds, 16, 0, 0);
}

// A block of 4 waves makes a BM x BN tile of the product, each wave a quarter of it.  Per
// 128-byte block of the inner length both tiles are staged in LDS, 16-byte pieces of a row
// rotated by exclusive-or with the row so that eight lanes read eight rows without a bank
// conflict; the staged loads are rotated on the global side, as they land in lane order.
// Block products start from zero and enter the running sums by one multiply-add with the
// scales' product, so sums and scales stay in 32 bits.  The table side (b) is the matrix
// instruction's row side: a lane holds four neighbouring columns of one row of c, with one
// scale of a.
template <int BM, int BN, bool SQUARE, class OT>
__global__ __launch_bounds__(256, 2) void ung_fp8_tile_product_kernel(const uint8_t *a, const float *a_scale,
                                                                      const uint8_t *b, const float *b_scale,
                                                                      uint64_t m, uint64_t n, uint32_t kblocks, OT *c,
                                                                      uint64_t c_stride, uint32_t m_tiles,
                                                                      uint32_t n_tiles, int vector_stores)
{
    constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 16, TN = WN / 16;
    __shared__ alignas(16) uint8_t as[2][BM * KB];
    __shared__ alignas(16) uint8_t bs[2][BN * KB];
    __shared__ float sa[2][BM], sb[2][BN];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t wm = (wave & 1) * WM, wn = (wave >> 1) * WN;
    const uint32_t tm = blockIdx.x % m_tiles, tn = blockIdx.x / m_tiles;
    const uint64_t m0 = (uint64_t)tm * BM, n0 = (uint64_t)tn * BN, kp = (uint64_t)kblocks * KB;
    (void)n_tiles;

    // rows past the end repeat the last one; their results are not stored
    auto stage = [&](uint32_t kb, int buf) {
        const uint32_t piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) {
            const uint32_t r = (wave * (BM / 32) + i) * 8 + (lane >> 3);
            const uint64_t row = min(m0 + r, m - 1);
            to_lds(a + row * kp + (uint64_t)kb * KB + piece * 16, &as[buf][(wave * (BM / 32) + i) * 1024]);
        }
#pragma unroll
        for (int i = 0; i < BN / 32; ++i) {
            const uint32_t r = (wave * (BN / 32) + i) * 8 + (lane >> 3);
            const uint64_t row = min(n0 + r, n - 1);
            to_lds(b + row * kp + (uint64_t)kb * KB + piece * 16, &bs[buf][(wave * (BN / 32) + i) * 1024]);
        }
        for (uint32_t t = threadIdx.x; t < BM; t += 256)
            sa[buf][t] = a_scale[min(m0 + t, m - 1) * kblocks + kb];
        for (uint32_t t = threadIdx.x; t < BN; t += 256) {
            const uint64_t row = min(n0 + t, n - 1);
            sb[buf][t] = b_scale[(SQUARE ? row / KB : row) * kblocks + kb];
        }
    };
    auto fragment = [&](const uint8_t *tile, uint32_t row0) {
        const uint32_t r = row0 + (lane & 15), g = lane >> 4;
        Frag f;
        f.h[0] = *reinterpret_cast<const uint4 *>(tile + r * KB + ((g ^ (r & 7)) * 16));
        f.h[1] = *reinterpret_cast<const uint4 *>(tile + r * KB + (((g + 4) ^ (r & 7)) * 16));
        if constexpr (sizeof(OT) == 4)
            return widen(f);
        else
            return f;
    };
    using Part = decltype(fragment(nullptr, 0));

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    if (kblocks)
        stage(0, 0);
    for (uint32_t kb = 0; kb < kblocks; ++kb) {
        const int buf = kb & 1;
        // loads into LDS are counted as memory loads, which a barrier alone does not await
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads(); // this block's tiles have landed; the other buffer is free
        if (kb + 1 < kblocks)
            stage(kb + 1, buf ^ 1);
        Part af[TM], bf[TN];
        float s[TM];
        f32x4 sn[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            af[i] = fragment(as[buf], wm + i * 16);
            s[i] = sa[buf][wm + i * 16 + (lane & 15)];
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            bf[j] = fragment(bs[buf], wn + j * 16);
            sn[j] = *reinterpret_cast<const f32x4 *>(&sb[buf][wn + j * 16 + (lane >> 4) * 4]);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const f32x4 p = block_product(bf[j], af[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[i][j][e] = __builtin_fmaf(p[e], s[i] * sn[j][e], acc[i][j][e]);
            }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const uint64_t row = m0 + wm + i * 16 + (lane & 15);
        if (row >= m)
            continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const uint64_t col = n0 + wn + j * 16 + (lane >> 4) * 4;
            OT o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = from_float<OT>(acc[i][j][e]);
            OT *to = c + row * c_stride + col;
            if (vector_stores && col + 4 <= n) {
                if constexpr (sizeof(OT) == 2)
                    *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(o);
                else
                    *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(o);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < n)
                        to[e] = o[e];
            }
        }
    }
}

} // namespace

extern "C" {

int ung_hip_fp8_quantize(const void *x, int type, uint64_t rows, uint64_t cols, uint64_t row_stride, int square,
                         uint8_t *q, float *scale, uint8_t *qt, float *scale_t, void *stream)
{
    clear_error();
    if (!known_type(type)) {
        set_error("ung_hip_fp8_quantize: unknown element type %d", type);
        return UNG_HIP_EINVAL;
    }
    if (rows == 0 || cols == 0)
        return UNG_HIP_OK;
    if (!x || (!q && !qt) || (q && !scale) || (qt && !scale_t) || (square && !q)) {
        set_error("ung_hip_fp8_quantize: null argument");
        return UNG_HIP_EINVAL;
    }
    if (rows > 1 && row_stride < cols) {
        set_error("ung_hip_fp8_quantize: row_stride %llu is less than %llu columns", (unsigned long long)row_stride,
                  (unsigned long long)cols);
        return UNG_HIP_EINVAL;
    }
    const uint64_t cb = ceil_div(cols, KB), rb = ceil_div(rows, KB);
    if (rows > UINT32_MAX || cols > UINT32_MAX || cb * rb > INT32_MAX) {
        set_error("ung_hip_fp8_quantize: %llu x %llu elements are too many", (unsigned long long)rows,
                  (unsigned long long)cols);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)q % 16 || (uintptr_t)qt % 16 || (uintptr_t)x % type_size(type)) {
        set_error("ung_hip_fp8_quantize: q and qt need 16-byte alignment, x that of its elements");
        return UNG_HIP_EINVAL;
    }
    const hipStream_t st = (hipStream_t)stream;
    const bool aligned = (uintptr_t)x % 16 == 0 && (rows == 1 || row_stride * type_size(type) % 16 == 0);
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const T *p = (const T *)x;
        if (!square && !qt) {
            const uint64_t groups = ceil_div(rows * cb, 16);
            const uint32_t grid = (uint32_t)(groups < 8192 ? groups : 8192);
            if (aligned)
                ung_fp8_rows_kernel<T, true><<<grid, 256, 0, st>>>(p, rows, cols, row_stride, (uint32_t)cb, q, scale);
            else
                ung_fp8_rows_kernel<T, false><<<grid, 256, 0, st>>>(p, rows, cols, row_stride, (uint32_t)cb, q, scale);
        } else {
            auto go = [&](auto kernel) {
                kernel<<<(uint32_t)(cb * rb), 256, 0, st>>>(p, rows, cols, row_stride, (uint32_t)cb, (uint32_t)rb, q,
                                                            scale, qt, scale_t);
            };
            if (square)
                aligned ? go(ung_fp8_tile_kernel<T, true, true>) : go(ung_fp8_tile_kernel<T, false, true>);
            else
                aligned ? go(ung_fp8_tile_kernel<T, true, false>) : go(ung_fp8_tile_kernel<T, false, false>);
        }
        return launched("ung_hip_fp8_quantize");
    });
}

int ung_hip_fp8_matmul_workspace(uint64_t m, uint64_t n, uint64_t kp, uint64_t *bytes)
{
    clear_error();
    if (!bytes) {
        set_error("ung_hip_fp8_matmul_workspace: null bytes");
        return UNG_HIP_EINVAL;
    }
    (void)m;
    (void)n;
    (void)kp;
    *bytes = 0;
    return UNG_HIP_OK;
}

int ung_hip_fp8_matmul(const uint8_t *a, const float *a_scale, const uint8_t *b, const float *b_scale, int b_square,
                       uint64_t m, uint64_t n, uint64_t kp, void *c, int type, uint64_t c_stride, void *workspace,
                       uint64_t workspace_bytes, void *stream)
{
    clear_error();
    if (!known_type(type)) {
        set_error("ung_hip_fp8_matmul: unknown element type %d", type);
        return UNG_HIP_EINVAL;
    }
    if (kp % KB) {
        set_error("ung_hip_fp8_matmul: inner length %llu is no multiple of %d", (unsigned long long)kp, KB);
        return UNG_HIP_EINVAL;
    }
    if (m == 0 || n == 0)
        return UNG_HIP_OK;
    if (!c || (kp && (!a || !a_scale || !b || !b_scale))) {
        set_error("ung_hip_fp8_matmul: null argument");
        return UNG_HIP_EINVAL;
    }
    if (m > 1 && c_stride < n) {
        set_error("ung_hip_fp8_matmul: c_stride %llu is less than %llu columns", (unsigned long long)c_stride,
                  (unsigned long long)n);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)a % 16 || (uintptr_t)b % 16 || (uintptr_t)a_scale % 4 || (uintptr_t)b_scale % 4 ||
        (uintptr_t)c % type_size(type)) {
        set_error("ung_hip_fp8_matmul: a and b need 16-byte alignment, the rest that of its elements");
        return UNG_HIP_EINVAL;
    }
    const uint64_t mt = ceil_div(m, 128), nt = ceil_div(n, 128);
    if (m > UINT32_MAX || n > UINT32_MAX || kp / KB > UINT32_MAX || mt * nt > INT32_MAX) {
        set_error("ung_hip_fp8_matmul: a %llu x %llu x %llu product is too large", (unsigned long long)m,
                  (unsigned long long)n, (unsigned long long)kp);
        return UNG_HIP_EINVAL;
    }
    (void)workspace;
    (void)workspace_bytes;
    const hipStream_t st = (hipStream_t)stream;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const int vec = (uintptr_t)c % (4 * sizeof(T)) == 0 && (m == 1 || c_stride % 4 == 0);
        auto go = [&](auto kernel) {
            kernel<<<(uint32_t)(mt * nt), 256, 0, st>>>(a, a_scale, b, b_scale, m, n, (uint32_t)(kp / KB), (T *)c,
                                                        c_stride, (uint32_t)mt, (uint32_t)nt, vec);
        };
        b_square ? go(ung_fp8_tile_product_kernel<128, 128, true, T>)
                 : go(ung_fp8_tile_product_kernel<128, 128, false, T>);
        return launched("ung_hip_fp8_matmul");
    });
}

} // extern "C"
