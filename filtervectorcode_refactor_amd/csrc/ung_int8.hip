// ung_int8.hip -- rows in 8-bit whole numbers with a scale a row, and their product, on gfx950:
// the kernels and the entry points ung_hip_int8_* of include/ung_hip.h.
//
// An operand holds rows of whole numbers -127..127, padded with zeros to whole chunks of 128; an
// element's value is its number times its row's scale, s = max(largest magnitude, 2^-64) *
// (1 / 127).  A row's scale leaves the sum, C_ij = s_i s_j sum_k q_ik q_jk, so the sum is one of
// whole numbers: exact, the same in any order, and shares of it may be joined in any way.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ung_elements.h"
#include "ung_hip.h"
#include "ung_internal.h"
#include "ung_tiles.h"

using namespace ung;

namespace {

constexpr float LARGEST = 127.0f;
constexpr float SMALLEST = 0x1p-64f; // a row's largest magnitude counts as this at least
static_assert(UNG_HIP_INT8_CHUNK == CHUNK, "");
static_assert((uint64_t)UNG_HIP_INT8_LONGEST * 128 * 128 < 1ull << 31 && UNG_HIP_INT8_LONGEST % CHUNK == 0, "");

// ---- quantisation --------------------------------------------------------------------

__device__ inline float scale_of(uint32_t most)
{
    return __uint_as_float(max(most, __float_as_uint(SMALLEST))) * (1.0f / LARGEST);
}

template <class T>
__device__ inline uint32_t most_of(const Vec<T> &v, uint32_t most)
{
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e)
        most = max(most, magnitude(v.get(e)));
    return most;
}

// The vector's whole numbers: x / s rounded as a 32-bit division rounds, then to nearest even.
template <class T>
__device__ inline void store_numbers(const Vec<T> &v, Divisor by, uint8_t *to)
{
    constexpr int N = Vec<T>::N;
    uint32_t w[N / 4];
#pragma unroll
    for (int x = 0; x < N / 4; ++x) {
        w[x] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[x] |= ((uint32_t)(int)__builtin_rintf(quotient(v.get(x * 4 + e), by)) & 0xFFu) << (e * 8);
    }
    __builtin_memcpy(__builtin_assume_aligned(to, N), w, N);
}

// A wave takes one row: its largest magnitude, then the quotients.  Up to NV vectors a lane stay in
// registers between the two (one read of the row); NV = 0: rows of any length, read again.  Memory bounds
// it: 200000 x 768 float32 144 us, 5.3 TB/s; 4096 x 4096 bf16 11 us, 4.6.
template <class T, int NV>
__global__ __launch_bounds__(256) void ung_int8_rows_kernel(const T *x, uint64_t rows, uint64_t cols, uint64_t stride,
                                                            uint64_t chunks, uint8_t *q, float *scale)
{
    constexpr uint64_t N = Vec<T>::N, KEPT = NV ? NV : 1;
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t cp = chunks * CHUNK;
    for (uint64_t row = blockIdx.x * 4ull + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4ull) {
        const T *from = x + row * stride;
        uint8_t *to = q + row * cp;
        Vec<T> v[KEPT];
        uint32_t most = 0;
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                v[i] = load_row(from, (i * 64 + lane) * N, cols);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                most = most_of(v[i], most);
        } else {
            for (uint64_t c = lane * N; c < cols; c += 64 * N)
                most = most_of(load_row(from, c, cols), most);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            most = max(most, (uint32_t)__shfl_xor((int)most, o));
        const bool finite = most < 0x7F800000u;
        const float s = scale_of(most);
        if (lane == 0)
            scale[row] = finite ? s : __uint_as_float(0x7FC00000u);
        const Divisor by(finite ? s : 1.0f);
        auto put = [&](Vec<T> u, uint64_t c) {
            if (!finite) // its products are NaN by the scale
                u.w[0] = u.w[1] = u.w[2] = u.w[3] = 0;
            store_numbers(u, by, to + c);
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint64_t c = (i * 64 + lane) * N;
                if (c < cp)
                    put(v[i], c);
            }
        } else {
            for (uint64_t c = lane * N; c < cp; c += 64 * N)
                put(load_row(from, c, cols), c);
        }
    }
}

// ---- product -------------------------------------------------------------------------

// The sum, exact in 32 bits, times the rows' scales: a 32-bit number, whatever follows (the
// compiler would make one instruction of the product and its rounding to fp16, which rounds once
// less than where it does not).
__device__ inline float scaled(int sum, float by)
{
    float y = (float)sum * by;
    asm("" : "+v"(y));
    return y;
}

// Sums to results.  With it the product 4096 x 4096 of 4096 takes 61 us, 2250 TOPS (the library's large
// products 2430; in a card's first calls 67 us, and 2090); 77 x 30001 of 768 9.3 us by 64 x 128 tiles, two a CU.
template <class T>
struct Scaled : Plainly {
    const float *a_scale, *b_scale;
    T *c;
    uint64_t c_stride, m, n;
    int vectors;

    template <int TM>
    __device__ inline void operator()(const Tile &t, const uint8_t *, i32x4 (&acc)[TM][4], uint8_t *lds) const
    {
        const uint32_t r = t.lane & 15, g = t.lane >> 4;
        const uint64_t col0 = t.n0 + t.wn;
        if (col0 >= n)
            return;
        f32x4 sb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sb[j][e] = b_scale[min(col0 + g * 16 + j * 4 + e, n - 1)];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const uint64_t row0 = t.m0 + t.wm + i * 16;
            if (row0 >= m)
                return;
            const uint32_t rows = (uint32_t)min(m - row0, (uint64_t)16);
            const float sa = a_scale[min(row0 + r, m - 1)];
            Vec<T> o[16 / Vec<T>::N];
#pragma unroll
            for (int e = 0; e < 16; e += 2)
                o[e / Vec<T>::N].put2(e % Vec<T>::N, scaled(acc[i][e / 4][e % 4], sa * sb[e / 4][e % 4]),
                                      scaled(acc[i][e / 4][e % 4 + 1], sa * sb[e / 4][e % 4 + 1]));
            store_rows(c + row0 * c_stride + col0, c_stride, rows, n - col0, vectors, o, lds + t.wave * turn_bytes(sizeof(T)), t.lane);
            __builtin_amdgcn_sched_barrier(0); // 16 rows at a time: all of them need more registers than there are
        }
    }
};

// The sums of a share of the inner length, as they are.
struct Shares : Plainly {
    float *part; // whole numbers, moved as 32-bit elements
    uint64_t stride, m, n;

    template <int TM>
    __device__ inline void operator()(const Tile &t, const uint8_t *, i32x4 (&acc)[TM][4], uint8_t *lds) const
    {
        const uint64_t col0 = t.n0 + t.wn;
        if (col0 >= n)
            return;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const uint64_t row0 = t.m0 + t.wm + i * 16;
            if (row0 >= m)
                return;
            Vec<float> o[4];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                o[e / 4].w[e % 4] = (uint32_t)acc[i][e / 4][e % 4];
            store_rows(part + (t.split * m + row0) * stride + col0, stride, (uint32_t)min(m - row0, (uint64_t)16),
                       stride - col0, true, o, lds + t.wave * turn_bytes(4), t.lane);
        }
    }
};

// Up to FEW short rows x against many rows of b in whole numbers, in one launch.  The blocks stay: a wave
// brings a row of x to whole numbers in LDS, while its first chunks of b are under way, and then
// takes 64 rows of b at a time, past LDS and without barriers.  4 x 384 against 1000 rows 6.4 us, in two
// launches 7.1; 100000 rows 10.5 and 11.9; 1000000 rows 94 and 87.  With longer rows the first step costs
// more than the launch: 1 x 1536 against 1000 rows 14.7 and 9.8.
constexpr uint32_t FEW = 4, FEW_LONG = 512, FEW_TABLE = 200000;
static_assert(FEW_LONG == 4 * CHUNK, "a row is two loads of two chunks");

template <class X, class T>
__global__ __launch_bounds__(256) void ung_int8_few_rows_kernel(const X *x, uint64_t cols, uint64_t stride, uint32_t m,
                                                                Operand b, uint32_t strips, Scaled<T> finish)
{
    constexpr uint32_t PITCH = FEW_LONG + 16;
    __shared__ alignas(16) uint8_t numbers[FEW * PITCH];
    __shared__ alignas(16) uint8_t turned[4 * turn_bytes(sizeof(T))];
    __shared__ float scales[FEW];
    Tile at = {};
    at.high = 16;
    at.strips = 1;
    at.lane = threadIdx.x & 63;
    at.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t strip = blockIdx.x * 4 + at.wave;
    Stream<int8_t> right;
    u32x4 y[2][2][2][4]; // the first two chunks of a row and the others
    auto load = [&](int set) {
        right.load(y[set][0]);
        right.load(y[set][1]);
        __builtin_amdgcn_sched_barrier(0); // not where their registers are needed next
    };
    auto begin = [&]() {
        right.begin(b, (uint64_t)strip * 64, at.lane);
        load(0);
    };
    if (strip < strips)
        begin();
    if (at.wave < m) {
        constexpr uint32_t N = Vec<X>::N, NV = FEW_LONG / (64 * N);
        const X *from = x + at.wave * stride;
        Vec<X> v[NV];
        uint32_t most = 0;
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i)
            v[i] = load_row(from, (i * 64 + at.lane) * N, cols);
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i)
            most = most_of(v[i], most);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            most = max(most, (uint32_t)__shfl_xor((int)most, o));
        const bool finite = most < 0x7F800000u;
        const float s = scale_of(most);
        const Divisor by(finite ? s : 1.0f);
        if (at.lane == 0)
            scales[at.wave] = finite ? s : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (uint32_t i = 0; i < NV; ++i) {
            if (!finite)
                v[i].w[0] = v[i].w[1] = v[i].w[2] = v[i].w[3] = 0;
            store_numbers(v[i], by, numbers + at.wave * PITCH + (i * 64 + at.lane) * N);
        }
    }
    __syncthreads();
    finish.a_scale = scales;
    // lanes of rows past the last one take another's; their results are not stored
    const uint8_t *row = numbers + (at.lane & (FEW - 1)) * PITCH + (at.lane >> 4) * 16;
    for (; strip < strips; strip += gridDim.x * 4) {
        i32x4 acc[1][4];
        finish.start(at, acc);
        auto multiply = [&](int set, uint32_t first) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const u32x4 f = *reinterpret_cast<const u32x4 *>(row + first * CHUNK + h * 64);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[0][j] = Matrix<int8_t>::mul(y[set][h / 2][h % 2][j], f, acc[0][j]);
            }
        };
        load(1); // chunks past the end are zeros of b, and of x's numbers
        multiply(0, 0);
        multiply(1, 2);
        at.n0 = (uint64_t)strip * 64;
        if (strip + gridDim.x * 4 < strips) {
            strip += gridDim.x * 4;
            begin();
            strip -= gridDim.x * 4;
        }
        finish(at, nullptr, acc, turned);
    }
}

template <class T>
__global__ __launch_bounds__(256) void ung_int8_join_kernel(const int *part, uint32_t splits, uint64_t m, uint64_t n,
                                                            uint64_t stride, const float *a_scale, const float *b_scale,
                                                            T *c, uint64_t c_stride)
{
    const uint64_t quads = stride / 4;
    for (uint64_t at = blockIdx.x * 256ull + threadIdx.x; at < m * quads; at += gridDim.x * 256ull) {
        const uint64_t row = at / quads, col = (at - row * quads) * 4;
        i32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
        for (uint32_t s = 0; s < splits; ++s)
            sum += *reinterpret_cast<const i32x4 *>(part + (s * m + row) * stride + col);
        const float sa = a_scale[row];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < n)
                c[row * c_stride + col + e] = from_float<T>(scaled(sum[e], sa * b_scale[col + e]));
    }
}

// ---- choice of the kernel ----------------------------------------------------------------

struct Plan {
    uint32_t high, wide, splits;
};

Plan plan_of(uint64_t m, uint64_t n, uint64_t kp)
{
    const uint64_t chunks = kp / CHUNK, cus = cu_count();
    Plan p = {128, 128, 1};
    if (m == 0 || n == 0 || chunks == 0)
        return p;
    if (m > 128 && n > 128) {
        const uint64_t tiles = ceil_div(m, BIG) * ceil_div(n, BIG);
        if (tiles * 8 > ceil_div(tiles, cus) * cus * 5)
            return {BIG, BIG, 1};
    }
    const bool few_tiles = ceil_div(m, 64) * ceil_div(n, 128) <= 3 * cus;
    p.high = m <= 32 ? 32 : m <= 64 || few_tiles ? 64 : 128;
    const uint64_t tiles = ceil_div(m, p.high) * ceil_div(n, 128);
    const double traffic = (double)m * (double)n * 8 / 3e6;
    double best = 0.6 * (double)chunks;
    for (uint64_t s = 2; s * tiles <= 2 * cus && s * 2 <= chunks; ++s) {
        const double cost = 0.6 * (double)ceil_div(chunks, s) + 4.0 + (0.1 + traffic) * (double)s;
        if (cost < best) {
            best = cost;
            p.splits = (uint32_t)s;
        }
    }
    return p;
}

uint64_t share_stride(uint64_t n) { return ceil_div(n, 64) * 64; }
uint64_t share_bytes(uint64_t m, uint64_t n, uint32_t splits)
{
    return splits > 1 ? (uint64_t)splits * m * share_stride(n) * 4 : 0;
}

int check_product(const char *what, uint64_t m, uint64_t n, uint64_t kp, int type)
{
    if (!known_type(type)) {
        set_error("%s: unknown element type %d", what, type);
        return UNG_HIP_EINVAL;
    }
    if (kp % CHUNK || kp > UNG_HIP_INT8_LONGEST) {
        set_error("%s: inner length %llu is no multiple of %u up to %u", what, (unsigned long long)kp, CHUNK,
                  (unsigned)UNG_HIP_INT8_LONGEST);
        return UNG_HIP_EINVAL;
    }
    if (m && n && (m > INT32_MAX || n > INT32_MAX || ceil_div(m, 32) * ceil_div(n, 128) > most_blocks(256))) {
        set_error("%s: a %llu x %llu x %llu product is too large", what, (unsigned long long)m, (unsigned long long)n,
                  (unsigned long long)kp);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}


// ---- the calls' checks and launches ----------------------------------------------------------

int check_rows(const char *what, const void *x, int type, uint64_t rows, uint64_t cols, uint64_t row_stride)
{
    if (!known_type(type)) {
        set_error("%s: unknown element type %d", what, type);
        return UNG_HIP_EINVAL;
    }
    if (rows && cols && !x) {
        set_error("%s: null argument", what);
        return UNG_HIP_EINVAL;
    }
    if (rows > 1 && row_stride < cols) {
        set_error("%s: row_stride %llu is less than %llu columns", what, (unsigned long long)row_stride,
                  (unsigned long long)cols);
        return UNG_HIP_EINVAL;
    }
    if (rows > UINT32_MAX || cols > UINT32_MAX) {
        set_error("%s: %llu x %llu elements are too many", what, (unsigned long long)rows, (unsigned long long)cols);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

// The other side of a product and its results.
int check_results(const char *what, const int8_t *b, const float *b_scale, uint64_t m, uint64_t n, uint64_t kp,
                  const void *c, int type, uint64_t c_stride)
{
    if (!c || !b_scale || (kp && !b)) {
        set_error("%s: null argument", what);
        return UNG_HIP_EINVAL;
    }
    if (m > 1 && c_stride < n) {
        set_error("%s: c_stride %llu is less than %llu columns", what, (unsigned long long)c_stride,
                  (unsigned long long)n);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)b % 16 || (uintptr_t)b_scale % 4 || (uintptr_t)c % type_size(type)) {
        set_error("%s: whole numbers need 16-byte alignment, the rest that of its elements", what);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

int check_workspace(const char *what, uint64_t needed, const void *workspace, uint64_t bytes)
{
    if (needed && (!workspace || bytes < needed || (uintptr_t)workspace % 16)) {
        set_error("%s: needs %llu bytes of workspace at a 16-byte boundary (got %llu)", what, (unsigned long long)needed,
                  (unsigned long long)(workspace ? bytes : 0));
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

void quantize(const void *x, int type, uint64_t rows, uint64_t cols, uint64_t row_stride, int8_t *q, float *scale,
              hipStream_t st)
{
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const uint64_t chunks = ceil_div(cols, CHUNK), blocks = ceil_div(rows, 4), cp = chunks * CHUNK;
        const uint32_t grid = (uint32_t)(blocks < 8192 ? blocks : 8192);
        auto go = [&](auto kernel) {
            kernel<<<grid, 256, 0, st>>>((const T *)x, rows, cols, row_stride, chunks, (uint8_t *)q, scale);
        };
        constexpr uint64_t once = 64 * Vec<T>::N; // elements of a vector for each lane
        if (cp <= once)
            go(ung_int8_rows_kernel<T, 1>);
        else if (cp <= 2 * once)
            go(ung_int8_rows_kernel<T, 2>);
        else if (cp <= 4 * once)
            go(ung_int8_rows_kernel<T, 4>);
        else if (cp <= 8 * once)
            go(ung_int8_rows_kernel<T, 8>);
        else
            go(ung_int8_rows_kernel<T, 0>);
        return 0;
    });
}

bool vectors_at(const void *c, uint64_t c_stride, uint64_t m, uint64_t size)
{
    return (uintptr_t)c % 4 == 0 && (m == 1 || c_stride * size % 4 == 0);
}

void product(const int8_t *a, const float *a_scale, const int8_t *b, const float *b_scale, uint64_t m, uint64_t n,
             uint64_t kp, void *c, int type, uint64_t c_stride, const Plan &plan, void *workspace, hipStream_t st)
{
    const Operand oa = {a, kp, m, kp}, ob = {b, kp, n, kp};
    auto run = [&](auto finish) {
        auto tiles = [&](auto high, auto wm, auto wn) {
            constexpr int BM = decltype(high)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
            const Grid grid = {(uint32_t)ceil_div(m, BM), (uint32_t)ceil_div(n, WN * 64), plan.splits, kp / CHUNK,
                               plan.high == BIG ? 16u : 8u};
            ung_tile_kernel<int8_t, BM, WM, WN, false, false>
                <<<grid.m_tiles * grid.n_tiles * grid.splits, WM * WN * 64, 0, st>>>(oa, ob, grid, finish);
        };
        constexpr std::integral_constant<int, 1> one;
        constexpr std::integral_constant<int, 2> two;
        if (plan.high == 32)
            tiles(std::integral_constant<int, 32>{}, one, two);
        else if (plan.high == 64)
            tiles(std::integral_constant<int, 64>{}, two, two);
        else if (plan.high == 128)
            tiles(std::integral_constant<int, 128>{}, two, two);
        else
            tiles(std::integral_constant<int, BIG>{}, two, std::integral_constant<int, 4>{});
    };
    with_type(type, [&](auto zero) {
        using T = decltype(zero);
        if (plan.splits == 1) {
            run(Scaled<T>{{}, a_scale, b_scale, (T *)c, c_stride, m, n, vectors_at(c, c_stride, m, sizeof(T))});
        } else {
            const uint64_t stride = share_stride(n), blocks = ceil_div(m * (stride / 4), 256);
            run(Shares{{}, (float *)workspace, stride, m, n});
            ung_int8_join_kernel<T><<<(uint32_t)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(
                (const int *)workspace, plan.splits, m, n, stride, a_scale, b_scale, (T *)c, c_stride);
        }
        return 0;
    });
}

// How linear is made: few short rows in one launch, or brought to whole numbers in the workspace first.
struct Linear {
    uint64_t kp, at_scale = 0, at_shares = 0, bytes = 0;
    bool few;
    Plan plan;
    Linear(uint64_t m, uint64_t n, uint64_t cols) : kp(ceil_div(cols, CHUNK) * CHUNK)
    {
        few = m <= FEW && kp && kp <= FEW_LONG && n <= FEW_TABLE;
        plan = plan_of(m, n, kp);
        if (few || !m || !n)
            return;
        at_scale = ceil_div(m * kp, 16) * 16;
        at_shares = at_scale + ceil_div(m * 4, 16) * 16;
        bytes = at_shares + share_bytes(m, n, plan.splits);
    }
};

} // namespace

extern "C" {

int ung_hip_int8_quantize(const void *x, int type, uint64_t rows, uint64_t cols, uint64_t row_stride, int8_t *q,
                          float *scale, void *stream)
{
    static const char what[] = "ung_hip_int8_quantize";
    clear_error();
    if (const int rc = check_rows(what, x, type, rows, cols, row_stride))
        return rc;
    if (rows == 0)
        return UNG_HIP_OK;
    if ((cols && !q) || !scale) {
        set_error("%s: null argument", what);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)q % 16 || (uintptr_t)x % type_size(type) || (uintptr_t)scale % 4) {
        set_error("%s: q needs 16-byte alignment, x and scale that of their elements", what);
        return UNG_HIP_EINVAL;
    }
    quantize(x, type, rows, cols, row_stride, q, scale, (hipStream_t)stream);
    return launched(what);
}

int ung_hip_int8_matmul_workspace(uint64_t m, uint64_t n, uint64_t kp, int type, uint64_t *bytes)
{
    static const char what[] = "ung_hip_int8_matmul_workspace";
    clear_error();
    if (!bytes) {
        set_error("%s: null bytes", what);
        return UNG_HIP_EINVAL;
    }
    if (const int rc = check_product(what, m, n, kp, type))
        return rc;
    *bytes = share_bytes(m, n, plan_of(m, n, kp).splits);
    return UNG_HIP_OK;
}

int ung_hip_int8_matmul(const int8_t *a, const float *a_scale, const int8_t *b, const float *b_scale, uint64_t m,
                        uint64_t n, uint64_t kp, void *c, int type, uint64_t c_stride, void *workspace,
                        uint64_t workspace_bytes, void *stream)
{
    static const char what[] = "ung_hip_int8_matmul";
    clear_error();
    if (const int rc = check_product(what, m, n, kp, type))
        return rc;
    if (m == 0 || n == 0)
        return UNG_HIP_OK;
    if (!a_scale || (kp && !a)) {
        set_error("%s: null argument", what);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)a % 16 || (uintptr_t)a_scale % 4) {
        set_error("%s: whole numbers need 16-byte alignment, the rest that of its elements", what);
        return UNG_HIP_EINVAL;
    }
    if (const int rc = check_results(what, b, b_scale, m, n, kp, c, type, c_stride))
        return rc;
    const Plan plan = plan_of(m, n, kp);
    if (const int rc = check_workspace(what, share_bytes(m, n, plan.splits), workspace, workspace_bytes))
        return rc;
    product(a, a_scale, b, b_scale, m, n, kp, c, type, c_stride, plan, workspace, (hipStream_t)stream);
    return launched(what);
}

int ung_hip_int8_linear_workspace(uint64_t rows, uint64_t cols, uint64_t n, int type, uint64_t *bytes)
{
    static const char what[] = "ung_hip_int8_linear_workspace";
    clear_error();
    if (!bytes) {
        set_error("%s: null bytes", what);
        return UNG_HIP_EINVAL;
    }
    if (const int rc = check_product(what, rows, n, ceil_div(cols, CHUNK) * CHUNK, type))
        return rc;
    *bytes = Linear(rows, n, cols).bytes;
    return UNG_HIP_OK;
}

int ung_hip_int8_linear(const void *x, int type, uint64_t rows, uint64_t cols, uint64_t row_stride, const int8_t *b,
                        const float *b_scale, uint64_t n, void *c, int c_type, uint64_t c_stride, void *workspace,
                        uint64_t workspace_bytes, void *stream)
{
    static const char what[] = "ung_hip_int8_linear";
    clear_error();
    const uint64_t kp = ceil_div(cols, CHUNK) * CHUNK;
    if (const int rc = check_product(what, rows, n, kp, c_type))
        return rc;
    if (const int rc = check_rows(what, x, type, rows, cols, row_stride))
        return rc;
    if (rows == 0 || n == 0)
        return UNG_HIP_OK;
    if ((uintptr_t)x % type_size(type)) {
        set_error("%s: x needs to be aligned to its elements", what);
        return UNG_HIP_EINVAL;
    }
    if (const int rc = check_results(what, b, b_scale, rows, n, kp, c, c_type, c_stride))
        return rc;
    const Linear how(rows, n, cols);
    if (const int rc = check_workspace(what, how.bytes, workspace, workspace_bytes))
        return rc;
    const hipStream_t st = (hipStream_t)stream;
    if (!how.few) {
        uint8_t *ws = (uint8_t *)workspace;
        float *scale = (float *)(ws + how.at_scale);
        quantize(x, type, rows, cols, row_stride, (int8_t *)ws, scale, st);
        product((int8_t *)ws, scale, b, b_scale, rows, n, kp, c, c_type, c_stride, how.plan, ws + how.at_shares, st);
        return launched(what);
    }
    return with_type(type, [&](auto x_zero) {
        using X = decltype(x_zero);
        return with_type(c_type, [&](auto c_zero) {
            using T = decltype(c_zero);
            const Operand ob = {b, kp, n, kp};
            const Scaled<T> finish = {{}, nullptr, b_scale, (T *)c, c_stride, rows, n,
                                      vectors_at(c, c_stride, rows, sizeof(T))};
            const uint32_t strips = (uint32_t)ceil_div(n, 64), blocks = (uint32_t)ceil_div(strips, 4), most = 2 * cu_count();
            ung_int8_few_rows_kernel<X, T><<<blocks < most ? blocks : most, 256, 0, st>>>(
                (const X *)x, cols, row_stride, (uint32_t)rows, ob, strips, finish);
            return launched(what);
        });
    });
}

} // extern "C"
