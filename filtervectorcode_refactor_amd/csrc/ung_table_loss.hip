// ung_table_loss.hip -- cross entropy of hidden states against every row of a table, and its
// gradients, without a large batch's scores in memory, on gfx950: the kernels and the entry points
// ung_hip_table_loss_* of include/ung_hip.h.
//
//   z_ij = x_i . t_j / T   (j not left out by row i)        lse_i = log sum_j exp z_ij
//   loss_i = lse_i - z_i,id                                  0 for rows without a target
//   g_ij = w_i / T (exp(z_ij - lse_i) - [j = id_i])          dX = G T,  dT = G^T X
//
// The forward pass makes tiles of scores and keeps of each only its rows' largest score and sum
// of exponentials.  The backward pass makes the scores anew, a piece of the table's rows at a
// time: G of the piece goes to memory in the inputs' type, where two products read it.  Few scores of
// long rows go through memory as sums of shares of the inner length.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "ung_elements.h"
#include "ung_hip.h"
#include "ung_internal.h"
#include "ung_tiles.h"

using namespace ung;

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float INF = __builtin_huge_valf();
constexpr int WHOLE = 256; // columns that every tile's width divides

// ---- forward -------------------------------------------------------------------------

// A row's part of a tile of scores: sum 2^(c s - top) with c = log2(e) / T and `top` the whole number
// nearest to the largest c s.  So a term's exponent is rounded once, near 0 where it counts, and parts
// are joined with factors that are powers of two.
struct Part {
    float top, sum;
};
constexpr float NO_TOP = -INF; // of a part without a score

__device__ inline Part joined(Part a, Part b)
{
    const float top = fmaxf(a.top, b.top), from = top == NO_TOP ? 0.0f : top;
    return {top, a.sum * __builtin_amdgcn_exp2f(a.top - from) + b.sum * __builtin_amdgcn_exp2f(b.top - from)};
}

// Of a tile of scores (rows of x, columns: rows of the table): every row's part, and the
// target's score where the tile holds it.  A lane makes a part of its 16 columns; the block joins them.
//   A tile's begin and end bound it, when no wave of the CU's one block has products under way: its first
// loads, its exponentials and the join (4096 x 100000 of 384 bf16 359 us, 880 TFLOP/s, matrix instructions
// busy in 36 % of the cycles; 2000 x 50001 of 1024 216 us, 950 and 39 %, seven rounds of tiles, the last an
// eighth full; the library's large products 1610).
struct LogSum : Plainly {
    const int32_t *ids, *without;
    float *target; // [n]
    Part *parts;   // [tiles of the table][n]
    uint64_t n, v;
    float c; // log2(e) / T

    struct Columns { // of a row: the target's and the one left out
        int32_t id, out;
    };
    static constexpr uint32_t AHEAD = sizeof(Columns);
    __device__ inline void ahead(const Tile &t, uint8_t *side) const
    {
        if (threadIdx.x >= t.high)
            return;
        const uint64_t at = min(t.m0 + threadIdx.x, n - 1);
        reinterpret_cast<Columns *>(side)[threadIdx.x] = {ids[at], without ? without[at] : -1};
    }

    template <int TM>
    __device__ inline void operator()(const Tile &t, const uint8_t *side, f32x4 (&acc)[TM][4], uint8_t *lds) const
    {
        Part *red = reinterpret_cast<Part *>(lds); // [4 strips][rows of the tile]
        const uint32_t r = t.lane & 15, g = t.lane >> 4, high = t.high;
        const uint64_t col0 = t.n0 + t.wn + g * 16;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const uint64_t row = t.m0 + t.wm + i * 16 + r;
            const Columns of = reinterpret_cast<const Columns *>(side)[t.wm + i * 16 + r];
            const uint32_t id = (uint32_t)of.id - (uint32_t)col0, out = (uint32_t)of.out - (uint32_t)col0;
            if (__any(id < 16 || out < 16 || col0 + 16 > v)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if (id == e && row < n)
                        target[row] = acc[i][e / 4][e % 4];
                    if (out == e || col0 + e >= v)
                        acc[i][e / 4][e % 4] = -INF;
                }
            }
            float top = acc[i][0][0];
#pragma unroll
            for (int e = 1; e < 16; ++e)
                top = fmaxf(top, acc[i][e / 4][e % 4]);
            top = __builtin_rintf(top * c);
            const float from = top == NO_TOP ? 0.0f : -top;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][e / 4][e % 4], c, from));
            red[(t.wn / 16 + g) * high + t.wm + i * 16 + r] = {top, sum};
            __builtin_amdgcn_sched_barrier(0); // 16 rows at a time: all of them need more registers than there are
        }
        __syncthreads();
        const uint64_t row = t.m0 + threadIdx.x;
        if (threadIdx.x < high && row < n) {
            Part p = red[threadIdx.x];
            for (uint32_t w = 1; w < t.strips * 4; ++w)
                p = joined(p, red[w * high + threadIdx.x]);
            parts[t.n0 / (t.strips * 64) * n + row] = p;
        }
    }
};

__device__ inline bool has_target(int32_t id, const int32_t *without, uint64_t row, uint64_t v)
{
    return (uint64_t)(uint32_t)id < v && !(without && without[row] == id);
}

// R rows a block, 256 / R threads each: a row's parts to its log-sum-exp and loss.  A launch's latency and
// the few parts' bound it: 3.5 to 6.5 us from 1 to 4096 rows of up to 1563 parts.
template <int R>
__global__ __launch_bounds__(256) void ung_table_join_kernel(const Part *parts, uint64_t tiles, uint64_t n, uint64_t v,
                                                             const float *target, const int32_t *ids,
                                                             const int32_t *without, float c, float *loss, float *lse)
{
    __shared__ Part red[256];
    constexpr uint32_t EACH = 256 / R;
    constexpr float LN2 = 0.693147180559945309417f;
    const uint32_t in = threadIdx.x % R, which = threadIdx.x / R;
    const uint64_t row = (uint64_t)blockIdx.x * R + in;
    Part p = {NO_TOP, 0.0f};
    if (row < n) {
#pragma unroll 4
        for (uint64_t t = which; t < tiles; t += EACH)
            p = joined(p, parts[t * n + row]);
    }
    red[threadIdx.x] = p;
    __syncthreads();
#pragma unroll
    for (uint32_t half = EACH / 2; half; half /= 2) {
        if (which < half)
            red[threadIdx.x] = joined(red[threadIdx.x], red[threadIdx.x + half * R]);
        __syncthreads();
    }
    if (which || row >= n)
        return;
    p = red[in];
    const float log_sum = log2f(p.sum);
    const int32_t id = ids[row];
    const bool there = has_target(id, without, row, v);
    // as the logarithm of a quotient, which is 1 or more as the sum holds the target's term; as a
    // difference where that term is nothing beside the sum
    const float u = __builtin_fmaf(there ? target[row] : 0.0f, c, -p.top);
    const float nll = u > -100.0f ? log2f(p.sum / __builtin_amdgcn_exp2f(u)) : log_sum - u;
    loss[row] = there ? nll * LN2 : 0.0f;
    // in 64 bits, rounded once: half a step of 32 is 3e-5 of all the row's weights at a score of 1000
    lse[row] = (float)((double)p.top * 0.69314718055994530942 + log((double)p.sum));
}

// ---- backward ------------------------------------------------------------------------

// What the gradient needs of a row: the log-sum-exp in bits, in 32 bits and so off by some r; weight / T,
// as weight 2^-r, and `one` = 2^r in the place of the target's 1, so that r is in no share exp2(c s - lse2)
// weight; the target and the column left out.  A row without a target: weight 0, log-sum-exp +inf and zeros
// in the place of x, so that no number of a row of padding reaches the table's gradient.
struct alignas(16) Row {
    float lse2, weight, one;
    int32_t id, out;
};
__device__ inline Row row_of(float lse, float weight, int32_t id, int32_t out)
{
    const double bits = (double)lse * 1.44269504088896340736;
    const float lse2 = (float)bits, r = fabsf(lse2) < INF ? (float)(bits - (double)lse2) : 0.0f;
    return {lse2, weight * exp2f(-r), exp2f(r), id, out};
}

// fp16 holds no numbers below 2^-24: weights are brought to the top of its range by a power of
// two (G is at most 2 |w| / T), which the gradients are divided by at the end.  Weights of rows without a
// target do not count: padding of any size would take the others' numbers out of range.  scale: {by, 1 / by}.
// One block, 4.7 us for 2048 weights: a launch's latency, for fp16 alone.
__global__ __launch_bounds__(1024) void ung_table_range_kernel(const float *weight, uint64_t n, uint64_t v, const int32_t *ids,
                                                               const int32_t *without, float by, float *scale)
{
    __shared__ float red[16];
    float most = weight || !n ? 0.0f : 1.0f;
    if (weight)
        for (uint64_t i = threadIdx.x; i < n; i += 1024) {
            const float w = fabsf(weight[i]);
            if (w < INF && has_target(ids[i], without, i, v))
                most = fmaxf(most, w);
        }
    most = block_reduce<1024>(most, red, [](float a, float b) { return fmaxf(a, b); }) * by;
    if (threadIdx.x == 0) {
        int e = 0;
        if (most > 0.0f && most < INF)
            (void)frexpf(most, &e); // most < 2^e
        e = 14 - e;
        e = e > 100 ? 100 : e < -100 ? -100 : e;
        scale[0] = ldexpf(1.0f, e);
        scale[1] = ldexpf(1.0f, -e);
    }
}

// A wave a row: its numbers, and its elements as rows of whole vectors (`pitch`: elements, whole vectors).
// Latency bounds it: 3 us for 500 x 100 float32, 5.2 for 4096 x 384 bf16.
template <class E>
__global__ __launch_bounds__(256) void ung_table_rows_kernel(const E *x, uint64_t stride, uint64_t n, uint64_t v,
                                                             uint64_t d, const int32_t *ids, const int32_t *without,
                                                             const float *lse, const float *weight, float by,
                                                             const float *scale, Row *rows, int32_t *targets, E *to,
                                                             uint64_t pitch)
{
    const uint32_t lane = threadIdx.x & 63;
    for (uint64_t row = blockIdx.x * 4ull + (threadIdx.x >> 6); row < n; row += gridDim.x * 4ull) {
        const int32_t id = ids[row], out = without ? without[row] : -1;
        const bool there = has_target(id, without, row, v);
        if (lane == 0) {
            rows[row] = there ? row_of(lse[row], (weight ? weight[row] : 1.0f) * by * (scale ? scale[0] : 1.0f), id, out)
                              : Row{INF, 0.0f, 1.0f, -1, -1};
            targets[row] = there ? id : -1;
        }
        for (uint64_t c = lane * Vec<E>::N; c < pitch; c += 64 * Vec<E>::N)
            *reinterpret_cast<Vec<E> *>(to + row * pitch + c) = load_row(x + row * stride, c, there ? d : 0);
    }
}

// Rows of any stride and length as rows of whole vectors, `each` of them by a block at a time.  Memory
// bounds it: 100000 x 385 bf16 24 us, 100000 x 100 10; by single elements, a wave a row, 32 and 17.
template <class E>
__global__ __launch_bounds__(256) void ung_table_pack_kernel(const E *x, uint64_t stride, uint64_t rows, uint64_t d,
                                                             E *to, uint64_t pitch, uint32_t each)
{
    constexpr uint32_t N = Vec<E>::N;
    const uint32_t vectors = (uint32_t)(pitch / N);
    for (uint64_t row0 = (uint64_t)blockIdx.x * each; row0 < rows; row0 += (uint64_t)gridDim.x * each) {
        const uint32_t all = (uint32_t)min(rows - row0, (uint64_t)each) * vectors;
        for (uint32_t i = threadIdx.x; i < all; i += 256) {
            const uint32_t r = i / vectors, c = (i - r * vectors) * N;
            *reinterpret_cast<Vec<E> *>(to + (row0 + r) * pitch + c) = load_row(x + (row0 + r) * stride, c, d);
        }
    }
}

// A tile of scores to G, in the inputs' type: at most half a step of it, 2^-8 of an element in bf16 and
// 2^-11 in fp16, as far as the gradients' own rounding; the products that read it sum in 32 bits.  Of a row's
// weights the target's is the largest, and alone in most rows of dT: what its rounding leaves is kept in
// 32 bits and joins dX with the table's row at the end (Rest), dT with the products (Targets).  4096 x 100000 x
// 384 bf16 at T = 0.05: 0.0017 of the norm from dX and dT, which their own rounding makes; 0.0038 and 0.0024 without.
template <class E>
struct Weights : Plainly {
    const Row *rows;
    float *rest; // [n]
    E *g; // [n][pitch], pitch whole tiles: columns past the piece's end are zero
    uint64_t pitch, n, v0, v;
    float c;

    static constexpr uint32_t AHEAD = sizeof(Row);
    __device__ inline void ahead(const Tile &t, uint8_t *side) const
    {
        if (threadIdx.x < t.high)
            reinterpret_cast<Row *>(side)[threadIdx.x] = rows[min(t.m0 + threadIdx.x, n - 1)];
    }

    template <int TM>
    __device__ inline void operator()(const Tile &t, const uint8_t *side, f32x4 (&acc)[TM][4], uint8_t *) const
    {
        const uint32_t r = t.lane & 15, gr = t.lane >> 4;
        const uint64_t col0 = t.n0 + t.wn + gr * 16;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const uint64_t row = t.m0 + t.wm + i * 16 + r;
            const Row p = reinterpret_cast<const Row *>(side)[t.wm + i * 16 + r];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc[i][e / 4][e % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][e / 4][e % 4], c, -p.lse2));
            const uint32_t id = (uint32_t)p.id - (uint32_t)(v0 + col0), out = (uint32_t)p.out - (uint32_t)(v0 + col0);
            if (__any(id < 16 || out < 16 || col0 + 16 > v)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if (id == e) {
                        acc[i][e / 4][e % 4] -= p.one;
                        if (row < n) {
                            const float all = acc[i][e / 4][e % 4] * p.weight;
                            rest[row] = all - to_float(from_float<E>(all));
                        }
                    }
                    if (out == e || col0 + e >= v)
                        acc[i][e / 4][e % 4] = 0.0f;
                }
            }
            Vec<E> o[16 / Vec<E>::N];
#pragma unroll
            for (int e = 0; e < 16; e += 2)
                o[e / Vec<E>::N].put2(e % Vec<E>::N, acc[i][e / 4][e % 4] * p.weight, acc[i][e / 4][e % 4 + 1] * p.weight);
            if (row < n)
#pragma unroll
                for (int x = 0; x < 16 / Vec<E>::N; ++x)
                    *reinterpret_cast<Vec<E> *>(g + row * pitch + col0 + x * Vec<E>::N) = o[x];
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// ---- scores in shares of the inner length ------------------------------------------------------

// Where the rows are long and tiles of scores too few for the chip, the tiles' sums are made in shares
// (Sums), and these kernels take LogSum's and Weights' place: a wave four columns a lane of a row's 256,
// the shares added in order.  They cost a pass over the sums.  Both passes, us, with shares and
// without: 613 x 3520 of 4096 float32 679 and 851, 983 x 859 296 and 437; 3 x 145 of 1984 34 and 116;
// bf16 225 x 1269 of 4096 61 and 103, 3 x 5269 63 and 105.
__device__ inline f32x4 shares_sum(const float *part, uint32_t splits, uint64_t n, uint64_t stride, uint64_t row, uint64_t col)
{
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t k = 0; k < splits; ++k)
        s += *reinterpret_cast<const f32x4 *>(part + (k * n + row) * stride + col);
    return s;
}

__global__ __launch_bounds__(256) void ung_table_parts_kernel(const float *part, uint32_t splits, uint64_t stride, LogSum f)
{
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t strips = stride / WHOLE;
    for (uint64_t item = blockIdx.x * 4ull + (threadIdx.x >> 6); item < f.n * strips; item += gridDim.x * 4ull) {
        const uint64_t row = item / strips, strip = item - row * strips, col = strip * WHOLE + lane * 4;
        f32x4 s = shares_sum(part, splits, f.n, stride, row, col);
        const uint32_t id = (uint32_t)f.ids[row] - (uint32_t)col, out = (uint32_t)(f.without ? f.without[row] : -1) - (uint32_t)col;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (id == e)
                f.target[row] = s[e];
            if (out == e || col + e >= f.v)
                s[e] = -INF;
        }
        float top = wave_reduce(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), [](float a, float b) { return fmaxf(a, b); });
        top = __builtin_rintf(top * f.c);
        const float from = top == NO_TOP ? 0.0f : -top;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], f.c, from));
        sum = wave_reduce(sum, [](float a, float b) { return a + b; });
        if (lane == 0)
            f.parts[strip * f.n + row] = {top, sum};
    }
}

template <class E>
__global__ __launch_bounds__(256) void ung_table_weights_kernel(const float *part, uint32_t splits, uint64_t stride, Weights<E> f)
{
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t strips = stride / WHOLE;
    for (uint64_t item = blockIdx.x * 4ull + (threadIdx.x >> 6); item < f.n * strips; item += gridDim.x * 4ull) {
        const uint64_t row = item / strips, col = (item - row * strips) * WHOLE + lane * 4;
        const f32x4 s = shares_sum(part, splits, f.n, stride, row, col);
        const Row p = f.rows[row];
        const uint32_t id = (uint32_t)p.id - (uint32_t)(f.v0 + col), out = (uint32_t)p.out - (uint32_t)(f.v0 + col);
        alignas(4 * sizeof(E)) E o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], f.c, -p.lse2));
            if (id == e) {
                y -= p.one;
                const float all = y * p.weight;
                f.rest[row] = all - to_float(from_float<E>(all));
            }
            if (out == e || col + e >= f.v)
                y = 0.0f;
            o[e] = from_float<E>(y * p.weight);
        }
        __builtin_memcpy(__builtin_assume_aligned(f.g + row * f.pitch + col, sizeof o), o, sizeof o);
    }
}

// The rest of the targets' weights (rows null: none), added to dX.
template <class E>
struct Rest {
    const Row *rows;
    const float *rest;
    const E *table;
    uint64_t stride;

    // What the row's `N` columns from col get; those at or past `cols` are not read.
    template <int N>
    __device__ inline void add(uint64_t row, uint64_t col, uint64_t cols, float (&to)[N]) const
    {
        if (!rows)
            return;
        const int32_t id = rows[row].id;
        if (id < 0)
            return;
        const float r = rest[row];
        const E *from = table + (uint64_t)id * stride + col; // (rows of whole vectors)
        E t[N] = {};
        if (col + N <= cols)
            __builtin_memcpy(t, __builtin_assume_aligned(from, std::min<int>(sizeof t, 16)), sizeof t);
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (col + e < cols)
                    t[e] = from[e];
#pragma unroll
        for (int e = 0; e < N; ++e)
            to[e] = __builtin_fmaf(r, to_float(t[e]), to[e]);
    }
};

// The same for dT = G^T X: row i of x times its rest joins row id of dT.  So G has a second part with one
// element a row, of 16 bits too: what is left then is 2^-17 of a weight in bf16, 2^-22 in fp16.  A wave
// looks at 64 ids a chunk, and makes fragments of the second part for the halves of groups of 16 rows that
// hold some.  The backward pass with it and without, us: 4096 x 100000 of 384 bf16 1187 and 1181, 2000 x 2000
// of 768 58 and 52; where every chunk has targets, 4366 x 201 of 4096, 107 and 87.
template <class E>
struct Targets {
    static constexpr uint32_t MORE = 64 * 4; // of the chunk's rows: place among the wave's rows, and the rest
    const int32_t *targets;                  // [n], -1: none; one is there where n is 0
    const float *rest;
    uint32_t n, v0; // v0: row of the table that the product's first is

    struct Next {
        uint32_t k; // of the whole wave
        int32_t id;
        float rest;
    };
    __device__ inline void fetch(Next &next, uint32_t lane) const
    {
        const uint32_t at = next.k + lane < n ? next.k + lane : 0;
        next.id = targets[at]; // (looked at where the next chunk is: here it would be waited for)
        next.rest = rest[at];
    }
    __device__ inline void first(Next &next, uint32_t k, uint32_t lane) const
    {
        static_assert(sizeof(E) == 2 && CHUNK == 64 * sizeof(E), "a lane for each row of a chunk");
        next.k = k;
        fetch(next, lane);
    }
    template <int TM>
    __device__ inline uint32_t holds(Next &next, const Tile &t, uint8_t *own) const
    {
        const uint32_t place = next.k + t.lane < n ? (uint32_t)next.id - (v0 + (uint32_t)t.m0 + t.wm) : TM * 16;
        const uint32_t rounded = __builtin_bit_cast(uint16_t, from_float<E>(next.rest));
        next.k += 64;
        fetch(next, t.lane);
        uint32_t held = 0;
        if (__any(place < TM * 16)) {
            reinterpret_cast<uint32_t *>(own)[t.lane] = place < TM * 16 ? place << 16 | rounded : 0xFFFF0000u;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const uint64_t of = __ballot(place / 16 == i);
                held |= ((uint32_t)of ? 1u << i : 0u) | ((uint32_t)(of >> 32) ? 1u << (16 + i) : 0u);
            }
            wave_lds_fence();
        }
        return held;
    }
    __device__ inline u32x4 more(const uint8_t *own, int i, int half, uint32_t lane) const
    {
        const u32x4 *const at = reinterpret_cast<const u32x4 *>(own + (half * 32 + (lane >> 4) * 8) * 4);
        const u32x4 lo = at[0], hi = at[1];
        const uint32_t place = i * 16 + (lane & 15);
        u32x4 f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t a = q < 2 ? lo[q * 2] : hi[q * 2 - 4], b = q < 2 ? lo[q * 2 + 1] : hi[q * 2 - 3];
            f[q] = (a >> 16 == place ? a & 0xFFFFu : 0u) | (b >> 16 == place ? b << 16 : 0u);
        }
        return f;
    }
};
struct NoTargets {
    static constexpr uint32_t MORE = 0;
    struct Next {};
};
template <class E> // of dT: float32 weights are not rounded
using TargetsOf = std::conditional_t<sizeof(E) == 2, Targets<E>, NoTargets>;

// A gradient's tile in its own type.
template <class E, class More>
struct Whole : Plainly, More {
    using More::MORE;
    using Next = typename More::Next;
    E *c;
    uint64_t stride, m, n;
    const float *by;
    int vectors;
    Rest<E> rest;

    template <int TM>
    __device__ inline void operator()(const Tile &t, const uint8_t *, f32x4 (&acc)[TM][4], uint8_t *lds) const
    {
        const uint64_t col0 = t.n0 + t.wn;
        if (col0 >= n)
            return;
        const float s = by ? by[0] : 1.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const uint64_t row0 = t.m0 + t.wm + i * 16;
            if (row0 >= m)
                return;
            float all[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                all[e] = acc[i][e / 4][e % 4];
            if (row0 + (t.lane & 15) < m)
                rest.add(row0 + (t.lane & 15), col0 + (t.lane >> 4) * 16, n, all);
            Vec<E> o[16 / Vec<E>::N];
#pragma unroll
            for (int e = 0; e < 16; e += 2)
                o[e / Vec<E>::N].put2(e % Vec<E>::N, all[e] * s, all[e + 1] * s);
            store_rows(c + row0 * stride + col0, stride, (uint32_t)min(m - row0, (uint64_t)16), n - col0, vectors, o,
                       lds + t.wave * turn_bytes(sizeof(E)), t.lane);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// Sums of a share of the inner length in 32 bits, from 0 or (ADD) from an earlier piece's: dX, whose tiles
// are few and whose inner length is the table's.  4096 x 384 of 20224 bf16, 5 shares, 68 us (930 TFLOP/s),
// 72 onto an earlier piece's; 2048 x 768 of 32768 fp16 108 us (960): matrix instructions busy in 35 to 42 % of
// the cycles, a third of the LDS cycles bank conflicts of the transposing reads.
template <bool ADD, class More = NoTargets>
struct Sums : More {
    float *part;
    uint64_t stride, m; // stride: whole tiles

    static constexpr uint32_t AHEAD = 0;
    __device__ inline void ahead(const Tile &, uint8_t *) const {}
    __device__ inline f32x4 *at(const Tile &t, int i) const
    {
        const uint64_t row = min(t.m0 + t.wm + i * 16 + (t.lane & 15), m - 1);
        return reinterpret_cast<f32x4 *>(part + (t.split * m + row) * stride + t.n0 + t.wn + (t.lane >> 4) * 16);
    }
    template <int TM>
    __device__ inline void start(const Tile &t, f32x4 (&acc)[TM][4]) const
    {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = ADD ? at(t, i)[j] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    template <int TM>
    __device__ inline void operator()(const Tile &t, const uint8_t *, f32x4 (&acc)[TM][4], uint8_t *) const
    {
#pragma unroll
        for (int i = 0; i < TM; ++i)
            if (t.m0 + t.wm + i * 16 + (t.lane & 15) < m)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    at(t, i)[j] = acc[i][j];
    }
};

// The shares' sums in the gradient's type.  P threads add up every P-th share of four results, and are
// joined in order (1 x 384 results of 256 shares by one thread each 18.6 us).
template <class E, uint32_t P>
__global__ __launch_bounds__(256) void ung_table_sum_kernel(const float *part, uint32_t splits, uint64_t rows,
                                                            uint64_t cols, uint64_t part_stride, const float *by, E *c,
                                                            uint64_t c_stride, Rest<E> rest)
{
    constexpr uint32_t EACH = 256 / P; // quads of a block
    __shared__ f32x4 red[P > 1 ? 256 : 1];
    const uint64_t quads = (cols + 3) / 4, all = rows * quads;
    const uint32_t in = threadIdx.x % EACH, which = threadIdx.x / EACH;
    const float scale = by ? by[0] : 1.0f;
    for (uint64_t first = (uint64_t)blockIdx.x * EACH; first < all; first += (uint64_t)gridDim.x * EACH) {
        const uint64_t at = min(first + in, all - 1), row = at / quads, col = (at - row * quads) * 4;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (uint32_t s = which; s < splits; s += P)
            sum += *reinterpret_cast<const f32x4 *>(part + (s * rows + row) * part_stride + col);
        if constexpr (P > 1) {
            __syncthreads(); // the last round's sums are read
            red[threadIdx.x] = sum;
            __syncthreads();
            if (which)
                continue;
#pragma unroll
            for (uint32_t p = 1; p < P; ++p)
                sum += red[p * EACH + in];
        }
        if (first + in >= all)
            continue;
        float out[4] = {sum[0], sum[1], sum[2], sum[3]};
        rest.add(row, col, cols, out);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < cols)
                c[row * c_stride + col + e] = from_float<E>(out[e] * scale);
    }
}

// ---- plan and workspace ------------------------------------------------------------------

// How a product of m x n results is made: by tiles of `high` x `wide` in so many shares of the inner
// length, and about how long it takes.
struct Shape {
    uint32_t high, wide, splits;
    double us;
};

// The time of a chunk of a tile alone on its CU, or of each of the tiles there where they share its matrix
// instructions, and of a tile's begin and end: weights by which the faster plan is chosen, not times to
// be had.  Measured, us, bf16: 2048 x 32768 of 768 125 by 256 x 256, 137 by 128 x 128; 32768 x 768 of 2048
// 141 and 131 (1.5 rounds, 3 whole ones); 14336 x 384 of 4096 64 by 128 rows, 67 by 64; float32: 500 x
// 10001 of 100 24.4 by 128 rows, 19.6 by 64.
struct Weight {
    uint32_t high, wide, at_once; // tiles that fit a CU
    double alone, shared, ends;
};
// Tiles of 128 x 64 are for few columns: the backward pass of 1044 x 185304 of 64
// float32 1000 us (1304 by 128 columns), 2000 x 20000 of 64 bf16 78 (82), 3000 x 50000 of 192
// 339 (351), both passes of 6565 x 53 of 4096 float32 240 (283).
constexpr Weight WEIGHTS_16[] = {{BIG, BIG, 1, 1.75, 1.75, 5.0}, {128, 128, 2, 0.6, 0.52, 3.5}, {64, 128, 3, 0.55, 0.33, 3.0},
                                 {32, 128, 3, 0.5, 0.25, 2.5}, {128, 64, 3, 0.6, 0.40, 3.0}};
constexpr Weight WEIGHTS_32[] = {{128, 128, 2, 2.0, 1.95, 4.0}, {64, 128, 3, 1.1, 0.98, 3.0}, {32, 128, 3, 2.2, 0.8, 2.5},
                                 {128, 64, 3, 1.1, 0.98, 3.0}};

constexpr uint64_t MOST_SUMS = 64ull << 20;
// dT's tiles, which take Targets' fragments too: a tile of 256 x 256 has no registers to choose among its groups
// of rows, so every chunk with a target costs it all of them (backward pass of 8192 x 6000 of 768 bf16 365
// us, by 128 x 128 319).
constexpr uint32_t MOST_HIGH_T = 128;

// `shares`: sums may be made in shares of the inner length, joined by a pass of their own.  `most_high`: rows
// of the highest tile.
Shape shape_of(uint64_t m, uint64_t n, uint64_t k, int type, bool shares, uint32_t most_high = BIG)
{
    const uint64_t cus = cu_count(), chunks = ceil_div(k * type_size(type), CHUNK);
    Shape best = {32, 128, 1, 1e30};
    auto consider = [&](const Weight &w) {
        const uint64_t tiles = ceil_div(m, w.high) * ceil_div(n, w.wide);
        auto time = [&](uint64_t each, uint64_t steps) { // of a round with `each` tiles on a CU
            const double step = w.alone > w.shared * (double)each ? w.alone : w.shared * (double)each;
            return step * (double)steps + w.ends;
        };
        auto with = [&](uint64_t splits) {
            const uint64_t items = tiles * splits, places = w.at_once * cus, rounds = items / places, rest = items % places;
            const uint64_t steps = ceil_div(chunks, splits);
            Shape s = {w.high, w.wide, (uint32_t)splits, (double)rounds * time(w.at_once, steps)};
            if (rest)
                s.us += time(ceil_div(rest, cus), steps);
            if (splits > 1)
                s.us += 3.0 + (double)splits * (double)m * (double)n * 8 / 4e6;
            if (s.us < best.us)
                best = s;
        };
        if (!tiles || w.high > most_high)
            return;
        with(1);
        if (!shares)
            return;
        for (uint64_t each = 1; each <= w.at_once; ++each) {
            const uint64_t by_cu = each * cus / tiles, by_k = chunks / (w.high == BIG ? 8 : 2), most = by_cu < by_k ? by_cu : by_k;
            if (most > 1)
                with(most);
        }
        // rounds filled better by two to four shares of long rows: 49 x 72321 of 4096 float32 339 us, 383
        // without; in 16 bits the sums cost what they save (1200 x 3000 of 4096 bf16 50 us either way)
        for (uint64_t splits = 2; splits <= 4 && splits * 16 <= chunks; ++splits)
            if (type == UNG_HIP_F32 && splits * m * n * 4 <= MOST_SUMS)
                with(splits);
    };
    if (type == UNG_HIP_F32)
        for (const Weight &w : WEIGHTS_32)
            consider(w);
    else
        for (const Weight &w : WEIGHTS_16)
            consider(w);
    return best;
}

// dT and dX in one launch: the shape of dX, of whose height dT's tiles are too; us is 0 where two launches
// are faster.  Each alone leaves a part of the chip idle in its last or only round, and the second waits
// for the first's last tile.  The backward pass, us, by one launch and by two: 16 x 1000 of 64 bf16 12.7
// and 16.1, 500 x 10001 of 100 float32 62 and 72, 2000 x 2000 of 768 bf16 58 and 75, 300 x 20000 of 512 bf16
// 52 and 58.
Shape together_of(uint64_t n, uint64_t v, uint64_t d, int type, double two_us)
{
    const uint64_t cus = cu_count();
    const uint64_t x_chunks = ceil_div(v * type_size(type), CHUNK), t_chunks = ceil_div(n * type_size(type), CHUNK);
    Shape best = {0, 128, 1, two_us + 2.0};
    auto consider = [&](const Weight &w) {
        const uint64_t x_tiles = ceil_div(n, w.high) * ceil_div(d, w.wide), t_tiles = ceil_div(v, w.high) * ceil_div(d, w.wide);
        if (w.high == BIG || !x_tiles || !t_tiles)
            return;
        const double even = w.shared * (double)(x_tiles * x_chunks + t_tiles * t_chunks) / (double)cus;
        // dX in shares that leave every CU with the same number of tiles; the first CUs have the more of dT's
        const uint64_t of_t = ceil_div(t_tiles, cus);
        for (uint64_t each = of_t; each <= of_t + w.at_once; ++each) {
            const uint64_t splits = (each * cus - t_tiles) / x_tiles;
            if (splits < 2 || splits * 2 > x_chunks || splits > 256)
                continue;
            const uint64_t steps = ceil_div(x_chunks, splits);
            const double first = (double)(of_t * t_chunks + (each - of_t) * steps), longest = (double)std::max(steps, t_chunks);
            const double busy = each <= w.at_once ? w.shared * first : even + w.shared * (double)steps;
            const double us = std::max({even, busy, w.alone * longest}) + w.ends * (double)ceil_div(each, (uint64_t)w.at_once) +
                              3.0 + (double)splits * (double)n * (double)d * 8 / 4e6;
            if (us < best.us)
                best = {w.high, w.wide, (uint32_t)splits, us};
        }
        // few tiles in all: dX in shares as long as one of dT's
        const uint64_t splits = ceil_div(x_chunks, std::max<uint64_t>(t_chunks, 2));
        if (splits >= 2 && splits <= 256 && t_tiles + x_tiles * splits <= cus) {
            const double us = w.alone * (double)std::max<uint64_t>(t_chunks, 2) + w.ends + 3.0 +
                              (double)splits * (double)n * (double)d * 8 / 4e6;
            if (us < best.us)
                best = {w.high, w.wide, (uint32_t)splits, us};
        }
    };
    if (type == UNG_HIP_F32)
        for (const Weight &w : WEIGHTS_32)
            consider(w);
    else
        for (const Weight &w : WEIGHTS_16)
            consider(w);
    if (!best.high)
        best.us = 0.0;
    return best;
}

constexpr uint32_t FEW = 32; // rows that the table is streamed for

// How scores are made.  A wave of few rows takes 0.5 to 0.7 us for a chunk, one after the other.
Shape scores_shape(uint64_t n, uint64_t v, uint64_t d, int type)
{
    if (n > FEW)
        return shape_of(n, v, d, type, true);
    const uint64_t waves = ceil_div(v, 64), chunks = ceil_div(d * type_size(type), CHUNK);
    const uint64_t splits = chunks < 16 || !waves ? 1 : std::min<uint64_t>({4 * (uint64_t)cu_count() / waves, chunks / 4, 32});
    return {n <= 16 ? 16u : 32u, 64, splits > 1 ? (uint32_t)ceil_div(chunks, ceil_div(chunks, splits)) : 1, 0.0};
}

struct Inputs {
    const void *x, *table;
    uint64_t x_stride, table_stride;
    int type;
    uint64_t n, v, d;
};

// Where the parts of a workspace lie, all at 256-byte boundaries.
struct Layout {
    uint64_t bytes = 0;
    uint64_t take(uint64_t size)
    {
        const uint64_t at = bytes;
        bytes += ceil_div(size, 256) * 256;
        return at;
    }
};

struct Packed { // a side of the products, copied to rows of whole vectors where it does not lie so
    bool copy, loose; // loose: not in whole vectors where it lies
    uint64_t at, pitch; // bytes
};

// `as_it_lies`: where it is read at any alignment.
Packed packed(Layout &l, const void *p, uint64_t stride, uint64_t rows, uint64_t d, uint64_t size, bool always,
              bool as_it_lies = false)
{
    Packed o = {always, false, 0, ceil_div(d * size, 16) * 16};
    o.loose = (uintptr_t)p % 16 || d * size % 16 || (rows > 1 && stride * size % 16);
    if ((o.loose && !as_it_lies) || (rows > 1 && stride * size >= MOST_STRIDE))
        o.copy = true;
    if (o.copy)
        o.at = l.take(rows * o.pitch);
    return o;
}

struct Forward {
    Layout l;
    Packed x, table;
    Shape shape;
    uint64_t tiles, parts, target, sums, stride;
    bool loose;
    explicit Forward(const Inputs &in)
    {
        const uint64_t size = type_size(in.type);
        x = packed(l, in.x, in.x_stride, in.n, in.d, size, false, in.n <= FEW);
        table = packed(l, in.table, in.table_stride, in.v, in.d, size, false, in.n <= FEW);
        loose = (!x.copy && x.loose) || (!table.copy && table.loose);
        shape = scores_shape(in.n, in.v, in.d, in.type);
        stride = ceil_div(in.v, WHOLE) * WHOLE;
        tiles = ceil_div(in.v, shape.splits > 1 ? WHOLE : shape.wide);
        sums = shape.splits > 1 ? l.take(shape.splits * in.n * stride * 4) : 0;
        parts = l.take(tiles * in.n * sizeof(Part));
        target = l.take(in.n * 4);
    }
};

// G of a piece takes this much at most (it is read while it lies in the last-level cache), but for at
// least 1024 rows of the table.
constexpr uint64_t PIECE_BYTES = 168ull << 20;

struct Backward {
    Layout l;
    Packed x, table;
    uint64_t rows, scale, targets, rest, piece, pieces, g, g_sums, x_sums, t_sums, sum_stride;
    Shape g_shape, x_shape, t_shape;
    bool together = false; // dX and dT in one launch (where both are asked for)
    explicit Backward(const Inputs &in)
    {
        const uint64_t size = type_size(in.type);
        x = packed(l, in.x, in.x_stride, in.n, in.d, size, true);
        table = packed(l, in.table, in.table_stride, in.v, in.d, size, false);
        rows = l.take(in.n * sizeof(Row));
        scale = l.take(8);
        targets = l.take((in.n ? in.n : 1) * 4);
        rest = l.take((in.n ? in.n : 1) * 4);
        const uint64_t all = ceil_div(in.v, WHOLE) * WHOLE;
        uint64_t fits = PIECE_BYTES / ((in.n ? in.n : 1) * size) / WHOLE * WHOLE;
        fits = fits < 1024 ? 1024 : fits;
        // of the least number of pieces and half as many again, the one whose dT fills its rounds best
        // (4096 x 100000 x 384: 5 of 20224 rows 1596 us, 7 of 14336 1702, 4 of 25088 1686)
        const uint64_t least = all ? ceil_div(all, fits) : 1;
        piece = all;
        double best = 1e30;
        for (uint64_t p = least; p <= least + least / 2 && least > 1; ++p) {
            const uint64_t of_it = ceil_div(ceil_div(all, p), WHOLE) * WHOLE;
            const double us = (double)p * shape_of(of_it, in.d, in.n, in.type, true, MOST_HIGH_T).us;
            if (us < best * 0.98)
                best = us, piece = of_it;
        }
        pieces = all ? ceil_div(all, piece) : 1;
        sum_stride = ceil_div(in.d, WHOLE) * WHOLE;
        const uint64_t v = in.v < piece ? in.v : piece;
        g_shape = scores_shape(in.n, v, in.d, in.type);
        x_shape = shape_of(in.n, in.d, v, in.type, true);
        t_shape = shape_of(v, in.d, in.n, in.type, true, MOST_HIGH_T);
        if (pieces == 1) {
            const Shape both = together_of(in.n, v, in.d, in.type, x_shape.us + t_shape.us);
            together = both.us > 0.0;
            if (together)
                x_shape = both, t_shape = {both.high, both.wide, 1, 0.0};
        }
        g = l.take(in.n * piece * size);
        g_sums = x_sums = t_sums = 0;
        if (g_shape.splits > 1)
            g_sums = l.take(g_shape.splits * in.n * piece * 4);
        if (x_shape.splits > 1 || pieces > 1)
            x_sums = l.take(x_shape.splits * in.n * sum_stride * 4);
        if (t_shape.splits > 1)
            t_sums = l.take(t_shape.splits * piece * sum_stride * 4);
    }
};

int too_many(const char *what, const Inputs &in)
{
    set_error("%s: %llu rows of %llu elements against a table of %llu are too many", what, (unsigned long long)in.n,
              (unsigned long long)in.d, (unsigned long long)in.v);
    return UNG_HIP_EINVAL;
}

int check_inputs(const char *what, const Inputs &in)
{
    if (!known_type(in.type)) {
        set_error("%s: unknown element type %d", what, in.type);
        return UNG_HIP_EINVAL;
    }
    // (rows of a packed copy have to stay below 2^23 bytes)
    if (in.n > (1u << 27) || in.v > INT32_MAX - 256 || in.d > (1u << 20))
        return too_many(what, in);
    if ((in.n > 1 && in.x_stride < in.d) || (in.v > 1 && in.table_stride < in.d)) {
        set_error("%s: strides %llu and %llu are less than %llu columns", what, (unsigned long long)in.x_stride,
                  (unsigned long long)in.table_stride, (unsigned long long)in.d);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)in.x % type_size(in.type) || (uintptr_t)in.table % type_size(in.type)) {
        set_error("%s: x and table need to be aligned to their elements", what);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

// Whether the launch of a product of m x n results, and of `more` blocks beside it, has its threads counted in 32 bits.
bool fits_a_launch(Shape s, uint64_t m, uint64_t n, uint64_t more = 0)
{
    if (s.high <= FEW && s.wide == 64) // few rows, their shares along another axis
        return ceil_div(n, 64) <= most_blocks(64);
    const uint32_t threads = s.high == BIG ? 512 : s.high == 32 ? 128 : 256;
    return ceil_div(m, s.high) * ceil_div(n, s.wide) * s.splits + more <= most_blocks(threads);
}

// The launches of the passes: of the forward pass for both, as the backward pass needs what it makes.
int check_launches(const char *what, const Inputs &in, const Backward *b)
{
    bool fits = fits_a_launch(scores_shape(in.n, in.v, in.d, in.type), in.n, in.v);
    if (b) {
        const uint64_t v = in.v < b->piece ? in.v : b->piece;
        const uint64_t of_t = b->together ? ceil_div(v, b->t_shape.high) * ceil_div(in.d, b->t_shape.wide) : 0;
        fits = fits && fits_a_launch(b->g_shape, in.n, v) && fits_a_launch(b->x_shape, in.n, in.d, of_t) &&
               fits_a_launch(b->t_shape, v, in.d);
    }
    return fits ? UNG_HIP_OK : too_many(what, in);
}

int check_call(const char *what, const Inputs &in, const int32_t *ids, const int32_t *without, float temperature,
               uint64_t needed, const void *workspace, uint64_t bytes)
{
    if (!(temperature > 0.0f) || !(1.0f / temperature > 0.0f) || !(LOG2E / temperature < INF)) {
        set_error("%s: temperature %g is not a positive number with a reciprocal", what, (double)temperature);
        return UNG_HIP_EINVAL;
    }
    if ((in.n && !ids) || (in.n && in.d && !in.x) || (in.v && in.d && !in.table)) {
        set_error("%s: null argument", what);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)ids % 4 || (uintptr_t)without % 4) {
        set_error("%s: ids and without need to be aligned to their elements", what);
        return UNG_HIP_EINVAL;
    }
    if (needed && (!workspace || bytes < needed || (uintptr_t)workspace % 16)) {
        set_error("%s: needs %llu bytes of workspace at a 16-byte boundary (got %llu)", what, (unsigned long long)needed,
                  (unsigned long long)(workspace ? bytes : 0));
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

uint32_t some_blocks(uint64_t n) { return (uint32_t)(n < 1 ? 1 : n < 8192 ? n : 8192); }

Grid grid_of(const Operand &a, const Operand &b, Shape shape, uint64_t size)
{
    return {(uint32_t)ceil_div(a.rows, shape.high), (uint32_t)ceil_div(b.rows, shape.wide), shape.splits,
            ceil_div(a.k * size, CHUNK), shape.high == BIG ? 16u : 8u};
}

uint32_t items_of(const Grid &g) { return g.m_tiles * g.n_tiles * g.splits; }

// Few rows against many.
template <class E, bool LOOSE, class Finish>
void few_rows(const Operand &a, const Operand &b, Shape shape, const Finish &finish, hipStream_t st)
{
    const uint32_t each = (uint32_t)ceil_div(ceil_div(b.k * sizeof(E), CHUNK), shape.splits);
    const dim3 blocks((uint32_t)ceil_div(b.rows, 64), shape.splits);
    if (!blocks.x)
        return;
    if (shape.high == 16)
        ung_few_rows_kernel<E, 1, LOOSE><<<blocks, 64, 0, st>>>(a, b, each, finish);
    else
        ung_few_rows_kernel<E, 2, LOOSE><<<blocks, 64, 0, st>>>(a, b, each, finish);
}

// The product of two sides, its tiles finished by `finish`.
template <class E, bool A_ACROSS, bool B_ACROSS, class Finish>
void product(const Operand &a, const Operand &b, Shape shape, const Finish &finish, hipStream_t st)
{
    if constexpr (!A_ACROSS && !B_ACROSS) {
        if (shape.high <= FEW && shape.wide == 64) // (tiles of 64 columns are 128 high)
            return few_rows<E, false>(a, b, shape, finish, st);
    }
    const Grid grid = grid_of(a, b, shape, sizeof(E));
    const uint32_t items = items_of(grid);
    if (!items)
        return;
    if constexpr (A_ACROSS) {
        if (shape.high == 128 && shape.wide == 128 && grid.chunks == 1) {
            ung_one_chunk_kernel<E, A_ACROSS, B_ACROSS><<<items, 256, 0, st>>>(a, b, grid, finish);
            return;
        }
    }
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    auto tiles = [&](auto high, auto wm, auto wn) {
        constexpr int BM = decltype(high)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
        ung_tile_kernel<E, BM, WM, WN, A_ACROSS, B_ACROSS><<<items, WM * WN * 64, 0, st>>>(a, b, grid, finish);
    };
    if (shape.high == 32)
        tiles(std::integral_constant<int, 32>{}, one, two);
    else if (shape.high == 64)
        tiles(std::integral_constant<int, 64>{}, two, two);
    else if (shape.high == 128 && shape.wide == 128)
        tiles(std::integral_constant<int, 128>{}, two, two);
    else if (shape.high == 128)
        tiles(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{}, one);
    else if constexpr (sizeof(E) == 2 && !Finish::MORE)
        tiles(std::integral_constant<int, BIG>{}, two, std::integral_constant<int, 4>{});
}

// dT of G and X, and dX of G and the table, by one launch.
template <class E>
void both_products(const Operand &gt, const Operand &x, Shape t_shape, const Whole<E, TargetsOf<E>> &whole, const Operand &g,
                   const Operand &table, Shape x_shape, const Sums<false> &sums, hipStream_t st)
{
    const Grid t_grid = grid_of(gt, x, t_shape, sizeof(E)), x_grid = grid_of(g, table, x_shape, sizeof(E));
    const uint32_t items = items_of(t_grid) + items_of(x_grid);
    if (x_shape.high == 32)
        ung_two_products_kernel<E, 32, 1, 2, true, true, false, true>
            <<<items, 128, 0, st>>>(gt, x, t_grid, whole, g, table, x_grid, sums);
    else if (x_shape.high == 64)
        ung_two_products_kernel<E, 64, 2, 2, true, true, false, true>
            <<<items, 256, 0, st>>>(gt, x, t_grid, whole, g, table, x_grid, sums);
    else if (x_shape.wide == 64)
        ung_two_products_kernel<E, 128, 4, 1, true, true, false, true>
            <<<items, 256, 0, st>>>(gt, x, t_grid, whole, g, table, x_grid, sums);
    else
        ung_two_products_kernel<E, 128, 2, 2, true, true, false, true>
            <<<items, 256, 0, st>>>(gt, x, t_grid, whole, g, table, x_grid, sums);
}

template <class E>
Operand side(const Packed &p, const void *x, uint64_t stride, uint64_t rows, uint64_t d, uint8_t *ws, hipStream_t st,
             bool fill)
{
    if (!p.copy)
        return {x, rows > 1 ? stride * sizeof(E) : p.pitch, rows, d};
    if (fill && rows && p.pitch) {
        const uint64_t each = p.pitch < 8192 ? 8192 / p.pitch : 1; // two vectors a thread
        ung_table_pack_kernel<E><<<some_blocks(ceil_div(rows, each)), 256, 0, st>>>(
            (const E *)x, stride, rows, d, (E *)(ws + p.at), p.pitch / sizeof(E), (uint32_t)each);
    }
    return {ws + p.at, p.pitch, rows, d};
}

// The same rows with lines across the inner length: element k of `cols` columns, side by side.
Operand across(const Operand &o) { return {o.p, o.stride, o.k, o.rows}; }

} // namespace

extern "C" {

int ung_hip_table_loss_workspace(const void *x, uint64_t x_stride, const void *table, uint64_t table_stride, int type,
                                 uint64_t rows, uint64_t table_rows, uint64_t cols, int backward, uint64_t *bytes)
{
    static const char what[] = "ung_hip_table_loss_workspace";
    clear_error();
    if (!bytes) {
        set_error("%s: null bytes", what);
        return UNG_HIP_EINVAL;
    }
    const Inputs in = {x, table, x_stride, table_stride, type, rows, table_rows, cols};
    if (const int rc = check_inputs(what, in))
        return rc;
    if (!backward) {
        *bytes = Forward(in).l.bytes;
        return check_launches(what, in, nullptr);
    }
    const Backward f(in);
    *bytes = f.l.bytes;
    return check_launches(what, in, &f);
}

int ung_hip_table_loss_forward(const void *x, uint64_t x_stride, const void *table, uint64_t table_stride, int type,
                               uint64_t rows, uint64_t table_rows, uint64_t cols, const int32_t *ids,
                               const int32_t *without, float temperature, float *loss, float *lse, void *workspace,
                               uint64_t workspace_bytes, void *stream)
{
    static const char what[] = "ung_hip_table_loss_forward";
    clear_error();
    const Inputs in = {x, table, x_stride, table_stride, type, rows, table_rows, cols};
    if (const int rc = check_inputs(what, in))
        return rc;
    const Forward f(in);
    if (const int rc = check_launches(what, in, nullptr))
        return rc;
    if (const int rc = check_call(what, in, ids, without, temperature, f.l.bytes, workspace, workspace_bytes))
        return rc;
    if (rows == 0)
        return UNG_HIP_OK;
    if (!loss || !lse || (uintptr_t)loss % 4 || (uintptr_t)lse % 4) {
        set_error("%s: null or unaligned loss or lse", what);
        return UNG_HIP_EINVAL;
    }
    const hipStream_t st = (hipStream_t)stream;
    uint8_t *ws = (uint8_t *)workspace;
    return with_type(type, [&](auto zero) {
        using E = decltype(zero);
        const float c = LOG2E / temperature;
        const Operand a = side<E>(f.x, x, x_stride, rows, cols, ws, st, true);
        const Operand b = side<E>(f.table, table, table_stride, table_rows, cols, ws, st, true);
        Part *parts = (Part *)(ws + f.parts);
        float *target = (float *)(ws + f.target);
        const LogSum finish = {{}, ids, without, target, parts, rows, table_rows, c};
        auto scores = [&](const auto &finish) {
            if (f.loose)
                few_rows<E, true>(a, b, f.shape, finish, st);
            else
                product<E, false, false>(a, b, f.shape, finish, st);
        };
        if (f.shape.splits > 1) {
            float *const sums = (float *)(ws + f.sums);
            scores(Sums<false>{{}, sums, f.stride, rows});
            ung_table_parts_kernel<<<some_blocks(ceil_div(rows * f.tiles, 4)), 256, 0, st>>>(sums, f.shape.splits, f.stride, finish);
        } else
            scores(finish);
        auto join = [&](auto each) {
            constexpr int R = decltype(each)::value;
            ung_table_join_kernel<R><<<(uint32_t)ceil_div(rows, R), 256, 0, st>>>(parts, f.tiles, rows, table_rows, target,
                                                                              ids, without, c, loss, lse);
        };
        // threads enough for a row where there are few of them (16 rows of 1563 parts by one block 10 us more)
        if (rows < 128)
            join(std::integral_constant<int, 1>{});
        else if (rows < 2048)
            join(std::integral_constant<int, 4>{});
        else
            join(std::integral_constant<int, 16>{});
        return launched(what);
    });
}

int ung_hip_table_loss_backward(const void *x, uint64_t x_stride, const void *table, uint64_t table_stride, int type,
                                uint64_t rows, uint64_t table_rows, uint64_t cols, const int32_t *ids,
                                const int32_t *without, const float *lse, const float *weight, float temperature,
                                void *dx, uint64_t dx_stride, void *dtable, uint64_t dtable_stride, void *workspace,
                                uint64_t workspace_bytes, void *stream)
{
    static const char what[] = "ung_hip_table_loss_backward";
    clear_error();
    const Inputs in = {x, table, x_stride, table_stride, type, rows, table_rows, cols};
    if (const int rc = check_inputs(what, in))
        return rc;
    const Backward f(in);
    if (const int rc = check_launches(what, in, &f))
        return rc;
    if (const int rc = check_call(what, in, ids, without, temperature, f.l.bytes, workspace, workspace_bytes))
        return rc;
    if ((dx && rows > 1 && dx_stride < cols) || (dtable && table_rows > 1 && dtable_stride < cols)) {
        set_error("%s: strides %llu and %llu of the gradients are less than %llu columns", what,
                  (unsigned long long)dx_stride, (unsigned long long)dtable_stride, (unsigned long long)cols);
        return UNG_HIP_EINVAL;
    }
    if ((rows && !lse) || (uintptr_t)lse % 4 || (uintptr_t)weight % 4 || (uintptr_t)dx % type_size(type) ||
        (uintptr_t)dtable % type_size(type)) {
        set_error("%s: null lse, or lse, weight, dx or dtable not aligned to their elements", what);
        return UNG_HIP_EINVAL;
    }
    if (cols == 0 || (!dx && !dtable))
        return UNG_HIP_OK;
    const hipStream_t st = (hipStream_t)stream;
    uint8_t *ws = (uint8_t *)workspace;
    return with_type(type, [&](auto zero) {
        using E = decltype(zero);
        const float c = LOG2E / temperature, by = 1.0f / temperature;
        Row *row = (Row *)(ws + f.rows);
        float *scale = sizeof(E) == 2 && std::is_same_v<E, fp16_t> ? (float *)(ws + f.scale) : nullptr;
        const float *back = scale ? scale + 1 : nullptr;
        if (scale)
            ung_table_range_kernel<<<1, 1024, 0, st>>>(weight, rows, table_rows, ids, without, by, scale);
        const Operand a = side<E>(f.x, x, x_stride, rows, cols, ws, st, false);
        if (rows)
            ung_table_rows_kernel<E><<<some_blocks(ceil_div(rows, 4)), 256, 0, st>>>(
                (const E *)x, x_stride, rows, table_rows, cols, ids, without, lse, weight, by, scale, row,
                (int32_t *)(ws + f.targets), (E *)(ws + f.x.at), f.x.pitch / sizeof(E));
        const Operand t = side<E>(f.table, table, table_stride, table_rows, cols, ws, st, true);
        auto vectors = [](const void *p, uint64_t stride, uint64_t rows) {
            return (uintptr_t)p % 4 == 0 && (rows == 1 || stride * sizeof(E) % 4 == 0);
        };
        const Rest<E> none = {}, rest = sizeof(E) == 4 ? none : Rest<E>{row, (float *)(ws + f.rest), (const E *)t.p, t.stride / sizeof(E)};
        const Operand x_side = {a.p, a.stride, rows, cols};
        float *const x_sums = (float *)(ws + f.x_sums);
        auto sum = [&](const float *sums, uint32_t splits, uint64_t n, E *to, uint64_t stride, const Rest<E> &more) {
            const uint64_t quads = n * ceil_div(cols, 4);
            if (splits >= 16 && quads < 65536)
                ung_table_sum_kernel<E, 16><<<some_blocks(ceil_div(quads, 16)), 256, 0, st>>>(
                    sums, splits, n, cols, f.sum_stride, back, to, stride, more);
            else
                ung_table_sum_kernel<E, 1><<<some_blocks(ceil_div(quads, 256)), 256, 0, st>>>(
                    sums, splits, n, cols, f.sum_stride, back, to, stride, more);
        };
        // Of piece p: its rows of the table, and its G
        auto length = [&](uint64_t p) { return std::min(table_rows - p * f.piece, f.piece); };
        auto table_of = [&](uint64_t p) {
            return Operand{(const uint8_t *)t.p + p * f.piece * t.stride, t.stride, length(p), cols};
        };
        E *const g_at = (E *)(ws + f.g);
        auto g_of = [&](uint64_t p) { return Operand{g_at, f.piece * sizeof(E), rows, length(p)}; };
        auto weights = [&](uint64_t p) {
            return Weights<E>{{}, row, (float *)(ws + f.rest), g_at, f.piece, rows, p * f.piece, length(p), c};
        };
        auto targets = [&](uint64_t p) {
            if constexpr (sizeof(E) == 2)
                return Targets<E>{(const int32_t *)(ws + f.targets), (const float *)(ws + f.rest), (uint32_t)rows, (uint32_t)(p * f.piece)};
            else
                return NoTargets{};
        };
        auto whole = [&](uint64_t p) {
            E *to = (E *)dtable + p * f.piece * dtable_stride;
            return Whole<E, TargetsOf<E>>{{}, targets(p), to, dtable_stride, length(p), cols, back,
                                          vectors(to, dtable_stride, length(p)), none};
        };
        for (uint64_t p = 0; p < f.pieces; ++p) {
            const uint64_t v = length(p);
            const Operand part = table_of(p), g = g_of(p);
            if (f.g_shape.splits > 1 && rows && v) {
                float *const sums = (float *)(ws + f.g_sums);
                const uint64_t stride = ceil_div(v, WHOLE) * WHOLE;
                product<E, false, false>(x_side, part, f.g_shape, Sums<false>{{}, sums, stride, rows}, st);
                ung_table_weights_kernel<E><<<some_blocks(ceil_div(rows * (stride / WHOLE), 4)), 256, 0, st>>>(
                    sums, f.g_shape.splits, stride, weights(p));
            } else
                product<E, false, false>(x_side, part, f.g_shape, weights(p), st);
            if (f.together && dx && dtable) {
                both_products<E>(across(g), across(x_side), f.t_shape, whole(p), g, across(part), f.x_shape,
                                 Sums<false>{{}, x_sums, f.sum_stride, rows}, st);
                break;
            }
            if (dx && rows) {
                if (f.x_shape.splits == 1 && f.pieces == 1)
                    product<E, false, true>(g, across(part), f.x_shape,
                                            Whole<E, NoTargets>{{}, {}, (E *)dx, dx_stride, rows, cols, back, vectors(dx, dx_stride, rows), rest}, st);
                else if (p == 0)
                    product<E, false, true>(g, across(part), f.x_shape,
                                            Sums<false>{{}, x_sums, f.sum_stride, rows}, st);
                else
                    product<E, false, true>(g, across(part), f.x_shape,
                                            Sums<true>{{}, x_sums, f.sum_stride, rows}, st);
            }
            if (dtable && v) {
                if (f.t_shape.splits == 1)
                    product<E, true, true>(across(g), across(x_side), f.t_shape, whole(p), st);
                else {
                    E *to = (E *)dtable + p * f.piece * dtable_stride;
                    product<E, true, true>(across(g), across(x_side), f.t_shape,
                                           Sums<false, TargetsOf<E>>{targets(p), (float *)(ws + f.t_sums), f.sum_stride, v}, st);
                    sum((const float *)(ws + f.t_sums), f.t_shape.splits, v, to, dtable_stride, none);
                }
            }
        }
        if (dx && rows && (f.x_shape.splits > 1 || f.pieces > 1))
            sum(x_sums, f.x_shape.splits, rows, (E *)dx, dx_stride, rest);
        return launched(what);
    });
}

} // extern "C"
