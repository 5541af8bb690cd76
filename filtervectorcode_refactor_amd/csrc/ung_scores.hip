// ung_scores.hip -- operators on rows of scores, on gfx950: the first k of each row with its
// log-sum-exp, and the distillation loss against a teacher's top scores with its gradient
// (the entry points ung_hip_top_scores* and ung_hip_distill* of include/ung_hip.h).
//
// A row is read in 16-byte vectors from the 16-byte boundary at or before its first element:
// vectors wholly inside the row by one load, the at most two at its ends element by element,
// so rows may start anywhere and nothing outside them is read.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "ung_elements.h"
#include "ung_hip.h"
#include "ung_internal.h"

using namespace ung;

namespace {

constexpr int MAX_K = UNG_HIP_TOP_SCORES_MAX; // 128
constexpr float NEG_INF = -__builtin_inff();

template <class T>
struct RowRef {
    const T *row;
    uint32_t shift; // elements between the 16-byte boundary and the row's first one
    uint32_t len;
    __device__ RowRef(const T *r, uint32_t n)
        : row(r), shift((uint32_t)(((uintptr_t)r & 15) / sizeof(T))), len(n)
    {
    }
    // Vector i of the row; elements outside the row are -inf.
    __device__ Vec<T> load(uint32_t i) const
    {
        constexpr int N = Vec<T>::N;
        const int64_t j = (int64_t)i * N - shift;
        if (j >= 0 && j + N <= (int64_t)len)
            return *reinterpret_cast<const Vec<T> *>(row + j);
        Vec<T> v;
#pragma unroll
        for (int e = 0; e < N; ++e)
            v.v[e] = j + e >= 0 && j + e < (int64_t)len ? row[j + e] : (T)NEG_INF;
        return v;
    }
};

// Writes vector i of a row that starts `shift` elements after a 16-byte boundary of the
// source; `same`: the destination row lies the same way.
template <class T>
__device__ inline void store_vec(T *row, uint32_t shift, uint32_t len, uint32_t i, const Vec<T> &v, bool same)
{
    constexpr int N = Vec<T>::N;
    const int64_t j = (int64_t)i * N - shift;
    if (same && j >= 0 && j + N <= (int64_t)len) {
        *reinterpret_cast<Vec<T> *>(row + j) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < (int64_t)len)
            row[j + e] = v.v[e];
}

template <class T>
__device__ inline uint32_t vectors_of(uint32_t shift, uint32_t len)
{
    return (uint32_t)(((uint64_t)shift + len + Vec<T>::N - 1) / Vec<T>::N);
}

// ---- the first k of a row ------------------------------------------------------------

// (score, id) as one whole number that orders like it: larger scores first, of equal ones the
// lower id; NaN above every score, -0 as 0; 0 = no candidate (-inf).
__device__ inline uint64_t order_of(float x, uint32_t id)
{
    if (x == NEG_INF)
        return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);
    uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    if (x != x)
        k = 0xFFFFFFFFu;
    return (uint64_t)k << 32 | (uint32_t)~id;
}

__device__ inline float score_of(uint64_t o)
{
    const uint32_t k = (uint32_t)(o >> 32);
    return k == 0xFFFFFFFFu ? __builtin_nanf("") : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

constexpr int TOP_NT = 256;   // threads of a block
constexpr int TOP_CAP = 1024; // candidates a block ranks

struct TopShared {
    uint64_t cand[TOP_CAP];
    uint64_t most[TOP_NT];
    float red[TOP_NT / 64];
    uint32_t wave_count[TOP_NT / 64];
    uint32_t count;
    uint64_t limit;
};

// The k largest of the orders that a block holds (each(f) calls f with those of a thread; 0 =
// none) to sh.cand in descending order; returns how many there are.  The k-th largest of the threads'
// maxima is no larger than the k-th largest of all, and few orders lie between the two: those
// at or above it are collected and ranked by counting.  Where they do not fit (many equal
// scores, few threads with candidates), the k-th largest is first found bit by bit.
template <class Each>
__device__ inline uint32_t select_top(TopShared &sh, uint32_t k, uint64_t thread_most, Each each)
{
    const uint32_t tid = threadIdx.x;
    sh.most[tid] = thread_most;
    if (tid == 0) {
        sh.count = 0;
        sh.limit = 1;
    }
    __syncthreads();
    uint32_t rank = 0;
    for (uint32_t t = 0; t < TOP_NT; ++t)
        rank += sh.most[t] > thread_most || (sh.most[t] == thread_most && t < tid);
    if (rank == k - 1 && thread_most)
        sh.limit = thread_most;
    __syncthreads();
    uint64_t limit = sh.limit;
    auto collect = [&]() {
        each([&](uint64_t o) {
            if (o >= limit) {
                const uint32_t at = atomicAdd(&sh.count, 1u);
                if (at < TOP_CAP)
                    sh.cand[at] = o;
            }
        });
        __syncthreads();
    };
    collect();
    uint32_t found = sh.count;
    if (found > TOP_CAP) {
        // the largest limit with at least k orders at or above it; there are over k of them
        limit = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t trial = limit | 1ull << bit;
            uint32_t mine = 0;
            each([&](uint64_t o) { mine += o >= trial; });
#pragma unroll
            for (int o = 32; o > 0; o >>= 1)
                mine += __shfl_xor((int)mine, o);
            __syncthreads();
            if ((tid & 63) == 0)
                sh.wave_count[tid >> 6] = mine;
            __syncthreads();
            uint32_t all = 0;
#pragma unroll
            for (int w = 0; w < TOP_NT / 64; ++w)
                all += sh.wave_count[w];
            if (all >= k)
                limit = trial;
        }
        if (tid == 0)
            sh.count = 0;
        __syncthreads();
        collect(); // orders are distinct: k of them
        found = sh.count;
    }
    uint64_t mine[TOP_CAP / TOP_NT];
    uint32_t place[TOP_CAP / TOP_NT];
#pragma unroll
    for (int p = 0; p < TOP_CAP / TOP_NT; ++p) {
        const uint32_t i = p * TOP_NT + tid;
        place[p] = k;
        if (i < found) {
            mine[p] = sh.cand[i];
            uint32_t at = 0;
            for (uint32_t t = 0; t < found; ++t)
                at += sh.cand[t] > mine[p];
            place[p] = at;
        }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < TOP_CAP / TOP_NT; ++p)
        if (place[p] < k)
            sh.cand[place[p]] = mine[p];
    __syncthreads();
    return found < k ? found : k;
}

// What a block found: final rows, or partial ones (orders and (maximum, sum) pairs).
__device__ inline void put_top(const TopShared &sh, uint32_t found, uint32_t k, uint64_t row, bool final_,
                               float *values, int32_t *ids, float *lse, uint64_t *part, float2 *part_sum, float top,
                               float sum)
{
    const uint32_t tid = threadIdx.x;
    if (final_) {
        if (tid < k) {
            values[row * k + tid] = tid < found ? score_of(sh.cand[tid]) : NEG_INF;
            ids[row * k + tid] = tid < found ? (int32_t)~(uint32_t)sh.cand[tid] : -1;
        }
        if (tid == 0 && lse)
            lse[row] = fabsf(top) == __builtin_inff() ? top : top + logf(sum);
    } else {
        if (tid < k)
            part[row * k + tid] = tid < found ? sh.cand[tid] : 0;
        if (tid == 0)
            part_sum[row] = make_float2(top, sum);
    }
}

// The first k of one piece of a row (TOP_NT * NV vectors; the whole row if `pieces` is 1), its
// values held in registers: one read of the scores, bound by memory.
template <class T, int NV>
__global__ __launch_bounds__(TOP_NT) void ung_top_scores_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                                uint32_t pieces, uint32_t k, float inv_t,
                                                                float *values, int32_t *ids, float *lse,
                                                                uint64_t *part, float2 *part_sum)
{
    constexpr int N = Vec<T>::N;
    __shared__ TopShared sh;
    const uint64_t r = blockIdx.x / pieces;
    const uint32_t piece = (uint32_t)(blockIdx.x - r * pieces);
    const RowRef<T> ref(scores + r * stride, len);
    const uint32_t first = piece * (TOP_NT * NV) + threadIdx.x, end = vectors_of<T>(ref.shift, len);
    Vec<T> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i * TOP_NT < end)
            v[i] = ref.load(first + i * TOP_NT);
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                v[i].v[e] = (T)NEG_INF;
    float most = NEG_INF;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
            most = max_nan(most, to_float(v[i].v[e]));
    const float top = block_reduce<TOP_NT>(most, sh.red, max_nan);
    const float at = top == NEG_INF ? 0.0f : top;
    float sum = 0.0f;
    uint64_t thread_most = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float x = to_float(v[i].v[e]);
            sum += exp_neg((x - at) * inv_t);
            const uint64_t o = order_of(x, (first + i * TOP_NT) * N + e - ref.shift);
            thread_most = o > thread_most ? o : thread_most;
        }
    __syncthreads();
    sum = block_reduce<TOP_NT>(sum, sh.red, add);
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e)
                f(order_of(to_float(v[i].v[e]), (first + i * TOP_NT) * N + e - ref.shift));
    };
    const uint32_t found = select_top(sh, k, thread_most, each);
    put_top(sh, found, k, blockIdx.x, pieces == 1, values, ids, lse, part, part_sum, top * inv_t, sum);
}

constexpr uint32_t MERGE_LISTS = 64; // lists one block merges

// Merges up to MERGE_LISTS partial rows of a row.
__global__ __launch_bounds__(TOP_NT) void ung_top_merge_kernel(const uint64_t *part, const float2 *part_sum,
                                                               uint32_t lists, uint32_t groups, uint32_t k,
                                                               float *values, int32_t *ids, float *lse, uint64_t *out,
                                                               float2 *out_sum)
{
    __shared__ TopShared sh;
    const uint64_t r = blockIdx.x / groups;
    const uint32_t group = (uint32_t)(blockIdx.x - r * groups), first = group * MERGE_LISTS;
    const uint32_t n = (lists - first < MERGE_LISTS ? lists - first : MERGE_LISTS);
    const uint64_t *mine = part + (r * lists + first) * k;
    const uint32_t items = n * k;
    uint64_t thread_most = 0;
    for (uint32_t i = threadIdx.x; i < items; i += TOP_NT)
        thread_most = mine[i] > thread_most ? mine[i] : thread_most;
    auto each = [&](auto f) {
        for (uint32_t i = threadIdx.x; i < items; i += TOP_NT)
            f(mine[i]);
    };
    float2 s = make_float2(NEG_INF, 0.0f);
    if (threadIdx.x < n)
        s = part_sum[r * lists + first + threadIdx.x];
    const float top = block_reduce<TOP_NT>(s.x, sh.red, max_nan);
    float sum = s.y == 0.0f ? 0.0f : s.y * exp_neg(s.x - (top == NEG_INF ? 0.0f : top));
    __syncthreads();
    sum = block_reduce<TOP_NT>(sum, sh.red, add);
    const uint32_t found = select_top(sh, k, thread_most, each);
    put_top(sh, found, k, blockIdx.x, groups == 1, values, ids, lse, out, out_sum, top, sum);
}

// ---- distillation --------------------------------------------------------------------
//
// Of a row: q = softmax(s / T) over all its scores, p the teacher's distribution.  Without the
// teacher's log-sum-exp p is the softmax of its listed scores; with it p_k = exp(t_k / T - lse)
// and the rest of its mass, p_r = 1 - sum p_k, stands against the student's mass outside the
// list, Q_r (left out where that is 0).
//   loss   = sum p_k (log p_k - log q_k) + p_r (log p_r - log Q_r)
//   d/ds_j = weight / T * (W q_j - p_j - [j not listed] p_r q_j / Q_r),  W = sum p_k + p_r
// Q_r is summed over the columns outside the list and relative to the largest of them, not
// taken as 1 - sum q_k: that would cancel where the student's mass lies in the list, and
// vanish where its other scores are far below.  A bit for each column of the block's stretch,
// in LDS, tells them apart; where Q_r counts, listed columns leave the stretch's sums and
// enter the row's from the entries.  A row without a valid entry, or without a score above
// -inf, has loss and gradient 0.

// What the backward pass needs of a row besides its inputs.
struct alignas(16) Saved {
    float top;      // largest score / T of the whole row; EMPTY: no loss
    float inside;   // W / sum exp(s / T - top)
    float rest_top; // the same two of the columns outside the list: gradient = weight / T *
    float outside;  // exp(s / T - rest_top) * outside
    float shift;    // p_k = exp(t_k / T - shift)
    float unused[3];
};
static_assert(sizeof(Saved) == 4 * UNG_HIP_DISTILL_SAVED, "");

constexpr float EMPTY = __builtin_inff(); // Saved::top of a row without loss

struct DistillShared {
    float z[MAX_K];  // teacher's score / T; -inf = not there
    float s[MAX_K];  // the student's there / T
    uint32_t id[MAX_K];
    uint32_t first[MAX_K]; // the entry is the first one to name its column
    float red[2][16];
    Saved saved;
};

__device__ inline float max_of(float a, float b) { return fmaxf(a, b); }

// The teacher's row: entries into sh by the first k threads, with the student's scores of
// those whose columns lie in [from, to) (a block that writes the gradient over the scores
// reads no other block's stretch).
template <class T>
__device__ inline void load_entries(DistillShared &sh, const T *row, const int32_t *ids, const float *values,
                                    uint32_t k, uint32_t len, float inv_t, int64_t from, int64_t to)
{
    const uint32_t tid = threadIdx.x;
    if (tid < k) {
        const int32_t id = ids[tid];
        const float v = values[tid];
        const bool ok = (uint32_t)id < len && v != NEG_INF;
        sh.id[tid] = ok ? (uint32_t)id : 0xFFFFFFFFu;
        sh.z[tid] = ok ? v * inv_t : NEG_INF;
        sh.s[tid] = ok && id >= from && id < to ? to_float(row[id]) * inv_t : 0.0f;
        sh.first[tid] = ok;
    }
}

// Loss and Saved of a row, run by one wave: from its entries and the sums (maximum / T, sum of
// exp(s / T - maximum)) of its columns, with `lse` of those outside the list.  Returns the
// loss in every lane.
__device__ inline float finish_row(DistillShared &sh, uint32_t k, const float *lse, float2 sums, Saved &saved)
{
    const uint32_t lane = threadIdx.x & 63;
    float z[2], s[2], best = NEG_INF, top = sums.x;
    bool any = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = h * 64 + lane;
        z[h] = i < k ? sh.z[i] : NEG_INF;
        s[h] = i < k ? sh.s[i] : 0.0f;
        any |= z[h] != NEG_INF;
        best = max_nan(best, z[h]);
        if (lse && i < k && sh.first[i])
            top = max_of(top, s[h]);
    }
    any = __any(any);
    saved = Saved{EMPTY, 0.0f, 0.0f, 0.0f, 0.0f, {}};
    best = wave_reduce(best, max_nan);
    top = wave_reduce(top, max_of);
    const float at = top == NEG_INF ? 0.0f : top;
    float total = sums.y;
    if (lse) {
        float in = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (h * 64 + lane < k && sh.first[h * 64 + lane])
                in += expf(s[h] - at);
        total = wave_reduce(in, add) + (sums.y == 0.0f ? 0.0f : sums.y * expf(sums.x - at));
    }
    if (total != total) // a NaN among the scores, or +inf: the whole row is NaN
        top = total;
    if (!any || top == NEG_INF)
        return 0.0f;
    float shift;
    if (lse)
        shift = *lse;
    else {
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            sum += z[h] == NEG_INF ? 0.0f : expf(z[h] - best);
        shift = best + logf(wave_reduce(sum, add));
    }
    const float log_total = logf(total);
    float mass = 0.0f, loss = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (z[h] != NEG_INF) {
            const float log_p = z[h] - shift, p = expf(log_p);
            mass += p;
            if (!(p <= 0.0f))
                loss += p * (log_p - (s[h] - top - log_total));
        }
    mass = wave_reduce(mass, add);
    loss = wave_reduce(loss, add);
    saved = Saved{top, mass / total, top, mass / total, shift, {}};
    if (lse && !(sums.y <= 0.0f)) {
        const float rest = 1.0f - mass < 0.0f ? 0.0f : 1.0f - mass;
        saved.rest_top = sums.x;
        if (!(rest <= 0.0f)) {
            loss += rest * (logf(rest) - (sums.x - top + logf(sums.y) - log_total));
            saved.inside = (mass + rest) / total;
        }
        saved.outside = expf(sums.x - top) * saved.inside - rest / sums.y;
    }
    return loss;
}

// Gradient of a stretch of a row whose vectors are in registers, then of the listed columns
// that lie in it (in one more write: their scores were read before the first one).
template <class T, int NT, int NV>
__device__ inline void write_gradient(DistillShared &sh, const Vec<T> (&v)[NV], uint32_t begin, uint32_t shift,
                                      uint32_t len, uint32_t end, uint32_t k, float inv_t, const Saved &saved,
                                      float weight, T *grad)
{
    constexpr int N = Vec<T>::N;
    const bool same = ((uintptr_t)grad & 15) == shift * sizeof(T);
    const bool empty = saved.top == EMPTY;
    const float w = weight * inv_t, out = saved.outside * w;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t at = begin + threadIdx.x + i * NT;
        if (at >= end)
            break;
        Vec<T> g;
#pragma unroll
        for (int e = 0; e < N; ++e)
            g.v[e] = from_float<T>(empty ? 0.0f : exp_neg(to_float(v[i].v[e]) * inv_t - saved.rest_top) * out);
        store_vec(grad, shift, len, at, g, same);
    }
    if (empty)
        return;
    __syncthreads();
    if (threadIdx.x < k) {
        const uint32_t id = sh.id[threadIdx.x];
        const uint32_t at = (id + shift) / N;
        if (id != 0xFFFFFFFFu && at >= begin && at < begin + NT * NV) {
            float p = 0.0f; // of every entry that names this column
            for (uint32_t t = 0; t < k; ++t)
                p += sh.id[t] == id ? expf(sh.z[t] - saved.shift) : 0.0f;
            grad[id] = from_float<T>((exp_neg(sh.s[threadIdx.x] - saved.top) * saved.inside - p) * w);
        }
    }
}

// Sums of a stretch of a row in registers, in every thread: its maximum / T and the sum of
// exp(s / T - maximum).  With `tail` listed columns become -inf first.
template <class T, int NT, int NV>
__device__ inline float2 stretch_sums(DistillShared &sh, uint32_t *bits, Vec<T> (&v)[NV], uint32_t begin,
                                      uint32_t shift, uint32_t k, bool tail, float inv_t)
{
    constexpr int N = Vec<T>::N;
    const uint32_t tid = threadIdx.x;
    if (tail) {
        for (uint32_t i = tid; i < NT * NV * N / 32; i += NT)
            bits[i] = 0;
        __syncthreads();
        if (tid < k && sh.id[tid] != 0xFFFFFFFFu) {
            const uint64_t at = (uint64_t)sh.id[tid] + shift, from = (uint64_t)begin * N;
            if (at >= from && at < from + NT * NV * N) {
                const uint32_t bit = 1u << ((at - from) & 31);
                sh.first[tid] = !(atomicOr(&bits[(at - from) >> 5], bit) & bit);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t b = (tid + i * NT) * N;
            const uint32_t listed = bits[b >> 5] >> (b & 31) & ((1u << N) - 1);
            if (listed)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (listed >> e & 1)
                        v[i].v[e] = (T)NEG_INF;
        }
    }
    float most = NEG_INF;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
            most = max_of(most, to_float(v[i].v[e])); // a NaN shows in the sum
    const float top = block_reduce<NT>(most, sh.red[0], max_of) * inv_t;
    const float at = top == NEG_INF ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
            sum += exp_neg(to_float(v[i].v[e]) * inv_t - at);
    return make_float2(top, block_reduce<NT>(sum, sh.red[1], add));
}

template <class T, int NT, int NV>
__device__ inline void load_stretch(const RowRef<T> &ref, uint32_t first, uint32_t end, Vec<T> (&v)[NV])
{
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i * NT < end)
            v[i] = ref.load(first + i * NT);
        else
#pragma unroll
            for (int e = 0; e < Vec<T>::N; ++e)
                v[i].v[e] = (T)NEG_INF;
}

// A row by one block, its scores in registers: loss, and the gradient with `grad`.  One read
// of the scores and one write of the gradient, bound by memory.  `grad` may be the scores.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void ung_distill_row_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                             const int32_t *ids, const float *values, uint32_t k,
                                                             const float *lse, const float *weight, float inv_t,
                                                             float *loss, Saved *saved_out, T *grad,
                                                             uint64_t grad_stride)
{
    __shared__ DistillShared sh;
    __shared__ uint32_t bits[NT * NV * Vec<T>::N / 32];
    const uint64_t r = blockIdx.x;
    const RowRef<T> ref(scores + r * stride, len);
    const uint32_t end = vectors_of<T>(ref.shift, len);
    Vec<T> v[NV];
    load_stretch<T, NT, NV>(ref, threadIdx.x, end, v);
    load_entries(sh, ref.row, ids + r * k, values + r * k, k, len, inv_t, 0, len);
    const float2 sums = stretch_sums<T, NT, NV>(sh, bits, v, 0, ref.shift, k, lse != nullptr, inv_t);
    __syncthreads();
    if (threadIdx.x < 64) {
        Saved saved;
        const float l = finish_row(sh, k, lse ? lse + r : nullptr, sums, saved);
        if (threadIdx.x == 0) {
            loss[r] = l;
            if (saved_out)
                saved_out[r] = saved;
            sh.saved = saved;
        }
    }
    if (!grad)
        return;
    __syncthreads();
    write_gradient<T, NT, NV>(sh, v, 0, ref.shift, len, end, k, inv_t, sh.saved, weight ? weight[r] : 1.0f,
                              grad + r * grad_stride);
}

// Sums of one piece of a row (NT * NV vectors).
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void ung_distill_part_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                              const int32_t *ids, const float *values, uint32_t k,
                                                              int tail, float inv_t, uint32_t pieces, float2 *part)
{
    __shared__ DistillShared sh;
    __shared__ uint32_t bits[NT * NV * Vec<T>::N / 32];
    const uint64_t r = blockIdx.x / pieces;
    const uint32_t begin = (uint32_t)(blockIdx.x - r * pieces) * (NT * NV);
    const RowRef<T> ref(scores + r * stride, len);
    Vec<T> v[NV];
    load_stretch<T, NT, NV>(ref, begin + threadIdx.x, vectors_of<T>(ref.shift, len), v);
    if (tail)
        load_entries(sh, ref.row, ids + r * k, values + r * k, k, len, inv_t, 0, 0);
    const float2 sums = stretch_sums<T, NT, NV>(sh, bits, v, begin, ref.shift, k, tail, inv_t);
    if (threadIdx.x == 0)
        part[blockIdx.x] = sums;
}

// A row's loss from its pieces' sums; one wave a row.
template <class T>
__global__ __launch_bounds__(128) void ung_distill_join_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                               const int32_t *ids, const float *values, uint32_t k,
                                                               const float *lse, float inv_t, uint32_t pieces,
                                                               const float2 *part, float *loss, Saved *saved_out)
{
    __shared__ DistillShared sh;
    const uint64_t r = blockIdx.x;
    load_entries(sh, scores + r * stride, ids + r * k, values + r * k, k, len, inv_t, 0, len);
    __syncthreads();
    if (lse && threadIdx.x < k) {
        const uint32_t id = sh.id[threadIdx.x];
        for (uint32_t t = 0; t < threadIdx.x; ++t)
            if (sh.id[t] == id)
                sh.first[threadIdx.x] = 0;
    }
    __syncthreads();
    if (threadIdx.x >= 64)
        return;
    const float2 *mine = part + r * pieces;
    float top = NEG_INF, sum = 0.0f;
    for (uint32_t i = threadIdx.x; i < pieces; i += 64)
        top = max_of(top, mine[i].x);
    top = wave_reduce(top, max_of);
    const float at = top == NEG_INF ? 0.0f : top;
    for (uint32_t i = threadIdx.x; i < pieces; i += 64)
        sum += mine[i].y == 0.0f ? 0.0f : mine[i].x == NEG_INF ? mine[i].y : mine[i].y * expf(mine[i].x - at);
    sum = wave_reduce(sum, add);
    Saved saved;
    const float l = finish_row(sh, k, lse ? lse + r : nullptr, make_float2(top, sum), saved);
    if (threadIdx.x == 0) {
        loss[r] = l;
        saved_out[r] = saved;
    }
}

// Gradient of one piece of a row from what its forward pass saved.  `grad` may be the scores.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void ung_distill_grad_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                              const int32_t *ids, const float *values, uint32_t k,
                                                              const Saved *saved, const float *weight, float inv_t,
                                                              uint32_t pieces, T *grad, uint64_t grad_stride)
{
    __shared__ DistillShared sh;
    const uint64_t r = blockIdx.x / pieces;
    const uint32_t begin = (uint32_t)(blockIdx.x - r * pieces) * (NT * NV);
    const RowRef<T> ref(scores + r * stride, len);
    const uint32_t end = vectors_of<T>(ref.shift, len);
    Vec<T> v[NV];
    load_stretch<T, NT, NV>(ref, begin + threadIdx.x, end, v);
    const int64_t from = (int64_t)begin * Vec<T>::N - ref.shift;
    load_entries(sh, ref.row, ids + r * k, values + r * k, k, len, inv_t, from, from + NT * NV * Vec<T>::N);
    __syncthreads(); // the entries' scores are read before this block writes
    write_gradient<T, NT, NV>(sh, v, begin, ref.shift, len, end, k, inv_t, saved[r],
                              weight ? weight[r] : 1.0f, grad + r * grad_stride);
}

} // namespace

namespace {

// Rows all of whose 16-byte vectors start at a boundary need no vector more for their ends.
template <class T>
uint32_t vectors_at_most(const void *p, uint64_t rows, uint64_t stride, uint64_t len)
{
    const bool aligned = (uintptr_t)p % 16 == 0 && (rows == 1 || stride * sizeof(T) % 16 == 0);
    return (uint32_t)ceil_div(len + (aligned ? 0 : Vec<T>::N - 1), Vec<T>::N);
}

int check_scores(const char *what, const void *scores, int type, uint64_t rows, uint64_t len, uint64_t stride)
{
    if (!known_type(type)) {
        set_error("%s: unknown element type %d", what, type);
        return UNG_HIP_EINVAL;
    }
    if (len > (1ull << 31) - 64 || rows > INT32_MAX) {
        set_error("%s: %llu rows of %llu scores are too many", what, (unsigned long long)rows, (unsigned long long)len);
        return UNG_HIP_EINVAL;
    }
    if (rows && len && !scores) {
        set_error("%s: null scores", what);
        return UNG_HIP_EINVAL;
    }
    if (rows > 1 && stride < len) {
        set_error("%s: row_stride %llu is less than %llu scores", what, (unsigned long long)stride,
                  (unsigned long long)len);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)scores % type_size(type)) {
        set_error("%s: scores are not aligned to their elements", what);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

int check_temperature(const char *what, float t)
{
    if (t > 0.0f && t < __builtin_inff())
        return UNG_HIP_OK;
    set_error("%s: temperature %g is not a positive number", what, (double)t);
    return UNG_HIP_EINVAL;
}

int check_k(const char *what, uint32_t k, uint32_t least)
{
    if (k >= least && k <= (uint32_t)MAX_K)
        return UNG_HIP_OK;
    set_error("%s: k=%u outside %u..%d", what, k, least, MAX_K);
    return UNG_HIP_EINVAL;
}

int check_grid(const char *what, uint64_t blocks)
{
    if (blocks <= INT32_MAX)
        return UNG_HIP_OK;
    set_error("%s: too many scores (%llu blocks)", what, (unsigned long long)blocks);
    return UNG_HIP_EINVAL;
}

int check_workspace(const char *what, const void *workspace, uint64_t bytes, uint64_t needed)
{
    if (needed == 0 || (workspace && bytes >= needed && (uintptr_t)workspace % 16 == 0))
        return UNG_HIP_OK;
    set_error("%s: needs %llu bytes of workspace at a 16-byte boundary (got %llu)", what, (unsigned long long)needed,
              (unsigned long long)(workspace ? bytes : 0));
    return UNG_HIP_EINVAL;
}

// Vectors a thread holds, and pieces a row is cut into.
struct Cut {
    uint32_t nv, pieces;
};

Cut top_cut(uint64_t rows, uint32_t vectors)
{
    uint32_t nv = 16;
    while (nv > 1 && (TOP_NT * (nv / 2) >= vectors || rows * ceil_div(vectors, TOP_NT * nv) < 512))
        nv /= 2;
    const uint64_t pieces = ceil_div(vectors, TOP_NT * nv);
    return Cut{nv, (uint32_t)(pieces ? pieces : 1)};
}

uint64_t top_bytes(uint64_t rows, uint32_t pieces, uint32_t k)
{
    uint64_t bytes = 0;
    for (uint64_t lists = pieces; lists > 1; lists = ceil_div(lists, MERGE_LISTS))
        bytes += ceil_div(rows * lists * k * 8, 16) * 16 + ceil_div(rows * lists * 8, 16) * 16;
    return bytes;
}

template <class F>
void with_nv(uint32_t nv, F f)
{
    if (nv == 1)
        f(std::integral_constant<int, 1>{});
    else if (nv == 2)
        f(std::integral_constant<int, 2>{});
    else if (nv == 4)
        f(std::integral_constant<int, 4>{});
    else if (nv == 8)
        f(std::integral_constant<int, 8>{});
    else
        f(std::integral_constant<int, 16>{});
}

constexpr int ROW_NT = 512;   // threads of a block that holds a whole row
constexpr int PIECE_NT = 256; // ... a piece of one

bool whole_rows(uint64_t rows, uint32_t vectors) { return vectors <= ROW_NT * 16 && (rows >= 128 || vectors <= ROW_NT * 2); }

Cut row_cut(uint32_t vectors)
{
    uint32_t nv = 1;
    while (ROW_NT * nv < vectors)
        nv *= 2;
    return Cut{nv, 1};
}

Cut piece_cut(uint64_t rows, uint32_t vectors)
{
    uint32_t nv = 8;
    while (nv > 1 && (PIECE_NT * (nv / 2) >= vectors || rows * ceil_div(vectors, PIECE_NT * nv) < 512))
        nv /= 2;
    const uint64_t pieces = ceil_div(vectors, PIECE_NT * nv);
    return Cut{nv, (uint32_t)(pieces ? pieces : 1)};
}

uint64_t part_bytes(uint64_t rows, uint32_t pieces) { return ceil_div(rows * pieces * 8, 16) * 16; }

int check_distill(const char *what, const void *scores, int type, uint64_t rows, uint64_t len, uint64_t stride,
                  const int32_t *ids, const float *values, uint32_t k, float temperature)
{
    int rc;
    if ((rc = check_scores(what, scores, type, rows, len, stride)) || (rc = check_k(what, k, 0)) ||
        (rc = check_temperature(what, temperature)))
        return rc;
    if (rows && k && (!ids || !values)) {
        set_error("%s: null ids/values", what);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

int check_grad(const char *what, const void *grad, int type, uint64_t rows, uint64_t len, uint64_t grad_stride)
{
    if (rows && len && !grad) {
        set_error("%s: null gradient", what);
        return UNG_HIP_EINVAL;
    }
    if (rows > 1 && grad_stride < len) {
        set_error("%s: grad_stride %llu is less than %llu scores", what, (unsigned long long)grad_stride,
                  (unsigned long long)len);
        return UNG_HIP_EINVAL;
    }
    if ((uintptr_t)grad % type_size(type)) {
        set_error("%s: the gradient is not aligned to its elements", what);
        return UNG_HIP_EINVAL;
    }
    return UNG_HIP_OK;
}

// Forward pass: loss and saved rows, and the gradient too with `grad`.
int distill(const char *what, const void *scores, int type, uint64_t rows, uint64_t len, uint64_t stride,
            const int32_t *ids, const float *values, uint32_t k, const float *lse, const float *weight,
            float temperature, float *loss, Saved *saved, void *grad, uint64_t grad_stride, void *workspace,
            uint64_t workspace_bytes, hipStream_t st)
{
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const T *p = (const T *)scores;
        const float inv_t = 1.0f / temperature;
        const uint32_t vectors = vectors_at_most<T>(scores, rows, stride, len);
        int rc;
        if (whole_rows(rows, vectors)) {
            with_nv(row_cut(vectors).nv, [&](auto nv) {
                ung_distill_row_kernel<T, ROW_NT, nv.value><<<(uint32_t)rows, ROW_NT, 0, st>>>(
                    p, (uint32_t)len, stride, ids, values, k, lse, weight, inv_t, loss, saved, (T *)grad, grad_stride);
            });
            return launched(what);
        }
        const Cut cut = piece_cut(rows, vectors);
        const uint64_t parts = part_bytes(rows, cut.pieces), blocks = rows * cut.pieces;
        if ((rc = check_grid(what, blocks)) ||
            (rc = check_workspace(what, workspace, workspace_bytes, parts + (saved ? 0 : rows * sizeof(Saved)))))
            return rc;
        float2 *part = (float2 *)workspace;
        Saved *kept = saved ? saved : (Saved *)((char *)workspace + parts);
        with_nv(cut.nv, [&](auto nv) {
            ung_distill_part_kernel<T, PIECE_NT, nv.value><<<(uint32_t)blocks, PIECE_NT, 0, st>>>(
                p, (uint32_t)len, stride, ids, values, k, lse != nullptr, inv_t, cut.pieces, part);
        });
        ung_distill_join_kernel<T><<<(uint32_t)rows, 128, 0, st>>>(p, (uint32_t)len, stride, ids, values, k, lse,
                                                                   inv_t, cut.pieces, part, loss, kept);
        if (grad)
            with_nv(cut.nv, [&](auto nv) {
                ung_distill_grad_kernel<T, PIECE_NT, nv.value><<<(uint32_t)blocks, PIECE_NT, 0, st>>>(
                    p, (uint32_t)len, stride, ids, values, k, kept, weight, inv_t, cut.pieces, (T *)grad, grad_stride);
            });
        return launched(what);
    });
}

} // namespace

extern "C" {

int ung_hip_top_scores_workspace(const void *scores, int type, uint64_t rows, uint64_t len, uint64_t row_stride,
                                 uint32_t k, uint64_t *bytes)
{
    static const char what[] = "ung_hip_top_scores_workspace";
    clear_error();
    int rc;
    if ((rc = check_scores(what, scores, type, rows, len, row_stride)) || (rc = check_k(what, k, 1)))
        return rc;
    if (!bytes) {
        set_error("%s: null bytes", what);
        return UNG_HIP_EINVAL;
    }
    return with_type(type, [&](auto zero) {
        const uint32_t v = vectors_at_most<decltype(zero)>(scores, rows, row_stride, len);
        *bytes = rows ? top_bytes(rows, top_cut(rows, v).pieces, k) : 0;
        return UNG_HIP_OK;
    });
}

int ung_hip_top_scores(const void *scores, int type, uint64_t rows, uint64_t len, uint64_t row_stride, uint32_t k,
                       float temperature, float *values, int32_t *ids, float *lse, void *workspace,
                       uint64_t workspace_bytes, void *stream)
{
    static const char what[] = "ung_hip_top_scores";
    clear_error();
    int rc;
    if ((rc = check_scores(what, scores, type, rows, len, row_stride)) || (rc = check_k(what, k, 1)) ||
        (rc = check_temperature(what, temperature)))
        return rc;
    if (rows == 0)
        return UNG_HIP_OK;
    if (!values || !ids) {
        set_error("%s: null values/ids", what);
        return UNG_HIP_EINVAL;
    }
    const hipStream_t st = (hipStream_t)stream;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const Cut cut = top_cut(rows, vectors_at_most<T>(scores, rows, row_stride, len));
        int rc;
        if ((rc = check_grid(what, rows * cut.pieces)) ||
            (rc = check_workspace(what, workspace, workspace_bytes, top_bytes(rows, cut.pieces, k))))
            return rc;
        char *at = (char *)workspace;
        auto take = [&](uint64_t bytes) {
            void *p = at;
            at += ceil_div(bytes, 16) * 16;
            return p;
        };
        uint64_t lists = cut.pieces;
        uint64_t *part = nullptr;
        float2 *sums = nullptr;
        if (lists > 1) {
            part = (uint64_t *)take(rows * lists * k * 8);
            sums = (float2 *)take(rows * lists * 8);
        }
        with_nv(cut.nv, [&](auto nv) {
            ung_top_scores_kernel<T, nv.value><<<(uint32_t)(rows * lists), TOP_NT, 0, st>>>(
                (const T *)scores, (uint32_t)len, row_stride, (uint32_t)lists, k, 1.0f / temperature, values, ids, lse,
                part, sums);
        });
        while (lists > 1) {
            const uint64_t groups = ceil_div(lists, MERGE_LISTS);
            uint64_t *out = nullptr;
            float2 *out_sums = nullptr;
            if (groups > 1) {
                out = (uint64_t *)take(rows * groups * k * 8);
                out_sums = (float2 *)take(rows * groups * 8);
            }
            ung_top_merge_kernel<<<(uint32_t)(rows * groups), TOP_NT, 0, st>>>(
                part, sums, (uint32_t)lists, (uint32_t)groups, k, values, ids, lse, out, out_sums);
            part = out;
            sums = out_sums;
            lists = groups;
        }
        return launched(what);
    });
}

int ung_hip_distill_workspace(const void *scores, int type, uint64_t rows, uint64_t len, uint64_t row_stride,
                              uint64_t *bytes)
{
    static const char what[] = "ung_hip_distill_workspace";
    clear_error();
    int rc;
    if ((rc = check_scores(what, scores, type, rows, len, row_stride)))
        return rc;
    if (!bytes) {
        set_error("%s: null bytes", what);
        return UNG_HIP_EINVAL;
    }
    return with_type(type, [&](auto zero) {
        const uint32_t v = vectors_at_most<decltype(zero)>(scores, rows, row_stride, len);
        *bytes = whole_rows(rows, v) ? 0 : part_bytes(rows, piece_cut(rows, v).pieces) + rows * sizeof(Saved);
        return UNG_HIP_OK;
    });
}

int ung_hip_distill_forward(const void *scores, int type, uint64_t rows, uint64_t len, uint64_t row_stride,
                            const int32_t *ids, const float *values, uint32_t k, const float *teacher_lse,
                            float temperature, float *loss, float *saved, void *workspace, uint64_t workspace_bytes,
                            void *stream)
{
    static const char what[] = "ung_hip_distill_forward";
    clear_error();
    int rc;
    if ((rc = check_distill(what, scores, type, rows, len, row_stride, ids, values, k, temperature)))
        return rc;
    if (rows == 0)
        return UNG_HIP_OK;
    if (!loss || !saved || (uintptr_t)saved % 16) {
        set_error("%s: null loss/saved, or saved not at a 16-byte boundary", what);
        return UNG_HIP_EINVAL;
    }
    return distill(what, scores, type, rows, len, row_stride, ids, values, k, teacher_lse, nullptr, temperature, loss,
                   (Saved *)saved, nullptr, 0, workspace, workspace_bytes, (hipStream_t)stream);
}

int ung_hip_distill_backward(const void *scores, int type, uint64_t rows, uint64_t len, uint64_t row_stride,
                             const int32_t *ids, const float *values, uint32_t k, const float *saved,
                             const float *weight, float temperature, void *grad, uint64_t grad_stride, void *stream)
{
    static const char what[] = "ung_hip_distill_backward";
    clear_error();
    int rc;
    if ((rc = check_distill(what, scores, type, rows, len, row_stride, ids, values, k, temperature)) ||
        (rc = check_grad(what, grad, type, rows, len, grad_stride)))
        return rc;
    if (rows == 0 || len == 0)
        return UNG_HIP_OK;
    if (!saved || (uintptr_t)saved % 16) {
        set_error("%s: null saved, or not at a 16-byte boundary", what);
        return UNG_HIP_EINVAL;
    }
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        const Cut cut = piece_cut(rows, vectors_at_most<T>(scores, rows, row_stride, len));
        int rc;
        if ((rc = check_grid(what, rows * cut.pieces)))
            return rc;
        with_nv(cut.nv, [&](auto nv) {
            ung_distill_grad_kernel<T, PIECE_NT, nv.value><<<(uint32_t)(rows * cut.pieces), PIECE_NT, 0,
                                                             (hipStream_t)stream>>>(
                (const T *)scores, (uint32_t)len, row_stride, ids, values, k, (const Saved *)saved, weight,
                1.0f / temperature, cut.pieces, (T *)grad, grad_stride);
        });
        return launched(what);
    });
}

int ung_hip_distill_step(const void *scores, int type, uint64_t rows, uint64_t len, uint64_t row_stride,
                         const int32_t *ids, const float *values, uint32_t k, const float *teacher_lse,
                         const float *weight, float temperature, float *loss, void *grad, uint64_t grad_stride,
                         void *workspace, uint64_t workspace_bytes, void *stream)
{
    static const char what[] = "ung_hip_distill_step";
    clear_error();
    int rc;
    if ((rc = check_distill(what, scores, type, rows, len, row_stride, ids, values, k, temperature)) ||
        (rc = check_grad(what, grad, type, rows, len, grad_stride)))
        return rc;
    if (rows == 0)
        return UNG_HIP_OK;
    if (!loss) {
        set_error("%s: null loss", what);
        return UNG_HIP_EINVAL;
    }
    return distill(what, scores, type, rows, len, row_stride, ids, values, k, teacher_lse, weight, temperature, loss,
                   nullptr, grad, grad_stride, workspace, workspace_bytes, (hipStream_t)stream);
}

} // extern "C"
