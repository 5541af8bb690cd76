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
constexpr double LOG2E = 1.4426950408889634;

struct Temperature {
    float inv, c; // 1 / T, log2(e) / T
};

__device__ inline float max_of(float a, float b) { return fmaxf(a, b); }

template <class T>
struct RowRef {
    static constexpr uint32_t N = Vec<T>::N;
    const T *row;
    uint32_t shift;        // elements between the 16-byte boundary and the row's first one
    uint32_t len;
    uint32_t whole, wholes; // the first vector wholly inside the row, and how many there are
    uint32_t end;          // vectors in all
    __device__ RowRef(const T *r, uint32_t n)
        : row(r), shift((uint32_t)(((uintptr_t)r & 15) / sizeof(T))), len(n), whole(shift ? 1 : 0),
          wholes((shift + n) / N > whole ? (shift + n) / N - whole : 0), end((shift + n + N - 1) / N)
    {
    }
    __device__ bool inside(uint32_t i) const { return i - whole < wholes; }
    // Vector i of the row; elements outside the row are -inf.
    __device__ Vec<T> load(uint32_t i) const
    {
        if (inside(i))
            return reinterpret_cast<const Vec<T> *>(row - shift)[i];
        Vec<T> v;
        v.fill_neg_inf();
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) {
            const uint32_t j = i * N + e - shift; // wraps below the row
            if (j < len)
                v.set(e, row[j]);
        }
        return v;
    }
    // Elements of vector i to a row of the same length, but for those whose bits are in `skip`.
    __device__ void store_elements(T *to, uint32_t i, const Vec<T> &v, uint32_t skip) const
    {
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) {
            const uint32_t j = i * N + e - shift;
            if (j < len && !(skip >> e & 1))
                to[j] = v.element(e);
        }
    }
};

// A stretch of a row, NT * NV vectors from `begin` on, in a block's registers: a thread holds
// the vectors begin + thread + i NT that lie wholly inside the row (-inf elsewhere), and its
// first two threads the vectors across the row's ends, if the stretch has them.
template <class T, int NT, int NV>
struct Stretch {
    Vec<T> v[NV], edge;
    uint32_t first, edge_at;
    bool has_edge;
    __device__ Stretch(const RowRef<T> &ref, uint32_t begin) : first(begin + threadIdx.x)
    {
        const Vec<T> *from = reinterpret_cast<const Vec<T> *>(ref.row - ref.shift);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i].fill_neg_inf();
            if (ref.inside(first + i * NT))
                v[i] = from[first + i * NT];
        }
        edge_at = threadIdx.x ? ref.end - 1 : 0;
        has_edge = threadIdx.x < 2 && edge_at - begin < NT * NV && edge_at < ref.end && !ref.inside(edge_at) &&
                   (threadIdx.x == 0 || edge_at > 0 || ref.end == 0);
        if (has_edge)
            edge = ref.load(edge_at);
    }
    // f(vector, its place in the row) for every vector of the thread
    template <class F>
    __device__ void each(F f)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            // keeps the compiler from holding the 32-bit values from pass to pass: 16-bit rows
            // would take twice the registers
            if constexpr (sizeof(T) == 2)
                asm volatile("" : "+v"(v[i].w[0]), "+v"(v[i].w[1]), "+v"(v[i].w[2]), "+v"(v[i].w[3]));
            f(v[i], first + i * NT);
        }
        if (has_edge)
            f(edge, edge_at);
    }
};

// ---- the first k of a row ------------------------------------------------------------

// A score as a whole number that orders like it: NaN above every score, -0 as 0, and 0 for no
// candidate (-inf).  With the id in the lower half, of equal scores the lower id is the larger
// number.
__device__ inline uint32_t key_of(float x)
{
    if (x == NEG_INF)
        return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0xFFFFFFFFu : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline uint64_t order_of(float x, uint32_t id)
{
    const uint32_t k = key_of(x);
    return k ? (uint64_t)k << 32 | (uint32_t)~id : 0;
}
__device__ inline float score_of(uint32_t key)
{
    return key == 0xFFFFFFFFu ? __builtin_nanf("") : __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

constexpr int TOP_NT = 256;   // threads of a block
constexpr int TOP_CAP = 1024; // candidates a block ranks

struct TopShared {
    alignas(16) uint64_t cand[TOP_CAP];
    uint32_t most[TOP_NT];
    float red[2][TOP_NT / 64];
    uint32_t wave_count[TOP_NT / 64];
    uint32_t count;
    uint32_t limit;
};

// The largest key with at least k of the threads' maxima at or above it, found bit by bit by
// one wave that holds all of them (a count is a ballot); the lowest LOW bits are left 0, which
// keys of 16-bit scores do not need told apart.  No larger than the k-th largest key of all,
// and few keys lie between the two.  0: fewer than k threads have a candidate.
template <int LOW>
__device__ inline uint32_t limit_of(const uint32_t *most, uint32_t k)
{
    uint32_t m[TOP_NT / 64], limit = 0;
#pragma unroll
    for (int i = 0; i < TOP_NT / 64; ++i)
        m[i] = most[i * 64 + (threadIdx.x & 63)];
#pragma unroll 4
    for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t trial = limit | 1u << bit;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < TOP_NT / 64; ++i)
            n += __popcll(__ballot(m[i] >= trial));
        limit = n >= k ? trial : limit;
    }
    return limit;
}

// The k-th largest of the orders that a block holds (each(f) calls f with those of a thread; 0
// = none), bit by bit over the whole block: for rows of many equal scores, where the
// candidates above the threads' limit do not fit.  0: there are fewer than k.  Each bit reads the
// row again: 4096 x 32768, k = 64, all but ten scores of a row at the type's lowest value bf16 3.9 ms
// (different scores 81 us), float32 5.6 ms (114 us); 1 x 100000, k = 32, bf16 91 us (15).
//   The bit moves down by shifts of one, not 1 << n: v_lshlrev_b64 with n in the last vector
// register of a wave's allocation (v103 of 104, float32 rows of 4 vectors a thread) shifted by
// something else in waves beside another block's, and waves searched with different trials (228
// of 600 such rows wrong; right in builds where n lay in another register).
template <class Each>
__device__ inline uint64_t kth_order(TopShared &sh, uint32_t k, Each each)
{
    uint64_t limit = 0;
    for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
        const uint64_t trial = limit | bit;
        uint32_t mine = 0;
        each([&](uint64_t o) { mine += o >= trial; });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            mine += __shfl_xor((int)mine, o);
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
            sh.wave_count[threadIdx.x >> 6] = mine;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (int w = 0; w < TOP_NT / 64; ++w)
            all += sh.wave_count[w];
        if (all >= k)
            limit = trial;
    }
    return limit;
}

// The k-th largest key of up to TOP_CAP candidates, by one wave as in limit_of; 0 if there are
// fewer than k.
template <int LOW>
__device__ inline uint32_t kth_key(const uint64_t *cand, uint32_t found, uint32_t k)
{
    uint32_t m[TOP_CAP / 64], limit = 0;
#pragma unroll
    for (int i = 0; i < TOP_CAP / 64; ++i)
        m[i] = i * 64 + (threadIdx.x & 63) < found ? (uint32_t)(cand[i * 64 + (threadIdx.x & 63)] >> 32) : 0;
    for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t trial = limit | 1u << bit;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < TOP_CAP / 64; ++i)
            n += __popcll(__ballot(m[i] >= trial));
        limit = n >= k ? trial : limit;
    }
    return limit;
}

__device__ inline void add_candidate(TopShared &sh, uint64_t order)
{
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < TOP_CAP)
        sh.cand[at] = order;
}

// Results of a row (or of a part of one) whose first k orders are among sh.cand[0..count):
// each candidate's place is the number of candidates above it.  Where the candidates did not
// fit, they are collected anew from the k-th order on.
template <int LOW, class Each>
__device__ inline void finish_top(TopShared &sh, uint32_t k, Each each, uint64_t row, bool last, float *values,
                                  int32_t *ids, float *lse, uint64_t *part, float2 *part_sum, float top, float sum,
                                  Temperature t)
{
    const uint32_t tid = threadIdx.x;
    uint32_t found = sh.count;
    if (found > TOP_CAP) {
        const uint64_t limit = kth_order(sh, k, each);
        if (tid == 0)
            sh.count = 0;
        __syncthreads();
        each([&](uint64_t o) {
            if (o && o >= limit) // limit 0: fewer than k
                add_candidate(sh, o);
        });
        __syncthreads();
        found = sh.count; // k at most: orders are distinct
    } else if (found > 320) {
        // ranking compares every two candidates: with the k-th key of them, few are left
        uint64_t mine[TOP_CAP / TOP_NT];
#pragma unroll
        for (int i = 0; i < TOP_CAP / TOP_NT; ++i)
            mine[i] = i * TOP_NT + tid < found ? sh.cand[i * TOP_NT + tid] : 0;
        __syncthreads(); // every wave has read the count, or a late one would find it reset
        if (tid < 64) {
            const uint32_t limit = kth_key<LOW>(sh.cand, found, k);
            if (tid == 0) {
                sh.limit = limit;
                sh.count = 0;
            }
        }
        __syncthreads();
        const uint64_t least = sh.limit ? (uint64_t)sh.limit << 32 : 1;
#pragma unroll
        for (int i = 0; i < TOP_CAP / TOP_NT; ++i)
            if (mine[i] >= least)
                add_candidate(sh, mine[i]);
        __syncthreads();
        found = sh.count;
    }
    auto put = [&](uint32_t place, uint64_t o) {
        if (last) {
            values[row * k + place] = o ? score_of((uint32_t)(o >> 32)) : NEG_INF;
            ids[row * k + place] = o ? (int32_t)~(uint32_t)o : -1;
        } else
            part[row * k + place] = o;
    };
    for (uint32_t i = tid; i < found; i += TOP_NT) {
        const uint64_t mine = sh.cand[i];
        uint32_t place = 0;
#pragma unroll 8
        for (uint32_t o = 0; o < found; ++o)
            place += sh.cand[o] > mine;
        if (place < k)
            put(place, mine);
    }
    if (tid >= found && tid < k)
        put(tid, 0);
    if (tid == 0) {
        if (!last)
            part_sum[row] = make_float2(top, sum);
        else if (lse)
            lse[row] = fabsf(top) == __builtin_inff() ? top : top * t.inv + logf(sum);
    }
}

// The first k of one piece of a row (TOP_NT * NV vectors; the whole row if `pieces` is 1), its
// values held in registers: one read of the scores, bound by memory.  While one wave finds
// the limit from the threads' maxima, the others sum the weights exp((s - maximum) / T).
template <class T, int NV>
__global__ __launch_bounds__(TOP_NT, 4) void ung_top_scores_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                                   uint32_t pieces, uint32_t k, Temperature t,
                                                                   float *values, int32_t *ids, float *lse,
                                                                   uint64_t *part, float2 *part_sum)
{
    constexpr int N = Vec<T>::N;
    constexpr int LOW = std::is_same_v<T, bf16_t> ? 16 : std::is_same_v<T, fp16_t> ? 13 : 0;
    __shared__ TopShared sh;
    const uint64_t r = blockIdx.x / pieces;
    const uint32_t piece = (uint32_t)(blockIdx.x - r * pieces), tid = threadIdx.x;
    const RowRef<T> ref(scores + r * stride, len);
    Stretch<T, TOP_NT, NV> x(ref, piece * (TOP_NT * NV));
    float most = NEG_INF, most_of[NV + 1];
    int n = 0;
    x.each([&](const Vec<T> &v, uint32_t) {
        float m = v.get(0);
#pragma unroll
        for (int e = 1; e < N; ++e)
            m = fmaxf(m, v.get(e)); // a NaN shows in the sum
        most_of[n++] = m;
        most = fmaxf(most, m);
    });
    sh.most[tid] = key_of(most);
    if (tid == 0)
        sh.count = 0;
    const float top = block_reduce<TOP_NT>(most, sh.red[0], max_of);
    if (tid < 64) {
        const uint32_t limit = limit_of<LOW>(sh.most, k);
        if (tid == 0)
            sh.limit = limit;
    }
    const float at = top == NEG_INF ? 0.0f : top;
    float sum = 0.0f;
    x.each([&](const Vec<T> &v, uint32_t) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            sum += weight_of(v.get(e), at, t.c);
    });
    sum = block_reduce<TOP_NT>(sum, sh.red[1], add);
    // the rest looks at few vectors, and reads those again
    const uint32_t shift = ref.shift, first = x.first, edge_at = x.edge_at, slots = NV + (x.has_edge ? 1 : 0);
    auto scan = [=](uint32_t i, auto f) {
        const uint32_t at = i < NV ? first + i * TOP_NT : edge_at;
        const Vec<T> v = ref.load(at); // -inf outside the row
#pragma unroll
        for (int e = 0; e < N; ++e)
            f(v.get(e), at * N + e - shift);
    };
    auto each = [=](auto f) {
        for (uint32_t i = 0; i < slots; ++i)
            if (i >= NV || ref.inside(first + i * TOP_NT))
                scan(i, [&](float x, uint32_t id) { f(order_of(x, id)); });
    };
    if (sum == sum) {
        // scores at or above the limit; -inf is below every float
        const float least = sh.limit ? score_of(sh.limit) : -3.402823466e38f;
        uint32_t hit = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            hit |= most_of[i] >= least ? 1u << i : 0u;
        if (x.has_edge && most_of[NV] >= least)
            hit |= 1u << NV;
        for (; hit; hit &= hit - 1)
            scan((uint32_t)__ffs((int)hit) - 1, [&](float x, uint32_t id) {
                if (x >= least)
                    add_candidate(sh, order_of(x, id));
            });
    } else if (tid == 0)
        sh.count = TOP_CAP + 1; // a NaN or +inf: the maxima do not tell
    __syncthreads();
    float out_sum = sum, out_top = top;
    if (sum != sum) { // +inf alone has the log-sum-exp +inf
        float any = 0.0f;
        each([&](uint64_t o) { any = (uint32_t)(o >> 32) == 0xFFFFFFFFu ? 1.0f : any; });
        any = block_reduce<TOP_NT>(any, sh.red[0], add);
        out_top = any > 0.0f ? sum : __builtin_inff();
    }
    finish_top<LOW>(sh, k, each, blockIdx.x, pieces == 1, values, ids, lse, part, part_sum, out_top, out_sum, t);
}

constexpr uint32_t MERGE_LISTS = 64; // lists one block merges

// Merges up to MERGE_LISTS partial rows of a row, NI orders a thread.
template <int NI>
__global__ __launch_bounds__(TOP_NT) void ung_top_merge_kernel(const uint64_t *part, const float2 *part_sum,
                                                               uint32_t lists, uint32_t groups, uint32_t k,
                                                               float *values, int32_t *ids, float *lse, uint64_t *out,
                                                               float2 *out_sum, Temperature t)
{
    __shared__ TopShared sh;
    const uint64_t r = blockIdx.x / groups;
    const uint32_t tid = threadIdx.x;
    const uint32_t first = (uint32_t)(blockIdx.x - r * groups) * MERGE_LISTS;
    const uint32_t n = lists - first < MERGE_LISTS ? lists - first : MERGE_LISTS, items = n * k;
    const uint64_t *mine = part + (r * lists + first) * k;
    uint64_t v[NI];
    // lists are sorted: each is turned by its own amount, or some threads would hold all the
    // large orders and their maxima tell little (k = 128: 55 us)
    const float per_k = 1.0f / (float)k;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const uint32_t j = i * TOP_NT + tid, list = (uint32_t)(((float)j + 0.5f) * per_k);
        const uint32_t turned = j - list * k + __umulhi(list * 0x9E3779B1u, k);
        v[i] = j < items ? mine[list * k + (turned < k ? turned : turned - k)] : 0;
    }
    float2 s = make_float2(NEG_INF, 0.0f);
    if (tid < n)
        s = part_sum[r * lists + first + tid];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i)
        most = max(most, (uint32_t)(v[i] >> 32));
    sh.most[tid] = most;
    if (tid == 0)
        sh.count = 0;
    const float top = block_reduce<TOP_NT>(s.x, sh.red[0], max_nan);
    if (tid < 64) {
        const uint32_t limit = limit_of<0>(sh.most, k);
        if (tid == 0)
            sh.limit = limit;
    }
    const float sum = block_reduce<TOP_NT>(s.y == 0.0f ? 0.0f : s.y * weight_of(s.x, top == NEG_INF ? 0.0f : top, t.c),
                                           sh.red[1], add);
    const uint64_t least = sh.limit ? (uint64_t)sh.limit << 32 : 1;
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            f(v[i]);
    };
    each([&](uint64_t o) {
        if (o >= least)
            add_candidate(sh, o);
    });
    __syncthreads();
    finish_top<0>(sh, k, each, blockIdx.x, groups == 1, values, ids, lse, out, out_sum, top, sum, t);
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
// enter the row's from the entries.  Their gradients come from the entries too, and the
// vectors that hold them go out without them, so that no store waits for another.  A row
// without a valid entry, or without a score above -inf, has loss and gradient 0.

// What the backward pass needs of a row besides its inputs.
struct alignas(16) Saved {
    float top;      // largest score of the whole row; EMPTY: no loss
    float inside;   // W / sum exp((s - top) / T)
    float rest_top; // the same two of the columns outside the list: gradient = weight / T *
    float outside;  // exp((s - rest_top) / T) * outside
    float base, log; // p_k = exp((t_k - base) / T - log)
    float unused[2];
};
static_assert(sizeof(Saved) == 4 * UNG_HIP_DISTILL_SAVED, "");

constexpr float EMPTY = __builtin_inff(); // Saved::top of a row without loss

struct DistillShared {
    float z[MAX_K]; // the teacher's score; -inf = not there
    float s[MAX_K]; // the student's there
    float p[MAX_K]; // p_k
    uint32_t id[MAX_K];
    uint32_t first[MAX_K]; // the entry is the first one to name its column
    float red[2][16];
    float base, log, mass; // as in Saved; sum of p_k
    uint32_t any, twice;   // entries there are; a column that several of them name
    Saved saved;
};

// One entry of the teacher's row, loaded by each of the first k threads: ahead of the scores,
// which it would else have to wait for.
struct Entry {
    int32_t id;
    float value;
    __device__ Entry(const int32_t *ids, const float *values, uint32_t k)
        : id(threadIdx.x < k ? ids[threadIdx.x] : -1), value(threadIdx.x < k ? values[threadIdx.x] : NEG_INF)
    {
    }
};

// Entries into sh, with the student's scores of those whose columns lie in [from, to) (a block
// that writes the gradient over the scores reads no other block's stretch).
template <class T>
__device__ inline void keep_entries(DistillShared &sh, const Entry &e, const T *row, uint32_t k, uint32_t len,
                                    int64_t from, int64_t to)
{
    const uint32_t tid = threadIdx.x;
    if (tid == 0)
        sh.twice = 0;
    if (tid < k) {
        const bool ok = (uint32_t)e.id < len && e.value != NEG_INF;
        sh.id[tid] = ok ? (uint32_t)e.id : 0xFFFFFFFFu;
        sh.z[tid] = ok ? e.value : NEG_INF;
        sh.s[tid] = ok && e.id >= from && e.id < to ? to_float(row[e.id]) : 0.0f;
        sh.first[tid] = ok;
    }
}

// sh.first by the order of the entries (of equal ones a fixed one, whichever thread came first).
__device__ inline void find_first(DistillShared &sh, uint32_t k)
{
    const uint32_t tid = threadIdx.x;
    if (tid < k) {
        const uint32_t id = sh.id[tid];
        bool first = id != 0xFFFFFFFFu;
        for (uint32_t o = 0; o < tid; ++o)
            first &= sh.id[o] != id;
        sh.first[tid] = first;
    }
    __syncthreads();
}

// Bits of the listed columns among the `vectors` vectors from `begin` on, and sh.first and
// sh.twice of the entries there.  Begins and ends with the block together.
template <int N, int NT>
__device__ inline void mark_listed(DistillShared &sh, uint32_t *bits, uint32_t begin, uint32_t vectors,
                                   uint32_t shift, uint32_t k)
{
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = tid; i < vectors * N / 32; i += NT)
        bits[i] = 0;
    __syncthreads();
    if (tid < k && sh.id[tid] != 0xFFFFFFFFu) {
        const uint64_t at = (uint64_t)sh.id[tid] + shift, from = (uint64_t)begin * N;
        if (at >= from && at < from + (uint64_t)vectors * N) {
            const uint32_t bit = 1u << ((at - from) & 31);
            if (atomicOr(&bits[(at - from) >> 5], bit) & bit)
                sh.twice = 1;
        }
    }
    __syncthreads();
    if (sh.twice)
        find_first(sh, k);
}

// Listed columns of one vector, a bit for each.
template <int N>
__device__ inline uint32_t listed_of(const uint32_t *bits, uint32_t begin, uint32_t at)
{
    const uint32_t b = (at - begin) * N;
    return bits[b >> 5] >> (b & 31) & ((1u << N) - 1);
}

// The teacher's side of a row, run by one wave.
__device__ inline void teacher_row(DistillShared &sh, uint32_t k, const float *lse, Temperature t)
{
    const uint32_t lane = threadIdx.x & 63;
    float z[2], best = NEG_INF, base = 0.0f, log_base = 0.0f;
    bool any = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        z[h] = h * 64 + lane < k ? sh.z[h * 64 + lane] : NEG_INF;
        any |= z[h] != NEG_INF;
        best = max_nan(best, z[h]);
    }
    any = __any(any);
    if (lse)
        log_base = *lse;
    else if (any) {
        float sum = 0.0f;
        base = wave_reduce(best, max_nan);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            sum += z[h] == NEG_INF ? 0.0f : expf((z[h] - base) * t.inv);
        log_base = logf(wave_reduce(sum, add));
    }
    float mass = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float p = z[h] == NEG_INF ? 0.0f : expf((z[h] - base) * t.inv - log_base);
        mass += p;
        if (h * 64 + lane < k)
            sh.p[h * 64 + lane] = p;
    }
    mass = wave_reduce(mass, add);
    if (lane == 0) {
        sh.any = any;
        sh.base = base;
        sh.log = log_base;
        sh.mass = mass;
    }
}

// Loss and Saved of a row, run by the wave that made the teacher's side: from that, the entries
// and the sums (maximum, sum of exp((s - maximum) / T)) of the row's columns, with `lse` of
// those outside the list.  Returns the loss in every lane.
__device__ inline float finish_row(DistillShared &sh, uint32_t k, bool tail, float2 sums, Temperature t, Saved &saved)
{
    const uint32_t lane = threadIdx.x & 63;
    float s[2], top = sums.x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = h * 64 + lane;
        s[h] = i < k ? sh.s[i] : 0.0f;
        if (tail && i < k && sh.first[i])
            top = max_of(top, s[h]);
    }
    saved = Saved{EMPTY, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, {}};
    top = wave_reduce(top, max_of);
    const float at = top == NEG_INF ? 0.0f : top;
    float total = sums.y;
    if (tail) {
        float in = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (h * 64 + lane < k && sh.first[h * 64 + lane])
                in += weight_of(s[h], at, t.c);
        total = wave_reduce(in, add) + (sums.y == 0.0f ? 0.0f : sums.y * weight_of(sums.x, at, t.c));
    }
    if (total != total) // a NaN among the scores, or +inf: the whole row is NaN
        top = total;
    if (!sh.any || top == NEG_INF)
        return 0.0f;
    const float log_total = logf(total), mass = sh.mass;
    float loss = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t i = h * 64 + lane;
        if (i < k && sh.z[i] != NEG_INF) {
            const float p = sh.p[i], log_p = (sh.z[i] - sh.base) * t.inv - sh.log;
            if (!(p <= 0.0f))
                loss += p * (log_p - ((s[h] - top) * t.inv - log_total));
        }
    }
    loss = wave_reduce(loss, add);
    saved = Saved{top, mass / total, top, mass / total, sh.base, sh.log, {}};
    if (tail && !(sums.y <= 0.0f)) {
        const float rest = 1.0f - mass < 0.0f ? 0.0f : 1.0f - mass;
        saved.rest_top = sums.x;
        if (!(rest <= 0.0f)) {
            loss += rest * (logf(rest) - ((sums.x - top) * t.inv + logf(sums.y) - log_total));
            saved.inside = (mass + rest) / total;
        }
        saved.outside = weight_of(sums.x, top, t.c) * saved.inside - rest / sums.y;
    }
    return loss;
}

// Gradient of a stretch of a row whose vectors are in registers: of the listed columns (marked
// in `bits`) from their entries, of the others from the vectors.
template <class T, int NT, int NV>
__device__ inline void write_gradient(DistillShared &sh, const uint32_t *bits, const RowRef<T> &ref,
                                      Stretch<T, NT, NV> &x, uint32_t begin, uint32_t k, Temperature t,
                                      const Saved saved, float weight, T *grad)
{
    constexpr int N = Vec<T>::N;
    const bool same = ((uintptr_t)grad & 15) == ref.shift * sizeof(T);
    const float c = t.c, w = weight * t.inv, out = saved.outside * w;
    const float rest_top = saved.rest_top;
    auto put = [&](const Vec<T> &g, uint32_t at, uint32_t skip) {
        const bool inside = ref.inside(at);
        if (same && inside && !skip)
            reinterpret_cast<Vec<T> *>(grad - ref.shift)[at] = g;
        else if (inside || (x.has_edge && at == x.edge_at)) // an end is written by its holder alone
            ref.store_elements(grad, at, g, skip);
    };
    if (saved.top == EMPTY) {
        x.each([&](const Vec<T> &, uint32_t at) { put(Vec<T>{}, at, 0); });
        return;
    }
    const uint32_t id = threadIdx.x < k && sh.first[threadIdx.x] ? sh.id[threadIdx.x] : 0xFFFFFFFFu;
    const uint32_t at = (id + ref.shift) / N;
    if (id != 0xFFFFFFFFu && at >= begin && at < begin + NT * NV) {
        float p = sh.p[threadIdx.x];
        if (sh.twice) { // of every entry that names this column
            p = 0.0f;
            for (uint32_t o = 0; o < k; ++o)
                p += sh.id[o] == id ? sh.p[o] : 0.0f;
        }
        const float e = weight_of(sh.s[threadIdx.x], saved.top, t.c);
        grad[id] = from_float<T>((e * saved.inside - p) * w);
    }
    x.each([&](const Vec<T> &v, uint32_t at) {
        Vec<T> g;
#pragma unroll
        for (int e = 0; e < N; e += 2)
            g.put2(e, weight_of(v.get(e), rest_top, c) * out, weight_of(v.get(e + 1), rest_top, c) * out);
        put(g, at, listed_of<N>(bits, begin, at));
    });
}

// Sums of a stretch of a row in registers, in every thread: its maximum and the sum of
// exp((s - maximum) / T).  With `tail` listed columns become -inf first.
template <class T, int NT, int NV>
__device__ inline float2 stretch_sums(DistillShared &sh, const uint32_t *bits, Stretch<T, NT, NV> &x, uint32_t begin,
                                      bool tail, float c)
{
    constexpr int N = Vec<T>::N;
    if (tail)
        x.each([&](Vec<T> &v, uint32_t at) {
            const uint32_t listed = listed_of<N>(bits, begin, at);
            if (listed)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (listed >> e & 1)
                        v.set(e, (T)NEG_INF);
        });
    float most = NEG_INF;
    x.each([&](const Vec<T> &v, uint32_t) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            most = max_of(most, v.get(e)); // a NaN shows in the sum
    });
    const float top = block_reduce<NT>(most, sh.red[0], max_of);
    const float at = top == NEG_INF ? 0.0f : top;
    float sum = 0.0f;
    x.each([&](const Vec<T> &v, uint32_t) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            sum += weight_of(v.get(e), at, c);
    });
    return make_float2(top, block_reduce<NT>(sum, sh.red[1], add));
}

// A row by one block, its scores in registers: loss, and the gradient with `grad`.  One read
// of the scores and one write of the gradient, bound by memory: 4096 x 32768, k = 64, bf16 130
// us (4.1 TB/s), float32 214 (5.0; a copy of it 4.9); 64 x 10000 8.2.  `grad` may be the scores.
// One wave makes the teacher's side while the others await the scores.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT, NV <= 8 ? 8 : 4) void ung_distill_row_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                             const int32_t *ids, const float *values, uint32_t k,
                                                             const float *lse, const float *weight, Temperature t,
                                                             float *loss, Saved *saved_out, T *grad,
                                                             uint64_t grad_stride)
{
    __shared__ DistillShared sh;
    __shared__ uint32_t bits[NT * NV * Vec<T>::N / 32];
    const uint64_t r = blockIdx.x;
    const RowRef<T> ref(scores + r * stride, len);
    const Entry entry(ids + r * k, values + r * k, k);
    Stretch<T, NT, NV> x(ref, 0);
    keep_entries(sh, entry, ref.row, k, len, 0, len);
    mark_listed<Vec<T>::N, NT>(sh, bits, 0, NT * NV, ref.shift, k);
    if (threadIdx.x < 64)
        teacher_row(sh, k, lse ? lse + r : nullptr, t);
    const float2 sums = stretch_sums<T, NT, NV>(sh, bits, x, 0, lse != nullptr, t.c);
    if (threadIdx.x < 64) {
        Saved saved;
        const float l = finish_row(sh, k, lse != nullptr, sums, t, saved);
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
    write_gradient<T, NT, NV>(sh, bits, ref, x, 0, k, t, sh.saved, weight ? weight[r] : 1.0f, grad + r * grad_stride);
}

// Sums of one piece of a row (NT * NV vectors).
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void ung_distill_part_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                              const int32_t *ids, const float *values, uint32_t k,
                                                              int tail, Temperature t, uint32_t pieces, float2 *part)
{
    __shared__ DistillShared sh;
    __shared__ uint32_t bits[NT * NV * Vec<T>::N / 32];
    const uint64_t r = blockIdx.x / pieces;
    const uint32_t begin = (uint32_t)(blockIdx.x - r * pieces) * (NT * NV);
    const RowRef<T> ref(scores + r * stride, len);
    const Entry entry(ids + r * k, values + r * k, tail ? k : 0);
    Stretch<T, NT, NV> x(ref, begin);
    if (tail) {
        keep_entries(sh, entry, ref.row, k, len, 0, 0);
        mark_listed<Vec<T>::N, NT>(sh, bits, begin, NT * NV, ref.shift, k);
    }
    const float2 sums = stretch_sums<T, NT, NV>(sh, bits, x, begin, tail, t.c);
    if (threadIdx.x == 0)
        part[blockIdx.x] = sums;
}

// A row's loss from its pieces' sums; one wave a row.
template <class T>
__global__ __launch_bounds__(128) void ung_distill_join_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                               const int32_t *ids, const float *values, uint32_t k,
                                                               const float *lse, Temperature t, uint32_t pieces,
                                                               const float2 *part, float *loss, Saved *saved_out)
{
    __shared__ DistillShared sh;
    const uint64_t r = blockIdx.x;
    keep_entries(sh, Entry(ids + r * k, values + r * k, k), scores + r * stride, k, len, 0, len);
    __syncthreads();
    if (lse)
        find_first(sh, k);
    if (threadIdx.x < 64)
        teacher_row(sh, k, lse ? lse + r : nullptr, t);
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
        sum += mine[i].y == 0.0f ? 0.0f : mine[i].x == NEG_INF ? mine[i].y : mine[i].y * weight_of(mine[i].x, at, t.c);
    sum = wave_reduce(sum, add);
    Saved saved;
    const float l = finish_row(sh, k, lse != nullptr, make_float2(top, sum), t, saved);
    if (threadIdx.x == 0) {
        loss[r] = l;
        saved_out[r] = saved;
    }
}

// Gradient of one piece of a row from what its forward pass saved.  `grad` may be the scores.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void ung_distill_grad_kernel(const T *scores, uint32_t len, uint64_t stride,
                                                              const int32_t *ids, const float *values, uint32_t k,
                                                              const Saved *saved, const float *weight, Temperature t,
                                                              uint32_t pieces, T *grad, uint64_t grad_stride)
{
    __shared__ DistillShared sh;
    __shared__ uint32_t bits[NT * NV * Vec<T>::N / 32];
    const uint64_t r = blockIdx.x / pieces;
    const uint32_t begin = (uint32_t)(blockIdx.x - r * pieces) * (NT * NV);
    const RowRef<T> ref(scores + r * stride, len);
    const Entry entry(ids + r * k, values + r * k, k);
    const Saved row = saved[r];
    Stretch<T, NT, NV> x(ref, begin);
    const int64_t from = (int64_t)begin * Vec<T>::N - ref.shift;
    keep_entries(sh, entry, ref.row, k, len, from, from + NT * NV * Vec<T>::N);
    if (threadIdx.x < k)
        sh.p[threadIdx.x] = sh.z[threadIdx.x] == NEG_INF ? 0.0f : expf((sh.z[threadIdx.x] - row.base) * t.inv - row.log);
    // and the entries' scores are read before this block writes
    mark_listed<Vec<T>::N, NT>(sh, bits, begin, NT * NV, ref.shift, k);
    write_gradient<T, NT, NV>(sh, bits, ref, x, begin, k, t, row, weight ? weight[r] : 1.0f, grad + r * grad_stride);
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

Temperature temperature_of(float t) { return Temperature{1.0f / t, (float)(LOG2E / t)}; }

int check_temperature(const char *what, float t)
{
    if (t > 0.0f && t < __builtin_inff() && temperature_of(t).c < __builtin_inff())
        return UNG_HIP_OK;
    set_error("%s: temperature %g is not a positive number with a reciprocal in 32 bits", what, (double)t);
    return UNG_HIP_EINVAL;
}

int check_k(const char *what, uint32_t k, uint32_t least)
{
    if (k >= least && k <= (uint32_t)MAX_K)
        return UNG_HIP_OK;
    set_error("%s: k=%u outside %u..%d", what, k, least, MAX_K);
    return UNG_HIP_EINVAL;
}

int check_grid(const char *what, uint64_t blocks, uint32_t threads)
{
    if (blocks <= most_blocks(threads))
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

// A row by one block where it fits one (64 x 10000 float32 8.9 us, in pieces 12.2; 1 x 10000 6.7,
// 10.1; 256 x 16000 9.5, 14.3).  Longer rows in pieces, shorter ones where blocks are few, but
// no more than one pass merges (1 x 100000 in 49 pieces 13.6, in 98 18.5).
Cut top_cut(uint64_t rows, uint32_t vectors)
{
    uint32_t nv = 16;
    if (vectors <= TOP_NT * 16) {
        while (nv > 1 && TOP_NT * (nv / 2) >= vectors)
            nv /= 2;
        return Cut{nv, 1};
    }
    while (nv > 1 && rows * ceil_div(vectors, TOP_NT * nv) < 512 &&
           ceil_div(vectors, TOP_NT * (nv / 2)) <= MERGE_LISTS)
        nv /= 2;
    return Cut{nv, (uint32_t)ceil_div(vectors, TOP_NT * nv)};
}

uint64_t top_bytes(uint64_t rows, uint32_t pieces, uint32_t k)
{
    uint64_t bytes = 0;
    for (uint64_t lists = pieces; lists > 1; lists = ceil_div(lists, MERGE_LISTS))
        bytes += ceil_div(rows * lists * k * 8, 16) * 16 + ceil_div(rows * lists * 8, 16) * 16;
    return bytes;
}

// f with nv, one of 1, 2, 4 .. MOST, as a constant.
template <int MOST, class F>
void with_nv(uint32_t nv, F f)
{
    if (nv == 1)
        f(std::integral_constant<int, 1>{});
    else if (nv == 2)
        f(std::integral_constant<int, 2>{});
    else if (nv == 4)
        f(std::integral_constant<int, 4>{});
    else if (MOST == 8 || nv == 8)
        f(std::integral_constant<int, 8>{});
    else
        f(std::integral_constant<int, MOST>{});
}

constexpr int ROW_NT = 512;   // threads of a block that holds a whole row
constexpr int PIECE_NT = 256; // ... a piece of one

// A row by one block if it fits a block's registers, unless few long rows would leave most CUs
// without work: then pieces of rows, in three launches.  Loss and gradient, us, whole against in
// pieces: 64 x 10000 bf16 8.2, 13; 64 x 32768 12.6, 15; 120 x 65000 21.4, 22; 64 x 65000 18.7, 15.9.
bool whole_rows(uint64_t rows, uint32_t vectors)
{
    return vectors <= ROW_NT * 8 || (vectors <= ROW_NT * 16 && rows >= 128);
}

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

// Whether an element of `rows` rows of len elements at a is one of such rows at b, by their
// addresses in elements; strides are len at least where there are several rows.
bool rows_meet(uint64_t a, uint64_t a_stride, uint64_t b, uint64_t b_stride, uint64_t rows, uint64_t len)
{
    const uint64_t a_end = a + (rows - 1) * a_stride + len, b_end = b + (rows - 1) * b_stride + len;
    if (a >= b_end || b >= a_end)
        return false;
    if (rows == 1)
        return true;
    if (a_stride == b_stride) { // rows i of the later ones begin `in` after rows i + `by` of the earlier
        const uint64_t from = a < b ? b - a : a - b, by = from / a_stride, in = from % a_stride;
        return (in < len && by < rows) || (in + len > a_stride && by + 1 < rows);
    }
    for (uint64_t i = 0, j = 0; i < rows && j < rows;) {
        const uint64_t x = a + i * a_stride, y = b + j * b_stride;
        if (x + len <= y)
            ++i;
        else if (y + len <= x)
            ++j;
        else
            return true;
    }
    return false;
}

int check_grad(const char *what, const void *scores, uint64_t stride, const void *grad, int type, uint64_t rows,
               uint64_t len, uint64_t grad_stride)
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
    // in place a block writes what it alone reads; elsewhere among the scores others still read
    const bool in_place = grad == scores && (rows == 1 || grad_stride == stride);
    if (rows && len && !in_place &&
        rows_meet((uintptr_t)scores / type_size(type), stride, (uintptr_t)grad / type_size(type), grad_stride, rows, len)) {
        set_error("%s: the gradient overlaps the scores without being in their place", what);
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
        const Temperature t = temperature_of(temperature);
        const uint32_t vectors = vectors_at_most<T>(scores, rows, stride, len);
        int rc;
        if (whole_rows(rows, vectors)) {
            if ((rc = check_grid(what, rows, ROW_NT)))
                return rc;
            with_nv<16>(row_cut(vectors).nv, [&](auto nv) {
                ung_distill_row_kernel<T, ROW_NT, nv.value><<<(uint32_t)rows, ROW_NT, 0, st>>>(
                    p, (uint32_t)len, stride, ids, values, k, lse, weight, t, loss, saved, (T *)grad, grad_stride);
            });
            return launched(what);
        }
        const Cut cut = piece_cut(rows, vectors);
        const uint64_t parts = part_bytes(rows, cut.pieces), blocks = rows * cut.pieces;
        if ((rc = check_grid(what, blocks, PIECE_NT)) ||
            (rc = check_workspace(what, workspace, workspace_bytes, parts + (saved ? 0 : rows * sizeof(Saved)))))
            return rc;
        float2 *part = (float2 *)workspace;
        Saved *kept = saved ? saved : (Saved *)((char *)workspace + parts);
        with_nv<8>(cut.nv, [&](auto nv) {
            ung_distill_part_kernel<T, PIECE_NT, nv.value><<<(uint32_t)blocks, PIECE_NT, 0, st>>>(
                p, (uint32_t)len, stride, ids, values, k, lse != nullptr, t, cut.pieces, part);
        });
        ung_distill_join_kernel<T><<<(uint32_t)rows, 128, 0, st>>>(p, (uint32_t)len, stride, ids, values, k, lse,
                                                                   t, cut.pieces, part, loss, kept);
        if (grad)
            with_nv<8>(cut.nv, [&](auto nv) {
                ung_distill_grad_kernel<T, PIECE_NT, nv.value><<<(uint32_t)blocks, PIECE_NT, 0, st>>>(
                    p, (uint32_t)len, stride, ids, values, k, kept, weight, t, cut.pieces, (T *)grad, grad_stride);
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
        if ((rc = check_grid(what, rows * cut.pieces, TOP_NT)) ||
            (rc = check_workspace(what, workspace, workspace_bytes, top_bytes(rows, cut.pieces, k))))
            return rc;
        const Temperature t = temperature_of(temperature);
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
        with_nv<16>(cut.nv, [&](auto nv) {
            ung_top_scores_kernel<T, nv.value><<<(uint32_t)(rows * lists), TOP_NT, 0, st>>>(
                (const T *)scores, (uint32_t)len, row_stride, (uint32_t)lists, k, t, values, ids, lse,
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
            auto merge = [&](auto kernel) {
                kernel<<<(uint32_t)(rows * groups), TOP_NT, 0, st>>>(part, sums, (uint32_t)lists, (uint32_t)groups, k,
                                                                     values, ids, lse, out, out_sums, t);
            };
            const uint64_t items = (lists < MERGE_LISTS ? lists : MERGE_LISTS) * k;
            if (items <= TOP_NT * 4)
                merge(ung_top_merge_kernel<4>);
            else if (items <= TOP_NT * 12)
                merge(ung_top_merge_kernel<12>);
            else
                merge(ung_top_merge_kernel<MERGE_LISTS * MAX_K / TOP_NT>);
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
        (rc = check_grad(what, scores, row_stride, grad, type, rows, len, grad_stride)))
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
        if ((rc = check_grid(what, rows * cut.pieces, PIECE_NT)))
            return rc;
        with_nv<8>(cut.nv, [&](auto nv) {
            ung_distill_grad_kernel<T, PIECE_NT, nv.value><<<(uint32_t)(rows * cut.pieces), PIECE_NT, 0,
                                                             (hipStream_t)stream>>>(
                (const T *)scores, (uint32_t)len, row_stride, ids, values, k, (const Saved *)saved, weight,
                temperature_of(temperature), cut.pieces, (T *)grad, grad_stride);
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
        (rc = check_grad(what, scores, row_stride, grad, type, rows, len, grad_stride)))
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
