// ung_gradients.hip -- the norm of many gradients together, and the gradients scaled to a largest
// norm, on gfx950: the kernels and the entry points ung_hip_gradient_* and ung_hip_clip_gradients
// of include/ung_hip.h.
//
//   norm = sqrt(sum of all squares),  out = g * min(1, largest / norm)
//
// Squares and sums are made in 64 bits: the square of every 32-bit number is one there without
// overflow or underflow, and neither the order nor the number of elements shows in 32 bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <vector>

#include "ung_elements.h"
#include "ung_hip.h"
#include "ung_internal.h"

using namespace ung;

namespace {

// A launch takes up to 64 tensors by its arguments, cut into chunks; a block takes every
// gridDim.x-th chunk, so the elements that a partial sum holds, and its order, are fixed.
constexpr uint32_t LIST = 64, CHUNK = 8192, NT = 256, MOST_BLOCKS = 1024;

struct List {
    const void *from[LIST];
    void *to[LIST];
    uint64_t size[LIST];
    uint32_t first[LIST + 1]; // chunk that a tensor begins with
    uint8_t type[LIST];
    uint32_t count;
};

__device__ inline uint32_t tensor_of(const List &list, uint32_t chunk)
{
    uint32_t lo = 0, hi = list.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (list.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// f(vector, first element) over a chunk's whole vectors, g(element) over what is left of its end.
template <class T, uint32_t THREADS, class F, class G>
__device__ inline void over(uint64_t size, uint64_t at, F f, G g)
{
    constexpr uint64_t N = Vec<T>::N;
    const uint64_t end = min(at + CHUNK, size), whole = at + (end - at) / N * N;
#pragma unroll 4
    for (uint64_t i = at + threadIdx.x * N; i < whole; i += THREADS * N)
        f(i);
    if (whole + threadIdx.x < end)
        g(whole + threadIdx.x);
}

template <class F>
__device__ inline void by_type(int type, F f)
{
    if (type == UNG_HIP_F32)
        f(float{});
    else if (type == UNG_HIP_F16)
        f(fp16_t{});
    else
        f(bf16_t{});
}

template <uint32_t THREADS>
__device__ inline double block_sum(double v, double *red)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (uint32_t w = 1; w < THREADS / 64; ++w)
        v += red[w];
    return v;
}

// A thread's squares of the chunks from `first` on, every `by`-th one.
template <uint32_t THREADS>
__device__ inline double squares(const List &list, uint32_t first, uint32_t by)
{
    double sum = 0.0;
    const uint32_t chunks = list.first[list.count];
    for (uint32_t chunk = first; chunk < chunks; chunk += by) {
        const uint32_t t = tensor_of(list, chunk);
        const uint64_t at = (uint64_t)(chunk - list.first[t]) * CHUNK, size = list.size[t];
        by_type(list.type[t], [&](auto zero) {
            using T = decltype(zero);
            const T *from = (const T *)list.from[t];
            auto add = [&](float x) { sum = __builtin_fma((double)x, (double)x, sum); };
            over<T, THREADS>(
                size, at,
                [&](uint64_t i) {
                    const Vec<T> v = load_loose(from + i);
#pragma unroll
                    for (int e = 0; e < Vec<T>::N; ++e)
                        add(v.get(e));
                },
                [&](uint64_t i) { add(to_float(from[i])); });
        });
    }
    return sum;
}

// What a norm and the largest one make of the gradients.  A norm past 32 bits, in which the caller gets it, is
// an infinite one.
struct Factor {
    bool less;
    float by;
    __device__ Factor(double norm, double most)
        : less(norm > most && (float)norm < __builtin_huge_valf()), by(less ? (float)(most / norm) : 1.0f)
    {
    }
};

template <uint32_t THREADS>
__device__ inline void scale(const List &list, uint32_t first, uint32_t step, Factor f)
{
    const uint32_t chunks = list.first[list.count];
    for (uint32_t chunk = first; chunk < chunks; chunk += step) {
        const uint32_t t = tensor_of(list, chunk);
        const uint64_t at = (uint64_t)(chunk - list.first[t]) * CHUNK, size = list.size[t];
        if (!f.less && list.to[t] == list.from[t])
            continue;
        by_type(list.type[t], [&](auto zero) {
            using T = decltype(zero);
            const T *from = (const T *)list.from[t];
            T *to = (T *)list.to[t];
            over<T, THREADS>(
                size, at,
                [&](uint64_t i) {
                    const Vec<T> v = load_loose(from + i);
                    Vec<T> o;
#pragma unroll
                    for (int e = 0; e < Vec<T>::N; e += 2)
                        o.put2(e, v.get(e) * f.by, v.get(e + 1) * f.by);
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        o.w[w] = f.less ? o.w[w] : v.w[w];
                    store_loose(to + i, o);
                },
                [&](uint64_t i) { to[i] = f.less ? from_float<T>(to_float(from[i]) * f.by) : from[i]; });
        });
    }
}

// Every block's chunks to one partial sum.  Memory bounds it: 60 tensors, 54 million elements of
// 4 and 2 bytes, 23 us (6.1 TB/s).
__global__ __launch_bounds__(NT) void ung_gradient_squares_kernel(List list, double *part)
{
    __shared__ double red[NT / 64];
    const double sum = block_sum<NT>(squares<NT>(list, blockIdx.x, gridDim.x), red);
    if (threadIdx.x == 0)
        part[blockIdx.x] = sum;
}

// The sum of all partial sums, in an order that their number decides.
__device__ inline double sum_of(const double *part, uint32_t count, double *red)
{
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < count; i += NT)
        sum += part[i];
    return block_sum<NT>(sum, red);
}

// For the norm alone, and where there are more partial sums than every block can add up for itself.
__global__ __launch_bounds__(NT) void ung_gradient_join_kernel(const double *part, uint32_t count, double *whole,
                                                               float *norm)
{
    __shared__ double red[NT / 64];
    const double sum = sum_of(part, count, red);
    if (threadIdx.x == 0) {
        whole[0] = sum;
        if (norm)
            norm[0] = (float)sqrt(sum);
    }
}

// Every block adds up the partial sums for itself: up to SUMS of them cost it less than a launch
// between the two passes would.  Memory bounds it, where part of what the first pass read still lies
// in the last-level cache: the same 60 tensors 45 us, 6.2 TB/s of reads and writes.
constexpr uint32_t SUMS = 2048;
__global__ __launch_bounds__(NT) void ung_gradient_scale_kernel(List list, const double *part, uint32_t count, double most,
                                                                float *to_norm)
{
    __shared__ double red[NT / 64];
    const double norm = sqrt(sum_of(part, count, red));
    if (to_norm && blockIdx.x == 0 && threadIdx.x == 0)
        to_norm[0] = (float)norm;
    scale<NT>(list, blockIdx.x, gridDim.x, Factor(norm, most));
}

// All of a few small tensors by one block, without a launch between the two passes: two of 8192 elements
// 12.8 us a call, in two launches 15.1.
constexpr uint32_t FEW_CHUNKS = 4, FEW_NT = 1024;
__global__ __launch_bounds__(FEW_NT) void ung_gradient_few_kernel(List list, int scaled, double most, float *norm)
{
    __shared__ double red[FEW_NT / 64];
    const double all = sqrt(block_sum<FEW_NT>(squares<FEW_NT>(list, 0, 1), red));
    if (norm && threadIdx.x == 0)
        norm[0] = (float)all;
    if (scaled)
        scale<FEW_NT>(list, 0, 1, Factor(all, most));
}

uint64_t chunks_of(uint64_t size) { return ceil_div(size, CHUNK); }
uint32_t blocks_of(uint64_t chunks) { return (uint32_t)(chunks < MOST_BLOCKS ? chunks : MOST_BLOCKS); }

// Partial sums of all launches of a call.
uint64_t parts_of(const uint64_t *sizes, uint32_t count)
{
    uint64_t parts = 0, chunks = 0;
    for (uint32_t i = 0, in = 0; i < count; ++i) {
        if (sizes[i]) {
            chunks += chunks_of(sizes[i]);
            ++in;
        }
        if (in == LIST || i + 1 == count) {
            parts += blocks_of(chunks);
            chunks = in = 0;
        }
    }
    return parts;
}

uint64_t bytes_of(const uint64_t *sizes, uint32_t count) { return (2 + parts_of(sizes, count)) * 8; }

int check_list(const char *what, const void *const *grads, void *const *out, const int *types, const uint64_t *sizes,
               uint32_t count)
{
    if (count && (!grads || !types || !sizes)) {
        set_error("%s: null argument", what);
        return UNG_HIP_EINVAL;
    }
    for (uint32_t i = 0; i < count; ++i) {
        if (!known_type(types[i])) {
            set_error("%s: unknown element type %d of tensor %u", what, types[i], i);
            return UNG_HIP_EINVAL;
        }
        if (sizes[i] > 1ull << 40) {
            set_error("%s: %llu elements of tensor %u are too many", what, (unsigned long long)sizes[i], i);
            return UNG_HIP_EINVAL;
        }
        const uintptr_t from = (uintptr_t)grads[i], to = out ? (uintptr_t)out[i] : from;
        if (sizes[i] && (!from || !to || from % type_size(types[i]) || to % type_size(types[i]))) {
            set_error("%s: tensor %u is null or not aligned to its elements", what, i);
            return UNG_HIP_EINVAL;
        }
    }
    return UNG_HIP_OK;
}

// Whether what a call writes overlaps anything else of it (an element scaled twice, or read after
// it is written).
bool overlaps(const void *const *grads, void *const *out, const int *types, const uint64_t *sizes, uint32_t count)
{
    struct Range {
        uintptr_t begin, end;
        bool written;
    };
    std::vector<Range> all;
    all.reserve(2 * (size_t)count);
    for (uint32_t i = 0; i < count; ++i) {
        if (!sizes[i])
            continue;
        const uintptr_t from = (uintptr_t)grads[i], to = out ? (uintptr_t)out[i] : from;
        const uint64_t bytes = sizes[i] * type_size(types[i]);
        all.push_back({to, to + bytes, true});
        if (to != from)
            all.push_back({from, from + bytes, false});
    }
    std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    uintptr_t written = 0, read = 0; // ends of what came before
    for (const Range &r : all) {
        if (r.begin < written || (r.written && r.begin < read))
            return true;
        uintptr_t &end = r.written ? written : read;
        end = std::max(end, r.end);
    }
    return false;
}

// f(list, its chunks) for every launch's worth of tensors.
template <class F>
int lists(const void *const *grads, void *const *out, const int *types, const uint64_t *sizes, uint32_t count, F f)
{
    List list;
    list.count = 0;
    uint64_t chunks = 0;
    for (uint32_t i = 0; i < count; ++i) {
        if (sizes[i]) {
            const uint32_t at = list.count++;
            list.from[at] = grads[i];
            list.to[at] = out ? out[i] : const_cast<void *>(grads[i]);
            list.size[at] = sizes[i];
            list.type[at] = (uint8_t)types[i];
            list.first[at] = (uint32_t)chunks;
            chunks += chunks_of(sizes[i]);
            list.first[at + 1] = (uint32_t)chunks;
        }
        if (list.count && (list.count == LIST || i + 1 == count)) {
            if (chunks > UINT32_MAX)
                return UNG_HIP_EINVAL;
            f(list, blocks_of(chunks));
            list.count = 0;
            chunks = 0;
        }
    }
    return UNG_HIP_OK;
}

int run(const char *what, const void *const *grads, void *const *out, const int *types, const uint64_t *sizes,
        uint32_t count, bool scaled, float most, float *norm, void *workspace, uint64_t workspace_bytes, void *stream)
{
    clear_error();
    if (const int rc = check_list(what, grads, out, types, sizes, count))
        return rc;
    if (scaled && !(most >= 0.0f)) {
        set_error("%s: largest norm %g is negative or NaN", what, (double)most);
        return UNG_HIP_EINVAL;
    }
    if ((!scaled && !norm) || (uintptr_t)norm % 4) {
        set_error("%s: null or unaligned norm", what);
        return UNG_HIP_EINVAL;
    }
    const uint64_t needed = bytes_of(sizes, count);
    if (!workspace || workspace_bytes < needed || (uintptr_t)workspace % 16) {
        set_error("%s: needs %llu bytes of workspace at a 16-byte boundary (got %llu)", what, (unsigned long long)needed,
                  (unsigned long long)(workspace ? workspace_bytes : 0));
        return UNG_HIP_EINVAL;
    }
    try {
        if (scaled && overlaps(grads, out, types, sizes, count)) {
            set_error("%s: gradients or outputs overlap", what);
            return UNG_HIP_EINVAL;
        }
    } catch (const std::exception &e) {
        set_error("%s: %s", what, e.what());
        return UNG_HIP_EDEVICE;
    }
    const hipStream_t st = (hipStream_t)stream;
    double *whole = (double *)workspace, *part = whole + 2;
    uint32_t parts = 0, launches = 0;
    uint64_t chunks = 0;
    int rc = lists(grads, out, types, sizes, count, [&](const List &list, uint32_t) {
        ++launches;
        chunks += list.first[list.count];
    });
    if (rc) {
        set_error("%s: too many elements", what);
        return rc;
    }
    if (launches == 1 && chunks <= FEW_CHUNKS) {
        (void)lists(grads, out, types, sizes, count, [&](const List &list, uint32_t) {
            ung_gradient_few_kernel<<<1, FEW_NT, 0, st>>>(list, scaled, (double)most, norm);
        });
        return launched(what);
    }
    rc = lists(grads, out, types, sizes, count, [&](const List &list, uint32_t blocks) {
        ung_gradient_squares_kernel<<<blocks, NT, 0, st>>>(list, part + parts);
        parts += blocks;
    });
    const bool joined = !scaled || parts > SUMS || parts == 0;
    if (joined)
        ung_gradient_join_kernel<<<1, NT, 0, st>>>(part, parts, whole, norm);
    if (scaled) {
        float *to_norm = joined ? nullptr : norm;
        rc = lists(grads, out, types, sizes, count, [&](const List &list, uint32_t blocks) {
            ung_gradient_scale_kernel<<<blocks, NT, 0, st>>>(list, joined ? whole : part, joined ? 1 : parts, (double)most,
                                                             to_norm);
            to_norm = nullptr;
        });
    }
    return launched(what);
}

} // namespace

extern "C" {

int ung_hip_gradient_workspace(const uint64_t *sizes, uint32_t count, uint64_t *bytes)
{
    clear_error();
    if (!bytes || (count && !sizes)) {
        set_error("ung_hip_gradient_workspace: null argument");
        return UNG_HIP_EINVAL;
    }
    *bytes = bytes_of(sizes, count);
    return UNG_HIP_OK;
}

int ung_hip_gradient_norm(const void *const *grads, const int *types, const uint64_t *sizes, uint32_t count,
                          float *norm, void *workspace, uint64_t workspace_bytes, void *stream)
{
    return run("ung_hip_gradient_norm", grads, nullptr, types, sizes, count, false, 0.0f, norm, workspace,
               workspace_bytes, stream);
}

int ung_hip_clip_gradients(const void *const *grads, void *const *out, const int *types, const uint64_t *sizes,
                           uint32_t count, float max_norm, float *norm, void *workspace, uint64_t workspace_bytes,
                           void *stream)
{
    return run("ung_hip_clip_gradients", grads, out, types, sizes, count, true, max_norm, norm, workspace,
               workspace_bytes, stream);
}

} // extern "C"
