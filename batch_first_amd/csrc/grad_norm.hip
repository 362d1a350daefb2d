// The norm over many tensors, and scaling them to a limit:
//
//     norm = sqrt(sum over tensors and elements of g^2)        g <- g * min(1, limit / (norm + 1e-6))
//
// Squares and sums are float64: float32 would overflow from 1.8e19 on and lose the small tensors beside the large.
// Bound by reading (and, to scale, reading again and writing): a workgroup walks a run of 16 KB chunks, through however
// many tensors it spans, with 16-byte accesses and four of them in flight a thread, and leaves one partial sum; every
// workgroup of the scaling pass adds the partial sums up by itself, in the same fixed order, which spares a launch between the two.
// The scaling pass walks its run backwards, so that it begins with what the first pass has left in the caches (100 M float32
// elements clipped in 208 us; forwards 253).  The norm of 268 M float32 elements takes 181 us, 5.9 TB/s; clipping 307
// bfloat16 tensors of 60 M elements 83 us, of which 77 on the GPU, 4.7 TB/s for reading twice and writing once.  A few
// chunks, as a head's own gradient, take one workgroup and one launch.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/batchfirst.h"
#include "bf_train.h"

namespace bf {
namespace {

constexpr int kThreads = 256;
constexpr int kInFlight = 4;                                        // 16-byte accesses a thread and chunk
constexpr size_t kChunkBytes = (size_t)kThreads * kInFlight * 16;
constexpr int kTable = 160;        // tensors a launch: their table travels in the kernel's arguments, of which there are 4 KB
// Workgroups a launch, four a compute unit: eight leave every workgroup of the scaling pass more partial sums to add up
// (150 M float32 elements clipped in 348 in place of 334 us), two keep fewer loads in flight.
constexpr unsigned kGroups = 1024;
constexpr int kTypeShift = 56;

struct Table {
    char* ptr[kTable];
    unsigned long long count[kTable];      // elements; the type in the top byte
    unsigned first[kTable + 1];            // first chunk of each tensor, and the end
    int n;
};
static_assert(sizeof(Table) <= 3600, "kernel arguments");

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// A tensor of elements T as 16-byte pieces of memory; the pieces at its ends may lie partly outside.
template <typename T>
struct Pieces {
    static constexpr int kPer = 16 / sizeof(T);
    T* base;                 // 16-byte aligned, at or before the tensor
    long long lo, hi;        // the tensor's elements are base[lo ... hi)
    __device__ __forceinline__ Pieces(char* p, unsigned long long count) {
        const unsigned skip = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u);
        base = reinterpret_cast<T*>(p - skip);
        lo = skip / sizeof(T);
        hi = lo + (long long)count;
    }
};

template <typename T>
__device__ __forceinline__ double square(T v) {
    const double d = (double)(float)v;
    return d * d;
}

// One chunk of a tensor by kThreads threads: whole(where, piece) for the pieces inside it, part(element) for the elements
// of those that its ends cut.
template <typename T, typename Whole, typename Part>
__device__ __forceinline__ void chunk_of(char* p, unsigned long long count, unsigned chunk, Whole&& whole, Part&& part) {
    typedef T piece_t __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int kPer = Pieces<T>::kPer;
    const Pieces<T> t(p, count);
    const long long at = (long long)chunk * (kThreads * kInFlight) + threadIdx.x % kThreads;
    piece_t v[kInFlight];
    bool in[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
        const long long e = (at + i * kThreads) * kPer;
        in[i] = e >= t.lo && e + kPer <= t.hi;
        if (in[i]) v[i] = *reinterpret_cast<const piece_t*>(t.base + e);
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
        const long long e = (at + i * kThreads) * kPer;
        if (in[i]) whole(reinterpret_cast<piece_t*>(t.base + e), v[i]);
        else if (e < t.hi)
            for (long long k = max(e, t.lo); k < min(e + kPer, t.hi); ++k) part(t.base + k);
    }
}

template <typename T>
__device__ __forceinline__ double squares(char* p, unsigned long long count, unsigned chunk) {
    constexpr int kPer = Pieces<T>::kPer;
    double a[2] = {0.0, 0.0};
    chunk_of<T>(p, count, chunk,
                [&](auto*, auto& v) {
#pragma unroll
                    for (int k = 0; k < kPer; ++k) a[k & 1] = fma((double)(float)v[k], (double)(float)v[k], a[k & 1]);
                },
                [&](T* e) { a[0] += square(*e); });
    return a[0] + a[1];
}

template <typename T>
__device__ __forceinline__ void scale(char* p, unsigned long long count, unsigned chunk, float f) {
    chunk_of<T>(p, count, chunk,
                [&](auto* at, auto& v) {
#pragma unroll
                    for (int k = 0; k < Pieces<T>::kPer; ++k) v[k] = (T)((float)v[k] * f);
                    *at = v;
                },
                [&](T* e) { *e = (T)((float)*e * f); });
}

// Chunk c of the table, which belongs to tensor k.
__device__ __forceinline__ double squares_of(const Table& t, int k, unsigned c) {
    const unsigned long long count = t.count[k] & ((1ull << kTypeShift) - 1);
    const int type = (int)(t.count[k] >> kTypeShift);
    if (type == BF_TYPE_F32) return squares<float>(t.ptr[k], count, c - t.first[k]);
    if (type == BF_TYPE_BF16) return squares<__bf16>(t.ptr[k], count, c - t.first[k]);
    return squares<_Float16>(t.ptr[k], count, c - t.first[k]);
}
__device__ __forceinline__ void scale_of(const Table& t, int k, unsigned c, float f) {
    const unsigned long long count = t.count[k] & ((1ull << kTypeShift) - 1);
    const int type = (int)(t.count[k] >> kTypeShift);
    if (type == BF_TYPE_F32) scale<float>(t.ptr[k], count, c - t.first[k], f);
    else if (type == BF_TYPE_BF16) scale<__bf16>(t.ptr[k], count, c - t.first[k], f);
    else scale<_Float16>(t.ptr[k], count, c - t.first[k], f);
}

// The sum over the workgroup's WAVES waves, the same in every thread.
template <int WAVES>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double red[WAVES];
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double a = red[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) a += red[i];
    return a;
}

// min(1, limit / (norm + 1e-6)): a norm of NaN gives a factor of NaN, one of infinity a factor of 0, as the formula has it
__device__ __forceinline__ float factor(float norm, float limit) {
    const float f = limit / (norm + 1e-6f);
    return f >= 1.0f ? 1.0f : f;
}

// The tensor that a chunk belongs to.
__device__ __forceinline__ int find(const Table& t, unsigned chunk) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ void run_of(const Table& t, unsigned& lo, unsigned& hi) {
    const unsigned long long chunks = t.first[t.n];
    lo = (unsigned)(chunks * blockIdx.x / gridDim.x);
    hi = (unsigned)(chunks * (blockIdx.x + 1) / gridDim.x);
}

__global__ __launch_bounds__(kThreads) void k_squares(Table t, double* __restrict__ part) {
    unsigned lo, hi;
    run_of(t, lo, hi);
    double a = 0.0;
    int k = find(t, lo);
    for (unsigned c = lo; c < hi; ++c) {
        while (c >= t.first[k + 1]) ++k;
        a += squares_of(t, k, c);
    }
    a = block_sum<kThreads / 64>(a);
    if (threadIdx.x == 0) part[blockIdx.x] = a;
}

__device__ __forceinline__ float norm_of(const double* __restrict__ part, unsigned parts) {
    double a = 0.0;
    for (unsigned i = threadIdx.x; i < parts; i += kThreads) a += part[i];
    return (float)sqrt(block_sum<kThreads / 64>(a));
}

__global__ __launch_bounds__(kThreads) void k_norm(const double* __restrict__ part, unsigned parts, float* __restrict__ norm) {
    const float v = norm_of(part, parts);
    if (threadIdx.x == 0) *norm = v;
}

__global__ __launch_bounds__(kThreads) void k_scale(Table t, const double* __restrict__ part, unsigned parts, float limit,
                                                    float* __restrict__ norm) {
    const float v = norm_of(part, parts);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
    const float f = factor(v, limit);
    if (f == 1.0f) return;   // within the limit: every product would be the value itself
    unsigned lo, hi;
    run_of(t, lo, hi);
    if (lo == hi) return;
    int k = find(t, hi - 1);
    for (unsigned c = hi; c-- > lo;) {
        while (c < t.first[k]) --k;
        scale_of(t, k, c, f);
    }
}

// Both passes over a few chunks by one workgroup, four chunks at a time: 2.9 us on the GPU and 6.7 a call where the two
// launches take 4.1 and 10.8, as long on the GPU (4.9 us) at twelve chunks, longer from there on.
constexpr int kSmallThreads = 1024;
constexpr unsigned kSmallChunks = 12;
__global__ __launch_bounds__(kSmallThreads) void k_small(Table t, bool clip, float limit, float* __restrict__ norm) {
    constexpr unsigned kAtOnce = kSmallThreads / kThreads;
    const unsigned chunks = t.first[t.n], mine = threadIdx.x / kThreads;
    double a = 0.0;
    for (unsigned c = mine; c < chunks; c += kAtOnce) a += squares_of(t, find(t, c), c);
    const float v = (float)sqrt(block_sum<kSmallThreads / 64>(a));
    if (threadIdx.x == 0) *norm = v;
    const float f = clip ? factor(v, limit) : 1.0f;
    if (f == 1.0f) return;
    for (unsigned c = mine; c < chunks; c += kAtOnce) scale_of(t, find(t, c), c, f);
}

size_t chunks_of(const void* ptr, size_t count, int type) {
    const size_t bytes = (reinterpret_cast<uintptr_t>(ptr) & 15u) + count * (type == BF_TYPE_F32 ? 4 : 2);
    return (bytes + kChunkBytes - 1) / kChunkBytes;
}

// Calls launch(table, workgroups) for the non-empty tensors, kTable at a time; returns the first error.
template <typename F>
hipError_t tables(void* const* ptrs, const size_t* counts, const int* types, size_t n_tensors, F launch) {
    Table t;
    t.n = 0;
    t.first[0] = 0;
    for (size_t i = 0; i < n_tensors; ++i) {
        if (counts[i]) {
            t.ptr[t.n] = static_cast<char*>(ptrs[i]);
            t.count[t.n] = (unsigned long long)counts[i] | (unsigned long long)types[i] << kTypeShift;
            t.first[t.n + 1] = t.first[t.n] + (unsigned)chunks_of(ptrs[i], counts[i], types[i]);
            ++t.n;
        }
        if (t.n && (t.n == kTable || i + 1 == n_tensors)) {
            launch(t, std::min(t.first[t.n], kGroups));
            if (hipError_t e = hipGetLastError()) return e;
            t.n = 0;
        }
    }
    return hipSuccess;
}

}  // namespace

size_t grad_norm_workspace(size_t n_tensors) { return std::max<size_t>((n_tensors + kTable - 1) / kTable, 1) * kGroups * sizeof(double); }

hipError_t launch_grad_norm(void* const* ptrs, const size_t* counts, const int* types, size_t n_tensors, bool clip, float limit,
                            float* d_norm, void* workspace, hipStream_t s) {
    size_t chunks = 0, filled = 0;
    for (size_t i = 0; i < n_tensors; ++i)
        if (counts[i]) chunks += chunks_of(ptrs[i], counts[i], types[i]), ++filled;
    if (chunks <= kSmallChunks && filled) {      // no more tensors than chunks
        static_assert(kSmallChunks <= kTable, "one table");
        return tables(ptrs, counts, types, n_tensors, [&](const Table& t, unsigned) {
            hipLaunchKernelGGL(k_small, dim3(1), dim3(kSmallThreads), 0, s, t, clip, limit, d_norm);
        });
    }
    double* part = static_cast<double*>(workspace);
    unsigned parts = 0;
    hipError_t e = tables(ptrs, counts, types, n_tensors, [&](const Table& t, unsigned groups) {
        hipLaunchKernelGGL(k_squares, dim3(groups), dim3(kThreads), 0, s, t, part + parts);
        parts += groups;
    });
    if (e != hipSuccess) return e;
    if (!clip || !parts) {
        hipLaunchKernelGGL(k_norm, dim3(1), dim3(kThreads), 0, s, part, parts, d_norm);
        return hipGetLastError();
    }
    return tables(ptrs, counts, types, n_tensors, [&](const Table& t, unsigned groups) {
        hipLaunchKernelGGL(k_scale, dim3(groups), dim3(kThreads), 0, s, t, part, parts, limit, d_norm);
        d_norm = nullptr;    // the first launch writes it
    });
}

}  // namespace bf
