// The norm over many tensors, and scaling them to a limit:
//
//     norm = sqrt(sum over tensors and elements of g^2)        g <- g * min(1, limit / (norm + 1e-6))
//
// Squares and sums are float64: float32 would overflow from 1.8e19 on and lose the small tensors beside the large.
#include <hip/hip_runtime.h>

#include "../../include/batchfirst.h"
#include "bf_train.h"

namespace bf {
namespace {

constexpr int kThreads = 256;
constexpr size_t kChunk = 65536;   // elements a workgroup
constexpr int kTable = 96;         // tensors a launch: the table travels in the kernel's arguments

struct Table {
    void* ptr[kTable];
    unsigned long long count[kTable];
    unsigned first[kTable];        // first workgroup of the tensor, within the launch
    unsigned char type[kTable];
    int n;
};

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double red[kThreads / 64];
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ int find(const Table& t, unsigned block) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ double squares(const T* g, size_t n) {
    double a = 0.0;
    for (size_t i = threadIdx.x; i < n; i += kThreads) {
        const double v = (double)(float)g[i];
        a = fma(v, v, a);
    }
    return a;
}

__global__ __launch_bounds__(kThreads) void k_squares(Table t, double* __restrict__ part) {
    const int k = find(t, blockIdx.x);
    const size_t at = (size_t)(blockIdx.x - t.first[k]) * kChunk;
    const size_t n = min((size_t)t.count[k] - at, kChunk);
    double a;
    if (t.type[k] == BF_TYPE_F32) a = squares(static_cast<const float*>(t.ptr[k]) + at, n);
    else if (t.type[k] == BF_TYPE_BF16) a = squares(static_cast<const __bf16*>(t.ptr[k]) + at, n);
    else a = squares(static_cast<const _Float16*>(t.ptr[k]) + at, n);
    a = block_sum(a);
    if (threadIdx.x == 0) part[blockIdx.x] = a;
}

__global__ __launch_bounds__(kThreads) void k_norm(const double* __restrict__ part, size_t parts, float limit,
                                                   float* __restrict__ norm, float* __restrict__ scale) {
    double a = 0.0;
    for (size_t i = threadIdx.x; i < parts; i += kThreads) a += part[i];
    a = block_sum(a);
    if (threadIdx.x == 0) {
        const float v = (float)sqrt(a);
        *norm = v;
        // a norm of NaN gives a scale of NaN, one of infinity a scale of 0, as the formula has it
        const float f = limit / (v + 1e-6f);
        *scale = f > 1.0f ? 1.0f : f;
    }
}

template <typename T>
__device__ __forceinline__ void scale_all(T* g, size_t n, float f) {
    for (size_t i = threadIdx.x; i < n; i += kThreads) g[i] = (T)((float)g[i] * f);
}

__global__ __launch_bounds__(kThreads) void k_scale(Table t, const float* __restrict__ scale) {
    const float f = *scale;
    if (f == 1.0f) return;   // within the limit: every product would be the value itself
    const int k = find(t, blockIdx.x);
    const size_t at = (size_t)(blockIdx.x - t.first[k]) * kChunk;
    const size_t n = min((size_t)t.count[k] - at, kChunk);
    if (t.type[k] == BF_TYPE_F32) scale_all(static_cast<float*>(t.ptr[k]) + at, n, f);
    else if (t.type[k] == BF_TYPE_BF16) scale_all(static_cast<__bf16*>(t.ptr[k]) + at, n, f);
    else scale_all(static_cast<_Float16*>(t.ptr[k]) + at, n, f);
}

// Calls launch(table, workgroups) for the non-empty tensors, kTable at a time.
template <typename F>
hipError_t tables(void* const* ptrs, const size_t* counts, const int* types, size_t n_tensors, F launch) {
    Table t;
    t.n = 0;
    unsigned blocks = 0;
    for (size_t i = 0; i < n_tensors; ++i) {
        if (counts[i]) {
            t.ptr[t.n] = ptrs[i];
            t.count[t.n] = counts[i];
            t.type[t.n] = (unsigned char)types[i];
            t.first[t.n++] = blocks;
            blocks += (unsigned)((counts[i] + kChunk - 1) / kChunk);
        }
        if (t.n && (t.n == kTable || i + 1 == n_tensors)) {
            launch(t, blocks);
            if (hipError_t e = hipGetLastError()) return e;
            t.n = 0;
            blocks = 0;
        }
    }
    return hipSuccess;
}

}  // namespace

size_t grad_norm_workspace(const size_t* counts, size_t n_tensors) {
    size_t parts = 0;
    for (size_t i = 0; i < n_tensors; ++i) parts += (counts[i] + kChunk - 1) / kChunk;
    return 16 + parts * sizeof(double);
}

hipError_t launch_grad_norm(void* const* ptrs, const size_t* counts, const int* types, size_t n_tensors, bool clip, float limit,
                            float* d_norm, void* workspace, hipStream_t s) {
    float* scale = static_cast<float*>(workspace);
    double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
    size_t parts = 0;
    hipError_t e = tables(ptrs, counts, types, n_tensors, [&](const Table& t, unsigned blocks) {
        hipLaunchKernelGGL(k_squares, dim3(blocks), dim3(kThreads), 0, s, t, part + parts);
        parts += blocks;
    });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(kThreads), 0, s, part, parts, limit, d_norm, scale);
    if ((e = hipGetLastError()) != hipSuccess || !clip) return e;
    return tables(ptrs, counts, types, n_tensors, [&](const Table& t, unsigned blocks) {
        hipLaunchKernelGGL(k_scale, dim3(blocks), dim3(kThreads), 0, s, t, scale);
    });
}

}  // namespace bf
