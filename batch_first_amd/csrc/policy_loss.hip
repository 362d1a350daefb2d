// Losses of the move-scoring head and their gradients.
//
// A board's features X [32][64] and the logit kernel W [32][73] give the logits l[f][s] = sum_c W[c][f] X[c][s] of its
// move vocabulary (73 filters x 64 from-squares = 4 672).  With target t and weight w of the board,
//
//     loss  = log sum exp l - l[t]                         d = w (softmax(l) - onehot(t))
//     dX[c][s] = sum_f W[c][f] d[f][s]                     dW[c][f] = sum over boards and s of X[c][s] d[f][s]
//
// where the softmax runs over the whole vocabulary (k_policy_loss) or over the board's own list of moves
// (k_policy_move_loss).  A board without a target has loss 0 and no part in the gradients.
#include <hip/hip_runtime.h>

#include "../../include/batchfirst.h"
#include "bf_train.h"

namespace bf {
namespace {

constexpr int kC = 32, kS = 64, kF = 73, kVocab = kF * kS, kXW = kC * kF;
constexpr int kThreads = 256;
constexpr unsigned kMaxGrid = 1024;   // workgroups of a gradient call: as many partial kernel gradients

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// Over the workgroup's four waves, in fixed order; `red` holds four floats.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* red) {
    v = MAX ? wave_max(v) : wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return MAX ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T, bool GRAD>
__global__ __launch_bounds__(kThreads) void k_policy_loss(const T* __restrict__ x, const T* __restrict__ w, size_t n,
                                                          const int64_t* __restrict__ targets, const float* __restrict__ weights,
                                                          unsigned weight_step, float* __restrict__ loss, T* __restrict__ dx,
                                                          float* __restrict__ dw_part, int* __restrict__ err) {
    __shared__ float sx[kC * kS], sw[kXW], sp[kVocab], red[4];
    const int tid = threadIdx.x;
    for (int i = tid; i < kXW; i += kThreads) sw[i] = (float)w[i];
    float acc[(kXW + kThreads - 1) / kThreads] = {};
    for (size_t b = blockIdx.x; b < n; b += gridDim.x) {
        __syncthreads();
        for (int i = tid; i < kC * kS; i += kThreads) sx[i] = (float)x[b * (kC * kS) + i];
        __syncthreads();
        float top = -INFINITY;
        for (int i = tid; i < kVocab; i += kThreads) {
            float l = 0.0f;
            for (int c = 0; c < kC; ++c) l = fmaf(sw[c * kF + (i >> 6)], sx[c * kS + (i & 63)], l);
            sp[i] = l;
            top = fmaxf(top, l);
        }
        top = block_reduce<true>(top, red);
        float z = 0.0f;
        for (int i = tid; i < kVocab; i += kThreads) z += expf(sp[i] - top);
        z = block_reduce<false>(z, red);
        const int64_t t = targets[b];
        const bool has = t >= 0 && t < kVocab;
        if (tid == 0) {
            if (t < -1 || t >= kVocab) atomicOr(err, 8);
            if (loss) loss[b] = has ? logf(z) + top - sp[t] : 0.0f;
        }
        if (!GRAD) continue;
        __syncthreads();
        const float wb = has ? weights[b * weight_step] : 0.0f;
        for (int i = tid; i < kVocab; i += kThreads) sp[i] = has ? (expf(sp[i] - top) / z - (i == t ? 1.0f : 0.0f)) * wb : 0.0f;
        __syncthreads();
        if (dx)
            for (int i = tid; i < kC * kS; i += kThreads) {
                float a = 0.0f;
                for (int f = 0; f < kF; ++f) a = fmaf(sw[(i >> 6) * kF + f], sp[f * kS + (i & 63)], a);
                dx[b * (kC * kS) + i] = (T)a;
            }
        if (dw_part && has)
            for (int k = 0, i = tid; i < kXW; i += kThreads, ++k)
                for (int s = 0; s < kS; ++s) acc[k] = fmaf(sx[(i / kF) * kS + s], sp[(i % kF) * kS + s], acc[k]);
    }
    if (GRAD && dw_part)
        for (int k = 0, i = tid; i < kXW; i += kThreads, ++k) dw_part[(size_t)blockIdx.x * kXW + i] = acc[k];
}

// start[b] = moves of the boards before b, start[n] = all moves; one workgroup.
__global__ __launch_bounds__(1024) void k_move_starts(const uint8_t* __restrict__ per, size_t n, size_t n_moves,
                                                      uint64_t* __restrict__ start, int* __restrict__ err) {
    __shared__ unsigned s[1024];
    uint64_t base = 0;
    for (size_t lo = 0; lo < n; lo += 1024) {
        const unsigned mine = lo + threadIdx.x < n ? per[lo + threadIdx.x] : 0u;
        s[threadIdx.x] = mine;
        __syncthreads();
        for (int o = 1; o < 1024; o <<= 1) {
            const unsigned v = (int)threadIdx.x >= o ? s[threadIdx.x - o] : 0u;
            __syncthreads();
            s[threadIdx.x] += v;
            __syncthreads();
        }
        if (lo + threadIdx.x < n) start[lo + threadIdx.x] = base + s[threadIdx.x] - mine;
        base += s[1023];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        start[n] = base;
        if (base != n_moves) atomicOr(err, 8);
    }
}

template <typename T, bool GRAD>
__global__ __launch_bounds__(kThreads) void k_policy_move_loss(const T* __restrict__ x, const T* __restrict__ w, size_t n,
                                                               const uint8_t* __restrict__ from, const uint8_t* __restrict__ filter,
                                                               size_t n_moves, const uint64_t* __restrict__ start,
                                                               const int64_t* __restrict__ targets, const float* __restrict__ weights,
                                                               unsigned weight_step, float* __restrict__ loss, T* __restrict__ dx,
                                                               float* __restrict__ dw_part, int* __restrict__ err) {
    __shared__ float sx[kC * kS], sw[kXW], sd[kThreads], red[4];
    __shared__ int ss[kThreads], sf[kThreads];
    const int tid = threadIdx.x;
    for (int i = tid; i < kXW; i += kThreads) sw[i] = (float)w[i];
    float acc[(kXW + kThreads - 1) / kThreads] = {};
    for (size_t b = blockIdx.x; b < n; b += gridDim.x) {
        __syncthreads();
        for (int i = tid; i < kC * kS; i += kThreads) sx[i] = (float)x[b * (kC * kS) + i];
        __syncthreads();
        const uint64_t lo = min(start[b], (uint64_t)n_moves), hi = min(start[b + 1], (uint64_t)n_moves);
        const int cnt = (int)(hi - lo);   // at most 255
        float l = -INFINITY;
        if (tid < cnt) {
            int s = from[lo + tid], f = filter[lo + tid];
            if (s >= kS || f >= kF) atomicOr(err, 8);
            s = min(s, kS - 1);
            f = min(f, kF - 1);
            l = 0.0f;
            for (int c = 0; c < kC; ++c) l = fmaf(sw[c * kF + f], sx[c * kS + s], l);
            ss[tid] = s;
            sf[tid] = f;
        }
        const float top = block_reduce<true>(l, red);
        const float e = tid < cnt ? expf(l - top) : 0.0f;
        const float z = block_reduce<false>(e, red);
        const int64_t t = targets[b];
        const bool has = t >= 0 && t < cnt;
        if (tid == 0) {
            if (t < -1 || t >= cnt) atomicOr(err, 8);
            if (loss && !has) loss[b] = 0.0f;
        }
        if (loss && has && tid == t) loss[b] = logf(z) + top - l;
        if (!GRAD) continue;
        sd[tid] = has ? (e / z - (tid == t ? 1.0f : 0.0f)) * weights[b * weight_step] : 0.0f;
        __syncthreads();
        if (dx)
            for (int i = tid; i < kC * kS; i += kThreads) {
                float a = 0.0f;
                for (int m = 0; m < cnt; ++m)
                    if (ss[m] == (i & 63)) a = fmaf(sw[(i >> 6) * kF + sf[m]], sd[m], a);
                dx[b * (kC * kS) + i] = (T)a;
            }
        if (dw_part && has)
            for (int k = 0, i = tid; i < kXW; i += kThreads, ++k)
                for (int m = 0; m < cnt; ++m)
                    if (sf[m] == i % kF) acc[k] = fmaf(sx[(i / kF) * kS + ss[m]], sd[m], acc[k]);
    }
    if (GRAD && dw_part)
        for (int k = 0, i = tid; i < kXW; i += kThreads, ++k) dw_part[(size_t)blockIdx.x * kXW + i] = acc[k];
}

// The partial kernel gradients of the workgroups, added up in fixed order.
template <typename T>
__global__ __launch_bounds__(64) void k_sum_parts(const float* __restrict__ part, unsigned parts, T* __restrict__ dw) {
    const int i = blockIdx.x * 64 + threadIdx.x;
    if (i >= kXW) return;
    double a = 0.0;
    for (unsigned p = 0; p < parts; ++p) a += part[(size_t)p * kXW + i];
    dw[i] = (T)(float)a;
}

unsigned grid_for(size_t n) { return (unsigned)(n < kMaxGrid ? n : kMaxGrid); }

template <typename T>
hipError_t launch(const PolicyLossArgs& a, hipStream_t s) {
    const T *x = static_cast<const T*>(a.features), *w = static_cast<const T*>(a.kernel);
    T* dx = static_cast<T*>(a.d_features);
    const bool grad = a.d_features || a.d_kernel;
    const unsigned grid = grid_for(a.n);
    const unsigned step = a.n_weights > 1 ? 1u : 0u;
    uint64_t* start = static_cast<uint64_t*>(a.workspace);
    float* part = a.d_kernel ? reinterpret_cast<float*>(a.per_board ? start + (a.n + 2) / 2 * 2 : start) : nullptr;
    if (grid && a.per_board) {
        hipLaunchKernelGGL(k_move_starts, dim3(1), dim3(1024), 0, s, a.per_board, a.n, a.n_moves, start, a.err);
        if (grad)
            hipLaunchKernelGGL((k_policy_move_loss<T, true>), dim3(grid), dim3(kThreads), 0, s, x, w, a.n, a.from, a.filter, a.n_moves,
                               start, a.targets, a.weights, step, a.loss, dx, part, a.err);
        else
            hipLaunchKernelGGL((k_policy_move_loss<T, false>), dim3(grid), dim3(kThreads), 0, s, x, w, a.n, a.from, a.filter, a.n_moves,
                               start, a.targets, nullptr, 0u, a.loss, nullptr, nullptr, a.err);
    } else if (grid) {
        if (grad)
            hipLaunchKernelGGL((k_policy_loss<T, true>), dim3(grid), dim3(kThreads), 0, s, x, w, a.n, a.targets, a.weights, step, a.loss,
                               dx, part, a.err);
        else
            hipLaunchKernelGGL((k_policy_loss<T, false>), dim3(grid), dim3(kThreads), 0, s, x, w, a.n, a.targets, nullptr, 0u, a.loss,
                               nullptr, nullptr, a.err);
    }
    if (a.d_kernel)
        hipLaunchKernelGGL(k_sum_parts<T>, dim3((kXW + 63) / 64), dim3(64), 0, s, part, grid, static_cast<T*>(a.d_kernel));
    return hipGetLastError();
}

}  // namespace

size_t policy_loss_workspace(size_t n, bool moves, bool kernel_grad) {
    return (moves ? (n + 2) / 2 * 2 * sizeof(uint64_t) : 0) + (kernel_grad ? (size_t)grid_for(n) * kXW * sizeof(float) : 0);
}

hipError_t launch_policy_loss(const PolicyLossArgs& a, hipStream_t stream) {
    if (a.type == BF_TYPE_F32) return launch<float>(a, stream);
    if (a.type == BF_TYPE_BF16) return launch<__bf16>(a, stream);
    return launch<_Float16>(a, stream);
}

}  // namespace bf
