// Launch wrappers of the training kernels (policy_loss.hip, grad_norm.hip).  All of them only enqueue.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bf {

// Losses of the move-scoring head and their gradients (policy_loss.hip).  per_board null: over the whole vocabulary;
// otherwise over the board's own moves.  d_features / d_kernel null: not wanted; with both null no weights are read.
struct PolicyLossArgs {
    const void* features;         // [n][32][64] of `type`
    const void* kernel;           // [32][73]
    int type;                     // BF_TYPE_*
    size_t n;
    const uint8_t* from;          // [n_moves]
    const uint8_t* filter;        // [n_moves]
    const uint8_t* per_board;     // [n]
    size_t n_moves;
    const int64_t* targets;       // [n]
    const float* weights;         // [n_weights], 1 or n
    size_t n_weights;
    float* loss;                  // [n], may be null beside a gradient
    void* d_features;
    void* d_kernel;
    void* workspace;              // with d_kernel: policy_loss_workspace bytes, 16-byte aligned
    int* err;                     // sticky flag: a target or a move list is out of range
};
size_t policy_loss_workspace(size_t n);
hipError_t launch_policy_loss(const PolicyLossArgs& args, hipStream_t stream);

// The norm over tensors of mixed types, and with `clip` scaling them in place to `limit` (grad_norm.hip).
size_t grad_norm_workspace(size_t n_tensors);
hipError_t launch_grad_norm(void* const* ptrs, const size_t* counts, const int* types, size_t n_tensors, bool clip, float limit,
                            float* d_norm, void* workspace, hipStream_t stream);

}  // namespace bf
