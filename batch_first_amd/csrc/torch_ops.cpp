// The training operators of torch.ops.batchfirst in C++: checks, outputs and workspace from torch's allocator on its
// current stream, and one call into the C ABI each.  Their kernels take 5 to 20 us where a batch is small, and the same
// bodies in Python take that long again (14 us for one board's loss, 170 us for clipping 307 gradients).
//
// The library is whichever one batch_first_amd/_lib.py has loaded: bf_torch_bind hands over its functions.  Contexts are
// known by their handle, as in batch_first_amd/ops.py, which announces them (bf_torch_context).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <algorithm>
#include <mutex>
#include <unordered_map>
#include <vector>

#include "../../include/batchfirst.h"

namespace {

struct Library {
    decltype(&bf_last_error) last_error;
    decltype(&bf_policy_loss) loss;
    decltype(&bf_policy_loss_grad) loss_grad;
    decltype(&bf_policy_loss_workspace) loss_workspace;
    decltype(&bf_policy_move_loss) move_loss;
    decltype(&bf_policy_move_loss_grad) move_loss_grad;
    decltype(&bf_global_norm) global_norm;
    decltype(&bf_clip_grad_norm) clip_grad_norm;
    decltype(&bf_grad_norm_workspace) norm_workspace;
};
Library lib{};

std::mutex contexts_mu;
std::unordered_map<int64_t, int> contexts;       // handle -> device

struct Context {
    bf_ctx* ctx;
    c10::Device device;
};
Context context(int64_t handle) {
    std::lock_guard<std::mutex> lock(contexts_mu);
    const auto it = contexts.find(handle);
    TORCH_CHECK_VALUE(it != contexts.end(), "unknown batchfirst context handle ", handle);
    return {reinterpret_cast<bf_ctx*>(handle), c10::Device(c10::kCUDA, (c10::DeviceIndex)it->second)};
}

void check(int rc) {
    if (rc == BF_OK) return;
    if (rc == BF_E_ARG || rc == BF_E_FORMAT) C10_THROW_ERROR(ValueError, lib.last_error());
    TORCH_CHECK(false, lib.last_error());
}

void* stream(const Context& c) { return c10::hip::getCurrentHIPStream(c.device.index()).stream(); }

at::Tensor on_device(const at::Tensor& t, at::ScalarType type, const char* name, const Context& c) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a device tensor");
    TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must have dtype ", type);
    // the kernels run on the context's GPU: a pointer and a stream from another one must not reach them
    TORCH_CHECK_VALUE(t.device() == c.device, name, " is on ", t.device(), ", but the context lives on ", c.device);
    return t.contiguous();
}
// The kernels load 16 bytes at a time; a view may start anywhere.
at::Tensor aligned(at::Tensor t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t; }

int type_of(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return BF_TYPE_F32;
        case at::kBFloat16: return BF_TYPE_BF16;
        case at::kHalf: return BF_TYPE_F16;
        default: C10_THROW_ERROR(ValueError, c10::str(name, " must be float32, bfloat16 or float16"));
    }
}

at::Tensor workspace(size_t bytes, const Context& c) {
    return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(c.device));
}

// Checked inputs of a loss; the move lists are undefined where it is over the whole vocabulary.
struct Head {
    Context c;
    at::Tensor x, w, t, from, filter, per;
    int type;
    size_t n;
    Head(int64_t handle, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& targets) : c(context(handle)) {
        type = type_of(features, "features");
        x = on_device(features, features.scalar_type(), "features", c);
        const bool planes = x.dim() == 4 && x.size(1) == 32 && x.size(2) == 8 && x.size(3) == 8;
        TORCH_CHECK_VALUE(planes || (x.dim() == 3 && x.size(1) == 32 && x.size(2) == 64), "features must have shape [N, 32, 8, 8] or [N, 32, 64]");
        w = on_device(kernel, features.scalar_type(), "logit_kernel", c);
        const bool hwio = w.dim() == 4 && w.size(0) == 1 && w.size(1) == 1 && w.size(2) == 32 && w.size(3) == 73;
        TORCH_CHECK_VALUE(hwio || (w.dim() == 2 && w.size(0) == 32 && w.size(1) == 73), "logit_kernel must have shape [32, 73] or [1, 1, 32, 73]");
        t = on_device(targets, at::kLong, "targets", c);
        TORCH_CHECK_VALUE(t.dim() == 1 && t.numel() == x.size(0), "targets needs one entry per board");
        x = aligned(x);
        w = aligned(w);
        n = (size_t)x.size(0);
    }
    void moves(const at::Tensor& from_squares, const at::Tensor& move_filters, const at::Tensor& moves_per_board) {
        from = on_device(from_squares, at::kByte, "from_squares", c);
        filter = on_device(move_filters, at::kByte, "move_filters", c);
        per = on_device(moves_per_board, at::kByte, "moves_per_board", c);
        TORCH_CHECK_VALUE(per.numel() == (int64_t)n && from.numel() == filter.numel(),
                          "moves_per_board needs one entry per board, from_squares and move_filters one per move");
    }
};

at::Tensor run_loss(const Head& h) {
    at::Tensor loss = at::empty({(int64_t)h.n}, h.x.options().dtype(at::kFloat));
    const auto* t = h.t.const_data_ptr<int64_t>();
    if (!h.per.defined())
        check(lib.loss(h.c.ctx, h.x.const_data_ptr(), h.type, h.n, h.w.const_data_ptr(), t, loss.data_ptr<float>(), stream(h.c)));
    else
        check(lib.move_loss(h.c.ctx, h.x.const_data_ptr(), h.type, h.n, h.w.const_data_ptr(), h.from.const_data_ptr<uint8_t>(),
                            h.filter.const_data_ptr<uint8_t>(), h.per.const_data_ptr<uint8_t>(), (size_t)h.from.numel(), t,
                            loss.data_ptr<float>(), stream(h.c)));
    return loss;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> run_grad(const Head& h, const at::Tensor& board_weights, bool features_grad, bool kernel_grad) {
    at::Tensor g = board_weights;
    // one weight for all boards: what a mean's or a sum's gradient is
    if (g.dim() == 1 && g.numel() > 1 && g.stride(0) == 0) g = g.narrow(0, 0, 1);
    g = on_device(g, at::kFloat, "board_weights", h.c);
    TORCH_CHECK_VALUE(g.dim() <= 1 && (g.numel() == 1 || g.numel() == (int64_t)h.n), "board_weights needs one entry, or one per board");
    at::Tensor loss = at::empty({(int64_t)h.n}, h.x.options().dtype(at::kFloat));
    at::Tensor dx = features_grad ? at::empty_like(h.x) : at::empty({0}, h.x.options());
    at::Tensor dw = kernel_grad ? at::empty_like(h.w) : at::empty({0}, h.w.options());
    const at::Tensor work = kernel_grad ? workspace(lib.loss_workspace(h.n), h.c) : at::Tensor();
    void *pdx = features_grad ? dx.data_ptr() : nullptr, *pdw = kernel_grad ? dw.data_ptr() : nullptr;
    void* pwork = kernel_grad ? work.data_ptr() : nullptr;
    const size_t bytes = kernel_grad ? (size_t)work.numel() : 0, weights = (size_t)g.numel();
    const auto* t = h.t.const_data_ptr<int64_t>();
    if (!h.per.defined())
        check(lib.loss_grad(h.c.ctx, h.x.const_data_ptr(), h.type, h.n, h.w.const_data_ptr(), t, g.const_data_ptr<float>(), weights,
                            loss.data_ptr<float>(), pdx, pdw, pwork, bytes, stream(h.c)));
    else
        check(lib.move_loss_grad(h.c.ctx, h.x.const_data_ptr(), h.type, h.n, h.w.const_data_ptr(), h.from.const_data_ptr<uint8_t>(),
                                 h.filter.const_data_ptr<uint8_t>(), h.per.const_data_ptr<uint8_t>(), (size_t)h.from.numel(), t,
                                 g.const_data_ptr<float>(), weights, loss.data_ptr<float>(), pdx, pdw, pwork, bytes, stream(h.c)));
    return {loss, dx, dw};
}

at::Tensor policy_loss(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& targets) {
    return run_loss(Head(ctx, features, kernel, targets));
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> policy_loss_grad(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel,
                                                                const at::Tensor& targets, const at::Tensor& board_weights,
                                                                bool features_grad, bool kernel_grad) {
    return run_grad(Head(ctx, features, kernel, targets), board_weights, features_grad, kernel_grad);
}
at::Tensor policy_move_loss(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& from_squares,
                            const at::Tensor& move_filters, const at::Tensor& moves_per_board, const at::Tensor& targets) {
    Head h(ctx, features, kernel, targets);
    h.moves(from_squares, move_filters, moves_per_board);
    return run_loss(h);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> policy_move_loss_grad(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel,
                                                                     const at::Tensor& from_squares, const at::Tensor& move_filters,
                                                                     const at::Tensor& moves_per_board, const at::Tensor& targets,
                                                                     const at::Tensor& board_weights, bool features_grad,
                                                                     bool kernel_grad) {
    Head h(ctx, features, kernel, targets);
    h.moves(from_squares, move_filters, moves_per_board);
    return run_grad(h, board_weights, features_grad, kernel_grad);
}

// ---- autograd ------------------------------------------------------------------------------------------------------

// A result that refuses to be differentiated.
at::Tensor refusing(at::Tensor t, const char* why) {
    if (!at::GradMode::is_enabled() || !t.defined()) return t;
    t = t.detach().set_requires_grad(true);
    auto refuse = std::make_shared<torch::autograd::DelayedError>(why, 1);
    return (*refuse)({t})[0];
}
at::Tensor once(at::Tensor g) { return refusing(g, "the gradient of a batchfirst loss cannot be differentiated"); }
bool any_requires_grad(at::ArrayRef<at::Tensor> inputs) {
    return at::GradMode::is_enabled() && std::any_of(inputs.begin(), inputs.end(), [](const at::Tensor& t) { return t.requires_grad(); });
}

// The capture a stream belongs to, 0 if none.  The default stream never belongs to one and must not be asked during one.
unsigned long long capture_of(hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (!s || hipStreamGetCaptureInfo(s, &status, &id) != hipSuccess) return 0;
    return status == hipStreamCaptureStatusActive ? id : 0;
}
// Called in a backward pass.  While it is captured, its gradients can go to nodes of the same capture only.  A leaf's
// accumulator stays on its first stream as long as any graph over the leaf lives: with an eager graph still there the
// engine would make the eager stream wait for the captured one, and the process ends in the engine's threads.
void check_receivers(torch::autograd::AutogradContext* ac, const Context& c) {
    const auto here = c10::hip::getCurrentHIPStream(c.device.index());
    const unsigned long long capture = capture_of(here.stream());
    const auto node = capture ? torch::autograd::get_current_node() : nullptr;
    if (!node) return;
    for (size_t i = 0; i < 2; ++i) {
        const auto& edge = node->next_edge(i);
        if (!ac->needs_input_grad(i) || !edge.is_valid()) continue;
        const auto there = edge.function->stream();
        if (!there) continue;
        // torch names a GPU's streams after CUDA's devices, the HIP stream class wants its own name
        const auto receiver = c10::hip::HIPStream::unpack3(there->id(), there->device_index(), c10::kHIP);
        TORCH_CHECK(receiver == here || capture_of(receiver.stream()) == capture,
                    "a captured backward pass would hand its gradient to another stream outside the capture: drop the eager graphs "
                    "of the same leaves first, or run them on the captured stream");
    }
}

// Forward-mode derivatives are not implemented: a result without a tangent would read as a derivative of zero.
void no_tangents(at::ArrayRef<at::Tensor> inputs, const char* what) {
    for (const at::Tensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "forward-mode derivatives of ", what, " are not implemented");
}

using Lists = std::optional<at::Tensor>;         // from-squares, move filters, moves per board: all three or none
struct Loss : torch::autograd::Function<Loss> {
    static at::Tensor forward(torch::autograd::AutogradContext* ac, int64_t ctx, const at::Tensor& features, const at::Tensor& kernel,
                              const at::Tensor& targets, const Lists& from, const Lists& filter, const Lists& per) {
        at::AutoDispatchBelowADInplaceOrView below;
        ac->saved_data["ctx"] = ctx;
        if (!per) {
            ac->save_for_backward({features, kernel, targets});
            return policy_loss(ctx, features, kernel, targets);
        }
        ac->save_for_backward({features, kernel, targets, *from, *filter, *per});
        return policy_move_loss(ctx, features, kernel, *from, *filter, *per, targets);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ac, torch::autograd::variable_list grads) {
        const auto saved = ac->get_saved_variables();
        const bool fg = ac->needs_input_grad(0), kg = ac->needs_input_grad(1);   // counts tensors only
        std::tuple<at::Tensor, at::Tensor, at::Tensor> out;
        if (grads[0].defined()) {
            no_tangents(grads[0], "a batchfirst loss's gradient");
            at::AutoDispatchBelowADInplaceOrView below;
            const int64_t ctx = ac->saved_data["ctx"].toInt();
            check_receivers(ac, context(ctx));
            out = saved.size() > 3 ? policy_move_loss_grad(ctx, saved[0], saved[1], saved[3], saved[4], saved[5], saved[2], grads[0], fg, kg)
                                     : policy_loss_grad(ctx, saved[0], saved[1], saved[2], grads[0], fg, kg);
        }
        return {at::Tensor(), fg ? once(std::get<1>(out)) : at::Tensor(), kg ? once(std::get<2>(out)) : at::Tensor(), at::Tensor(),
                at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

at::Tensor policy_loss_autograd(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& targets) {
    no_tangents({features, kernel}, "policy_loss");
    if (any_requires_grad({features, kernel})) return Loss::apply(ctx, features, kernel, targets, Lists(), Lists(), Lists());
    at::AutoDispatchBelowADInplaceOrView below;
    return policy_loss(ctx, features, kernel, targets);
}
at::Tensor policy_move_loss_autograd(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& from_squares,
                                     const at::Tensor& move_filters, const at::Tensor& moves_per_board, const at::Tensor& targets) {
    no_tangents({features, kernel}, "policy_move_loss");
    if (any_requires_grad({features, kernel})) return Loss::apply(ctx, features, kernel, targets, Lists(from_squares), Lists(move_filters), Lists(moves_per_board));
    at::AutoDispatchBelowADInplaceOrView below;
    return policy_move_loss(ctx, features, kernel, from_squares, move_filters, moves_per_board, targets);
}
// The one-pass forms: their gradients come without a graph, as those that a backward pass leaves; their losses would end one
// without a word, and refuse instead.
using Grads = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
Grads refusing_loss(Grads out, at::ArrayRef<at::Tensor> inputs) {
    if (any_requires_grad(inputs))
        std::get<0>(out) = refusing(std::get<0>(out), "the loss of a batchfirst _grad form cannot be differentiated: its gradients are beside it");
    return out;
}
Grads policy_loss_grad_autograd(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& targets,
                                const at::Tensor& board_weights, bool features_grad, bool kernel_grad) {
    no_tangents({features, kernel, board_weights}, "policy_loss_grad");
    Grads out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = policy_loss_grad(ctx, features, kernel, targets, board_weights, features_grad, kernel_grad);
    }
    return refusing_loss(std::move(out), {features, kernel, board_weights});
}
Grads policy_move_loss_grad_autograd(int64_t ctx, const at::Tensor& features, const at::Tensor& kernel, const at::Tensor& from_squares,
                                     const at::Tensor& move_filters, const at::Tensor& moves_per_board, const at::Tensor& targets,
                                     const at::Tensor& board_weights, bool features_grad, bool kernel_grad) {
    no_tangents({features, kernel, board_weights}, "policy_move_loss_grad");
    Grads out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = policy_move_loss_grad(ctx, features, kernel, from_squares, move_filters, moves_per_board, targets, board_weights,
                                    features_grad, kernel_grad);
    }
    return refusing_loss(std::move(out), {features, kernel, board_weights});
}

// ---- norms ---------------------------------------------------------------------------------------------------------

// Host tables of many tensors.  The elements' order does not matter, so a dense tensor is taken as it lies; one with
// gaps or repeats is copied.
struct Tables {
    Context c;
    std::vector<at::Tensor> copies;              // of the tensors with gaps, undefined for the others
    std::vector<void*> ptrs;
    std::vector<size_t> counts;
    std::vector<int> types;
    at::Tensor work, norm;
    Tables(int64_t handle, at::TensorList tensors) : c(context(handle)) {
        ptrs.reserve(tensors.size()), counts.reserve(tensors.size()), types.reserve(tensors.size());
        for (const at::Tensor& t : tensors) {
            types.push_back(type_of(t, "tensors"));
            const void* p;
            if (t.device() == c.device && (t.is_contiguous() || t.is_non_overlapping_and_dense())) {
                p = t.const_data_ptr();
            } else {
                copies.resize(tensors.size());
                copies[types.size() - 1] = on_device(t, t.scalar_type(), "tensors", c);
                p = copies[types.size() - 1].const_data_ptr();
            }
            ptrs.push_back(const_cast<void*>(p));
            counts.push_back((size_t)t.numel());
        }
        work = workspace(lib.norm_workspace(ptrs.size()), c);
        norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(c.device));
    }
};

// The library refuses dense tensors that overlap; tensors with gaps reach it as copies and are looked at here.
void check_gapped(at::TensorList tensors) {
    auto span = [](const at::Tensor& t) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        const uintptr_t at = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        return std::make_pair(at, at + (size_t)(last + 1) * t.element_size());
    };
    for (size_t i = 0; i < tensors.size(); ++i) {
        const at::Tensor& t = tensors[i];
        if (t.numel() == 0 || t.is_contiguous() || t.is_non_overlapping_and_dense()) continue;
        for (int64_t d = 0; d < t.dim(); ++d)
            TORCH_CHECK_VALUE(t.stride(d) != 0 || t.size(d) == 1, "a tensor to clip must not be expanded");
        const auto a = span(t);
        for (size_t j = 0; j < tensors.size(); ++j) {
            if (j == i || tensors[j].numel() == 0) continue;
            const auto b = span(tensors[j]);
            TORCH_CHECK_VALUE(b.first >= a.second || a.first >= b.second, "two of the tensors to clip overlap or interleave");
        }
    }
}

at::Tensor global_norm(int64_t ctx, at::TensorList tensors) {
    const Tables t(ctx, tensors);
    check(lib.global_norm(t.c.ctx, t.ptrs.data(), t.counts.data(), t.types.data(), t.ptrs.size(), t.norm.data_ptr<float>(),
                          t.work.data_ptr(), (size_t)t.work.numel(), stream(t.c)));
    return t.norm;
}

at::Tensor clip_grad_norm_(int64_t ctx, at::TensorList tensors, double max_norm) {
    for (const at::Tensor& t : tensors) {
        TORCH_CHECK_VALUE(!t.requires_grad(), "tensors to clip are gradients: they must not require grad themselves");
        // torch says so itself, but only where the new version is noted, with the tensors scaled already
        TORCH_CHECK_VALUE(!t.is_inference() || c10::InferenceMode::is_enabled(), "an inference tensor cannot be clipped outside inference mode");
    }
    check_gapped(tensors);
    const Tables t(ctx, tensors);
    check(lib.clip_grad_norm(t.c.ctx, t.ptrs.data(), t.counts.data(), t.types.data(), t.ptrs.size(), (float)max_norm,
                             t.norm.data_ptr<float>(), t.work.data_ptr(), (size_t)t.work.numel(), stream(t.c)));
    for (size_t i = 0; i < tensors.size(); ++i) {
        if (i < t.copies.size() && t.copies[i].defined()) tensors[i].copy_(t.copies[i]);
        else tensors[i].unsafeGetTensorImpl()->bump_version();
    }
    return t.norm;
}

at::Tensor global_norm_autograd(int64_t ctx, at::TensorList tensors) {
    no_tangents(tensors, "global_norm");
    at::Tensor norm;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        norm = global_norm(ctx, tensors);
    }
    return any_requires_grad(tensors) ? refusing(norm, "global_norm cannot be differentiated") : norm;
}
at::Tensor clip_grad_norm_autograd(int64_t ctx, at::TensorList tensors, double max_norm) {
    no_tangents(tensors, "clip_grad_norm_");
    at::AutoDispatchBelowADInplaceOrView below;
    return clip_grad_norm_(ctx, tensors, max_norm);
}

}  // namespace

extern "C" {
// The library's functions, in struct Library's order.
void bf_torch_bind(void* const* functions) { std::copy_n(functions, sizeof(Library) / sizeof(void*), reinterpret_cast<void**>(&lib)); }
// Announces a context; device < 0 takes it back.
void bf_torch_context(void* handle, int device) {
    std::lock_guard<std::mutex> lock(contexts_mu);
    if (device < 0) contexts.erase(reinterpret_cast<int64_t>(handle));
    else contexts[reinterpret_cast<int64_t>(handle)] = device;
}
}

TORCH_LIBRARY_FRAGMENT(batchfirst, m) {
    m.def("policy_loss(int ctx, Tensor features, Tensor logit_kernel, Tensor targets) -> Tensor");
    m.def("policy_loss_grad(int ctx, Tensor features, Tensor logit_kernel, Tensor targets, Tensor board_weights, "
          "bool features_grad=True, bool kernel_grad=True) -> (Tensor, Tensor, Tensor)");
    m.def("policy_move_loss(int ctx, Tensor features, Tensor logit_kernel, Tensor from_squares, Tensor move_filters, "
          "Tensor moves_per_board, Tensor targets) -> Tensor");
    m.def("policy_move_loss_grad(int ctx, Tensor features, Tensor logit_kernel, Tensor from_squares, Tensor move_filters, "
          "Tensor moves_per_board, Tensor targets, Tensor board_weights, bool features_grad=True, bool kernel_grad=True) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("global_norm(int ctx, Tensor[] tensors) -> Tensor");
    m.def("clip_grad_norm_(int ctx, Tensor(a!)[] tensors, float max_norm) -> Tensor");
}
// one body for every device, so that the wrong one is refused in the framework's words
TORCH_LIBRARY_IMPL(batchfirst, CompositeExplicitAutograd, m) {
    m.impl("policy_loss", policy_loss);
    m.impl("policy_loss_grad", policy_loss_grad);
    m.impl("policy_move_loss", policy_move_loss);
    m.impl("policy_move_loss_grad", policy_move_loss_grad);
    m.impl("global_norm", global_norm);
    m.impl("clip_grad_norm_", clip_grad_norm_);
}
TORCH_LIBRARY_IMPL(batchfirst, Autograd, m) {
    m.impl("policy_loss", policy_loss_autograd);
    m.impl("policy_move_loss", policy_move_loss_autograd);
    // not differentiable
    m.impl("policy_loss_grad", policy_loss_grad_autograd);
    m.impl("policy_move_loss_grad", policy_move_loss_grad_autograd);
    m.impl("global_norm", global_norm_autograd);
    m.impl("clip_grad_norm_", clip_grad_norm_autograd);
}
