"""PyTorch-ROCm custom ops over the C ABI: device tensors in, device tensors out, on torch's
current stream.  PyTorch is plumbing here (allocator, streams, torch.distributed); every op body
is one call into libbatchfirst_hip.so.

    torch.ops.batchfirst.eval_wire(ctx, piece_filters u8[B], occupied_bbs i64[N]) -> f32[N]
    torch.ops.batchfirst.eval_structs(ctx, records u8[N, stride])                 -> f32[N]
    torch.ops.batchfirst.eval_mailbox(ctx, mailbox u8[N, 32])                      -> f32[N]
    torch.ops.batchfirst.encode_planes_wire(ctx, piece_filters, occupied_bbs)      -> f32[N,15,8,8]
    torch.ops.batchfirst.encode_planes_structs(ctx, records)                       -> f32[N,15,8,8]
    torch.ops.batchfirst.encode_mailbox_wire / encode_mailbox_structs              -> u8[N,32]
    torch.ops.batchfirst.policy_features_wire / policy_features_structs            -> f32[N,32,8,8]
    torch.ops.batchfirst.policy_scores(ctx, features, from_squares, move_filters, moves_per_board) -> f32[M]

and, for training the move-scoring head on those features (float32, bfloat16 or float16; the kernel [32,73] of the
features' type):

    torch.ops.batchfirst.policy_loss(ctx, features, logit_kernel, targets i64[N])  -> f32[N]
    torch.ops.batchfirst.policy_move_loss(ctx, features, logit_kernel, from_squares, move_filters, moves_per_board,
                                          targets)                                 -> f32[N]
    torch.ops.batchfirst.policy_loss_grad / policy_move_loss_grad(..., board_weights, features_grad=True,
                                          kernel_grad=True) -> (f32[N], grad of features, grad of logit_kernel)
    torch.ops.batchfirst.global_norm(ctx, tensors)                                 -> f32[]
    torch.ops.batchfirst.clip_grad_norm_(ctx, tensors, max_norm)                   -> f32[], tensors scaled in place

The two losses are differentiable in the features and the kernel; the ``_grad`` forms give loss and gradients in one
pass where the boards' weights in the total are known beforehand.

``ctx`` is the integer handle of a :class:`DeviceContext`.  occupied_bbs travels as int64
because torch has no first-class uint64; only the bits matter (the reference's placeholder is
int64 too, ann_creation_helper.py:51).
"""
import ctypes
from typing import Tuple

import numpy as np
import torch

from . import _lib
from .chestimator import _as_blob, _as_policy_blob

_contexts = {}


class DeviceContext:
    """Owns a bf_ctx on one GPU; ``handle`` is what the ops take."""

    def __init__(self, weights, device=0, dtype="f32"):
        self._lib = _lib.load()
        blob = _as_blob(weights)
        ctx = ctypes.c_void_p()
        _lib.check(self._lib.bf_ctx_create_ex(ctypes.byref(ctx), int(device), blob.ctypes.data, blob.size,
                                              _lib.precision_code(dtype)))
        self._ctx = ctx
        self.device = torch.device("cuda", int(device))
        self.handle = int(ctx.value)
        _contexts[self.handle] = self

    def set_policy(self, policy_weights):
        blob = _as_policy_blob(policy_weights)
        _lib.check(self._lib.bf_ctx_set_policy(self._ctx, blob.ctypes.data, blob.size))

    def check_policy(self):
        _lib.check(self._lib.bf_policy_check(self._ctx, _stream(self.device)))

    def check(self):
        """Synchronise the current stream and raise ValueError if a wire input was malformed."""
        _lib.check(self._lib.bf_ctx_check(self._ctx, _stream(self.device)))

    def close(self):
        if self._ctx is not None:
            _contexts.pop(self.handle, None)
            self._lib.bf_ctx_destroy(self._ctx)
            self._ctx = None


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _ctx(handle):
    try:
        return _contexts[int(handle)]
    except KeyError:
        raise ValueError("unknown batchfirst context handle %r" % (handle,))


def _dev(t, dtype, name, c=None):
    if not t.is_cuda:
        raise ValueError("%s must be a device tensor" % name)
    if t.dtype != dtype:
        raise ValueError("%s must have dtype %s" % (name, dtype))
    if c is not None and t.device != c.device:
        # the kernels run on the context's GPU: a pointer and a stream from another one must not reach them
        raise ValueError("%s is on %s, but the context lives on %s" % (name, t.device, c.device))
    return t.contiguous()


def _records(t, c):
    recs = _dev(t, torch.uint8, "records", c)
    if recs.dim() != 2 or recs.shape[1] < 82:
        raise ValueError("records must be uint8[N, stride] with stride >= 82")
    return recs


@torch.library.custom_op("batchfirst::eval_wire", mutates_args=())
def eval_wire(ctx: int, piece_filters: torch.Tensor, occupied_bbs: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    pf = _dev(piece_filters, torch.uint8, "piece_filters", c)
    occ = _dev(occupied_bbs, torch.int64, "occupied_bbs", c)
    out = torch.empty(occ.numel(), dtype=torch.float32, device=occ.device)
    _lib.check(c._lib.bf_eval_wire(c._ctx, pf.data_ptr(), pf.numel(), occ.data_ptr(), occ.numel(), out.data_ptr(),
                                   _stream(occ.device)))
    return out


@torch.library.custom_op("batchfirst::eval_structs", mutates_args=())
def eval_structs(ctx: int, records: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    recs = _records(records, c)
    out = torch.empty(recs.shape[0], dtype=torch.float32, device=recs.device)
    _lib.check(c._lib.bf_eval_structs(c._ctx, recs.data_ptr(), recs.shape[1], recs.shape[0], out.data_ptr(),
                                      _stream(recs.device)))
    return out


@torch.library.custom_op("batchfirst::eval_mailbox", mutates_args=())
def eval_mailbox(ctx: int, mailbox: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    mb = _dev(mailbox, torch.uint8, "mailbox", c)
    if mb.dim() != 2 or mb.shape[1] != 32:
        raise ValueError("mailbox must be uint8[N, 32]")
    out = torch.empty(mb.shape[0], dtype=torch.float32, device=mb.device)
    _lib.check(c._lib.bf_eval_mailbox(c._ctx, mb.data_ptr(), mb.shape[0], out.data_ptr(), _stream(mb.device)))
    return out


@torch.library.custom_op("batchfirst::encode_planes_wire", mutates_args=())
def encode_planes_wire(ctx: int, piece_filters: torch.Tensor, occupied_bbs: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    pf = _dev(piece_filters, torch.uint8, "piece_filters", c)
    occ = _dev(occupied_bbs, torch.int64, "occupied_bbs", c)
    out = torch.empty((occ.numel(), 15, 8, 8), dtype=torch.float32, device=occ.device)
    _lib.check(c._lib.bf_encode_planes_wire(c._ctx, pf.data_ptr(), pf.numel(), occ.data_ptr(), occ.numel(),
                                            out.data_ptr(), _stream(occ.device)))
    return out


@torch.library.custom_op("batchfirst::encode_planes_structs", mutates_args=())
def encode_planes_structs(ctx: int, records: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    recs = _records(records, c)
    out = torch.empty((recs.shape[0], 15, 8, 8), dtype=torch.float32, device=recs.device)
    _lib.check(c._lib.bf_encode_planes_structs(c._ctx, recs.data_ptr(), recs.shape[1], recs.shape[0],
                                               out.data_ptr(), _stream(recs.device)))
    return out


@torch.library.custom_op("batchfirst::encode_mailbox_wire", mutates_args=())
def encode_mailbox_wire(ctx: int, piece_filters: torch.Tensor, occupied_bbs: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    pf = _dev(piece_filters, torch.uint8, "piece_filters", c)
    occ = _dev(occupied_bbs, torch.int64, "occupied_bbs", c)
    out = torch.empty((occ.numel(), 32), dtype=torch.uint8, device=occ.device)
    _lib.check(c._lib.bf_encode_mailbox_wire(c._ctx, pf.data_ptr(), pf.numel(), occ.data_ptr(), occ.numel(),
                                             out.data_ptr(), _stream(occ.device)))
    return out


@torch.library.custom_op("batchfirst::encode_mailbox_structs", mutates_args=())
def encode_mailbox_structs(ctx: int, records: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    recs = _records(records, c)
    out = torch.empty((recs.shape[0], 32), dtype=torch.uint8, device=recs.device)
    _lib.check(c._lib.bf_encode_mailbox_structs(c._ctx, recs.data_ptr(), recs.shape[1], recs.shape[0],
                                                out.data_ptr(), _stream(recs.device)))
    return out


@torch.library.custom_op("batchfirst::policy_features_wire", mutates_args=())
def policy_features_wire(ctx: int, piece_filters: torch.Tensor, occupied_bbs: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    pf = _dev(piece_filters, torch.uint8, "piece_filters", c)
    occ = _dev(occupied_bbs, torch.int64, "occupied_bbs", c)
    out = torch.empty((occ.numel(), 32, 8, 8), dtype=torch.float32, device=occ.device)
    _lib.check(c._lib.bf_policy_features_wire(c._ctx, pf.data_ptr(), pf.numel(), occ.data_ptr(), occ.numel(),
                                              out.data_ptr(), _stream(occ.device)))
    return out


@torch.library.custom_op("batchfirst::policy_features_structs", mutates_args=())
def policy_features_structs(ctx: int, records: torch.Tensor) -> torch.Tensor:
    c = _ctx(ctx)
    recs = _records(records, c)
    out = torch.empty((recs.shape[0], 32, 8, 8), dtype=torch.float32, device=recs.device)
    _lib.check(c._lib.bf_policy_features_structs(c._ctx, recs.data_ptr(), recs.shape[1], recs.shape[0],
                                                 out.data_ptr(), _stream(recs.device)))
    return out


@torch.library.custom_op("batchfirst::policy_scores", mutates_args=())
def policy_scores(ctx: int, features: torch.Tensor, from_squares: torch.Tensor, move_filters: torch.Tensor,
                  moves_per_board: torch.Tensor) -> torch.Tensor:
    """Stage 2: one score per move; the three move tensors are uint8 device tensors."""
    c = _ctx(ctx)
    x9 = _dev(features, torch.float32, "features", c)
    frm = _dev(from_squares, torch.uint8, "from_squares", c)
    flt = _dev(move_filters, torch.uint8, "move_filters", c)
    per = _dev(moves_per_board, torch.uint8, "moves_per_board", c)
    n = x9.shape[0]
    if per.numel() != n or frm.numel() != flt.numel():
        raise ValueError("moves_per_board needs one entry per board, from_squares and move_filters one per move")
    # np.repeat of the board index, as numpy_style_repeat_1d_creator does (ann_creation_helper.py:488-510)
    board_index = torch.repeat_interleave(torch.arange(n, device=x9.device, dtype=torch.int32), per.to(torch.int64))
    if board_index.numel() != frm.numel():
        raise ValueError("moves_per_board sums to %d, but %d moves were given" % (board_index.numel(), frm.numel()))
    out = torch.empty(frm.numel(), dtype=torch.float32, device=x9.device)
    _lib.check(c._lib.bf_policy_scores(c._ctx, x9.data_ptr(), n, board_index.data_ptr(), frm.data_ptr(), flt.data_ptr(),
                                       frm.numel(), out.data_ptr(), _stream(x9.device)))
    return out


_TYPES = {torch.float32: _lib.BF_TYPE_F32, torch.bfloat16: _lib.BF_TYPE_BF16, torch.float16: _lib.BF_TYPE_F16}


def _aligned(t):
    """The kernels load 16 bytes at a time; a view may start anywhere."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _head(c, features, logit_kernel, targets):
    """Checked (features, kernel, targets) of a loss."""
    if features.dtype not in _TYPES:
        raise ValueError("features must be float32, bfloat16 or float16")
    x = _dev(features, features.dtype, "features", c)
    if tuple(x.shape[1:]) not in ((32, 8, 8), (32, 64)):
        raise ValueError("features must have shape [N, 32, 8, 8] or [N, 32, 64]")
    w = _dev(logit_kernel, features.dtype, "logit_kernel", c)
    if tuple(w.shape) not in ((32, 73), (1, 1, 32, 73)):
        raise ValueError("logit_kernel must have shape [32, 73] or [1, 1, 32, 73]")
    t = _dev(targets, torch.int64, "targets", c)
    if t.dim() != 1 or t.numel() != x.shape[0]:
        raise ValueError("targets needs one entry per board")
    return _aligned(x), _aligned(w), t


def _move_lists(c, from_squares, move_filters, moves_per_board, n):
    frm = _dev(from_squares, torch.uint8, "from_squares", c)
    flt = _dev(move_filters, torch.uint8, "move_filters", c)
    per = _dev(moves_per_board, torch.uint8, "moves_per_board", c)
    if per.numel() != n or frm.numel() != flt.numel():
        raise ValueError("moves_per_board needs one entry per board, from_squares and move_filters one per move")
    return frm, flt, per


def _board_weights(c, board_weights, n):
    g = board_weights
    if g.dim() == 1 and g.numel() > 1 and g.stride(0) == 0:
        g = g[:1]                     # one weight for all boards: what a mean's or a sum's gradient is
    g = _dev(g, torch.float32, "board_weights", c)
    if g.dim() > 1 or g.numel() not in (1, n):
        raise ValueError("board_weights needs one entry, or one per board")
    return g


def _loss(name, c, x, w, t, lists):
    n = x.shape[0]
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    _lib.check(getattr(c._lib, name)(c._ctx, x.data_ptr(), _TYPES[x.dtype], n, w.data_ptr(), *lists, t.data_ptr(), loss.data_ptr(),
                                     _stream(x.device)))
    return loss


def _loss_grad(name, c, x, w, t, lists, board_weights, features_grad, kernel_grad):
    n = x.shape[0]
    g = _board_weights(c, board_weights, n)
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x) if features_grad else x.new_empty(0)
    dw = torch.empty_like(w) if kernel_grad else w.new_empty(0)
    work = torch.empty(c._lib.bf_policy_loss_workspace(n) if kernel_grad else 0, dtype=torch.uint8, device=x.device)
    _lib.check(getattr(c._lib, name + "_grad")(
        c._ctx, x.data_ptr(), _TYPES[x.dtype], n, w.data_ptr(), *lists, t.data_ptr(), g.data_ptr(), g.numel(), loss.data_ptr(),
        dx.data_ptr() if features_grad else None, dw.data_ptr() if kernel_grad else None, work.data_ptr(), work.numel(),
        _stream(x.device)))
    return loss, dx, dw


@torch.library.custom_op("batchfirst::policy_loss", mutates_args=())
def policy_loss(ctx: int, features: torch.Tensor, logit_kernel: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Softmax cross entropy of one target a board over the 73 x 64 move vocabulary; a target is
    move_filter * 64 + from_square in the mover's frame, or -1 (loss 0).  Targets out of range count as -1 and are
    reported by :meth:`DeviceContext.check_policy`."""
    c = _ctx(ctx)
    return _loss("bf_policy_loss", c, *_head(c, features, logit_kernel, targets), ())


@torch.library.custom_op("batchfirst::policy_loss_grad", mutates_args=())
def policy_loss_grad(ctx: int, features: torch.Tensor, logit_kernel: torch.Tensor, targets: torch.Tensor,
                     board_weights: torch.Tensor, features_grad: bool = True,
                     kernel_grad: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(loss[N], gradients of sum(board_weights * loss)) in one pass; board_weights float32[N] or [1].  A gradient that
    is not asked for comes back empty."""
    c = _ctx(ctx)
    return _loss_grad("bf_policy_loss", c, *_head(c, features, logit_kernel, targets), (), board_weights, features_grad, kernel_grad)


@torch.library.custom_op("batchfirst::policy_move_loss", mutates_args=())
def policy_move_loss(ctx: int, features: torch.Tensor, logit_kernel: torch.Tensor, from_squares: torch.Tensor,
                     move_filters: torch.Tensor, moves_per_board: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """The same over each board's own moves, as :func:`policy_scores` takes them; a target is a place in the board's
    list, or -1 (a board without moves has no other).  Lists that do not add up, squares, filters or targets out of
    range are reported by :meth:`DeviceContext.check_policy`; the call itself never waits for the device."""
    c = _ctx(ctx)
    x, w, t = _head(c, features, logit_kernel, targets)
    frm, flt, per = _move_lists(c, from_squares, move_filters, moves_per_board, x.shape[0])
    return _loss("bf_policy_move_loss", c, x, w, t, (frm.data_ptr(), flt.data_ptr(), per.data_ptr(), frm.numel()))


@torch.library.custom_op("batchfirst::policy_move_loss_grad", mutates_args=())
def policy_move_loss_grad(ctx: int, features: torch.Tensor, logit_kernel: torch.Tensor, from_squares: torch.Tensor,
                          move_filters: torch.Tensor, moves_per_board: torch.Tensor, targets: torch.Tensor,
                          board_weights: torch.Tensor, features_grad: bool = True,
                          kernel_grad: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    c = _ctx(ctx)
    x, w, t = _head(c, features, logit_kernel, targets)
    frm, flt, per = _move_lists(c, from_squares, move_filters, moves_per_board, x.shape[0])
    return _loss_grad("bf_policy_move_loss", c, x, w, t, (frm.data_ptr(), flt.data_ptr(), per.data_ptr(), frm.numel()), board_weights,
                      features_grad, kernel_grad)


def _save_inputs(ctx, inputs, output):
    ctx.handle = inputs[0]
    ctx.save_for_backward(*inputs[1:])


def _backward_of(grad_op, lists):
    def backward(ctx, g):
        # the registered op, so that differentiating a second time is refused instead of silently wrong
        _, dx, dw = grad_op(ctx.handle, *ctx.saved_tensors, g, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return (None, dx if ctx.needs_input_grad[1] else None, dw if ctx.needs_input_grad[2] else None) + (None,) * (lists + 1)
    return backward


policy_loss.register_autograd(_backward_of(policy_loss_grad, 0), setup_context=_save_inputs)
policy_move_loss.register_autograd(_backward_of(policy_move_loss_grad, 3), setup_context=_save_inputs)


def _dense(t):
    return t.is_contiguous() or torch._prims_common.is_non_overlapping_and_dense(t)


def _span(t):
    last = sum((k - 1) * s for k, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _norm_tables(c, tensors):
    """Flat tensors and the host tables of their pointers, element counts and types.  The elements' order does not
    matter, so a dense tensor is taken as it lies; one with gaps or repeats is copied."""
    try:
        types = np.array([_TYPES[t.dtype] for t in tensors], np.int32)
    except KeyError:
        raise ValueError("tensors must be float32, bfloat16 or float16") from None
    index, flat = c.device.index, tensors
    if not all([t.get_device() == index and t.is_contiguous() for t in tensors]):
        flat = [t if t.get_device() == index and _dense(t) else _dev(t, t.dtype, "tensors", c) for t in tensors]
    ptrs = np.array([t.data_ptr() for t in flat], np.uint64)
    counts = np.array([t.numel() for t in flat], np.uint64)
    n = len(flat)
    work = torch.empty(c._lib.bf_grad_norm_workspace(n), dtype=torch.uint8, device=c.device)
    return flat, (ptrs, counts, types), (ptrs.ctypes.data, counts.ctypes.data, types.ctypes.data, n), work


def _check_gapped(tensors):
    """The library refuses dense tensors that overlap; tensors with gaps reach it as copies and are checked here."""
    if all([t.is_contiguous() for t in tensors]):
        return
    for i, t in enumerate(tensors):
        if t.numel() == 0 or _dense(t):
            continue
        if any(s == 0 and k > 1 for s, k in zip(t.stride(), t.shape)):
            raise ValueError("a tensor to clip must not be expanded")
        lo, hi = _span(t)
        for j, o in enumerate(tensors):
            if j != i and o.numel() and _span(o)[0] < hi and lo < _span(o)[1]:
                raise ValueError("two of the tensors to clip overlap or interleave")


# Registered by hand: custom_op's wrappers visit every tensor of a list in Python several times over, 118 us for 307
# tensors where these take 20.
_lists = torch.library.Library("batchfirst", "FRAGMENT")
_lists.define("global_norm(int ctx, Tensor[] tensors) -> Tensor")
_lists.define("clip_grad_norm_(int ctx, Tensor(a!)[] tensors, float max_norm) -> Tensor")


@torch.library.impl(_lists, "global_norm", "CompositeExplicitAutograd")
def global_norm(ctx, tensors):
    """The 2-norm over all elements of all tensors, a float32 scalar on the device; not differentiable."""
    c = _ctx(ctx)
    flat, _keep, tables, work = _norm_tables(c, tensors)
    norm = torch.empty((), dtype=torch.float32, device=c.device)
    _lib.check(c._lib.bf_global_norm(c._ctx, *tables, norm.data_ptr(), work.data_ptr(), work.numel(), _stream(c.device)))
    return norm


@torch.library.impl(_lists, "clip_grad_norm_", "CompositeExplicitAutograd")
def clip_grad_norm_(ctx, tensors, max_norm):
    """Scale all tensors in place by min(1, max_norm / (norm + 1e-6)); returns the norm before."""
    c = _ctx(ctx)
    if any([t.requires_grad for t in tensors]):
        raise ValueError("tensors to clip are gradients: they must not require grad themselves")
    _check_gapped(tensors)
    flat, _keep, tables, work = _norm_tables(c, tensors)
    norm = torch.empty((), dtype=torch.float32, device=c.device)
    _lib.check(c._lib.bf_clip_grad_norm(c._ctx, *tables, max_norm, norm.data_ptr(), work.data_ptr(), work.numel(), _stream(c.device)))
    torch.autograd.graph.increment_version(tensors)
    if flat is not tensors:
        for t, f in zip(tensors, flat):
            if f is not t:
                t.copy_(f)
    return norm


def eval_mailbox_debug(ctx, mailbox):
    """Scores plus every intermediate activation (testing aid; not a registered op)."""
    c = _ctx(ctx)
    mb = _dev(mailbox, torch.uint8, "mailbox", c)
    n = mb.shape[0]
    per = c._lib.bf_debug_floats_per_board()
    scores = torch.empty(n, dtype=torch.float32, device=mb.device)
    dbg = torch.zeros((n, per), dtype=torch.float32, device=mb.device)
    _lib.check(c._lib.bf_eval_mailbox_debug(c._ctx, mb.data_ptr(), n, scores.data_ptr(), dbg.data_ptr(),
                                            _stream(mb.device)))
    return scores, dbg


def records_to_tensor(structs, device):
    """View a NumPy array of node records as a uint8[N, stride] device tensor."""
    raw = np.ascontiguousarray(structs).view(np.uint8).reshape(len(structs), -1)
    return torch.from_numpy(raw.copy()).to(device)
