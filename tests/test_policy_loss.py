"""Softmax cross entropy of the move-scoring head and its gradients (ops.policy_loss, ops.policy_move_loss) against the
definitions in float64 (oracle/losses.py).

Tolerances, with u = 2^-24 (half a step of float32), eps(t) / 2 half a step of the output's type t:
  a logit adds 32 products in float32:  dl = 40 u logit_size  (32 sums, the products, what splitting into bf16 terms drops)
  a loss is log(z) + top - l[target]:   2 dl + 16 u (1 + loss + top)
  a probability exp(l - top) / z:       relative 2 dl + u (2 spread + 100)     (exp's argument, z's sum in at most 90 steps)
  a gradient adds 73 (features) or 64 a board (kernel, at most 8 boards a partial sum) products of these, and is rounded
  once:                                 (2 dl + u (2 spread + 100) + u k + split) size + eps(t) / 2 |value|,  k = 80 / 600,
                                        split = 2^-17 where the probabilities travel as two bf16 terms (16-bit types)
  A probability below float32's smallest normal number 2^-126, or a bf16 term of one, may be flushed to zero: up to three
  flushes a product, 3 * 2^-126 * weight * |factor|, summed over the 73 filters / the boards' 64 squares.
  Operands in two float16 terms are scaled so that the largest lies in [2^13, 2^14) or above and end at float16's last
  step, 2^-24: what is below 2^-37 of the largest is lost.  The largest gradient of a board's logits is the target's, 1 - exp(-loss)
  (counted as 2^-17 where smaller); their magnitudes sum to at most twice that.  So a gradient may miss 2^-37 times
  2 weight (1 - exp(-loss)) times the largest factor, for either operand's loss, and for the logits' gradients as many
  times as there are terms: 73 or 64.
"""
import ctypes
import os

import numpy as np
import pytest
import torch

from batch_first_amd import _lib
from oracle import losses

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}.get
gpu = pytest.mark.gpu


def moves_for(n, rng, longest=60, empty=0.1):
    per = rng.integers(1, longest + 1, n)
    per[rng.random(n) < empty] = 0
    m = int(per.sum())
    return (rng.integers(0, 64, m).astype(np.uint8), rng.integers(0, 73, m).astype(np.uint8), per.astype(np.uint8))


def make(n, dtype, seed=0, moves=False, longest=60, scale=1.0):
    """Host inputs as a dict: features and kernel in `dtype`."""
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(np.maximum(rng.standard_normal((n, 32, 8, 8)), 0).astype(np.float32) * np.float32(scale)).to(dtype)
    k = torch.from_numpy((rng.standard_normal((32, 73)) * 0.28).astype(np.float32)).to(dtype)
    case = {"x": x, "k": k, "w": torch.from_numpy(rng.uniform(0.1, 1.0, n).astype(np.float32)), "moves": None}
    if moves:
        case["moves"] = moves_for(n, rng, longest)
        per = case["moves"][2].astype(np.int64)
        t = np.where(per > 0, (rng.random(n) * per).astype(np.int64), -1)
    else:
        t = rng.integers(0, 4672, n)
    t[rng.random(n) < 0.1] = -1
    case["t"] = torch.from_numpy(t)
    return case


def reference(case, weights=None):
    w = case["w"] if weights is None else weights
    return losses.policy_loss(case["x"].double().numpy(), case["k"].double().numpy(), case["t"].numpy(),
                              np.broadcast_to(w.double().numpy(), len(case["t"])), case["moves"])


def limits(ref, case):
    """(loss, d_features, d_kernel) tolerances."""
    dtype = case["x"].dtype
    flush = 3 * 2.0 ** -126 * float(case["w"].max())
    dl = 40 * U * ref["logit_size"]
    x, k = np.abs(case["x"].double().numpy().reshape(-1, 32, 64)), float(case["k"].abs().max())
    x = np.nan_to_num(x, posinf=0.0).max((1, 2), initial=0.0)
    lost = 2.0 ** -37 * np.broadcast_to(case["w"].double().numpy(), len(x)) * np.maximum(-np.expm1(-ref["loss"]), 2.0 ** -17)
    p = 2 * dl + U * (2 * ref["spread"] + 100)
    split = 0.0 if dtype == torch.float32 else 2.0 ** -17
    half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return (2 * dl + 16 * U * (1 + np.abs(ref["loss"]) + ref["top"]),
            (p[:, None, None] + U * 80 + split) * ref["d_features_size"] + half * np.abs(ref["d_features"]) + least
            + flush * 73 * k + (lost * 75 * k)[:, None, None],
            (p.max(initial=0.0) + U * 600 + split) * ref["d_kernel_size"] + half * np.abs(ref["d_kernel"]) + least
            + flush * 64 * len(x) * x.max(initial=0.0) + (lost * 66 * x).sum())


def close(got, want, tol, what):
    got = got.double().cpu().numpy().reshape(want.shape)
    off = np.abs(got - want) - tol
    assert np.all(off <= 0), "%s: off by %g over the tolerance at %s" % (what, off.max(), np.unravel_index(off.argmax(), off.shape))


# ---- without a GPU ---------------------------------------------------------------------------------------------------

def test_oracle_gradients_are_the_differences_of_its_losses():
    rng = np.random.default_rng(3)
    for moves in (False, True):
        case = make(4, torch.float32, 5, moves=moves)
        ref = reference(case)

        def total(x, k):
            r = losses.policy_loss(x, k, case["t"].numpy(), case["w"].numpy(), case["moves"])
            return float((r["loss"] * case["w"].double().numpy()).sum())

        x, k = case["x"].double().numpy().reshape(4, 32, 64), case["k"].double().numpy()
        dx, dk = rng.standard_normal(x.shape), rng.standard_normal(k.shape)
        h = 1e-5
        diff = (total(x + h * dx, k + h * dk) - total(x - h * dx, k - h * dk)) / (2 * h)
        # the third difference is below 100 here and the loss is known to 1e-14: h^2 * 100 / 6 + 1e-14 / h
        assert abs(diff - (ref["d_features"] * dx).sum() - (ref["d_kernel"] * dk).sum()) < 1e-8


def _fake_context():
    """Memory that stands for a context: the checks look at nothing in it, and every call here is refused by them."""
    return ctypes.cast(ctypes.create_string_buffer(1 << 16), ctypes.c_void_p)


def test_refusals_of_the_c_entry_points():
    lib, ctx = _lib.load(), _fake_context()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) & ~255
    big = lib.bf_policy_loss_workspace(2)

    def refused(rc, text):
        assert rc == _lib.BF_E_ARG and text in lib.bf_last_error().decode(), lib.bf_last_error()

    def loss(ctx=ctx, x=p, type_=0, n=2, k=p, t=p, out=p):
        return lib.bf_policy_loss(ctx, x, type_, n, k, t, out, None)

    refused(loss(ctx=None), "null context")
    refused(loss(type_=3), "element type 3")
    refused(loss(n=(1 << 26) + 1), "exceeds the limit")
    for name in ("x", "k", "t", "out"):
        refused(loss(**{name: None}), "null pointer")
    refused(loss(x=p + 4), "aligned")
    refused(loss(k=p + 8), "aligned")
    assert loss(n=0, x=None, k=None, t=None, out=p) == 0

    def grad(n=2, w=p, nw=2, out=p, dx=p, dk=p, ws=p, size=big):
        return lib.bf_policy_loss_grad(ctx, p, 0, n, p, p, w, nw, out, dx, dk, ws, size, None)

    refused(grad(w=None), "null pointer")
    refused(grad(nw=3), "3 weights for 2 boards")
    refused(grad(nw=0), "0 weights")
    refused(grad(out=None, dx=None, dk=None), "no output")
    refused(grad(dx=p + 2), "aligned")
    refused(grad(ws=p + 8), "aligned")
    refused(grad(size=big - 1), "workspace")
    refused(grad(ws=None), "workspace")

    def moves(n=2, frm=p, flt=p, per=p, m=4):
        return lib.bf_policy_move_loss(ctx, p, 0, n, p, frm, flt, per, m, p, p, None)

    refused(moves(frm=None), "null pointer")
    refused(moves(flt=None), "null pointer")
    refused(moves(per=None), "null pointer")
    refused(moves(m=(1 << 31) + 1), "2^31")
    refused(moves(n=0, per=None), "moves given without boards")
    refused(lib.bf_policy_move_loss_grad(ctx, p, 0, 2, p, p, p, p, 4, p, p, 2, p, p, p, p, big - 1, None),
            "workspace")


def test_ops_refuse_host_tensors_and_unknown_contexts():
    from batch_first_amd import ops
    o = torch.ops.batchfirst
    x, k, t = torch.zeros(2, 32, 8, 8), torch.zeros(32, 73), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="unknown batchfirst context"):
        o.policy_loss(1, x, k, t)
    ops._torch.bf_torch_context(1, 0)
    try:
        with pytest.raises(ValueError, match="device tensor"):
            o.policy_loss(1, x, k, t)
        with pytest.raises(ValueError, match="device tensor"):
            o.policy_loss(1, x.requires_grad_(), k, t)
        with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
            o.policy_loss_grad(1, x.double(), k, t, torch.ones(1))
    finally:
        ops._torch.bf_torch_context(1, -1)
    with pytest.raises(ValueError, match="unknown batchfirst context"):
        o.policy_loss(1, x, k, t)


def refuses_tangents(handle, device):
    """Every form, given a tensor with a tangent, in place of a result without one (a derivative of zero)."""
    import torch.autograd.forward_ad as fwad
    o = torch.ops.batchfirst
    x, k, t = torch.zeros(2, 32, 8, 8, device=device), torch.zeros(32, 73, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    u8 = torch.ones(2, dtype=torch.uint8, device=device)
    w = torch.ones(2, device=device)
    calls = {"policy_loss": lambda x, k, w: o.policy_loss(handle, x, k, t),
             "policy_move_loss": lambda x, k, w: o.policy_move_loss(handle, x, k, u8, u8, u8, t),
             "policy_loss_grad": lambda x, k, w: o.policy_loss_grad(handle, x, k, t, w),
             "policy_move_loss_grad": lambda x, k, w: o.policy_move_loss_grad(handle, x, k, u8, u8, u8, t, w)}
    for name, call_ in calls.items():
        for i in range(3 if name.endswith("grad") else 2):
            for leaf in (False, True):
                args = [a.clone().requires_grad_(leaf) for a in (x, k, w)]
                with fwad.dual_level():
                    args[i] = fwad.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(NotImplementedError, match="forward-mode derivatives of %s " % name):
                        call_(*args)
                    with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode derivatives"):
                        call_(*args)
        with pytest.raises(NotImplementedError, match="forward-mode derivatives of %s " % name):
            torch.func.jvp(lambda k: call_(x, k, w), (k,), (torch.ones_like(k),))


def test_forward_mode_is_refused():
    from batch_first_amd import ops                # noqa: F401  registers the operators
    refuses_tangents(1, "cpu")


@pytest.mark.parametrize("library", ["missing", "unloadable"])
def test_evaluation_ops_need_no_training_library(tmp_path, library):
    """Without libbatchfirst_torch.so, or with one that does not load, the other ops are there and these say what is wrong."""
    import subprocess
    import sys
    path = tmp_path / "libbatchfirst_torch.so"
    if library == "unloadable":
        path.write_bytes(b"not a library")
    code = """
import torch
from batch_first_amd import _lib
_lib.TORCH_PATH = %r
from batch_first_amd import ops
assert torch.ops.batchfirst.eval_structs is not None and callable(ops.policy_scores)
try:
    torch.ops.batchfirst.eval_structs(1, torch.zeros(1, 82, dtype=torch.uint8))
except ValueError as e:
    assert "unknown batchfirst context" in str(e)
ops._announce(None, 0)
for name in ("policy_loss", "policy_loss_grad", "policy_move_loss", "policy_move_loss_grad", "global_norm", "clip_grad_norm_"):
    try:
        getattr(ops, name)(1, [])
        raise SystemExit(name)
    except ImportError as e:
        assert "training operators are not available" in str(e) and _lib.TORCH_PATH in str(e), e
""" % str(path)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]


# ---- on the GPU ------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def ctx():
    from batch_first_amd import ops, weights
    c = ops.DeviceContext(weights.make_weights(seed=7))
    yield c
    c.close()


def on_gpu(case):
    out = {k: v.cuda() for k, v in case.items() if torch.is_tensor(v)}
    out["lists"] = () if case["moves"] is None else tuple(torch.from_numpy(a).cuda() for a in case["moves"])
    return out


def call(ctx, d, **kw):
    """(loss, d_features, d_kernel) of the one-pass form."""
    o = torch.ops.batchfirst
    op = o.policy_move_loss_grad if d["lists"] else o.policy_loss_grad
    return op(ctx.handle, d["x"], d["k"], *d["lists"], d["t"], d["w"], **kw)


def forward(ctx, d):
    o = torch.ops.batchfirst
    op = o.policy_move_loss if d["lists"] else o.policy_loss
    return op(ctx.handle, d["x"], d["k"], *d["lists"], d["t"])


def check_all(ctx, case):
    ref = reference(case)
    tol = limits(ref, case)
    d = on_gpu(case)
    loss = forward(ctx, d)
    close(loss, ref["loss"], tol[0], "loss")
    got = call(ctx, d)
    assert torch.equal(got[0], loss)
    for g, name, t in zip(got[1:], ("d_features", "d_kernel"), tol[1:]):
        assert g.dtype == case["x"].dtype
        close(g, ref[name], t, name)
    again = call(ctx, d)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    ctx.check_policy()
    return got


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n", [1, 2, 3, 7, 64, 301])
def test_losses_and_gradients(ctx, n, dtype, moves):
    check_all(ctx, make(n, dtype, seed=n, moves=moves))


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_boards_beyond_one_round_of_workgroups(ctx, dtype, moves):
    check_all(ctx, make(2049, dtype, seed=9, moves=moves, longest=20))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_steep_logits(ctx, dtype, moves):
    """Logits of a hundred and more: exp of them overflows, of their differences from the largest it does not."""
    case = make(9, dtype, seed=4, moves=moves, scale=60.0)
    ref = reference(case)
    assert ref["top"].max() > 89      # where exp passes the largest float32
    d = on_gpu(case)
    close(forward(ctx, d), ref["loss"], limits(ref, case)[0], "loss")
    got = call(ctx, d)
    for g, name, t in zip(got[1:], ("d_features", "d_kernel"), limits(ref, case)[1:]):
        close(g, ref[name], t, name)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_lists_of_every_length(ctx, dtype):
    """0 to 255 moves a board, the same move several times over, targets at both ends."""
    rng = np.random.default_rng(2)
    case = make(256, dtype, seed=2, moves=True)
    per = rng.permutation(256).astype(np.uint8)
    m = int(per.sum())
    sq, fl = rng.integers(0, 64, m).astype(np.uint8), rng.integers(0, 73, m).astype(np.uint8)
    sq[::3], fl[::3] = 63, 72
    case["moves"] = sq, fl, per
    case["t"] = torch.from_numpy(np.where(rng.random(256) < 0.5, 0, per.astype(np.int64) - 1))
    case["t"][torch.from_numpy(per == 0)] = -1
    check_all(ctx, case)


@gpu
@pytest.mark.parametrize("n", [1023, 1024, 1025, 4095, 4096, 4097, 9000])
def test_list_starts(ctx, n):
    """Boards at the borders of whatever the prefix sum of the list lengths is cut into."""
    case = make(n, torch.float32, seed=n, moves=True, longest=3)
    want = check_all(ctx, case)
    d = on_gpu(case)
    odd = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    odd[5:5 + n] = d["lists"][2]
    d["lists"] = d["lists"][:2] + (odd[5:5 + n],)
    assert all(torch.equal(a, b) for a, b in zip(call(ctx, d), want))


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_boards_without_a_target(ctx, moves):
    """They take no part whatever they hold; a NaN in a board that has a target stays in that board and the kernel."""
    case = make(5, torch.float32, seed=1, moves=moves)
    case["t"] = torch.tensor([3 if not moves else 0, -1, -1, 5 if not moves else 0, -1])
    if moves:
        case["moves"] = (case["moves"][0][:6].repeat(4), case["moves"][1][:6].repeat(4), np.array([6, 6, 0, 6, 6], np.uint8))
    clean = check_all(ctx, case)
    case["x"][1], case["x"][2], case["x"][4] = float("nan"), float("inf"), -float("inf")
    d = on_gpu(case)
    got = call(ctx, d)
    assert torch.equal(forward(ctx, d), clean[0])
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    assert not got[1][[1, 2, 4]].any()
    case["x"][3] = float("nan")
    got = call(ctx, on_gpu(case))
    assert got[0][3].isnan() and torch.equal(got[0][:3], clean[0][:3])
    assert got[1][3].isnan().any() and torch.equal(got[1][:3], clean[1][:3]) and got[2].isnan().any()
    case["t"][:] = -1
    got = call(ctx, on_gpu(case))
    assert not any(g.any() for g in got)
    ctx.check_policy()


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_no_boards(ctx, moves):
    case = make(3, torch.float32, moves=moves)
    d = on_gpu(case)
    d["x"], d["t"], d["w"], d["lists"] = d["x"][:0], d["t"][:0], d["w"][:0], tuple(a[:0] for a in d["lists"])
    assert forward(ctx, d).shape == (0,)
    d["w"] = torch.ones(1, device="cuda")
    loss, dx, dk = call(ctx, d)
    assert loss.shape == (0,) and dx.shape == (0, 32, 8, 8) and dk.shape == (32, 73) and not dk.any()
    o = torch.ops.batchfirst
    k = d["k"].clone().requires_grad_()
    (o.policy_move_loss if moves else o.policy_loss)(ctx.handle, d["x"], k, *d["lists"], d["t"]).sum().backward()
    assert not k.grad.any()


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_layouts_and_weights(ctx, moves):
    """Strided, misaligned and permuted inputs, a kernel with the blob's shape, one weight for all boards."""
    case = make(10, torch.bfloat16, seed=6, moves=moves)
    d = on_gpu(case)
    want = call(ctx, d)
    other = dict(d)
    other["x"] = d["x"].to(memory_format=torch.channels_last)
    assert not other["x"].is_contiguous()
    other["t"] = torch.stack([d["t"], d["t"]], 1)[:, 0]
    room = torch.empty(d["k"].numel() + 1, dtype=torch.bfloat16, device="cuda")
    room[1:] = d["k"].flatten()
    other["k"] = room[1:].view(1, 1, 32, 73)
    got = call(ctx, other)
    assert got[2].shape == (1, 1, 32, 73)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2].view(32, 73), want[2])
    other["x"] = d["x"].reshape(10, 32, 64)
    got = call(ctx, other)
    assert got[1].shape == (10, 32, 64) and torch.equal(got[1].view_as(want[1]), want[1])
    room = torch.empty(d["x"].numel() + 3, dtype=torch.bfloat16, device="cuda")
    room[3:] = d["x"].flatten()
    other["x"], other["k"] = room[3:].view_as(d["x"]), d["k"].t().contiguous().t()
    for i, a in enumerate(d["lists"]):           # bytes that start anywhere
        odd = torch.empty(a.numel() + 16, dtype=torch.uint8, device="cuda")
        odd[3 + 2 * i:][:a.numel()] = a
        other["lists"] = other["lists"][:i] + (odd[3 + 2 * i:][:a.numel()],) + other["lists"][i + 1:]
    assert all(torch.equal(a, b) for a, b in zip(call(ctx, other), want))
    d["w"] = torch.tensor([0.25], device="cuda")
    want = call(ctx, d)
    d["w"] = d["w"].expand(10)
    assert all(torch.equal(a, b) for a, b in zip(call(ctx, d), want))
    d["w"] = torch.full((10,), 0.25, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(call(ctx, d), want))
    only = call(ctx, d, kernel_grad=False)
    assert torch.equal(only[1], want[1]) and only[2].numel() == 0
    only = call(ctx, d, features_grad=False)
    assert torch.equal(only[2], want[2]) and only[1].numel() == 0


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_autograd(ctx, dtype, moves):
    case = make(21, dtype, seed=8, moves=moves)
    d = on_gpu(case)
    x, k = d["x"].clone().requires_grad_(), d["k"].clone().requires_grad_()
    o = torch.ops.batchfirst
    op = o.policy_move_loss if moves else o.policy_loss
    (op(ctx.handle, x, k, *d["lists"], d["t"]) * d["w"]).sum().backward()
    want = call(ctx, d)
    assert torch.equal(x.grad, want[1]) and torch.equal(k.grad, want[2])
    # a mean hands one expanded number down
    k.grad = None
    op(ctx.handle, d["x"], k, *d["lists"], d["t"]).mean().backward()
    d["w"] = torch.full((1,), 1 / 21, device="cuda")
    assert torch.equal(k.grad, call(ctx, d)[2])
    loss = op(ctx.handle, x, k, *d["lists"], d["t"]).sum()
    g, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_gradient_is_the_difference_of_the_losses(ctx, moves):
    """Along one direction, step h: the third derivative of a log-sum-exp along v is at most 0.2 r^3, r the spread of the
    logits' change; the losses are known to their tolerance."""
    case = make(6, torch.float32, seed=12, moves=moves)
    ref = reference(case, torch.ones(1))
    rng = np.random.default_rng(0)
    v = torch.from_numpy(rng.standard_normal(case["x"].shape).astype(np.float32))
    h = 2.0 ** -5
    d = on_gpu(case)
    d["w"] = torch.ones(1, device="cuda")
    g = call(ctx, d)[1].cpu().double()
    sides = []
    for sign in (1, -1):
        d["x"] = (case["x"] + sign * h * v).cuda()
        sides.append(forward(ctx, d).cpu().double())
    exactly = [losses.policy_loss((case["x"] + s * h * v).numpy(), case["k"].numpy(), case["t"].numpy(), np.ones(6), case["moves"]) for s in (1, -1)]
    r = np.abs(np.einsum("cf,ncs->nfs", case["k"].double().numpy(), v.double().numpy().reshape(6, 32, 64))).max((1, 2)) * 2
    tol = h * h / 6 * 0.2 * r ** 3 + (limits(exactly[0], case)[0] + limits(exactly[1], case)[0]) / (2 * h)
    along = (g * v.double()).flatten(1).sum(1)
    tol = tol + (limits(ref, case)[1] * np.abs(v.double().numpy().reshape(6, 32, 64))).sum((1, 2))
    assert np.all(np.abs(((sides[0] - sides[1]) / (2 * h) - along).numpy()) <= tol)


@gpu
def test_out_of_range_inputs_are_reported_once(ctx):
    case = make(4, torch.float32, seed=3)
    case["t"] = torch.tensor([1, 4672, -2, 7])
    d = on_gpu(case)
    loss, dx, dk = call(ctx, d)
    assert loss[1] == 0 and loss[2] == 0 and not dx[1:3].any()
    with pytest.raises(ValueError, match="out of range"):
        ctx.check_policy()
    ctx.check_policy()
    case["t"][1:3] = -1
    assert all(torch.equal(a, b) for a, b in zip((loss, dx, dk), call(ctx, on_gpu(case))))
    ctx.check_policy()

    case = make(3, torch.float32, seed=3, moves=True)
    case["moves"] = (np.array([1, 2, 3, 4, 5], np.uint8), np.array([0, 1, 2, 3, 4], np.uint8), np.array([2, 0, 3], np.uint8))
    case["t"] = torch.tensor([0, -1, 2])
    check_all(ctx, case)

    def reported(change):
        bad = dict(case)
        bad["t"] = case["t"].clone()
        bad["moves"] = tuple(a.copy() for a in case["moves"])
        change(bad)
        d = on_gpu(bad)
        got = call(ctx, d)
        with pytest.raises(ValueError, match="out of range"):
            ctx.check_policy()
        assert torch.equal(forward(ctx, d), got[0])
        with pytest.raises(ValueError, match="out of range"):
            ctx.check_policy()
        return got

    assert reported(lambda c: c["t"].__setitem__(2, 3))[0][2] == 0
    assert reported(lambda c: c["t"].__setitem__(1, 0))[0][1] == 0
    reported(lambda c: c["moves"][0].__setitem__(0, 64))
    reported(lambda c: c["moves"][1].__setitem__(0, 73))
    reported(lambda c: c["moves"][2].__setitem__(0, 1))        # one move too few
    reported(lambda c: c["moves"][2].__setitem__(2, 200))      # far too many: absent ones end the list
    ctx.check_policy()


@gpu
def test_a_loss_flag_does_not_reach_a_prediction(ctx):
    """Out-of-range inputs of a loss are bf_policy_check's to report, not the next move prediction's on the context."""
    from batch_first_amd import chestimator, ops, positions, weights
    pred, start, closer = chestimator.get_inference_functions(weights.make_weights(seed=7), policy_weights=weights.make_policy_weights(seed=1))
    try:
        from batch_first_amd.encoder import struct_array_to_ann_inputs
        structs = positions.test_set(4, seed=1)
        nib, occ = struct_array_to_ann_inputs(structs, structs[:0], np.ones(4, bool), np.zeros(0, bool), 4)
        moves = [np.array([1, 2, 3, 4], np.uint8), np.array([5, 6, 7, 8], np.uint8), np.ones(4, np.uint8)]
        want = start(nib, occ)(moves)
        handle = pred._handle()
        ops._torch.bf_torch_context(handle, 0)
        d = on_gpu(make(2, torch.float32))
        torch.ops.batchfirst.policy_loss(handle.value, d["x"], d["k"], torch.tensor([9999, 0], device="cuda"))
        torch.cuda.synchronize()
        assert np.array_equal(start(nib, occ)(moves), want)
        assert _lib.load().bf_policy_check(handle, None) == _lib.BF_E_FORMAT and b"loss input" in _lib.load().bf_last_error()
        assert _lib.load().bf_policy_check(handle, None) == 0
        ops._torch.bf_torch_context(handle, -1)
    finally:
        closer()


@gpu
def test_ops_refuse(ctx):
    o = torch.ops.batchfirst
    x, k, t = torch.zeros(2, 32, 8, 8, device="cuda"), torch.zeros(32, 73, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    u8 = torch.zeros(2, dtype=torch.uint8, device="cuda")
    w = torch.ones(2, device="cuda")
    for bad, match in (((x[:, :31], k, t), "shape"), ((x, k[:31], t), "shape"), ((x, k.t(), t), "shape"), ((x, k.bfloat16(), t), "dtype"),
                       ((x, k, t[:1]), "one entry"), ((x, k, t.int()), "dtype"), ((x.double(), k, t), "float32, bfloat16"),
                       ((x.cpu(), k, t), "device tensor"), ((x, k, t.cpu()), "device tensor")):
        with pytest.raises(ValueError, match=match):
            o.policy_loss(ctx.handle, *bad)
    for bad, match in ((w[:1].expand(2, 1), "board_weights"), (torch.ones(3, device="cuda"), "board_weights"), (w.double(), "dtype")):
        with pytest.raises(ValueError, match=match):
            o.policy_loss_grad(ctx.handle, x, k, t, bad)
    for bad, match in (((u8, u8[:1], u8), "one per move"), ((u8, u8, u8[:1]), "one entry per board"), ((u8.int(), u8, u8), "dtype")):
        with pytest.raises(ValueError, match=match):
            o.policy_move_loss(ctx.handle, x, k, *bad, t)


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_captured_and_replayed(ctx, moves):
    """Two graphs with their own workspaces, replayed in turn with other inputs and eager calls between."""
    cases = [make(300, torch.bfloat16, seed=s, moves=moves) for s in (1, 2)]
    if moves:      # a graph's lists keep their total
        cases[1]["moves"], cases[1]["t"] = cases[0]["moves"], cases[0]["t"]
    static = on_gpu(cases[0])
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        call(ctx, static)
        side.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(call(ctx, static))
            graphs.append(g)
    torch.cuda.synchronize()
    for turn in range(4):
        d = on_gpu(cases[turn % 2])
        want = call(ctx, d)
        for name in ("x", "k", "w", "t"):
            static[name].copy_(d[name])
        for g, out in zip(graphs, outs):
            for o in out:
                o.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn
    ctx.check_policy()


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_captured_backward(ctx, moves):
    """Loss and backward pass of leaves of their own in one graph, replayed with other features."""
    cases = [make(70, torch.float32, seed=s, moves=moves) for s in (3, 4)]
    if moves:
        cases[1]["moves"] = cases[0]["moves"]
    cases[1]["t"] = cases[0]["t"]
    d = on_gpu(cases[0])
    x, k = d["x"].clone().requires_grad_(), d["k"].clone().requires_grad_()
    o = torch.ops.batchfirst
    op = o.policy_move_loss if moves else o.policy_loss

    def step():
        x.grad, k.grad = None, None
        op(ctx.handle, x, k, *d["lists"], d["t"]).backward(d["w"])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        x.grad, k.grad = None, None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step()
    torch.cuda.synchronize()
    for turn in range(4):
        other = on_gpu(cases[turn % 2])
        want = call(ctx, other)
        with torch.no_grad():
            x.copy_(other["x"])
            k.copy_(other["k"])
            d["w"].copy_(other["w"])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, want[1]) and torch.equal(k.grad, want[2]), turn


@gpu
def test_captured_backward_beside_an_eager_graph(ctx):
    """Refused while an eager graph of another stream keeps a leaf's accumulator; once that is gone it is captured."""
    d = on_gpu(make(70, torch.float32, seed=5))
    x, k = d["x"].clone().requires_grad_(), d["k"].clone().requires_grad_()
    op = torch.ops.batchfirst.policy_loss
    want = call(ctx, d)
    eager = op(ctx.handle, x, k, d["t"])
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="outside the capture"):
            op(ctx.handle, x, k, d["t"]).backward(d["w"])
    assert x.grad is None and k.grad is None
    eager.backward(d["w"])                      # the eager one goes on as before
    assert torch.equal(x.grad, want[1]) and torch.equal(k.grad, want[2])
    del eager
    x.grad, k.grad = None, None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op(ctx.handle, x, k, d["t"]).backward(d["w"])
    for _ in range(3):
        x.grad.zero_()
        k.grad.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, want[1]) and torch.equal(k.grad, want[2])


@gpu
def test_two_threads(ctx):
    """Calls of one context from two threads, each on a stream of its own."""
    import threading
    cases = [on_gpu(make(400, torch.bfloat16, seed=s, moves=bool(s), longest=30)) for s in range(2)]
    want = [call(ctx, d) for d in cases]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = call(ctx, cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # noqa: BLE001  reported by the test
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@gpu
def test_streams_of_their_own(ctx):
    """Calls on two streams at once, each with its own workspace, give what they give alone."""
    cases = [on_gpu(make(700, torch.float32, seed=s, moves=s % 2 == 1, longest=30)) for s in range(4)]
    want = [call(ctx, d) for d in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None] * 4
    for _ in range(5):
        for i, (s, d) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i] = call(ctx, d)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@gpu
def test_unlisted_squares_may_hold_anything(ctx):
    """NaN and infinities in squares from which no move is listed change nothing but their own gradient's place: zero."""
    for dtype in TYPES:
        case = make(6, dtype, seed=13, moves=True, longest=20)
        sq, fl, per = case["moves"]
        sq[:] = sq % 32                          # squares 32 ... 63 of every board
        case["t"] = torch.from_numpy(np.where(per > 0, 0, -1).astype(np.int64))
        case["x"].view(6, 32, 64)[:, :, 32:] = 0
        clean = check_all(ctx, case)
        for bad in (float("nan"), float("inf"), -float("inf")):
            case["x"].view(6, 32, 64)[:, 5:9, 40:50] = bad
            d = on_gpu(case)
            got = call(ctx, d)
            assert all(torch.equal(a, b) for a, b in zip(got, clean)), (dtype, bad)
            assert torch.equal(forward(ctx, d), clean[0])


@gpu
def test_features_of_every_magnitude(ctx):
    """float32 features whose scale differs from board to board by 2^200, which no float16 term could hold unscaled."""
    rng = np.random.default_rng(1)
    case = make(40, torch.float32, seed=21)
    scale = torch.from_numpy(2.0 ** rng.integers(-100, 3, 40)).float()
    case["x"] = case["x"] * scale[:, None, None, None]
    case["t"] = torch.from_numpy(rng.integers(0, 4672, 40))
    check_all(ctx, case)
    # and of a kernel that makes up for it
    case = make(20, torch.float32, seed=22, moves=True)
    case["x"], case["k"] = case["x"] * 2.0 ** 60, case["k"] * 2.0 ** -60
    check_all(ctx, case)
    case["x"], case["k"] = case["x"] * 2.0 ** -120, case["k"] * 2.0 ** 120
    check_all(ctx, case)


@gpu
def test_a_board_that_is_almost_certain(ctx):
    """The target's probability within 1e-5 of one: the others' gradients keep their precision."""
    for moves in (False, True):
        for dtype in TYPES:
            case = make(8, dtype, seed=31, moves=moves)
            if moves:
                case["t"] = torch.zeros(8, dtype=torch.int64)
                sq, fl, per = case["moves"]
                per[:] = np.maximum(per, 2)
                m = int(per.sum())
                rng = np.random.default_rng(5)
                sq, fl = rng.integers(0, 64, m).astype(np.uint8), rng.integers(1, 73, m).astype(np.uint8)
                first = np.cumsum(per.astype(int)) - per
                sq[first], fl[first] = np.arange(8), 0
                case["moves"] = sq, fl, per
                at = [(b, b, 0) for b in range(8)]
            else:
                case["t"] = torch.tensor([64 * 0 + 3 * b for b in range(8)])
                at = [(b, 3 * b, 0) for b in range(8)]
            x, k = case["x"].view(8, 32, 64).float(), case["k"].float()
            k[0], k[0, 0] = 0.0, 4.0
            x[:, 0] = 0.0
            for b, s, f in at:
                x[b, 0, s] = 7.0                 # + 28 for the target's logit alone (filter 0, its square)
            case["x"], case["k"] = x.view(8, 32, 8, 8).to(dtype), k.to(dtype)
            ref = reference(case)
            assert ref["loss"].max() < 1e-5
            check_all(ctx, case)


@gpu
def test_features_beyond_four_gib(ctx):
    """More than 2^31 elements and 2^32 bytes of features: the last boards give what they give in a call of their own."""
    n = (1 << 20) + 3
    case = make(16, torch.bfloat16, seed=5)
    d = on_gpu(case)
    x = d["x"].repeat((n + 15) // 16, 1, 1, 1)[:n]
    t = d["t"].repeat((n + 15) // 16)[:n]
    one = torch.ones(1, device="cuda")
    loss, dx, _ = torch.ops.batchfirst.policy_loss_grad(ctx.handle, x, d["k"], t, one, kernel_grad=False)
    want = torch.ops.batchfirst.policy_loss_grad(ctx.handle, x[-16:].clone(), d["k"], t[-16:].clone(), one, kernel_grad=False)
    assert torch.equal(loss[-16:], want[0]) and torch.equal(dx[-16:], want[1])
    assert torch.equal(torch.ops.batchfirst.policy_loss(ctx.handle, x, d["k"], t)[-16:], want[0])
    per = torch.full((n,), 2, dtype=torch.uint8, device="cuda")
    frm = torch.arange(2 * n, device="cuda").remainder(64).to(torch.uint8)
    flt = torch.arange(2 * n, device="cuda").remainder(73).to(torch.uint8)
    t = torch.arange(n, device="cuda").remainder(3) - 1
    args = (frm, flt, per, t)
    loss, dx, _ = torch.ops.batchfirst.policy_move_loss_grad(ctx.handle, x, d["k"], *args, one, kernel_grad=False)
    last = (frm[-32:].clone(), flt[-32:].clone(), per[-16:].clone(), t[-16:].clone())
    want = torch.ops.batchfirst.policy_move_loss_grad(ctx.handle, x[-16:].clone(), d["k"], *last, one, kernel_grad=False)
    assert torch.equal(loss[-16:], want[0]) and torch.equal(dx[-16:], want[1])
    ctx.check_policy()


def whole_lists(case, shortest):
    """New lists of `shortest` moves a board at least."""
    rng = np.random.default_rng(1)
    per = np.maximum(case["moves"][2], shortest).astype(np.uint8)
    m = int(per.sum())
    case["moves"] = rng.integers(0, 64, m).astype(np.uint8), rng.integers(0, 73, m).astype(np.uint8), per
    return case["moves"]


@gpu
@pytest.mark.parametrize("value", [1e4, 1e8, 1e12, 1e20, 3e38])
def test_unlisted_squares_and_filters_of_any_size(ctx, value):
    """Finite values in squares and in columns of the kernel that no listed move uses change no bit, however large."""
    case = make(7, torch.float32, seed=17, moves=True, longest=40)
    sq, fl, per = whole_lists(case, 1)
    sq[:], fl[:] = sq % 32, fl % 60              # squares 32 ... 63 and filters 60 ... 72 of every board
    case["t"] = torch.zeros(7, dtype=torch.int64)
    case["x"].view(7, 32, 64)[:, :, 32:] = 0
    case["k"][:, 60:] = 0
    clean = check_all(ctx, case)
    for kind in ("square", "filter", "both"):
        big = dict(case, x=case["x"].clone(), k=case["k"].clone())
        if kind != "filter":
            big["x"].view(7, 32, 64)[:, 5:9, 40:50] = value
            big["x"].view(7, 32, 64)[:, 20, 33] = -value
        if kind != "square":
            big["k"][3:5, 61:70] = -value
            big["k"][17, 72] = value
        d = on_gpu(big)
        assert torch.equal(forward(ctx, d), clean[0]), kind
        # what the unlisted columns and squares hold takes no part in either gradient
        assert all(torch.equal(a, b) for a, b in zip(call(ctx, d), clean)), kind


def without(case, masked):
    """`case` with lists of the moves that `masked` (filter, square) leaves, for the oracle alone: targets as before."""
    n = len(case["t"])
    if case["moves"] is None:
        f, s = np.divmod(np.arange(4672), 64)
        boards = [(s, f)] * n
    else:
        ends = np.cumsum(case["moves"][2].astype(int))
        boards = [(case["moves"][0][a:b].astype(int), case["moves"][1][a:b].astype(int)) for a, b in zip(ends - case["moves"][2], ends)]
    out, sq, fl, per, targets = dict(case), [], [], [], []
    for (s, f), t in zip(boards, case["t"].tolist()):
        keep = ~masked(f, s)
        assert keep[t]
        sq.append(s[keep]), fl.append(f[keep]), per.append(int(keep.sum())), targets.append(int(keep[:t].sum()))
    out["moves"], out["t"] = (np.concatenate(sq), np.concatenate(fl), np.array(per)), torch.tensor(targets)
    return out


@gpu
@pytest.mark.parametrize("value", [1e5, 1e9, 1e20, 1e36])
@pytest.mark.parametrize("what", ["filter", "square"])
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_logits_far_below_the_others(ctx, moves, what, value):
    """Filters or squares whose logits a large negative value takes out of the softmax: the others keep their precision.

    The oracle sees them taken out of the lists: at -1e4 and below, exp is zero in 64 bits too."""
    case = make(9, torch.float32, seed=23, moves=moves)
    case["x"] += 0.25                            # every channel of every square counts
    x, k = case["x"].view(9, 32, 64), case["k"]
    if what == "filter":
        k[:, 7], k[:, 64] = -value, -value / 3
        masked = lambda f, s: (f == 7) | (f == 64)
    else:
        k[11] = -(k[11].abs() + 0.125)
        x[:, 11, 5], x[:, 11, 63] = value, value / 3
        masked = lambda f, s: (s == 5) | (s == 63)
    if moves:                                    # a target that is left, and one masked move at least
        sq, fl, per = whole_lists(case, 3)
        first = np.cumsum(per.astype(int)) - per
        sq[first], fl[first], sq[first + 1], fl[first + 1] = 5, 7, 9, 11
        case["t"] = torch.ones(9, dtype=torch.int64)
    else:
        case["t"] = torch.arange(9) * 65 + 66    # filters 1 ... 9, squares 2 ... 10
        case["t"][case["t"] // 64 == 7] = 66
        case["t"][case["t"] % 64 == 5] = 66
    left = without(case, masked)
    small = dict(left, x=case["x"].clone(), k=case["k"].clone())      # for the tolerances: values that take part
    if what == "filter":
        small["k"][:, 7] = small["k"][:, 64] = 0
    else:
        small["x"].view(9, 32, 64)[:, 11, 5] = small["x"].view(9, 32, 64)[:, 11, 63] = 0
    ref = reference(small)
    tol = limits(ref, small)
    d = on_gpu(case)
    loss = forward(ctx, d)
    close(loss, ref["loss"], tol[0], "loss")
    got = call(ctx, d)
    assert torch.equal(got[0], loss)
    close(got[1], ref["d_features"], tol[1], "d_features")
    close(got[2], ref["d_kernel"], tol[2], "d_kernel")
    only = call(ctx, d, kernel_grad=False), call(ctx, d, features_grad=False)
    assert torch.equal(only[0][1], got[1]) and torch.equal(only[1][2], got[2])
    ctx.check_policy()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_logits_of_minus_infinity(ctx, moves, dtype):
    """An infinity that makes a square's logits -inf takes them out of the softmax; only its channel's row of the kernel's
    gradient, 0 times infinity, is NaN, as by the formula.  One that makes a logit +inf makes its board's loss NaN."""
    case = make(5, dtype, seed=29, moves=moves)
    case["k"][11] = -(case["k"][11].float().abs() + 0.125).to(dtype)
    if moves:
        sq, fl, per = whole_lists(case, 3)
        first = np.cumsum(per.astype(int)) - per
        sq[first], fl[first], sq[first + 1], fl[first + 1] = 5, 7, 9, 11
        case["t"] = torch.ones(5, dtype=torch.int64)
    else:
        case["t"] = torch.arange(5) * 65 + 70     # squares 6 ... 10
    left = without(case, lambda f, s: s == 5)
    ref = reference(left)
    tol = limits(ref, left)
    case["x"].view(5, 32, 64)[:, 11, 5] = float("inf")
    d = on_gpu(case)
    close(forward(ctx, d), ref["loss"], tol[0], "loss")
    got = call(ctx, d)
    close(got[0], ref["loss"], tol[0], "loss")
    close(got[1], ref["d_features"], tol[1], "d_features")
    rest = torch.arange(32) != 11
    close(got[2][rest.cuda()], ref["d_kernel"][rest.numpy()], tol[2][rest.numpy()], "d_kernel")
    assert got[2][11].isnan().all()
    case["x"].view(5, 32, 64)[2, 11, 5] = -float("inf")
    got = call(ctx, on_gpu(case))[0].cpu()
    assert got[2].isnan() and not got[[0, 1, 3, 4]].isnan().any()


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
def test_logits_at_the_end_of_the_range(ctx, dtype, moves):
    """Logits near float32's largest, of either sign: their differences are what counts.  One channel makes the logits
    up: features 2^63 times powers of two, the kernel 2^62 ... 2^64; one place stands out and is the target or is not."""
    for sign in (1, -1):
        case = make(4, dtype, seed=3, moves=moves)
        case["x"].zero_(), case["k"].zero_()
        x, k = case["x"].view(4, 32, 64), case["k"]
        x[:, 6] = 2.0 ** 63
        k[6] = sign * 2.0 ** 64
        k[6, 3] = sign * (2.0 ** 64 + (2.0 ** 63 if sign > 0 else -(2.0 ** 63)))     # sign > 0: the largest, 1.5 * 2^127
        k[6, 4] = sign * 2.0 ** 62                                                  # sign < 0: the largest, -2^125
        best = 3 if sign > 0 else 4
        if moves:
            case["moves"] = (np.array([9, 8, 7] * 4, np.uint8), np.array([best, 5, 6] * 4, np.uint8), np.full(4, 3, np.uint8))
            case["t"] = torch.tensor([0, 1, 0, 2])
        else:
            x[:, 6, :] = 2.0 ** 62
            x[:, 6, 10] = 2.0 ** 63 if sign > 0 else 2.0 ** 61
            case["t"] = torch.tensor([64 * best + 10, 1, 64 * best + 10, 700])
        want = np.asarray(reference(case)["loss"])
        got = forward(ctx, on_gpu(case)).double().cpu().numpy()
        # exact products and one place that holds all of the probability: its loss is 0, the others' a difference
        # of two numbers of float32, rounded once
        with np.errstate(over="ignore"):
            assert np.array_equal(got, want.astype(np.float32).astype(np.float64)), (got, want)
        assert got[0] == 0 and got[1] > 1e30


@gpu
def test_forward_mode_is_refused_on_the_gpu(ctx):
    refuses_tangents(ctx.handle, "cuda")
    # nor in the backward pass, whose incoming gradient may have a tangent
    import torch.autograd.forward_ad as fwad
    d = on_gpu(make(3, torch.float32))
    k = d["k"].clone().requires_grad_()
    loss = forward(ctx, dict(d, k=k))
    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode derivatives"):
        loss.backward(fwad.make_dual(d["w"], torch.ones_like(d["w"])))
    assert k.grad is None


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_the_loss_of_a_grad_form_refuses_to_be_differentiated(ctx, moves):
    """It would end the graph without a word; the gradients beside it come without one, as a backward pass leaves them."""
    d = on_gpu(make(5, torch.float32, seed=2, moves=moves))
    want = call(ctx, d)
    for name in ("x", "k", "w"):
        loss, dx, dk = call(ctx, dict(d, **{name: d[name].clone().requires_grad_()}))
        assert all(torch.equal(a, b) for a, b in zip((loss.detach(), dx, dk), want))
        assert loss.requires_grad and not dx.requires_grad and not dk.requires_grad
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            loss.sum().backward()
        torch.ops.batchfirst.clip_grad_norm_(ctx.handle, [dk.clone()], 1.0)
        with torch.no_grad():
            assert not call(ctx, dict(d, **{name: d[name].clone().requires_grad_()}))[0].requires_grad
    assert not want[0].requires_grad


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n", [1, 70, 2600])
def test_one_gradient_alone(ctx, n, dtype, moves):
    """Either gradient without the other, and without the losses, is what both together give."""
    case = make(n, dtype, seed=40 + n, moves=moves, longest=80)
    case["t"][0] = 0 if not moves or case["moves"][2][0] else -1
    d = on_gpu(case)
    loss, dx, dk = call(ctx, d)
    one, other = call(ctx, d, kernel_grad=False), call(ctx, d, features_grad=False)
    assert torch.equal(one[0], loss) and torch.equal(one[1], dx) and one[2].numel() == 0
    assert torch.equal(other[0], loss) and other[1].numel() == 0 and torch.equal(other[2], dk)
    o = torch.ops.batchfirst
    op = o.policy_move_loss if moves else o.policy_loss
    for name, want in (("x", dx), ("k", dk)):
        leaf = d[name].clone().requires_grad_()
        e = dict(d, **{name: leaf})
        got, = torch.autograd.grad((op(ctx.handle, e["x"], e["k"], *d["lists"], d["t"]) * d["w"]).sum(), leaf)
        assert torch.equal(got, want)
    # the C entry may leave the losses out
    lib, p = _lib.load(), lambda t: ctypes.c_void_p(t.data_ptr())
    work = torch.empty(lib.bf_policy_loss_workspace(n), dtype=torch.uint8, device="cuda")
    again = torch.empty_like(dx), torch.empty_like(dk)
    type_ = TYPES.index(dtype)
    tail = (p(d["t"]), p(d["w"]), n, None, p(again[0]), p(again[1]), p(work), work.numel(),
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    if moves:
        sq, fl, per = d["lists"]
        rc = lib.bf_policy_move_loss_grad(ctypes.c_void_p(ctx.handle), p(d["x"]), type_, n, p(d["k"]), p(sq), p(fl), p(per), sq.numel(), *tail)
    else:
        rc = lib.bf_policy_loss_grad(ctypes.c_void_p(ctx.handle), p(d["x"]), type_, n, p(d["k"]), *tail)
    assert rc == 0 and torch.equal(again[0], dx) and torch.equal(again[1], dk)
    ctx.check_policy()


def check_on_gpu(ctx, case):
    """As check_all, with the definitions in float64 on the GPU: for many boards.

    The kernel's gradient adds a board's 64 products and then the boards of a wave, of 2 048, one by one, and the waves of a
    workgroup: 64 + n / 2048 + 8 roundings, which limits()' 600 covers up to a million boards."""
    n, dtype = len(case["t"]), case["x"].dtype
    assert n <= 1 << 20
    d = on_gpu(case)
    loss, dx, dk = call(ctx, d)
    k = d["k"].double()
    k_most = float(k.abs().max())
    flush = 3 * 2.0 ** -126 * float(case["w"].max())
    half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    split = 0.0 if dtype == torch.float32 else 2.0 ** -17
    want_dk, size_dk, p_most, x_most, lost_dk = torch.zeros_like(k), torch.zeros_like(k), 0.0, 0.0, 0.0
    starts = torch.cumsum(d["lists"][2].long(), 0) - d["lists"][2].long() if d["lists"] else None
    for lo in range(0, n, 4096):
        x = d["x"][lo:lo + 4096].double().reshape(-1, 32, 64)
        m = len(x)
        t, w = d["t"][lo:lo + m], d["w"][lo:lo + m].double()
        has = t >= 0
        logits, size = (torch.matmul(a.t().contiguous(), b).flatten(1) for a, b in ((k, x), (k.abs(), x.abs())))
        if starts is None:
            listed, target = torch.ones_like(logits), t.clamp(min=0)
        else:
            sq, fl, per = (a.long() for a in d["lists"])
            first, count = int(starts[lo]), int(per[lo:lo + m].sum())
            places = fl[first:first + count] * 64 + sq[first:first + count]
            board = torch.repeat_interleave(torch.arange(m, device="cuda"), per[lo:lo + m])
            listed = torch.zeros_like(logits).index_put_((board, places), torch.ones_like(places, dtype=torch.float64), accumulate=True)
            target = places[(starts[lo:lo + m] - first + t.clamp(min=0)).clamp(max=count - 1)]
            listed[~has, 0] = 1
        inside = listed > 0
        top = logits.masked_fill(~inside, -float("inf")).amax(1)
        spread = (top - logits.masked_fill(~inside, float("inf")).amin(1)) * has
        e = torch.where(inside, listed * torch.exp(torch.clamp(logits - top[:, None], max=0.0)), 0.0)
        z = e.sum(1, keepdim=True)
        hot = torch.zeros_like(e).scatter_(1, target[:, None], 1.0)
        want = torch.where(has, torch.log(z)[:, 0] + top - logits.gather(1, target[:, None])[:, 0], 0.0)
        dl = 40 * U * size.masked_fill(~inside, 0.0).amax(1) * has
        p = 2 * dl + U * (2 * spread + 100)
        off = (loss[lo:lo + m].double() - want).abs() - (2 * dl + 16 * U * (1 + want + (top * has).abs()))
        assert bool((off <= 0).all()), ("loss", float(off.max()))
        w = (w * has)[:, None]
        g, s = ((e / z - hot) * w).view(m, 73, 64), ((e / z + hot) * w.abs()).view(m, 73, 64)
        lost = 2.0 ** -37 * d["w"][lo:lo + m].double() * torch.clamp(-torch.expm1(-want), min=2.0 ** -17)
        want_dx = torch.matmul(k, g)
        tol = (p[:, None, None] + U * 80 + split) * torch.matmul(k.abs(), s) + half * want_dx.abs() + least + flush * 73 * k_most
        off = (dx[lo:lo + m].double().view(m, 32, 64) - want_dx).abs() - tol - (lost * 75 * k_most)[:, None, None]
        assert bool((off <= 0).all()), ("d_features", float(off.max()))
        want_dk += torch.matmul(x, g.transpose(1, 2).contiguous()).sum(0)
        size_dk += torch.matmul(x.abs(), s.transpose(1, 2).contiguous()).sum(0)
        most = x.abs().amax((1, 2))
        p_most, x_most, lost_dk = max(p_most, float(p.max())), max(x_most, float(most.max())), lost_dk + float((lost * 66 * most).sum())
    tol = (p_most + U * 600 + split) * size_dk + half * want_dk.abs() + least + flush * 64 * n * x_most + lost_dk
    off = (dk.double() - want_dk).abs() - tol
    assert bool((off <= 0).all()), ("d_kernel", float(off.max()))
    only = call(ctx, d, features_grad=False)
    assert torch.equal(only[0], loss) and torch.equal(only[2], dk)
    ctx.check_policy()


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_kernel_gradient_of_many_boards(ctx, dtype, moves):
    """Ten boards a wave, read ahead one by one."""
    check_on_gpu(ctx, make(20011, dtype, seed=51, moves=moves, longest=40))


@gpu
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_kernel_gradient_of_more_boards_than_a_round(ctx, moves):
    """A wave looks targets and lists up for 64 of its boards at a time; 2 048 waves begin another round beyond 131 072."""
    n = 131072 + 1027
    case = make(4001, torch.float32, seed=52, moves=moves, longest=9)
    again = -(-n // 4001)
    case["x"] = case["x"].repeat(again, 1, 1, 1)[:n]
    case["w"] = torch.from_numpy(np.random.default_rng(6).uniform(0.1, 1.0, n).astype(np.float32))
    case["t"] = case["t"].repeat(again)[:n]
    if moves:
        sq, fl, per = case["moves"]
        per = np.tile(per, again)[:n]
        m = int(per.astype(np.int64).sum())
        case["moves"] = np.tile(sq, again)[:m], np.tile(fl, again)[:m], per
    check_on_gpu(ctx, case)


@gpu
@pytest.mark.parametrize("value", [1e3, 1e6, 1e9, 1e20])
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_a_large_factor_of_zero(ctx, moves, value):
    """An element of the kernel, or a feature, that only meets zeros has no part in any logit, however large."""
    for what in ("kernel", "feature"):
        case = make(12, torch.float32, seed=61, moves=moves, longest=50)
        x, k = case["x"].view(12, 32, 64), case["k"]
        if what == "kernel":
            x[:, 11], k[11, 7:9] = 0, value
        else:
            k[11], x[:, 11, 20:24] = 0, value
        if moves:
            whole_lists(case, 4)
            sq, fl, per = case["moves"]
            first = np.cumsum(per.astype(int)) - per
            sq[first], fl[first], sq[first + 1], fl[first + 1] = 21, 30, 40, 7
            case["t"] = torch.from_numpy(np.arange(12) % 4)
        else:
            case["t"] = torch.from_numpy(np.arange(12) * 333 + 21)
        check_all(ctx, case)


@gpu
@pytest.mark.parametrize("what", ["filter", "square"])
@pytest.mark.parametrize("moves", [False, True], ids=["vocabulary", "moves"])
def test_large_values_beside_small_factors(ctx, moves, what):
    """As test_logits_far_below_the_others with products of ordinary size: values of 1e8 and more, taken out of the softmax,
    meet factors of 2^-20 and less.  The gradients of what is left have the ordinary values' precision."""
    case = make(9, torch.float32, seed=24, moves=moves)
    case["x"] += 0.25
    x, k = case["x"].view(9, 32, 64), case["k"]
    if what == "filter":
        x *= 2.0 ** -20
        k[:, 7], k[:, 64] = -1e8, -0.5e8         # 32 channels of 2^-22 and more: -380 and below
        masked = lambda f, s: (f == 7) | (f == 64)
    else:
        k *= 2.0 ** -20
        k[11] = -(k[11].abs() + 0.125 * 2.0 ** -20)
        x[:, 11, 5], x[:, 11, 63] = 4e9, 2e9     # -230 and below
        masked = lambda f, s: (s == 5) | (s == 63)
    if moves:
        sq, fl, per = whole_lists(case, 3)
        first = np.cumsum(per.astype(int)) - per
        sq[first], fl[first], sq[first + 1], fl[first + 1] = 5, 7, 9, 11
        case["t"] = torch.ones(9, dtype=torch.int64)
    else:
        case["t"] = torch.arange(9) + 64 * 20 + 10
    left = without(case, masked)
    small = dict(left, x=case["x"].clone(), k=case["k"].clone())
    if what == "filter":
        small["k"][:, 7] = small["k"][:, 64] = 0
    else:
        small["x"].view(9, 32, 64)[:, 11, 5] = small["x"].view(9, 32, 64)[:, 11, 63] = 0
    ref = reference(small)
    tol = limits(ref, small)
    d = on_gpu(case)
    # what is taken out has probabilities of e^-230 at most, times values of 4e9 below every tolerance
    close(forward(ctx, d), ref["loss"], tol[0], "loss")
    got = call(ctx, d)
    close(got[1], ref["d_features"], tol[1], "d_features")
    close(got[2], ref["d_kernel"], tol[2], "d_kernel")
    assert torch.equal(call(ctx, d, kernel_grad=False)[1], got[1]) and torch.equal(call(ctx, d, features_grad=False)[2], got[2])


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_unlisted_filters_may_hold_anything(ctx, dtype):
    """As unlisted squares: NaN and infinities in columns of the kernel that no listed move uses."""
    case = make(6, dtype, seed=14, moves=True, longest=20)
    sq, fl, per = whole_lists(case, 1)
    fl[:] = fl % 60
    case["t"] = torch.zeros(6, dtype=torch.int64)
    case["k"][:, 60:] = 0
    clean = check_all(ctx, case)
    for bad in (float("nan"), float("inf"), -float("inf")):
        case["k"][5:9, 62:70] = bad
        d = on_gpu(case)
        assert torch.equal(forward(ctx, d), clean[0]), bad
        assert all(torch.equal(a, b) for a, b in zip(call(ctx, d), clean)), bad
