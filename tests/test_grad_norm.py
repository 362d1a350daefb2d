"""The norm over many tensors and clipping to it (ops.global_norm, ops.clip_grad_norm_) against float64.

Tolerances, u = 2^-24: squares are exact and summed in float64, so the norm is the true one rounded once and its square
root's last float64 bit: u norm + 1e-13 norm.  The factor adds limit / (norm + 1e-6) in float32 (the norm's rounding, the sum's,
the quotient's, the limit's: 4 u), a product one more and the rounding to the tensor's type half a step of that.
"""
import ctypes

import numpy as np
import pytest
import torch

from batch_first_amd import _lib, spec
from oracle import losses

U = 2.0 ** -24
gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}.get


def check_against(norm, tensors, before, limit):
    want, scaled = losses.clip_grad_norm([t.double().cpu().numpy() for t in before], limit)
    assert abs(float(norm) - want) <= want * (U + 1e-13)
    for t, b, s in zip(tensors, before, scaled):
        info = torch.finfo(t.dtype)
        tol = np.abs(s) * (6 * U + info.eps / 2) + info.smallest_normal * info.eps
        assert t.dtype == b.dtype and t.shape == b.shape
        off = np.abs(t.double().cpu().numpy() - s) - tol
        assert off.size == 0 or off.max() <= 0, off.max()


# ---- without a GPU ---------------------------------------------------------------------------------------------------

def test_refusals_of_the_c_entry_points():
    lib = _lib.load()
    ctx = ctypes.cast(ctypes.create_string_buffer(1 << 16), ctypes.c_void_p)    # the checks look at nothing in it
    buf = ctypes.create_string_buffer(1 << 17)
    p = (ctypes.addressof(buf) + 255) & ~255

    def clip(ctx=ctx, ptrs=(p, p + 4096), counts=(8, 8), types=(0, 1), limit=1.0, norm=p + 8192, ws=p + 16384, size=1 << 15):
        n = len(ptrs)
        return lib.bf_clip_grad_norm(ctx, (ctypes.c_void_p * n)(*ptrs), (ctypes.c_size_t * n)(*counts), (ctypes.c_int * n)(*types), n,
                                     limit, norm, ws, size, None)

    def refused(rc, text):
        assert rc == _lib.BF_E_ARG and text in lib.bf_last_error().decode(), lib.bf_last_error()

    refused(clip(ctx=None), "null context")
    refused(clip(norm=None), "null pointer")
    refused(clip(ws=None), "null pointer")
    refused(clip(ws=p + 16384 + 8), "aligned")
    refused(clip(size=8), "workspace")
    refused(clip(types=(0, 3)), "tensor 1 has unknown element type 3")
    refused(clip(ptrs=(p, None)), "tensor 1 is a null pointer")
    refused(clip(ptrs=(p + 2, p + 4096)), "tensor 0 is not aligned")
    refused(clip(ptrs=(p, p + 4097)), "tensor 1 is not aligned")
    refused(clip(counts=(8, (1 << 37) + 1)), "2^37")
    refused(lib.bf_global_norm(ctx, p, p, p, (1 << 20) + 1, p, p, 4096, None), "2^20")
    for limit in (-1.0, float("nan")):
        refused(clip(limit=limit), "max_norm")
    refused(clip(ptrs=(p, p)), "overlap")
    refused(clip(ptrs=(p + 16, p), types=(0, 1), counts=(8, 9)), "overlap")
    refused(lib.bf_clip_grad_norm(ctx, None, None, None, 1, 1.0, p, p, 4096, None), "null pointer")
    refused(lib.bf_global_norm(ctx, None, None, None, 1, p, p, 4096, None), "null pointer")


def test_gapped_tensors_that_overlap_are_refused():
    """The check comes before the one that the tensors are on the context's device."""
    from batch_first_amd import ops
    clip, t = torch.ops.batchfirst.clip_grad_norm_, torch.zeros(8, 8)
    ops._torch.bf_torch_context(1, 0)
    try:
        for good in ([t, torch.zeros(4)], [t[:, :4], torch.zeros(4)], [t[:4, :4], t[4:, :4]], [t[:0, :4], t]):
            with pytest.raises(ValueError, match="device tensor"):
                clip(1, good, 1.0)
        for bad in ([t[:, :4], t], [t[:, :4], t[:, :4]], [t[::2], t[1::2]]):
            with pytest.raises(ValueError, match="overlap"):
                clip(1, bad, 1.0)
        with pytest.raises(ValueError, match="expanded"):
            clip(1, [torch.zeros(4, 1).expand(4, 4)], 1.0)
    finally:
        ops._torch.bf_torch_context(1, -1)


# ---- on the GPU ------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def ctx():
    from batch_first_amd import ops, weights
    c = ops.DeviceContext(weights.make_weights(seed=7))
    yield c
    c.close()


def randn(shape, dtype=torch.float32, seed=0, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def clip_and_check(ctx, tensors, limit):
    before = [t.clone() for t in tensors]
    o = torch.ops.batchfirst
    alone = o.global_norm(ctx.handle, tensors)
    assert all(torch.equal(t, b) for t, b in zip(tensors, before))
    norm = o.clip_grad_norm_(ctx.handle, tensors, limit)
    assert norm.shape == () and norm.dtype == torch.float32 and torch.equal(norm, alone)
    check_against(norm, tensors, before, limit)
    return float(norm)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 255, 2336, 4097, 32768, 49151, 49152, 49153, 65535, 65537, 98305, 200003, 1 << 20, 3000001])
def test_one_tensor(ctx, n, dtype):
    clip_and_check(ctx, [randn(n, dtype, n)], 0.3 * n ** 0.5)


@gpu
@pytest.mark.parametrize("count", [2, 5, 11, 12, 13, 14, 27, 159, 160, 161, 321, 1000])
def test_many_tensors_of_mixed_types_and_sizes(ctx, count):
    rng = np.random.default_rng(count)
    tensors = [randn(int(k), TYPES[i % 3], i, 0.1) for i, k in enumerate(np.exp(rng.uniform(0, 10, count)).astype(int))]
    tensors[1] = torch.empty(0, device="cuda")
    clip_and_check(ctx, tensors, 0.7)


@gpu
@pytest.mark.parametrize("count", [2, 3, 4, 11, 12, 13])
def test_few_small_tensors(ctx, count):
    """As many as one workgroup takes, and one more."""
    clip_and_check(ctx, [randn(700 + 31 * i, TYPES[i % 3], i, 0.1) for i in range(count)], 0.7)


@gpu
def test_the_networks_own_tensors(ctx):
    tensors = [randn(tuple(s), torch.float32, i, 0.01) for i, s in enumerate(spec.layer_shapes())]
    clip_and_check(ctx, tensors, 1.0)


@gpu
@pytest.mark.parametrize("offset", [1, 2, 3, 5])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_any_alignment_and_untouched_neighbours(ctx, dtype, offset):
    """Tensors that start and end anywhere within a buffer: what lies around them stays as it was."""
    sizes = [1, 3, 70001, 9, 4096, 131075]
    flat = randn(sum(sizes) + offset * (len(sizes) + 1), dtype, 5)
    was, at, tensors, inside = flat.clone(), offset, [], torch.zeros(flat.numel(), dtype=torch.bool, device="cuda")
    for k in sizes:
        tensors.append(flat[at:at + k])
        inside[at:at + k] = True
        at += k + offset
    clip_and_check(ctx, tensors, 1.0)
    assert torch.equal(flat[~inside], was[~inside]) and not torch.equal(flat[inside], was[inside])


@gpu
def test_strides(ctx):
    """Dense tensors in another order are scaled as they lie, gapped ones through a copy."""
    a = randn((6, 5, 4, 3)).to(memory_format=torch.channels_last)
    b = randn((40, 30), torch.bfloat16, 1).t()
    room = randn((50, 20), torch.float32, 2)
    was = room.clone()
    clip_and_check(ctx, [a, b, room[:, 3:9]], 1.0)
    room[:, 3:9] = was[:, 3:9]
    assert torch.equal(room, was)


@gpu
def test_within_the_limit_nothing_changes(ctx):
    t = [randn(70000), randn(33, torch.float16, 1)]
    was = [x.clone() for x in t]
    for limit in (1e4, float("inf")):
        torch.ops.batchfirst.clip_grad_norm_(ctx.handle, t, limit)
        assert all(torch.equal(a, b) for a, b in zip(t, was))
    zero = [torch.zeros(100, device="cuda")]
    assert float(torch.ops.batchfirst.clip_grad_norm_(ctx.handle, zero, 1.0)) == 0.0 and not zero[0].any()
    torch.ops.batchfirst.clip_grad_norm_(ctx.handle, t, 0.0)
    assert not t[0].any() and not t[1].any()
    assert float(torch.ops.batchfirst.global_norm(ctx.handle, [])) == 0.0
    assert float(torch.ops.batchfirst.clip_grad_norm_(ctx.handle, [torch.empty(0, device="cuda")], 1.0)) == 0.0


@gpu
def test_norms_that_float32_squares_would_lose(ctx):
    """1e30 squared is beyond float32 and 1e-30 squared below it; the norms are neither."""
    for size in (1e30, 1e-30):
        t = randn(5000, torch.float32, 3) * size
        norm = torch.ops.batchfirst.global_norm(ctx.handle, [t])
        want = float(t.double().norm())
        assert abs(float(norm) - want) <= want * (U + 1e-13)


@gpu
def test_infinities_and_nan(ctx):
    t = [randn(3000), randn(70000, torch.bfloat16, 1)]
    t[0][5] = float("inf")
    norm = torch.ops.batchfirst.clip_grad_norm_(ctx.handle, t, 1.0)
    assert float(norm) == float("inf")
    assert t[0][5].isnan() and int(t[0].isnan().sum()) == 1 and not t[0][6:].any() and not t[1].any()
    t = [randn(3000), randn(70000, torch.bfloat16, 1)]
    t[1][-1] = float("nan")
    norm = torch.ops.batchfirst.clip_grad_norm_(ctx.handle, t, 1.0)
    assert norm.isnan() and t[0].isnan().all() and t[1].isnan().all()


@gpu
def test_same_bits_every_time(ctx):
    t = [randn(500001, torch.float32, i) for i in range(5)]
    norms = {float(torch.ops.batchfirst.global_norm(ctx.handle, t)) for _ in range(5)}
    assert len(norms) == 1


@gpu
def test_refusals(ctx):
    o = torch.ops.batchfirst
    x = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        o.clip_grad_norm_(ctx.handle, [x, x], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        o.clip_grad_norm_(ctx.handle, [x[:33], x[32:]], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        o.clip_grad_norm_(ctx.handle, [x], -1.0)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        o.clip_grad_norm_(ctx.handle, [x.double()], 1.0)
    with pytest.raises(ValueError, match="device tensor"):
        o.global_norm(ctx.handle, [x, torch.ones(3)])
    with pytest.raises(ValueError, match="device tensor"):
        o.clip_grad_norm_(ctx.handle, [torch.ones(3)], 1.0)
    with pytest.raises(ValueError, match="require grad"):
        o.clip_grad_norm_(ctx.handle, [x, torch.ones(3, device="cuda", requires_grad=True)], 1.0)
    version = x._version
    o.global_norm(ctx.handle, [x])
    assert x._version == version
    o.clip_grad_norm_(ctx.handle, [x], 100.0)
    assert x._version == version + 1
    assert torch.equal(x, torch.ones(64, device="cuda"))
    assert float(o.global_norm(ctx.handle, [x, x])) == pytest.approx(128 ** 0.5)    # reading twice is fine


@gpu
def test_captured_and_replayed(ctx):
    """A graph whose tensors are refilled between replays, another one beside it on its own tensors."""
    sets = [[randn(k, torch.float32, k) for k in (2336, 120832, 7)], [randn(k, torch.bfloat16, k) for k in (300000, 5)]]
    o = torch.ops.batchfirst
    side = torch.cuda.Stream()
    graphs, norms = [], []
    with torch.cuda.stream(side):
        o.clip_grad_norm_(ctx.handle, [randn(10)], 1.0)
        side.synchronize()
        for s in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                norms.append(o.clip_grad_norm_(ctx.handle, s, 1.0))
            graphs.append(g)
    torch.cuda.synchronize()
    for turn in range(4):
        for s, g, norm in zip(sets, graphs, norms):
            for i, t in enumerate(s):
                t.copy_(randn(t.shape, t.dtype, 10 * turn + i, 1.0 + turn))
            before = [t.clone() for t in s]
            eager = [t.clone() for t in s]
            want = o.clip_grad_norm_(ctx.handle, eager, 1.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(s, eager))
            check_against(norm, s, before, 1.0)


@gpu
def test_tensor_beyond_four_gib(ctx):
    n = (1 << 31) + 12345
    t = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    t[-1] = 3.0
    norm = torch.ops.batchfirst.clip_grad_norm_(ctx.handle, [t], 0.5 * float(np.sqrt(np.float64(n))))
    want = np.sqrt((n - 1) * 0.25 + 9.0)
    assert abs(float(norm) - want) <= want * 2 * U
    # the factor is below 1 by 4e-9: one step of float32 or none, neither seen in bfloat16
    assert t[-1] == 3.0 and t[0] == 0.5 and t[n // 2] == 0.5
    torch.ops.batchfirst.clip_grad_norm_(ctx.handle, [t], 0.25 * float(np.sqrt(np.float64(n))))
    assert t[0] == 0.25 and t[-1] == 1.5 and t[n // 2] == 0.25 and t[-2] == 0.25


@gpu
def test_a_training_step_of_the_head(ctx):
    """Features of the context's own tower, the loss over the legal moves, clipping, a step, and back into the context:
    the scores that it then serves are those of the stepped kernel."""
    from batch_first_amd import ops, positions, weights
    structs = positions.test_set(48, seed=4)
    blob = weights.to_policy_blob(weights.make_policy_weights(seed=11))
    c = ops.DeviceContext(weights.make_weights(seed=7))
    try:
        c.set_policy(blob)
        records = ops.records_to_tensor(structs, "cuda")
        o = torch.ops.batchfirst
        x = o.policy_features_structs(c.handle, records)
        kernel = torch.from_numpy(blob[-32 * 73:].reshape(32, 73).copy()).cuda()
        rng = np.random.default_rng(0)
        per = rng.integers(1, 40, 48)
        m = int(per.sum())
        lists = [torch.from_numpy(a.astype(np.uint8)).cuda() for a in (rng.integers(0, 64, m), rng.integers(0, 73, m), per)]
        targets = torch.from_numpy((rng.random(48) * per).astype(np.int64)).cuda()
        weight = torch.full((1,), 1 / 48, device="cuda")
        loss, _, grad = o.policy_move_loss_grad(c.handle, x, kernel, *lists, targets, weight, features_grad=False)
        # the loss is of the scores that the context serves
        scores = o.policy_scores(c.handle, x, *lists).double().cpu().numpy()
        ends = np.cumsum(per)
        for b in range(48):
            mine = scores[ends[b] - per[b]:ends[b]]
            want = np.log(np.exp(mine - mine.max()).sum()) + mine.max() - mine[int(targets[b])]
            assert abs(want - float(loss[b])) <= 64 * U * (1 + 34 * np.abs(mine).max())
        ref = losses.policy_loss(x.double().cpu().numpy(), kernel.double().cpu().numpy(), targets.cpu().numpy(), np.full(48, 1 / 48),
                                 [a.cpu().numpy() for a in lists])
        norm = o.clip_grad_norm_(c.handle, [grad], 0.1)
        assert float(norm) == pytest.approx(float(np.linalg.norm(ref["d_kernel"])), rel=1e-4)
        assert float(o.global_norm(c.handle, [grad])) <= 0.1 * (1 + 8 * U)
        kernel -= 0.5 * grad
        blob[-32 * 73:] = kernel.cpu().numpy().ravel()
        c.set_policy(blob)
        assert torch.equal(o.policy_features_structs(c.handle, records), x)
        stepped = o.policy_scores(c.handle, x, *lists)
        want = torch.from_numpy(np.concatenate([ref_scores for ref_scores in _scores(x, kernel, lists)]))
        size = torch.from_numpy(np.concatenate([s for s in _scores(x.abs(), kernel.abs(), lists)]))
        assert bool(((stepped.double().cpu() - want).abs() <= 40 * U * size).all())
        c.check_policy()
    finally:
        c.close()


def _scores(x, kernel, lists):
    sq, fl, per = (a.cpu().numpy().astype(np.int64) for a in lists)
    xs, k, at = x.double().cpu().numpy().reshape(-1, 32, 64), kernel.double().cpu().numpy(), 0
    for b, p in enumerate(per):
        yield np.einsum("cm,cm->m", xs[b][:, sq[at:at + p]], k[:, fl[at:at + p]])
        at += p


def refuses_tangents(handle, device):
    import torch.autograd.forward_ad as fwad
    o, t = torch.ops.batchfirst, torch.ones(5, device=device)
    with fwad.dual_level():
        dual = fwad.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward-mode derivatives of global_norm "):
            o.global_norm(handle, [t, dual])
        with pytest.raises(NotImplementedError, match="forward-mode derivatives of clip_grad_norm_ "):
            o.clip_grad_norm_(handle, [dual, t], 1.0)
    with pytest.raises(NotImplementedError, match="forward-mode derivatives of global_norm "):
        torch.func.jvp(lambda a: o.global_norm(handle, [a]), (t,), (torch.ones_like(t),))
    assert torch.equal(t, torch.ones_like(t))


def test_forward_mode_is_refused():
    from batch_first_amd import ops                # noqa: F401  registers the operators
    refuses_tangents(1, "cpu")


@gpu
def test_forward_mode_is_refused_on_the_gpu(ctx):
    refuses_tangents(ctx.handle, "cuda")


@gpu
def test_the_norm_refuses_to_be_differentiated(ctx):
    """A norm without a graph in a sum of losses would train without its part."""
    o = torch.ops.batchfirst
    a, b = torch.randn(300, device="cuda"), torch.randn(20, 7, device="cuda", requires_grad=True)
    want = o.global_norm(ctx.handle, [a, b.detach()])
    norm = o.global_norm(ctx.handle, [a, b])
    assert not want.requires_grad and norm.requires_grad and torch.equal(norm.detach(), want) and norm.item() == want.item()
    with pytest.raises(RuntimeError, match="global_norm cannot be differentiated"):
        (b.sum() + norm).backward()
    with torch.no_grad():
        assert not o.global_norm(ctx.handle, [a, b]).requires_grad


def clips_no_inference_tensors(handle, device):
    """Outside inference mode they may not be changed in place; that is said before they are."""
    o = torch.ops.batchfirst
    with torch.inference_mode():
        t = torch.ones(6, device=device)
    for tensors in ([t], [torch.ones(3, device=device), t.view(2, 3).t()[:2]]):
        with pytest.raises(ValueError, match="inference tensor"):
            o.clip_grad_norm_(handle, tensors, 0.5)
    assert torch.equal(t.clone(), torch.ones(6, device=device))
    return t


def test_inference_tensors_are_not_clipped():
    from batch_first_amd import ops                # noqa: F401  registers the operators
    clips_no_inference_tensors(1, "cpu")


@gpu
def test_inference_tensors_are_clipped_in_inference_mode(ctx):
    t = clips_no_inference_tensors(ctx.handle, "cuda")
    with torch.inference_mode():
        norm = torch.ops.batchfirst.clip_grad_norm_(ctx.handle, [t], 0.5)
        assert float(norm) == pytest.approx(6 ** 0.5) and float(t.norm()) == pytest.approx(0.5, rel=1e-5)
