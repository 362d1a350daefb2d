"""The operators that train the move-scoring head, as cases to time: inputs, plain forms and definitions in 64 bits.

A board's move vocabulary is the 73 x 64 = 4 672 (move filter, from-square) pairs of the move-scoring network's logit
layer (index = filter * 64 + square).  Features are float [boards][32][8][8], what the network's tower leaves in front
of that layer; the logit kernel is [32][73].

    vocabulary   softmax cross entropy of one target move a board over the whole vocabulary (ops.policy_loss) and, in
                 one pass, with the gradients of the features and of the logit kernel (ops.policy_loss_grad)
    moves        the same over the board's own list of legal moves (ops.policy_move_loss, ops.policy_move_loss_grad)
    norm         the norm over many gradients (ops.global_norm), and clipping them to a limit (ops.clip_grad_norm_)
"""
import math
import random

import numpy as np
import torch

own = False

CHANNELS, SQUARES, FILTERS = 32, 64, 73
VOCABULARY = FILTERS * SQUARES
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
#: Clipping works in place, so a second pass over the same state meets gradients that the first has clipped.  A training
#: step's gradients arrive unclipped: every pass's limit lies a little below what the pass before it left.
LIMIT_FALL = 0.999

#: The move-scoring network's trained parameters, floats each: nine input convolutions and the batch-norm's shifts, eight
#: tower layers with theirs, the logit kernel.
NETWORK = ([9 * 15 * c for c in (64, 32, 20, 20, 18, 18, 16)] + [4 * 15 * 24] * 2 + [236]
           + [236 * 512, 512, 512 * 128, 128, 9 * 128 * 32, 32] + [9 * 32 * 32, 32] * 5 + [32 * 73])


def listed():
    return [
        # the loss of one played move: what an analysis asks for one position at a time
        {"name": "vocabulary_one_board", "op": "vocabulary", "grad": False, "boards": 1, "type": "f32", "weights": "mean"},
        # one training batch of the reference's size
        {"name": "vocabulary_step_512", "op": "vocabulary", "grad": True, "boards": 512, "type": "f32", "weights": "mean"},
        # a validation pass over a ragged rest of a data set, half precision
        {"name": "vocabulary_check_f16", "op": "vocabulary", "grad": False, "boards": 9001, "type": "f16", "weights": "mean"},
        # a large mixed-precision training batch
        {"name": "vocabulary_step_bf16", "op": "vocabulary", "grad": True, "boards": 32768, "type": "bf16", "weights": "each"},
        # the benchmark's batch, float32
        {"name": "vocabulary_step_65536", "op": "vocabulary", "grad": True, "boards": 65536, "type": "f32", "weights": "mean"},
        # the same four uses with the softmax over each board's legal moves
        {"name": "moves_one_board", "op": "moves", "grad": False, "boards": 1, "type": "f32", "weights": "mean"},
        {"name": "moves_step_512", "op": "moves", "grad": True, "boards": 512, "type": "f32", "weights": "mean"},
        {"name": "moves_step_bf16", "op": "moves", "grad": True, "boards": 8191, "type": "bf16", "weights": "each"},
        {"name": "moves_step_65536", "op": "moves", "grad": True, "boards": 65536, "type": "f32", "weights": "mean"},
        # every gradient of the move-scoring network, clipped
        {"name": "clip_network", "op": "norm", "grad": True, "tensors": 0, "elements": sum(NETWORK), "type": "f32"},
        # the gradients of a larger model, many tensors of odd sizes in 16 bits
        {"name": "clip_ragged_bf16", "op": "norm", "grad": True, "tensors": 307, "elements": 60_000_011, "type": "bf16"},
        # the norm alone of gradients larger than any cache
        {"name": "norm_large", "op": "norm", "grad": False, "tensors": 24, "elements": 268_435_456, "type": "f32"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["vocabulary", "moves", "norm"])
    case = {"op": op, "grad": rng.random() < 0.6, "type": rng.choice(list(TYPES))}
    if op == "norm":
        case["elements"] = _spread(rng, 1000, 200_000_000)
        case["tensors"] = min(_spread(rng, 1, 500), case["elements"])
    else:
        case["boards"] = _spread(rng, 1, 65536)
        case["weights"] = rng.choice(["mean", "each"])
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _sizes(case):
    """The tensors' element counts: the network's own, or ragged ones (a few large, many small) that add up."""
    if not case["tensors"]:
        return list(NETWORK)
    rng = random.Random(case["tensors"] * 1_000_003 + case["elements"])
    shares = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    room, total = case["elements"] - case["tensors"], sum(shares)
    sizes = [1 + int(room * s / total) for s in shares]
    sizes[0] += case["elements"] - sum(sizes)
    return sizes


def _moves(n, rng):
    """Move lists of n boards as a move generator gives them: grouped by from-square, all different, about 30 a board
    and up to 218; one board in fifty has none (mate, stalemate)."""
    per = np.clip(rng.gamma(5.0, 6.5, n), 1, 218).astype(np.int64)
    if n > 1:
        per[rng.random(n) < 0.02] = 0
    start = np.cumsum(per) - per
    board = np.repeat(np.arange(n), per)
    k = np.arange(board.size) - start[board]                      # place in the board's own list
    pieces = np.argsort(rng.random((n, SQUARES)), axis=1)[:, :16]
    squares = pieces[board, k * 16 // np.maximum(per[board], 1)]
    filters = (rng.integers(0, FILTERS, n)[board] + k * rng.integers(1, FILTERS, n)[board]) % FILTERS
    targets = np.where(per > 0, (rng.random(n) * per).astype(np.int64), -1)
    return squares.astype(np.uint8), filters.astype(np.uint8), per.astype(np.uint8), targets


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "norm":
        # gradients of the size that a mean over a batch gives
        # in one flat buffer, as data-parallel training keeps them, each from a multiple of 64 elements on
        sizes = _sizes(case)
        starts = np.cumsum([0] + [-(-k // 64) * 64 for k in sizes])
        state["flat"] = torch.zeros(int(starts[-1]), dtype=dtype, device=dev)
        state["tensors"] = [state["flat"][a:a + k] for a, k in zip(starts.tolist(), sizes)]
        for t in state["tensors"]:
            t.copy_(torch.randn(t.numel(), generator=gen, device=dev) * 0.02)
        state["limit"] = 0.013 * math.sqrt(case["elements"])
    else:
        n = case["boards"]
        # the tower ends in a ReLU: about half the features are zero; the kernel as the network initialises it
        state["features"] = torch.relu(torch.randn((n, CHANNELS, 8, 8), generator=gen, device=dev)).to(dtype)
        state["kernel"] = (torch.randn((CHANNELS, FILTERS), generator=gen, device=dev) * math.sqrt(2.6 / CHANNELS)).to(dtype)
        # a mean over the boards, or boards that count differently; float16 training scales its loss up
        scale = min(65536, 128 * n) if case["type"] == "f16" else 1.0
        if case["weights"] == "mean":
            state["weights"] = torch.full((1,), scale / n, device=dev)
        else:
            state["weights"] = torch.rand(n, generator=gen, device=dev) * (scale / n)
        if case["op"] == "vocabulary":
            targets = torch.randint(0, VOCABULARY, (n,), generator=gen, device=dev)
            if n > 1:                                             # boards without a played move
                targets[torch.rand(n, generator=gen, device=dev) < 0.02] = -1
            state["targets"] = targets
        else:
            lists = _moves(n, np.random.default_rng(seed))
            state["squares"], state["filters"], state["per"], state["targets"] = (torch.from_numpy(a).to(dev) for a in lists)
    if own:
        from batch_first_amd import ops, weights
        state["ctx"] = ops.DeviceContext(weights.make_weights())
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)(state["case"], state)


def _own(case, s):
    o = torch.ops.batchfirst
    ctx = s["ctx"].handle
    if case["op"] == "norm":
        if not case["grad"]:
            return o.global_norm(ctx, s["tensors"])
        norm = o.clip_grad_norm_(ctx, s["tensors"], s["limit"])
        s["limit"] *= LIMIT_FALL
        return norm, s["flat"]
    if case["op"] == "vocabulary":
        if not case["grad"]:
            return o.policy_loss(ctx, s["features"], s["kernel"], s["targets"])
        return o.policy_loss_grad(ctx, s["features"], s["kernel"], s["targets"], s["weights"])
    lists = s["squares"], s["filters"], s["per"], s["targets"]
    if not case["grad"]:
        return o.policy_move_loss(ctx, s["features"], s["kernel"], *lists)
    return o.policy_move_loss_grad(ctx, s["features"], s["kernel"], *lists, s["weights"])


def _plain(case, s):
    return {"vocabulary": _plain_vocabulary, "moves": _plain_moves, "norm": _plain_norm}[case["op"]](case, s)


def _plain_vocabulary(case, s):
    n = case["boards"]
    x = s["features"].float().reshape(n, CHANNELS, SQUARES)
    k = s["kernel"].float()
    logits = torch.matmul(k.t().contiguous(), x).reshape(n, VOCABULARY)
    valid = s["targets"] >= 0
    target = s["targets"].clamp(min=0)[:, None]
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    z = e.sum(1, keepdim=True)
    loss = torch.where(valid, (torch.log(z) + top - logits.gather(1, target))[:, 0], 0.0)
    if not case["grad"]:
        return loss
    d = e / z
    d.scatter_add_(1, target, torch.full_like(target, -1, dtype=torch.float32))
    d *= (s["weights"] * valid)[:, None]
    return (loss,) + _plain_gradients(s, x, k, d)


def _plain_gradients(s, x, k, d):
    """Of the features and of the kernel, from the logits' [boards][4672]."""
    d = d.reshape(-1, FILTERS, SQUARES)
    d_features = torch.matmul(k, d).reshape(-1, CHANNELS, 8, 8)
    d_kernel = torch.matmul(x, d.transpose(1, 2).contiguous()).sum(0, dtype=torch.float64)   # over up to 65 536 boards
    return d_features.to(s["features"].dtype), d_kernel.to(s["kernel"].dtype)


def _plain_moves(case, s):
    n, m = case["boards"], s["squares"].numel()
    dev = s["squares"].device
    x = s["features"].float().reshape(n, CHANNELS, SQUARES)
    k = s["kernel"].float()
    per = s["per"].long()
    start = torch.cumsum(per, 0) - per
    board = torch.repeat_interleave(torch.arange(n, device=dev), per, output_size=m)
    squares, filters = s["squares"].long(), s["filters"].long()
    logits = (x[board, :, squares] * k.t()[filters]).sum(1)
    valid = s["targets"] >= 0
    chosen = (start + s["targets"].clamp(min=0)).clamp(max=m - 1)
    top = torch.full((n,), -math.inf, device=dev).scatter_reduce(0, board, logits, "amax")
    e = torch.exp(logits - top[board])
    z = torch.zeros(n, device=dev).index_add(0, board, e)
    loss = torch.where(valid, torch.log(z) + top - logits[chosen], 0.0)
    if not case["grad"]:
        return loss
    d = e / z[board]
    d.index_add_(0, chosen, -valid.float())
    d *= (s["weights"] * valid)[board]
    places = (board * FILTERS + filters) * SQUARES + squares
    d = torch.zeros(n * VOCABULARY, device=dev).index_add(0, places, d)
    return (loss,) + _plain_gradients(s, x, k, d)


def _plain_norm(case, s):
    total = torch.stack([(t.float() * t.float()).sum(dtype=torch.float64) for t in s["tensors"]]).sum()
    norm = torch.sqrt(total).float()
    if not case["grad"]:
        return norm
    scale = torch.clamp(s["limit"] / (norm + 1e-6), max=1.0)
    s["limit"] *= LIMIT_FALL
    for t in s["tensors"]:
        t.copy_(t.float() * scale)
    return norm, s["flat"]


# ---- the bytes and operations that a pass cannot do without ---------------------------------------------------------

def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        n = case["elements"]
        return {"bytes": n * size * (2 if case["grad"] else 1) + 4, "flops": n * (3 if case["grad"] else 2)}
    n, passes = case["boards"], 3 if case["grad"] else 1
    features = n * CHANNELS * SQUARES * size
    kernel = CHANNELS * FILTERS * size
    bytes_ = (features + kernel) * (2 if case["grad"] else 1) + n * (8 + 4)
    if case["grad"]:
        bytes_ += 4 * (1 if case["weights"] == "mean" else n)
    if case["op"] == "vocabulary":
        return {"bytes": bytes_, "flops": passes * 2 * CHANNELS * VOCABULARY * n}
    moves = 32 * n                                                # the lists' mean length
    return {"bytes": bytes_ + n + 2 * moves, "flops": passes * 2 * CHANNELS * moves}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "norm":
        squares = sum(float(torch.dot(t.double(), t.double())) for t in s["tensors"])
        norm = torch.tensor(math.sqrt(squares), dtype=torch.float64)
        if not case["grad"]:
            return norm
        factor = min(1.0, s["limit"] / (math.sqrt(squares) + 1e-6))
        return norm, s["flat"].double() * factor
    n = case["boards"]
    weights = s["weights"].double().expand(n)
    k = s["kernel"].double()
    losses, grads, d_k = [], [], torch.zeros((CHANNELS, FILTERS), dtype=torch.float64, device=k.device)
    first = 0
    for lo in range(0, n, 2048):
        hi = min(lo + 2048, n)
        x = s["features"][lo:hi].double().flatten(2).permute(0, 2, 1).contiguous()      # [boards][64][32]
        logits = x @ k                                                                # [boards][64][73]
        t = s["targets"][lo:hi]
        has = t >= 0
        wanted = torch.zeros_like(logits)
        if case["op"] == "vocabulary":
            b = torch.arange(hi - lo, device=k.device)[has]
            wanted[b, t[has] % SQUARES, t[has] // SQUARES] = 1.0
            log_p = torch.log_softmax(logits.flatten(1), 1).view_as(logits)
            loss = -(log_p * wanted).sum((1, 2))
            d = (log_p.exp() - wanted) * (weights[lo:hi] * has)[:, None, None]
        else:
            # each board's list padded to the longest with moves of logit -inf
            per = s["per"][lo:hi].long()
            ends = torch.cumsum(per, 0) + first
            slot = torch.arange(max(1, int(per.max())), device=k.device)
            real = slot[None, :] < per[:, None]
            at = torch.where(real, (ends - per)[:, None] + slot[None, :], 0)
            first = int(ends[-1])
            if s["squares"].numel():
                sq, fl = s["squares"][at].long(), s["filters"][at].long()
            else:
                sq = fl = torch.zeros_like(at)
            flat = sq * FILTERS + fl
            score = logits.flatten(1).gather(1, flat).masked_fill(~real, -math.inf)
            score = torch.where((per > 0)[:, None], score, 0.0)
            log_p = torch.log_softmax(score, 1)
            picked = (slot[None, :] == t[:, None]) & real
            loss = -torch.where(picked, log_p, 0.0).sum(1)
            d = (torch.where(real, log_p.exp(), 0.0) - picked.double()) * (weights[lo:hi] * has)[:, None]
            d = torch.zeros_like(logits).flatten(1).scatter_add(1, flat, d).view_as(logits)
        losses.append(loss)
        if case["grad"]:
            grads.append((d @ k.t().contiguous()).permute(0, 2, 1).reshape(hi - lo, CHANNELS, 8, 8))
            d_k += x.reshape(-1, CHANNELS).t() @ d.reshape(-1, FILTERS)
    if not case["grad"]:
        return torch.cat(losses)
    return torch.cat(losses), torch.cat(grads), d_k
