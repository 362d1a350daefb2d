"""Losses of the move-scoring head, their gradients and gradient clipping from their definitions, in float64 on the CPU.

Beside each value comes the sum of the magnitudes that it adds up, which is what the rounding errors of a float32
evaluation scale with.
"""
import numpy as np

FILTERS, SQUARES = 73, 64


def _loss_of(logits, target, weight):
    """(loss, gradient of weight * loss by the logits, softmax) of one list of logits."""
    if target < 0:
        return 0.0, np.zeros_like(logits), np.zeros_like(logits)
    top = logits.max()
    e = np.exp(logits - top)
    p = e / e.sum()
    d = p.copy()
    d[target] -= 1.0
    return float(np.log(e.sum()) + top - logits[target]), d * weight, p


def policy_loss(features, kernel, targets, weights, moves=None):
    """``features`` [N, 32, 64], ``kernel`` [32, 73], ``weights`` [N].  ``moves``: None for the softmax over the whole
    vocabulary, or (from_squares, move_filters, moves_per_board) for each board's own list.

    Returns a dict of loss, d_features, d_kernel, and
      logit_size   [N]  largest sum over channels of |kernel * features| among the softmax's logits
      spread       [N]  largest difference of its logits from the largest
      top          [N]  the largest logit
      d_features_size, d_kernel_size   sums of |factor| * weight * (softmax + onehot)
    """
    x = np.asarray(features, np.float64).reshape(-1, 32, SQUARES)
    k = np.asarray(kernel, np.float64).reshape(32, FILTERS)
    n = len(x)
    out = {"loss": np.zeros(n), "d_features": np.zeros_like(x), "d_kernel": np.zeros_like(k), "logit_size": np.zeros(n),
           "spread": np.zeros(n), "top": np.zeros(n), "d_features_size": np.zeros_like(x), "d_kernel_size": np.zeros_like(k)}
    starts = None
    if moves is not None:
        sq, fl, per = (np.asarray(a).astype(np.int64) for a in moves)
        starts = np.concatenate([[0], np.cumsum(per)])
    for b in range(n):
        if targets[b] < 0:
            continue
        if moves is None:
            f, s = np.divmod(np.arange(FILTERS * SQUARES), SQUARES)
        else:
            s, f = sq[starts[b]:starts[b + 1]], fl[starts[b]:starts[b + 1]]
        logits = (k.T @ x[b])[f, s]
        out["loss"][b], d, p = _loss_of(logits, int(targets[b]), float(weights[b]))
        size = p * abs(float(weights[b]))
        size[targets[b]] += abs(float(weights[b]))
        for name, v, kk, xx in (("", d, k, x[b]), ("_size", size, np.abs(k), np.abs(x[b]))):
            full = np.zeros((FILTERS, SQUARES))
            np.add.at(full, (f, s), v)
            out["d_features" + name][b] = kk @ full
            out["d_kernel" + name] += xx @ full.T
        out["logit_size"][b] = (np.abs(k).T @ np.abs(x[b]))[f, s].max()
        out["spread"][b] = logits.max() - logits.min()
        out["top"][b] = abs(logits.max())
    return out


def clip_grad_norm(tensors, max_norm):
    """(norm, scaled tensors), all float64."""
    arrays = [np.asarray(t, np.float64) for t in tensors]
    norm = np.sqrt(sum(float(np.sum(a * a)) for a in arrays))
    with np.errstate(invalid="ignore"):
        return norm, [a * min(1.0, max_norm / (norm + 1e-6)) for a in arrays]
