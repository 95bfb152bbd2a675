"""Plain statements, in 64 bits, of the operators for a field of several experts (numpy, loops where loops are clearest)."""
import numpy as np
import torch

TORCH = {0: torch.float16, 1: torch.bfloat16, 2: torch.float32}
NAMES = {0: "f16", 1: "bf16", 2: "f32"}
TINY = {0: 2.0 ** -25, 1: 0.0, 2: 0.0}   # half of f16's smallest step: values below its normal range round absolutely


def half_step(dtype):
    """A rounding to the type is off by at most this share of the value."""
    return torch.finfo(TORCH[dtype]).eps / 2


def plan(ids, n_experts):
    """offsets, order, slot of a stable sort by expert; ids outside [0, n_experts) are dropped."""
    flat = np.asarray(ids, np.int64).reshape(-1)
    kept = np.flatnonzero((flat >= 0) & (flat < n_experts))
    by = kept[np.argsort(flat[kept], kind="stable")]
    offsets = np.zeros(n_experts + 1, np.int32)
    offsets[1:] = np.cumsum(np.bincount(flat[kept], minlength=n_experts))
    order = np.full(flat.size, -1, np.int32)
    order[: by.size] = by
    slot = np.full(flat.size, -1, np.int32)
    slot[by] = np.arange(by.size)
    return offsets, order, slot.reshape(np.asarray(ids).shape)


def combine(rows, weights, slot):
    """(sum, sum of magnitudes) per element"""
    n, k = slot.shape
    y = np.zeros((n, rows.shape[1]))
    size = np.zeros_like(y)
    for j in range(k):
        t = np.flatnonzero(slot[:, j] >= 0)
        part = rows[slot[t, j]].astype(np.float64) * (1.0 if weights is None else weights[t, j, None].astype(np.float64))
        y[t] += part
        size[t] += np.abs(part)
    return y, size


def combine_grad(dy, rows, weights, slot, drows):
    """drows (rows of no choice as given), dweights, and the magnitudes' sums of the latter"""
    n, k = slot.shape
    d = drows.astype(np.float64).copy()
    dw, size = np.zeros((n, k)), np.zeros((n, k))
    for j in range(k):
        t = np.flatnonzero(slot[:, j] >= 0)
        g = dy[t].astype(np.float64)
        d[slot[t, j]] = g * (1.0 if weights is None else weights[t, j, None].astype(np.float64))
        prod = g * rows[slot[t, j]].astype(np.float64)
        dw[t, j], size[t, j] = prod.sum(1), np.abs(prod).sum(1)
    return d, dw, size


def quantize(x):
    """(q int, scale f32) of f32 rows: the quotient 127 x / a is exact enough in 64 bits that its rounding is the definition's."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(1)
    top = np.abs(np.where(bad[:, None], np.float32(0), x)).max(1)
    a = np.maximum(top, np.float32(2.0 ** -100)).astype(np.float32)
    q = np.rint(127.0 * np.where(bad[:, None], 0.0, x).astype(np.float64) / a.astype(np.float64)[:, None]).astype(np.int64)
    scale = (a / np.float32(127)).astype(np.float32)
    return q, np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def linear(q, scale, w, w_scale, bias, relu):
    """(y, the magnitude before the bias plus the bias's) in 64 bits: q [r][k], w [c][k] whole numbers"""
    acc = np.matmul(q.astype(np.float64), w.astype(np.float64).T)   # whole numbers below 2^53: exact
    p = acc * scale.astype(np.float64)[:, None] * w_scale.astype(np.float64)[None]
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    y = p + b
    size = np.abs(p) + np.abs(b)
    return (np.where(y < 0, 0.0, y) if relu else y), size
