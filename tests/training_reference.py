"""The operators with a backward pass in 64 bits, straight from their definitions, and bounds of what rounding may do to them."""
import math

import numpy as np
from scipy.special import erf, expit

STEP = {"float16": 2.0 ** -11, "float32": 2.0 ** -24}  # half a step relative to the value: what one rounding to nearest may cost
TINY = {"float16": 2.0 ** -25, "float32": 2.0 ** -150}  # half a step where values are subnormal
FP32 = 2.0 ** -24


def bits(a, dtype):
    """Values -> the storage type, rounded to nearest (fp16 as bit patterns)."""
    a = np.ascontiguousarray(a, np.float32)
    return a.astype(np.float16).view(np.uint16) if dtype == "float16" else a


def numbers(a):
    a = np.asarray(a)
    return (a.view(np.float16) if a.dtype == np.uint16 else a).astype(np.float64)


def rounded(value, dtype):
    """What rounding `value` to the type once may add."""
    return STEP[dtype] * np.abs(value) + TINY[dtype]


def norm(x, epsilon):
    mean = x.mean(-1, keepdims=True)
    r = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + epsilon)
    return (x - mean) * r, r, mean


def layer_norm(x, w, b, epsilon):
    return norm(x, epsilon)[0] * w + b


def layer_norm_gradients(x, w, dy, epsilon):
    n, r, _ = norm(x, epsilon)
    g = dy * w
    return r * (g - g.mean(-1, keepdims=True) - n * (g * n).mean(-1, keepdims=True)), (dy * n).sum(0), dy.sum(0)


def norm_error(x, epsilon):
    """How far n may be off in 32 bits. A sum of C values goes through at most 16 additions in a thread, 6 in a wavefront and 16 across wavefronts, and a division: below 40 roundings of
    the mean of |x|; n takes that over r, and its own three operations and half the relative error of the variance, below 50 roundings together."""
    n, r, _ = norm(x, epsilon)
    length = 40 + x.shape[-1] / 256  # rows that do not fit the registers are summed by 256 threads
    off = length * FP32 * np.abs(x).mean(-1, keepdims=True) * r
    return off * (1 + np.abs(n)) + (10 + length) * FP32 * (np.abs(n) + 1)


def layer_norm_bound(x, w, b, epsilon, dtype):
    y = layer_norm(x, w, b, epsilon)
    return rounded(y, dtype) + np.abs(w) * norm_error(x, epsilon) + 2 * FP32 * (np.abs(y) + np.abs(b))


def layer_norm_gradient_bounds(x, w, dy, epsilon, dtype):
    n, r, _ = norm(x, epsilon)
    off = norm_error(x, epsilon)
    g = np.abs(dy * w)
    dx, dw, db = layer_norm_gradients(x, w, dy, epsilon)
    length = 60 + x.shape[-1] / 256
    mean_g, mean_gn = g.mean(-1, keepdims=True), (g * np.abs(n)).mean(-1, keepdims=True)
    # r is off by as much as n relative to itself; each mean by `length` roundings and by what n is off
    relative = off.max(-1, keepdims=True)
    dx_off = r * ((relative + length * FP32) * (g + mean_g + np.abs(n) * mean_gn) + off * mean_gn + np.abs(n) * (g * off).mean(-1, keepdims=True))
    # rows are added one after another in a thread, then over the workgroups: never more additions than rows, and 80 where they meet
    adds = (x.shape[0] + 80) * FP32
    return rounded(dx, dtype) + dx_off, rounded(dw, dtype) + adds * np.abs(dy * n).sum(0) + (np.abs(dy) * off).sum(0), rounded(db, dtype) + adds * np.abs(dy).sum(0)


GATES = ("sigmoid", "relu", "silu", "gelu")
# what the gates' functions may be off by, relative to 1 + |g| of their argument: a few steps of 2^-24, and in fp16 the hardware's exponential, whose argument is rounded too
GATE_ERROR = {"float16": 2.0 ** -19, "float32": 2.0 ** -21}


def gate(g, name):
    """a(g) and its derivative."""
    if name == "relu":
        return np.maximum(g, 0), (g > 0).astype(float)
    if name == "gelu":
        p = 0.5 * (1 + erf(g / math.sqrt(2)))
        return g * p, p + g * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = expit(g)
    return (s, s * (1 - s)) if name == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def product_error(a, b, dtype):
    """How far a @ b may be off when it is summed in 32 bits: an instruction adds 16 (fp16) or 2 (fp32) products to a sum, its own additions and the sum's may be cut off instead of rounded
    (2^-23 each); at most 16 of them inside, 8 where partial sums meet."""
    steps = a.shape[-1] / (16 if dtype == "float16" else 2) + 24
    return steps * 2 * FP32 * (np.abs(a) @ np.abs(b))


def gated(x, w, b, name):
    """y and the projections [rows, 2, hidden]."""
    p = np.stack((x @ w[0].T + b[0], x @ w[1].T + b[1]), 1)
    return gate(p[:, 0], name)[0] * p[:, 1], p


def gated_bounds(x, w, b, name, dtype):
    y, p = gated(x, w, b, name)
    off = np.stack((product_error(x, w[0].T, dtype), product_error(x, w[1].T, dtype)), 1) + FP32 * np.abs(p)
    a = gate(p[:, 0], name)[0]
    off_a = 1.2 * off[:, 0] + GATE_ERROR[dtype] * (1 + np.abs(p[:, 0]))  # no gate is steeper than 1.13
    return rounded(y, dtype) + off_a * (np.abs(p[:, 1]) + off[:, 1]) + np.abs(a) * off[:, 1] + FP32 * np.abs(y), rounded(p, dtype) + off


def gated_gradients(x, w, p, dy, name):
    a, slope = gate(p[:, 0], name)
    d = np.concatenate((dy * p[:, 1] * slope, dy * a), 1)
    return d @ w.reshape(-1, w.shape[2]), (d.T @ x).reshape(w.shape), d.sum(0).reshape(2, -1)


def gated_gradient_bounds(x, w, p, dy, name, dtype):
    a, slope = gate(p[:, 0], name)
    d = np.concatenate((dy * p[:, 1] * slope, dy * a), 1)
    off = np.concatenate((np.abs(dy * p[:, 1]) * (1 + np.abs(p[:, 0])), np.abs(dy) * (1 + np.abs(p[:, 0]))), 1) * 2 * GATE_ERROR[dtype] + 2 * FP32 * np.abs(d)
    stored = off + rounded(d, dtype)  # d goes to memory in the tensors' type
    dx, dw, db = gated_gradients(x, w, p, dy, name)
    flat = w.reshape(-1, w.shape[2])
    return (rounded(dx, dtype) + product_error(d, flat, dtype) + stored @ np.abs(flat),
            rounded(dw, dtype) + (product_error(d.T, x, dtype) + stored.T @ np.abs(x)).reshape(w.shape),
            rounded(db, dtype) + (off.sum(0) + (x.shape[0] + 80) * FP32 * np.abs(d).sum(0)).reshape(2, -1))


def cross_entropy(x, w, b, targets):
    """loss, lse and the logits; targets that are no class have loss 0."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        z = x @ w.T + b
        top = z.max(1, keepdims=True)
        lse = np.where(np.isfinite(top[:, 0]), top[:, 0] + np.log(np.exp(z - top).sum(1)), top[:, 0])
        kept = (targets >= 0) & (targets < w.shape[0])
        loss = np.where(kept, lse - z[np.arange(len(z)), np.where(kept, targets, 0)], 0.0)
    return loss, lse, z


def logit_error(x, w, z, dtype):
    return product_error(x, w.T, dtype) + FP32 * np.abs(z)


def cross_entropy_bounds(x, w, b, targets, dtype):
    """A logarithm of sums is off by the largest error of a logit; by its exponentials, (|z - top| + 2) 2^-22 relative each, where those with |z - top| > 40 are nothing beside the largest; and by less than 200
    additions."""
    loss, lse, z = cross_entropy(x, w, b, targets)
    off = logit_error(x, w, z, dtype)
    off_lse = off.max(1) + 42 * 2.0 ** -22 + 200 * FP32 + 2 * FP32 * np.abs(lse)
    return off_lse + off.max(1) + FP32 * np.abs(loss), off_lse


def cross_entropy_gradients(x, w, b, targets, dloss, lse=None):
    z = cross_entropy(x, w, b, targets)
    p = np.exp(z[2] - (z[1] if lse is None else lse)[:, None])
    kept = (targets >= 0) & (targets < w.shape[0])
    d = p * np.where(kept, dloss, 0)[:, None]
    at = np.nonzero(kept)[0]
    d[at, targets[at]] -= dloss[at]
    return d @ w, d.T @ x, d.sum(0)


def cross_entropy_gradient_bounds(x, w, b, targets, dloss, dtype):
    loss, lse, z = cross_entropy(x, w, b, targets)
    kept = (targets >= 0) & (targets < w.shape[0])
    weight = np.where(kept, np.abs(dloss), 0)[:, None]
    about = z - lse[:, None]
    p = np.exp(about)
    # the exponent is off by the logit's error, the lse's and its own rounding
    exponent = logit_error(x, w, z, dtype) + cross_entropy_bounds(x, w, b, targets, dtype)[1][:, None] + (np.abs(about) + 4) * 2.0 ** -22
    off = weight * (p * np.expm1(np.minimum(exponent, 1)) + 2 * FP32 * (p + 1e-30))
    d = p * weight
    at = np.nonzero(kept)[0]
    d[at, targets[at]] = np.abs(d[at, targets[at]] - np.abs(dloss[at]))
    off[at, targets[at]] += 2 * FP32 * np.abs(dloss[at])
    # d is kept in the tensors' type, times 2^15 over a power of two that is at most twice the largest |dloss|
    stored = off + STEP[dtype] * d + TINY[dtype] * 2.0 ** -14 * weight.max(initial=0)
    dx, dw, db = cross_entropy_gradients(x, w, b, targets, dloss)
    return (rounded(dx, dtype) + product_error(d, w, dtype) + stored @ np.abs(w), rounded(dw, dtype) + product_error(d.T, x, dtype) + stored.T @ np.abs(x),
            rounded(db, dtype) + off.sum(0) + (x.shape[0] + 80) * FP32 * d.sum(0))


def worst(got, want, bound):
    """The largest error in units of its bound; places that are not finite have to be the same. What rounds to more than fp16's largest value, 65504, is an infinity there: from half a step beyond, 65520,
    on; within the bound of that place either is right."""
    if np.asarray(got).dtype == np.uint16:
        over, near = np.abs(want) >= 65520, np.abs(np.abs(want) - 65520) <= bound
        want = np.where(over, np.copysign(np.inf, want), want)
        want = np.where(near & np.isinf(numbers(got)), numbers(got), want)
    got, want, bound = np.broadcast_arrays(numbers(got), want, bound)
    if not want.size:
        return 0.0
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    ratio = np.abs(got[finite] - want[finite]) / bound[finite]
    return float(ratio.max()) if ratio.size else 0.0
