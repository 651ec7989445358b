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


def worst(got, want, bound):
    """The largest error in units of its bound, and where; places that are not finite have to be the same."""
    got, want, bound = np.broadcast_arrays(numbers(got), want, bound)
    if not want.size:
        return 0.0
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    ratio = np.abs(got[finite] - want[finite]) / bound[finite]
    return float(ratio.max()) if ratio.size else 0.0
