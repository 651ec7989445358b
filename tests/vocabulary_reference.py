"""What a model over a vocabulary learns from, in 64 bits and straight from the definitions, and bounds of what rounding may do to it."""
import numpy as np

from training_reference import FP32, rounded


def embedding(tokens, table, scale):
    kept = (tokens >= 0) & (tokens < len(table))
    y = scale * table[np.where(kept, tokens, 0)]
    y[~kept] = 0
    return y


def embedding_bound(y, dtype):
    """One product in 32 bits, then the result's type."""
    return rounded(y, dtype) + rounded(y, "float32")


def embedding_gradient(tokens, dy, classes, scale):
    kept = (tokens >= 0) & (tokens < classes)
    total, size = np.zeros((classes, dy.shape[-1])), np.zeros((classes, dy.shape[-1]))
    np.add.at(total, tokens[kept], dy[kept])
    np.add.at(size, tokens[kept], np.abs(dy[kept]))
    counts = np.bincount(tokens[kept], minlength=classes)[:, None]
    return scale * total, abs(scale) * size * counts


def embedding_gradient_bound(gradient, weighted, old, dtype):
    """n rows of one class go through n - 1 additions in 32 bits at most, whatever their order; then the scale, what is added to, and the result's type."""
    return rounded(gradient + old, dtype) + FP32 * weighted + 3 * (rounded(gradient, "float32") + rounded(old, "float32"))


def policy(nll, old, reference, advantages, targets, classes, clip, kl_weight, average):
    """loss [4], weights [sequences], gradient of nll for a dloss of 1, and bounds of the three."""
    low, high = 1 - clip[0], 1 + clip[1]
    kept = (targets >= 0) & (targets < classes)
    a = np.broadcast_to(advantages if advantages.ndim == 2 else advantages[:, None], nll.shape)
    pick = lambda t: np.where(kept, t, 0.0)
    d, a, q = pick(old - nll), pick(a), pick(nll - reference) if reference is not None else np.zeros(nll.shape)
    r = np.exp(d)
    free, held = r * a, np.clip(r, low, high) * a
    clipped = free > held
    gain = np.minimum(free, held)
    kl, slope = np.expm1(q) - q, np.expm1(q)
    count = kept.sum(1)
    if average == "tokens":
        weights = (count > 0) / max(1, count.sum())
    else:
        weights = np.where(count > 0, 1 / np.maximum(count, 1), 0.0) / max(1, (count > 0).sum())
    each = weights[:, None] * kept
    mean = lambda t: (each * t).sum()
    parts = np.array([kl_weight * mean(kl) - mean(gain), -mean(gain), mean(kl), mean(clipped)])
    gradient = each * (np.where(clipped, 0, free) + kl_weight * slope)
    # the exponent is rounded once, the exponential is a step off, the product half of one
    gain_off = (np.abs(d) + 6) * FP32 * np.abs(free)
    # near zero a series of eight terms whose rounding counts less and less, about ten steps; else an exponential from which larger numbers are taken
    close = np.abs(q) < 0.5
    kl_off = np.where(close, 12 * FP32 * kl, FP32 * ((np.abs(q) + 4) * np.exp(q) + 2 * np.abs(q) + 2))
    slope_off = np.where(close, 12 * FP32 * np.abs(slope), FP32 * ((np.abs(q) + 4) * np.exp(q) + 2))
    off = np.array([mean(gain_off) + kl_weight * mean(kl_off), mean(gain_off), mean(kl_off), 0.0])
    size = np.array([abs(parts[1]) + kl_weight * parts[2]] + [abs(v) for v in parts[1:]])
    gradient_off = each * (gain_off + kl_weight * slope_off) + 6 * FP32 * each * (np.abs(free) + kl_weight * np.abs(slope))
    return (parts, weights, gradient), (off + 4 * FP32 * size + 1e-14, 2 * FP32 * weights, gradient_off + 2.0 ** -140)
