"""What a model over a vocabulary learns from, in 64 bits and straight from the definitions, and bounds of what rounding may do to it."""
import numpy as np

from minml_amd import core as ml
from training_reference import FP32, STEP, TINY, product_error, rounded


def workspace(ctx, size):
    """A workspace of `size` bytes that holds NaN in both types (nothing may be read before it was written), with as much behind it as tells whether a call kept to it."""
    return ml.toDevice(ctx, np.full(size + 4096, 0xff, np.uint8)).view((max(1, size),))


def check_workspace(ctx, space):
    assert (space._owner.copyToHost(ctx)[-4095:] == 0xff).all()


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


def teacher(classes, logits, total, temperature):
    """The teacher's distribution over all classes [rows, total], that of every place [rows, count], and which places count."""
    kept = (classes >= 0) & (classes < total) & ~np.isneginf(logits)
    with np.errstate(invalid="ignore", over="ignore"):
        v = np.where(kept, logits / temperature, -np.inf)
        top = v.max(1, keepdims=True)
        q = np.where(kept, np.exp(v - np.where(np.isfinite(top), top, 0)), 0)
    q = q / np.where(kept.any(1), q.sum(1), 1)[:, None]
    dense = np.zeros((len(classes), total))
    np.add.at(dense, (np.nonzero(kept)[0], classes[kept]), q[kept])
    return dense, q, kept


def distillation(x, w, b, classes, logits, temperature):
    """loss, lse, log p at the teacher's classes, and the scaled logits."""
    z = (x @ w.T + b) / temperature
    top = z.max(1, keepdims=True)
    lse = top[:, 0] + np.log(np.exp(z - top).sum(1))
    dense, _, kept = teacher(classes, logits, len(w), temperature)
    log_p = z - lse[:, None]
    loss = np.where(dense > 0, dense * (np.log(np.where(dense > 0, dense, 1)) - log_p), 0).sum(1)
    return loss, lse, np.where(kept, np.take_along_axis(log_p, np.where(kept, classes, 0), 1), 0), z


def share_error(classes, logits, total, temperature):
    """How far a probability of the teacher may be off, relative to it: the exponent's two numbers are rounded, the exponential is a step off, then a sum of `count` and a division."""
    _, _, kept = teacher(classes, logits, total, temperature)
    return FP32 * (4 * np.abs(np.where(kept, logits, 0) / temperature).max(1) + 24 + classes.shape[1] / 32)


def scaled_logit_error(x, w, b, z, temperature, dtype):
    return (product_error(x, w.T, dtype) + FP32 * np.abs(temperature * z)) / temperature + 3 * FP32 * np.abs(z)


def distillation_bounds(x, w, b, classes, logits, temperature, dtype):
    """As the cross entropy's; the loss is a mean over the teacher's probabilities, whose own errors it takes times what they weigh."""
    loss, lse, log_p, z = distillation(x, w, b, classes, logits, temperature)
    dense, q, kept = teacher(classes, logits, len(w), temperature)
    off = scaled_logit_error(x, w, b, z, temperature, dtype)
    off_lse = off.max(1) + 42 * 2.0 ** -22 + 200 * FP32 + 2 * FP32 * np.abs(lse)
    off_p = np.where(kept, np.take_along_axis(off, np.where(kept, classes, 0), 1) + off_lse[:, None] + FP32 * np.abs(log_p), 0)
    log_q = np.log(np.where(dense > 0, dense, 1))
    weighed = dense * (np.abs(log_q) + np.abs(z - lse[:, None]))
    relative = share_error(classes, logits, len(w), temperature)
    return (q * off_p).sum(1) + (relative + (classes.shape[1] / 32 + 20) * FP32) * (weighed.sum(1) + 1) + FP32 * np.abs(loss), off_lse, off_p


def distillation_gradients(x, w, b, classes, logits, temperature, dloss):
    z, lse = distillation(x, w, b, classes, logits, temperature)[3], distillation(x, w, b, classes, logits, temperature)[1]
    dense, _, kept = teacher(classes, logits, len(w), temperature)
    d = (np.exp(z - lse[:, None]) - dense) * np.where(kept.any(1), dloss, 0)[:, None] / temperature
    return d @ w, d.T @ x, d.sum(0)


def common_row(w, classes, logits):
    """The mean of up to 64 of the rows of W that the teacher names, by one of four places of 256 each."""
    named, places = np.where(np.isneginf(logits), -1, classes).reshape(-1), min(classes.size, 256)
    named = named[np.arange(places) * classes.size // places]
    named = np.pad(np.where((named >= 0) & (named < len(w)), named, -1), (0, 256 - places), constant_values=-1).reshape(4, 64)
    named = named[(named >= 0).argmax(0), np.arange(64)]
    return w[named[named >= 0]].mean(0) if (named >= 0).any() else None


def distillation_gradient_bounds(x, w, b, classes, logits, temperature, dloss, dtype):
    """dx in fp16: e_j is what rounding takes from d_j. For a, the class with the teacher's largest share, it is given back to W_a, for all others to c, the common row, or to W_a where no row is common. So dx is off by the
    sum over j other than a of e_j (W_j - c), by |e_j| (|W_j| + |c|) for each of them at most: the sums of d's errors with |W|, and their sum for the row times |c|."""
    _, lse, _, z = distillation(x, w, b, classes, logits, temperature)
    dense, _, kept = teacher(classes, logits, len(w), temperature)
    weight = np.where(kept.any(1), np.abs(dloss), 0)[:, None] / temperature
    about = z - lse[:, None]
    p = np.exp(about)
    exponent = scaled_logit_error(x, w, b, z, temperature, dtype) + distillation_bounds(x, w, b, classes, logits, temperature, dtype)[1][:, None] + (np.abs(about) + 4) * 2.0 ** -22
    off = weight * (p * np.expm1(np.minimum(exponent, 1)) + 4 * FP32 * (p + 1e-30) + dense * (share_error(classes, logits, len(w), temperature)[:, None] + 4 * FP32))
    d = np.abs(p - dense) * weight
    # d is kept in the tensors' type, times 2^15 over a power of two that is at most twice the largest |dloss|
    stored = off + STEP[dtype] * d + TINY[dtype] * 2.0 ** -14 * weight.max(initial=0)
    common = common_row(w, classes, logits)
    given_back = stored.sum(1, keepdims=True) * np.abs(w[dense.argmax(1)] if common is None else common) if dtype == "float16" else 0
    dx, dw, db = distillation_gradients(x, w, b, classes, logits, temperature, dloss)
    return (rounded(dx, dtype) + product_error(d, w, dtype) + stored @ np.abs(w) + given_back, rounded(dw, dtype) + product_error(d.T, x, dtype) + stored.T @ np.abs(x),
            rounded(db, dtype) + off.sum(0) + (x.shape[0] + 80) * FP32 * (weight * (p + dense)).sum(0))


def spacing(v):
    """From an fp16 number's size to the next."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -14))) - 10)


def distillation_input_noise(x, w, b, classes, logits, temperature, dloss):
    """The 2-norm that the error of dx in fp16 has where roundings are as good as random, evenly over a spacing, whose mean square is a twelfth: of every element of d but the largest share's, times W_j - c, and of dx."""
    dense, _, kept = teacher(classes, logits, len(w), temperature)
    _, lse, _, z = distillation(x, w, b, classes, logits, temperature)
    scale = 2.0 ** 15
    d = (np.exp(z - lse[:, None]) - dense) * np.where(kept.any(1), dloss, 0)[:, None] / temperature
    squares = (spacing(d * scale) / scale) ** 2
    squares[np.arange(len(d)), dense.argmax(1)] = 0
    squares[~kept.any(1)] = 0
    common = common_row(w, classes, logits)
    to = w[dense.argmax(1)] if common is None else np.broadcast_to(common, x.shape)
    away = (w ** 2).sum(1) - 2 * to @ w.T + (to ** 2).sum(1)[:, None]
    return np.sqrt(((squares * away).sum() + (spacing(d @ w) ** 2).sum()) / 12)
