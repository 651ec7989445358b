"""The operators of a transformer's token-wise half, in training and in answering, as plain cases: layer normalisation, the gated dense layer and
the softmax cross entropy over a large vocabulary, each with its gradients.

A case names an operator and its sizes:

  norm_forward    layerNormForward: every row normalised, scaled and shifted
  norm_backward   layerNormBackward: the gradient of the rows, and the sums over all rows that are the gradients of scale and shift
  gated_forward   gatedDenseForward: y = a(x Wg^T + bg) * (x Wu^T + bu); `keep`: the two projections are returned for the backward pass
  gated_backward  gatedDenseBackward: gradients of x, of both weights and of both biases from the projections that were kept
  loss            linearCrossEntropyForward: -log softmax(x W^T + b)[target] of every row, with the logarithm of the softmax's sum
  loss_gradient   the same, then linearCrossEntropyBackward: gradients of x, of W and of b

`own` chooses between elementary torch operations and the calls of minml_amd.
"""
import math

import torch

own = False

EPSILON = 1e-5
SIZE = {"float16": 2, "float32": 4}
TYPE = {"float16": torch.float16, "float32": torch.float32}
DEVICE = "cuda:0"


def listed():
    return [
        # one position of 15x15 in a network of 256 channels: the latency of a search that evaluates positions one by one
        dict(name="norm_forward_board", kind="norm_forward", dtype="float16", rows=225, columns=256),
        # 256 positions at once, self-play
        dict(name="norm_forward_batch", kind="norm_forward", dtype="float16", rows=57600, columns=256),
        # a training step of a wide model
        dict(name="norm_backward_wide", kind="norm_backward", dtype="float16", rows=16384, columns=4096),
        # full precision, rows that end anywhere
        dict(name="norm_backward_ragged", kind="norm_backward", dtype="float32", rows=7001, columns=1001),
        # one token is answered: the weights are read for a single row
        dict(name="gated_forward_token", kind="gated_forward", dtype="float16", rows=1, columns=4096, hidden=8192, gate="silu", keep=False),
        # the feed-forward half of the hybrid networks on 256 positions, in training
        dict(name="gated_forward_batch", kind="gated_forward", dtype="float16", rows=57600, columns=256, hidden=1024, gate="gelu", keep=True),
        # a training step of a wider model
        dict(name="gated_backward_wide", kind="gated_backward", dtype="float16", rows=8192, columns=2048, hidden=5504, gate="silu"),
        # full precision, no size a multiple of anything
        dict(name="gated_backward_ragged", kind="gated_backward", dtype="float32", rows=1111, columns=1000, hidden=2731, gate="sigmoid"),
        # the likelihood of a few given tokens: the vocabulary's matrix is read for them alone
        dict(name="loss_few", kind="loss", dtype="float16", rows=7, columns=2048, classes=65536),
        # the evaluation of a validation batch, a vocabulary of any size
        dict(name="loss_batch", kind="loss", dtype="float16", rows=4096, columns=1024, classes=50001),
        # a training step over a large vocabulary
        dict(name="loss_gradient_wide", kind="loss_gradient", dtype="float16", rows=4096, columns=2048, classes=65536),
        # full precision, ragged
        dict(name="loss_gradient_ragged", kind="loss_gradient", dtype="float32", rows=901, columns=520, classes=10007),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A row's length: mostly a multiple of 8 elements, sometimes any number."""
    n = _log_int(rng, low, high)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    """A case of the same ranges: one row to those of a full batch, narrow networks to wide ones, any length among them."""
    kind = rng.choice(("norm_forward", "norm_backward", "gated_forward", "gated_backward", "loss", "loss_gradient"))
    case = dict(kind=kind, dtype=rng.choice(("float16", "float16", "float32")), rows=_log_int(rng, 1, 65536))
    if kind.startswith("norm"):
        case["columns"] = _width(rng, 16, 16384)
    else:
        case["columns"] = _width(rng, 32, 4096)
        if kind.startswith("gated"):
            case["hidden"] = _width(rng, 32, 8192)
            case["gate"] = rng.choice(("sigmoid", "relu", "silu", "gelu"))
            if kind == "gated_forward":
                case["keep"] = case["rows"] > 64 and rng.random() < 0.5
        else:
            case["rows"] = _log_int(rng, 1, 8192)
            case["classes"] = _log_int(rng, 300, 131072)
    # no dearer than the largest listed case; products of full precision are counted at a sixteenth of the rate
    limit = {"norm": work(listed()[2]), "gate": work(listed()[6]), "loss": work(listed()[10])}[kind[:4]]
    slow = 16 if case["dtype"] == "float32" and not kind.startswith("norm") else 1

    def dear():
        w = work(case)
        return w["flops"] * slow > limit["flops"] or w["bytes"] > limit["bytes"]

    while dear() and case["rows"] > 1:
        case["rows"] = max(1, case["rows"] * 2 // 3)
    while dear():
        name = "classes" if "classes" in case else "hidden" if "hidden" in case else "columns"
        case[name] = max(32, case[name] * 2 // 3)
    return case


# ---- what a program has in hand -------------------------------------------------------------------------------------------------

def prepare(case, seed):
    draws = torch.Generator(device=DEVICE)
    draws.manual_seed(seed)
    dtype, rows, columns, kind = TYPE[case["dtype"]], case["rows"], case["columns"], case["kind"]

    def normal(*shape, sigma=1.0, mean=0.0):
        return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(mean, sigma, generator=draws).to(dtype)

    state = {"case": dict(case), "x": normal(rows, columns)}
    if kind.startswith("norm"):
        # a residual stream: channels of different scale about different means
        scale = torch.empty(columns, device=DEVICE).normal_(0, 0.5, generator=draws).exp()
        shift = torch.empty(columns, device=DEVICE).normal_(0, 0.5, generator=draws)
        state["x"] = (state["x"].float() * scale + shift).to(dtype)
        state["w"], state["b"] = normal(columns, sigma=0.1, mean=1.0), normal(columns, sigma=0.1)
        if kind == "norm_backward":
            state["dy"] = normal(rows, columns, sigma=0.1)
    elif kind.startswith("gated"):
        hidden = case["hidden"]
        state["w"], state["b"] = normal(2, hidden, columns, sigma=columns ** -0.5), normal(2, hidden, sigma=0.1)
        if kind == "gated_backward":
            state["projections"] = normal(rows, 2, hidden)  # as the forward pass keeps them: normalised rows give about N(0, 1)
            state["dy"] = normal(rows, hidden, sigma=0.1)
    else:
        classes = case["classes"]
        state["w"], state["b"] = normal(classes, columns, sigma=2 * columns ** -0.5), normal(classes, sigma=0.5)
        targets = torch.randint(0, classes, (rows,), generator=draws, device=DEVICE, dtype=torch.int32)
        padding = torch.rand(rows, generator=draws, device=DEVICE) < 0.05
        state["targets"] = torch.where(padding, torch.full_like(targets, -1), targets)
        if kind == "loss_gradient":  # weights of the tokens, scaled as losses in half precision are
            state["dloss"] = torch.empty(rows, device=DEVICE).uniform_(0.5, 2.0, generator=draws) * 4
    return state


# ---- the plain form -------------------------------------------------------------------------------------------------------------

def _gate(g, gate):
    """a(g) and its derivative."""
    if gate == "relu":
        return torch.clamp(g, min=0), (g > 0).to(g.dtype)
    if gate == "gelu":
        normal = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * normal, normal + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-g))
    if gate == "sigmoid":
        return s, s * (1 - s)
    return g * s, s * (1 + g * (1 - s))


def _norm(x):
    mean = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPSILON)
    return (x - mean) * r, r


def _plain(state):
    case = state["case"]
    kind, dtype = case["kind"], TYPE[case["dtype"]]
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    if kind == "norm_forward":
        return {"y": (_norm(x)[0] * w + b).to(dtype)}
    if kind == "norm_backward":
        dy = state["dy"].float()
        n, r = _norm(x)
        g = dy * w
        dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
        return {"dx": dx.to(dtype), "dw": (dy * n).sum(0).to(dtype), "db": dy.sum(0).to(dtype)}
    if kind == "gated_forward":
        g, u = x @ w[0].T + b[0], x @ w[1].T + b[1]
        out = {"y": (_gate(g, case["gate"])[0] * u).to(dtype)}
        if case["keep"]:
            out["projections"] = torch.stack((g, u), 1).to(dtype)
        return out
    if kind == "gated_backward":
        g, u, dy = state["projections"][:, 0].float(), state["projections"][:, 1].float(), state["dy"].float()
        a, slope = _gate(g, case["gate"])
        d = torch.cat((dy * u * slope, dy * a), 1)
        both = w.reshape(-1, w.shape[2])
        return {"dx": (d @ both).to(dtype), "dw": (d.T @ x).reshape(w.shape).to(dtype), "db": d.sum(0).reshape(b.shape).to(dtype)}
    z = x @ w.T + b
    top = z.max(1, keepdim=True).values
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(1))
    targets = state["targets"].long()
    kept = targets >= 0
    place = torch.clamp(targets, min=0)[:, None]
    loss = torch.where(kept, lse - torch.gather(z, 1, place)[:, 0], torch.zeros_like(lse))
    if kind == "loss":
        return {"loss": loss, "lse": lse}
    weight = torch.where(kept, state["dloss"], torch.zeros_like(lse))[:, None]
    d = torch.exp(z - lse[:, None]) * weight
    d.scatter_add_(1, place, -weight)
    return {"loss": loss, "lse": lse, "dx": (d @ w).to(dtype), "dw": (d.T @ x).to(dtype), "db": d.sum(0).to(dtype)}


# ---- the calls of the framework -------------------------------------------------------------------------------------------------

_context = None


class _Call:
    """One call as a program keeps it: the tensors of its inputs and results, and its workspace."""

    def __init__(self, state):
        from minml_amd import core as ml

        global _context
        if _context is None:
            _context = ml.Context(0)
        self.ml, self.results = ml, {}
        case = state["case"]
        dtype, rows, columns, kind = case["dtype"], case["rows"], case["columns"], case["kind"]
        for name in ("x", "w", "b", "dy", "projections", "targets", "dloss"):
            if name in state:
                setattr(self, name, self.over(state[name]))
        if kind == "norm_forward":
            self.y = self.new("y", (rows, columns), dtype)
        elif kind == "norm_backward":
            self.dx, self.dw, self.db = self.new("dx", (rows, columns), dtype), self.new("dw", (columns,), dtype), self.new("db", (columns,), dtype)
            self.space = self.workspace(ml.layerNormGetWorkspaceSize(_context, self.x))
        elif kind == "gated_forward":
            self.y = self.new("y", (rows, case["hidden"]), dtype)
            self.kept = self.new("projections", (rows, 2, case["hidden"]), dtype) if case["keep"] else None
            self.space = self.workspace(ml.gatedDenseGetWorkspaceSize(_context, self.x, self.w, False))
        elif kind == "gated_backward":
            self.dx = self.new("dx", (rows, columns), dtype)
            self.dw, self.db = self.new("dw", self.w.shape, dtype), self.new("db", self.b.shape, dtype)
            self.space = self.workspace(ml.gatedDenseGetWorkspaceSize(_context, self.x, self.w, True))
        else:
            self.loss, self.lse = self.new("loss", (rows,), "float32"), self.new("lse", (rows,), "float32")
            if kind == "loss_gradient":
                self.dx = self.new("dx", (rows, columns), dtype)
                self.dw, self.db = self.new("dw", self.w.shape, dtype), self.new("db", self.b.shape, dtype)
            self.space = self.workspace(ml.linearCrossEntropyGetWorkspaceSize(_context, self.x, self.w, kind == "loss_gradient"))

    def over(self, t):
        name = {torch.float16: "float16", torch.float32: "float32", torch.int32: "int32", torch.uint8: "uint8"}[t.dtype]
        return self.ml.Tensor.over(t.data_ptr(), t.shape, name, 0, t)

    def new(self, name, shape, dtype):
        self.results[name] = torch.empty(shape, dtype=TYPE[dtype], device=DEVICE)
        return self.over(self.results[name])

    def workspace(self, size):
        return self.over(torch.empty((max(size, 1),), dtype=torch.uint8, device=DEVICE))

    def __call__(self, case):
        ml, kind = self.ml, case["kind"]
        if kind == "norm_forward":
            ml.layerNormForward(_context, self.x, self.w, self.b, self.y, EPSILON)
        elif kind == "norm_backward":
            ml.layerNormBackward(_context, self.x, self.w, self.dy, 0.0, self.dx, 0.0, self.dw, self.db, self.space, EPSILON)
        elif kind == "gated_forward":
            ml.gatedDenseForward(_context, self.x, self.w, self.b, self.y, self.kept, case["gate"], self.space)
        elif kind == "gated_backward":
            ml.gatedDenseBackward(_context, self.x, self.w, self.projections, self.dy, 0.0, self.dx, 0.0, self.dw, self.db, case["gate"], self.space)
        else:
            ml.linearCrossEntropyForward(_context, self.x, self.w, self.b, self.targets, self.loss, self.lse, self.space)
            if kind == "loss_gradient":
                ml.linearCrossEntropyBackward(_context, self.x, self.w, self.b, self.targets, self.lse, self.dloss, 0.0, self.dx, 0.0, self.dw, self.db, self.space)
        return self.results


def run(state):
    if not own:
        return _plain(state)
    if "call" not in state:
        state["call"] = _Call(state)
    return state["call"](state["case"])


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    kind = case["kind"]
    if kind.startswith("norm"):
        centred = x - x.sum(1, keepdim=True) / x.shape[1]
        deviation = torch.sqrt(centred.square().sum(1, keepdim=True) / x.shape[1] + EPSILON)
        n = centred / deviation
        if kind == "norm_forward":
            return {"y": n * w + b}
        dy = s["dy"].double()
        # the Jacobian of a row is (1 - 1/C - n n^T / C) / deviation
        g = dy * w
        dx = (g - (g.sum(1, keepdim=True) + n * (g * n).sum(1, keepdim=True)) / x.shape[1]) / deviation
        return {"dx": dx, "dw": torch.einsum("rc,rc->c", dy, n), "db": dy.sum(0)}
    if kind.startswith("gated"):
        gate = case["gate"]
        if kind == "gated_forward":
            p = torch.matmul(x, w.reshape(-1, x.shape[1]).t()).reshape(x.shape[0], 2, -1) + b
        else:
            p = s["projections"].double()
        g, u = p[:, 0], p[:, 1]
        if gate == "relu":
            a, slope = g * (g > 0), (g > 0).double()
        elif gate == "gelu":
            half = 0.5 * torch.erfc(-g / math.sqrt(2.0))
            a, slope = g * half, half + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        else:
            half = torch.sigmoid(g)
            a, slope = (half, half * torch.sigmoid(-g)) if gate == "sigmoid" else (g * half, half + g * half * torch.sigmoid(-g))
        if kind == "gated_forward":
            return {"y": a * u, "projections": p} if case["keep"] else {"y": a * u}
        dy = s["dy"].double()
        dg, du = dy * u * slope, dy * a
        return {"dx": torch.matmul(dg, w[0]) + torch.matmul(du, w[1]), "dw": torch.stack((torch.matmul(dg.t(), x), torch.matmul(du.t(), x))),
                "db": torch.stack((dg.sum(0), du.sum(0)))}
    z = torch.addmm(b, x, w.t())
    lse = torch.logsumexp(z, 1)
    t = s["targets"].long()
    at = torch.nonzero(t >= 0)[:, 0]
    loss = torch.zeros_like(lse)
    loss[at] = lse[at] - z[at, t[at]]
    if kind == "loss":
        return {"loss": loss, "lse": lse}
    d = torch.exp(z - lse[:, None])
    d[at, t[at]] -= 1
    weight = torch.zeros_like(lse)
    weight[at] = s["dloss"].double()[at]
    d *= weight[:, None]
    return {"loss": loss, "lse": lse, "dx": torch.matmul(d, w), "dw": torch.matmul(d.t(), x), "db": d.sum(0)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    """Bytes: inputs and results once each. Flops: the products' (for the loss with its gradient: the logits once, and the two gradients),
    and about what a row's normalisation takes."""
    kind, s, rows, columns = case["kind"], SIZE[case["dtype"]], case["rows"], case["columns"]
    if kind == "norm_forward":
        return {"bytes": float(s * (2 * rows * columns + 2 * columns)), "flops": 8.0 * rows * columns}
    if kind == "norm_backward":
        return {"bytes": float(s * (3 * rows * columns + 3 * columns)), "flops": 14.0 * rows * columns}
    if kind.startswith("gated"):
        hidden = case["hidden"]
        weights = 2 * hidden * columns + 2 * hidden
        if kind == "gated_forward":
            return {"bytes": float(s * (rows * columns + weights + rows * hidden * (3 if case["keep"] else 1))), "flops": 4.0 * rows * columns * hidden}
        return {"bytes": float(s * (2 * rows * columns + 2 * weights + 3 * rows * hidden)), "flops": 8.0 * rows * columns * hidden}
    weights = case["classes"] * (columns + 1)
    if kind == "loss":
        return {"bytes": float(s * (rows * columns + weights) + 12 * rows), "flops": 2.0 * rows * columns * case["classes"]}
    return {"bytes": float(2 * s * (rows * columns + weights) + 16 * rows), "flops": 6.0 * rows * columns * case["classes"]}
