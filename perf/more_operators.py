"""What a model over a vocabulary learns from, beside the cross entropy of given tokens, as plain cases: the embedding it begins with and its gradient, the distillation of a teacher's top
logits into its last dense layer, and the clipped policy loss over the likelihoods of sampled tokens.

A case names an operator and its sizes:

  embed            embeddingForward: y = scale * table[token]; a token that is none of the table's gives zeros
  embed_gradient   embeddingBackward: the table's gradient, rows of equal tokens added up
  distil           linearDistillationForward: for every row the divergence of softmax((x W^T + b) / t) from the softmax of the teacher's logits / t over the classes the teacher gives for it
  distil_gradient  the same, then linearDistillationBackward: gradients of x, of W and of b
  policy           policyLossForward: the mean over tokens of -min(r A, clip(r) A) + kl_weight * KL, with r = exp(old - nll) and the estimate KL = exp(q) - q - 1, q = nll - reference
  policy_gradient  the same, then policyLossBackward: the gradient of every token's nll

`own` chooses between elementary torch operations and the calls of minml_amd.
"""
import math

import torch

own = False

SIZE = {"float16": 2, "float32": 4}
TYPE = {"float16": torch.float16, "float32": torch.float32}
DEVICE = "cuda:0"


def listed():
    return [
        # one token is answered: its row of the table
        dict(name="embed_token", kind="embed", dtype="float16", rows=1, columns=4096, classes=65536),
        # 256 positions of 15x15, every point a token of one of 400 patterns, in a network of 256 channels
        dict(name="embed_board", kind="embed", dtype="float16", rows=57600, columns=256, classes=400),
        # a training step of a wide model over a large vocabulary; a few tokens are in every line of text
        dict(name="embed_gradient_wide", kind="embed_gradient", dtype="float16", rows=16384, columns=4096, classes=65536),
        # a training step on positions: few rows of the table, each used hundreds of times
        dict(name="embed_gradient_board", kind="embed_gradient", dtype="float16", rows=57600, columns=256, classes=400),
        # full precision, rows that end anywhere
        dict(name="embed_gradient_ragged", kind="embed_gradient", dtype="float32", rows=20011, columns=1001, classes=5003),
        # how far a handful of tokens is from the teacher: the vocabulary's matrix is read for them alone
        dict(name="distil_few", kind="distil", dtype="float16", rows=3, columns=1024, classes=32000, top=16),
        # the evaluation of a validation batch
        dict(name="distil_batch", kind="distil", dtype="float16", rows=2048, columns=1024, classes=50001, top=32),
        # a training step over a large vocabulary
        dict(name="distil_gradient_wide", kind="distil_gradient", dtype="float16", rows=4096, columns=2048, classes=65536, top=64),
        # full precision, no size a multiple of anything
        dict(name="distil_gradient_ragged", kind="distil_gradient", dtype="float32", rows=701, columns=520, classes=10007, top=21),
        # a few games, one move at a time: the latency of an update
        dict(name="policy_few", kind="policy_gradient", sequences=4, length=113, average="sequences", per_token=False, reference=True),
        # the check of a batch of answers before its update
        dict(name="policy_batch", kind="policy", sequences=512, length=1024, average="tokens", per_token=False, reference=True),
        # an update on a large batch of long answers with an advantage of its own for every token
        dict(name="policy_gradient_long", kind="policy_gradient", sequences=1024, length=8191, average="tokens", per_token=True, reference=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A row's length: mostly a multiple of 8 elements, sometimes any number."""
    n = _log_int(rng, low, high)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    """A case of the same ranges: one row to those of a full batch, narrow tables to wide ones, any length among them."""
    kind = rng.choice(("embed", "embed_gradient", "distil", "distil_gradient", "policy", "policy_gradient"))
    case = dict(kind=kind)
    if kind.startswith("policy"):
        case.update(sequences=_log_int(rng, 1, 4096), length=_log_int(rng, 1, 16384), average=rng.choice(("tokens", "sequences")), per_token=rng.random() < 0.5, reference=rng.random() < 0.7)
        limit = listed()[11]
        while case["sequences"] * case["length"] > limit["sequences"] * limit["length"]:
            name = "sequences" if case["sequences"] > 1 and rng.random() < 0.5 else "length"
            case[name] = max(1, case[name] * 2 // 3)
        return case
    case["dtype"] = rng.choice(("float16", "float16", "float32"))
    if kind.startswith("embed"):
        case.update(rows=_log_int(rng, 1, 65536), columns=_width(rng, 16, 8192), classes=_log_int(rng, 2, 131072))
        limit = work(listed()[2])
    else:
        case.update(rows=_log_int(rng, 1, 8192), columns=_width(rng, 32, 4096), classes=_log_int(rng, 300, 131072), top=_log_int(rng, 1, 128))
        limit = work(listed()[7])
    # no dearer than the largest listed case; products of full precision are counted at a sixteenth of the rate
    slow = 16 if case["dtype"] == "float32" and kind.startswith("distil") else 1

    def dear():
        w = work(case)
        return w["flops"] * slow > limit["flops"] or w["bytes"] > limit["bytes"]

    while dear() and case["rows"] > 1:
        case["rows"] = max(1, case["rows"] * 2 // 3)
    while dear():
        case["classes"] = max(300, case["classes"] * 2 // 3)
        case["columns"] = max(32, case["columns"] * 2 // 3)
    return case


# ---- what a program has in hand -------------------------------------------------------------------------------------------------

TEMPERATURE = 2.0
CLIP = (0.2, 0.28)
KL_WEIGHT = 0.04


def prepare(case, seed):
    draws = torch.Generator(device=DEVICE)
    draws.manual_seed(seed)
    kind = case["kind"]
    state = {"case": dict(case)}

    def normal(*shape, sigma=1.0, mean=0.0):
        return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(mean, sigma, generator=draws)

    def uniform(*shape, low=0.0, high=1.0):
        return torch.empty(shape, dtype=torch.float32, device=DEVICE).uniform_(low, high, generator=draws)

    if kind.startswith("policy"):
        sequences, length = case["sequences"], case["length"]
        # what a model sampled: mostly likely tokens; the model moved a little since, and further from its reference
        old = torch.empty((sequences, length), dtype=torch.float32, device=DEVICE).exponential_(1.0, generator=draws)
        state["old"] = old
        state["nll"] = torch.clamp(old + normal(sequences, length, sigma=0.15), min=0)
        state["reference"] = torch.clamp(old + normal(sequences, length, sigma=0.4), min=0) if case["reference"] else None
        state["advantages"] = normal(sequences, length) if case["per_token"] else normal(sequences)
        # a prompt before and padding behind the sampled tokens; some sequences hold none
        places = torch.arange(length, device=DEVICE)[None]
        begin = (uniform(sequences, 1) * 0.3 * length).int()
        end = begin + (uniform(sequences, 1) * 1.1 * (length + 1)).int()
        targets = torch.randint(0, 50000, (sequences, length), generator=draws, device=DEVICE, dtype=torch.int32)
        state["targets"] = torch.where((places >= begin) & (places < end), targets, torch.full_like(targets, -1))
        state["dloss"] = torch.full((1,), 1024.0, device=DEVICE)  # scaled as losses in half precision are
        return state
    dtype, rows, columns, classes = TYPE[case["dtype"]], case["rows"], case["columns"], case["classes"]
    if kind.startswith("embed"):
        # the k-th most frequent token about as often as 1 / k
        place = torch.exp(uniform(rows) * math.log(classes + 1.0)).int() - 1
        tokens = torch.randperm(classes, generator=draws, device=DEVICE, dtype=torch.int32)[torch.clamp(place, 0, classes - 1).long()]
        state["tokens"] = torch.where(uniform(rows) < 0.03, torch.full_like(tokens, -1), tokens)
        state["scale"] = math.sqrt(columns)
        if kind == "embed":
            state["table"] = normal(classes, columns, sigma=columns ** -0.5).to(dtype)
        else:
            state["dy"] = normal(rows, columns, sigma=0.01).to(dtype)
            state["table"] = torch.empty((classes, columns), dtype=dtype, device=DEVICE).fill_(0.5)  # its values play no part
        return state
    top = min(case["top"], classes)
    w = normal(classes, columns, sigma=2 * columns ** -0.5).to(dtype)
    # the teacher's best classes, best first, no class twice; some rows are padding, some teachers name fewer
    first = torch.randint(0, classes, (rows, 1), generator=draws, device=DEVICE)
    step = 1 + (uniform(rows, 1) * (classes // top - 1)).long()
    given = (first + step * torch.arange(top, device=DEVICE)[None]) % classes
    gaps = torch.empty((rows, top), dtype=torch.float32, device=DEVICE).exponential_(2.0, generator=draws)
    logits = normal(rows, 1, mean=10.0) - torch.cumsum(gaps, 1)
    # a student that has learned some of it: rows lean towards the first classes' weights
    x = normal(rows, columns)
    for k in range(min(top, 3)):
        x += w[given[:, k]].float() * (1.5 / (k + 1))
    there = (torch.arange(top, device=DEVICE)[None] < 1 + (uniform(rows, 1) * 4 * top).int()) & (uniform(rows, 1) >= 0.05)
    state.update(x=x.to(dtype), w=w, b=normal(classes, sigma=0.5).to(dtype), given=torch.where(there, given, torch.full_like(given, -1)).int(), logits=logits.to(dtype))
    if kind == "distil_gradient":
        state["dloss"] = uniform(rows, low=0.5, high=2.0) * 4
    return state


# ---- the plain form -------------------------------------------------------------------------------------------------------------

def _plain_embedding(state):
    case, tokens = state["case"], state["tokens"].long()
    kept = (tokens >= 0) & (tokens < case["classes"])
    if case["kind"] == "embed":
        y = state["table"][torch.clamp(tokens, 0, case["classes"] - 1)].float() * state["scale"]
        return {"y": torch.where(kept[:, None], y, torch.zeros_like(y)).to(TYPE[case["dtype"]])}
    dy = torch.where(kept[:, None], state["dy"].float() * state["scale"], torch.zeros((), device=DEVICE))
    gradient = torch.zeros((case["classes"], case["columns"]), device=DEVICE)
    gradient.index_add_(0, torch.clamp(tokens, 0, case["classes"] - 1), dy)
    return {"dtable": gradient.to(TYPE[case["dtype"]])}


def _plain_distillation(state):
    case = state["case"]
    dtype = TYPE[case["dtype"]]
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    given = state["given"].long()
    kept = (given >= 0) & (given < case["classes"])
    place = torch.clamp(given, 0, case["classes"] - 1)
    v = torch.where(kept, state["logits"].float() / TEMPERATURE, torch.full((), -math.inf, device=DEVICE))
    some = kept.any(1)
    v = v - torch.where(some, v.max(1).values, torch.zeros((), device=DEVICE))[:, None]
    q = torch.exp(v)
    total = q.sum(1, keepdim=True)
    q = q / torch.where(some[:, None], total, torch.ones_like(total))
    z = (x @ w.T + b) / TEMPERATURE
    top = z.max(1, keepdim=True).values
    lse = top[:, 0] + torch.log(torch.exp(z - top).sum(1))
    log_p = torch.where(kept, torch.gather(z, 1, place) - lse[:, None], torch.zeros((), device=DEVICE))
    log_q = torch.where(kept, v - torch.log(total), torch.zeros((), device=DEVICE))
    out = {"loss": (q * (log_q - log_p)).sum(1), "lse": lse, "log_probabilities": log_p}
    if case["kind"] == "distil":
        return out
    weight = torch.where(some, state["dloss"] / TEMPERATURE, torch.zeros_like(lse))[:, None]
    d = torch.exp(z - lse[:, None]) * weight
    d.scatter_add_(1, place, -q * weight)
    return dict(out, dx=(d @ w).to(dtype), dw=(d.T @ x).to(dtype), db=d.sum(0).to(dtype))


def _plain_policy(state):
    case = state["case"]
    kept = state["targets"] >= 0
    nothing = torch.zeros((), device=DEVICE)
    # in 64 bits: differences of close numbers, tokens next to the clip's border and a sum whose terms have both signs
    d = torch.where(kept, state["old"].double() - state["nll"].double(), nothing.double())
    a = state["advantages"].double()
    a = a if case["per_token"] else a[:, None].expand_as(d)
    a = torch.where(kept, a, nothing.double())
    r = torch.exp(d)
    clipped = ((a > 0) & (d > math.log1p(CLIP[1]))) | ((a < 0) & (d < math.log1p(-CLIP[0])))
    limit = torch.where(a > 0, 1 + CLIP[1], 1 - CLIP[0])
    gain = torch.where(clipped, limit, r) * a
    if state["reference"] is not None:
        q = torch.where(kept, state["nll"].double() - state["reference"].double(), nothing.double())
        kl = torch.exp(q) - q - 1
    else:
        q = kl = torch.zeros_like(d)
    count = kept.sum(1).double()
    if case["average"] == "tokens":
        weight = torch.ones_like(count) / torch.clamp(count.sum(), min=1)
    else:
        weight = 1 / (torch.clamp(count, min=1) * torch.clamp((count > 0).sum(), min=1))
    weight = torch.where(count > 0, weight, torch.zeros_like(weight))
    mean = lambda t: (torch.where(kept, t, nothing.double()).sum(1) * weight).sum()
    gain, kl, share = mean(gain), mean(kl), mean(clipped.double())
    out = {"loss": torch.stack((KL_WEIGHT * kl - gain, -gain, kl, share)).float(), "weights": weight.float()}
    if case["kind"] == "policy":
        return out
    slope = torch.where(clipped, nothing.double(), r * a) + KL_WEIGHT * (torch.exp(q) - 1)
    return dict(out, dnll=torch.where(kept, slope * weight[:, None] * state["dloss"].double(), nothing.double()).float())


def _plain(state):
    kind = state["case"]["kind"]
    return (_plain_embedding if kind.startswith("embed") else _plain_distillation if kind.startswith("distil") else _plain_policy)(state)


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
        kind = case["kind"]
        for name, t in state.items():
            if isinstance(t, torch.Tensor):
                setattr(self, name, self.over(t))
        if kind == "embed":
            self.scale = state["scale"]
            self.y = self.new("y", (case["rows"], case["columns"]), case["dtype"])
        elif kind == "embed_gradient":
            self.scale = state["scale"]
            self.dtable = self.new("dtable", (case["classes"], case["columns"]), case["dtype"])
            self.space = self.workspace(ml.embeddingGetWorkspaceSize(_context, self.tokens, self.table))
        elif kind.startswith("distil"):
            rows, top = self.given.shape
            self.loss, self.lse, self.log_p = self.new("loss", (rows,), "float32"), self.new("lse", (rows,), "float32"), self.new("log_probabilities", (rows, top), "float32")
            if kind == "distil_gradient":
                self.dx = self.new("dx", self.x.shape, case["dtype"])
                self.dw, self.db = self.new("dw", self.w.shape, case["dtype"]), self.new("db", self.b.shape, case["dtype"])
            self.space = self.workspace(ml.linearDistillationGetWorkspaceSize(_context, self.x, self.w, top, kind == "distil_gradient"))
        else:
            if not case["reference"]:
                self.reference = None
            self.loss, self.weights = self.new("loss", (4,), "float32"), self.new("weights", (case["sequences"],), "float32")
            if kind == "policy_gradient":
                self.dnll = self.new("dnll", self.nll.shape, "float32")
            self.space = self.workspace(ml.policyLossGetWorkspaceSize(_context, self.nll))

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
        if kind == "embed":
            ml.embeddingForward(_context, self.tokens, self.table, self.scale, self.y)
        elif kind == "embed_gradient":
            ml.embeddingBackward(_context, self.tokens, self.dy, self.scale, 0.0, self.dtable, self.space)
        elif kind.startswith("distil"):
            ml.linearDistillationForward(_context, self.x, self.w, self.b, self.given, self.logits, TEMPERATURE, self.loss, self.lse, self.log_p, self.space)
            if kind == "distil_gradient":
                ml.linearDistillationBackward(_context, self.x, self.w, self.b, self.given, self.logits, TEMPERATURE, self.lse, self.log_p, self.dloss, 0.0, self.dx, 0.0, self.dw, self.db,
                                              self.space)
        else:
            ml.policyLossForward(_context, self.nll, self.old, self.reference, self.advantages, self.targets, 50000, CLIP, KL_WEIGHT, case["average"], self.loss, self.weights, self.space)
            if kind == "policy_gradient":
                ml.policyLossBackward(_context, self.nll, self.old, self.reference, self.advantages, self.targets, 50000, CLIP, KL_WEIGHT, self.weights, self.dloss, 0.0, self.dnll)
        return self.results


def run(state):
    if not own:
        return _plain(state)
    if "call" not in state:
        state["call"] = _Call(state)
    return state["call"](state["case"])


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------

def _exact_distillation(s):
    case = s["case"]
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    given = s["given"].long()
    rows, places = torch.nonzero((given >= 0) & (given < case["classes"]), as_tuple=True)
    classes = given[rows, places]
    taught = torch.full((x.shape[0], given.shape[1]), -math.inf, dtype=torch.float64, device=DEVICE)
    taught[rows, places] = s["logits"].double()[rows, places]
    log_q = torch.log_softmax(taught / TEMPERATURE, 1)[rows, places]  # rows without any class are not looked at
    z = torch.addmm(b, x, w.t())
    z /= TEMPERATURE
    lse = torch.logsumexp(z, 1)
    log_p = z[rows, classes] - lse[rows]
    loss = torch.zeros_like(lse).index_add(0, rows, torch.exp(log_q) * (log_q - log_p))
    kept = torch.zeros((x.shape[0], given.shape[1]), dtype=torch.float64, device=DEVICE)
    kept[rows, places] = log_p
    out = {"loss": loss, "lse": lse, "log_probabilities": kept}
    if case["kind"] == "distil":
        return out
    d = torch.softmax(z, 1)
    del z
    d[rows, classes] -= torch.exp(log_q)
    weight = torch.zeros_like(lse)
    weight[rows] = s["dloss"].double()[rows] / TEMPERATURE
    d *= weight[:, None]
    return dict(out, dx=torch.matmul(d, w), dw=torch.matmul(d.t(), x), db=d.sum(0))


def _exact_policy(s):
    case = s["case"]
    at = torch.nonzero(s["targets"] >= 0, as_tuple=True)
    nll = s["nll"].double()[at]
    ratio = torch.exp(s["old"].double()[at] - nll)
    a = s["advantages"].double()[at if case["per_token"] else at[0]]
    free, held = ratio * a, torch.clamp(ratio, 1 - CLIP[0], 1 + CLIP[1]) * a
    passes = (free <= held).double()
    gain = torch.minimum(free, held)
    kl = slope = torch.zeros_like(gain)
    if s["reference"] is not None:
        q = nll - s["reference"].double()[at]
        kl, slope = torch.expm1(q) - q, torch.expm1(q)
    count = torch.bincount(at[0], minlength=case["sequences"]).double()
    if case["average"] == "tokens":
        weights = (count > 0).double() / max(1.0, float(count.sum()))
    else:
        weights = torch.where(count > 0, 1 / count, 0.0) / max(1, int((count > 0).sum()))
    each = weights[at[0]]
    parts = [(each * t).sum() for t in (gain, kl, 1 - passes)]
    out = {"loss": torch.stack((KL_WEIGHT * parts[1] - parts[0], -parts[0], parts[1], parts[2])), "weights": weights}
    if case["kind"] == "policy":
        return out
    gradient = torch.zeros((case["sequences"], case["length"]), dtype=torch.float64, device=DEVICE)
    gradient[at] = (passes * free + KL_WEIGHT * slope) * each * s["dloss"].double()
    return dict(out, dnll=gradient)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("distil"):
        return _exact_distillation(s)
    if kind.startswith("policy"):
        return _exact_policy(s)
    at = torch.nonzero((s["tokens"] >= 0) & (s["tokens"] < case["classes"]))[:, 0]
    tokens = s["tokens"].long()[at]
    if kind == "embed":
        y = torch.zeros((case["rows"], case["columns"]), dtype=torch.float64, device=DEVICE)
        y[at] = torch.nn.functional.embedding(tokens, s["table"]).double() * s["scale"]
        return {"y": y}
    order = torch.argsort(tokens, stable=True)
    dtable = torch.zeros((case["classes"], case["columns"]), dtype=torch.float64, device=DEVICE)
    sums = torch.cumsum(s["dy"].double()[at[order]], 0)  # a token's rows lie together: the difference of two sums
    ends = torch.cumsum(torch.bincount(tokens, minlength=case["classes"]), 0)
    sums = torch.cat((torch.zeros((1, case["columns"]), dtype=torch.float64, device=DEVICE), sums))
    dtable += sums[ends]
    dtable[1:] -= sums[ends[:-1]]
    return {"dtable": dtable * s["scale"]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    """Bytes: inputs and results once each (of a table that is looked up: as many rows as tokens can name). Flops: the products' (with gradients: the logits once, and the two gradients), else
    about what an element takes."""
    kind = case["kind"]
    if kind.startswith("policy"):
        tokens = case["sequences"] * case["length"]
        reads = 12 + 4 * case["reference"] + 4 * case["per_token"]
        writes = 4 if kind == "policy_gradient" else 0
        return {"bytes": float(tokens * (reads + writes) + case["sequences"] * (4 if case["per_token"] else 8) + 16), "flops": float(tokens * (20 if kind == "policy" else 35))}
    s, rows, columns, classes = SIZE[case["dtype"]], case["rows"], case["columns"], case["classes"]
    if kind == "embed":
        return {"bytes": float(s * columns * (rows + min(rows, classes)) + 4 * rows), "flops": float(rows * columns)}
    if kind == "embed_gradient":
        return {"bytes": float(s * columns * (rows + classes) + 4 * rows), "flops": 2.0 * rows * columns}
    top = min(case["top"], classes)
    given = rows * top * (8 + s) + 8 * rows
    weights = classes * (columns + 1)
    if kind == "distil":
        return {"bytes": float(s * (rows * columns + weights) + given), "flops": 2.0 * rows * columns * classes}
    return {"bytes": float(2 * s * (rows * columns + weights) + given + 4 * rows), "flops": 6.0 * rows * columns * classes}
