"""No-GPU checks of the embedding and the policy loss: what the library and the mirror refuse, before anything reaches a device."""
import pytest

from minml_amd import backend as B
from minml_amd import core as ml
from test_training_refusals import NULL, fake, refused


class Ctx:
    handle = None


def test_embedding_refusals_of_the_library():
    t, w, y = fake((4,), "int32").desc(), fake((90, 16)).desc(), fake((4, 16)).desc()
    forward = lambda t=t, w=w, y=y, scale=2.0, why=None: refused("embedding_forward", t, w, scale, y, why=why)
    for scale in (float("inf"), float("nan")):
        forward(scale=scale, why="scale")
    forward(t=fake((4,), "float32").desc(), why="int32")
    forward(t=NULL)
    forward(t=ml.Tensor((4,), "int32", _ptr=0x7002).desc(), why="misaligned")
    forward(w=fake((90, 16), "int8").desc(), why="data type")
    forward(w=fake((2, 90, 16)).desc())
    forward(w=fake((0, 16)).desc())
    forward(y=fake((4, 15)).desc())
    forward(y=fake((3, 16)).desc())
    forward(y=fake((16, 4)).desc())
    forward(y=fake((4, 16), "float32").desc())
    forward(y=fake((90, 16)).view((4, 16), 16).desc(), w=w, why="null context")
    whole = fake((90, 16))
    forward(w=whole.desc(), y=whole.view((4, 16), 160).desc(), why="overlap")
    forward(why="null context")
    size = B.fn("embedding_get_workspace_size")(fake((5000,), "int32").shape_desc(), fake((90, 16)).shape_desc(), B.DTYPE_FLOAT16)
    assert size >= 5000 * 8
    t, dy = fake((5000,), "int32").desc(), fake((5000, 16)).desc()
    backward = lambda t=t, dy=dy, dw=w, space=0x7000, n=size, scale=1.0, why=None: refused("embedding_backward", t, dy, scale, 0.0, dw, space, n, why=why)
    for scale in (float("-inf"), float("nan")):
        backward(scale=scale, why="scale")
    backward(t=fake((4999,), "int32").desc())
    backward(dy=fake((5000, 8)).desc())
    backward(dy=fake((5000, 16), "int8").desc())
    backward(dw=fake((90, 17)).desc())
    backward(dw=fake((90,)).desc())
    backward(dw=fake((90, 16), "int32").desc())
    backward(dy=fake((5000, 16), "float32").desc())  # fp16 sums of fp32 rows
    backward(n=size - 1, why="workspace")
    backward(space=None, why="workspace")
    backward(space=0x7010, why="workspace")
    backward(dw=ml.Tensor((90, 16), "float16", _ptr=0x7000).desc(), why="overlap")
    rows = fake((5000, 16))
    backward(dy=rows.desc(), dw=rows.view((90, 16), 64).desc(), why="overlap")
    backward(why="null context")
    B.fn("embedding_backward")(None, t, dy, 1.0, 0.0, NULL, None, 0)  # nothing asked for


def test_embedding_refuses_what_its_counters_do_not_reach():
    shape = lambda *dims: B.make_shape(dims)
    for tokens, table in (((2 ** 28 + 1,), (8, 8)), ((8,), (2 ** 28 + 1, 8)), ((8,), (8, 2 ** 18 + 1))):
        with pytest.raises(ValueError, match="too many"):
            B.fn("embedding_get_workspace_size")(shape(*tokens), shape(*table), B.DTYPE_FLOAT32)
    for dtype in (B.DTYPE_INT8, B.DTYPE_INT32):
        with pytest.raises(ValueError):
            B.fn("embedding_get_workspace_size")(shape(8), shape(8, 8), dtype)


def test_embedding_workspace_of_fp32_is_enough_for_fp16():
    """A table's gradient in fp32 of rows in fp16: the size may be asked for with either type."""
    for rows in (1, 31, 33, 5000, 70000):
        for classes in (1, 300, 3000, 100000):
            for features in (1, 5, 64, 520, 1000, 1032, 2048, 4100):
                half, full = (B.fn("embedding_get_workspace_size")(B.make_shape((rows,)), B.make_shape((classes, features)), d) for d in (B.DTYPE_FLOAT16, B.DTYPE_FLOAT32))
                assert full >= half > 0


def test_embedding_refusals_of_the_mirror():
    t, w, y = fake((2, 3), "int32"), fake((90, 16)), fake((2, 3, 16))
    space = ml.Tensor((1 << 22,), "uint8", _ptr=1 << 50)
    for call in (lambda: ml.embeddingForward(Ctx, fake((2, 3)), w, 1.0, y), lambda: ml.embeddingForward(Ctx, t, w, 1.0, fake((2, 16))), lambda: ml.embeddingForward(Ctx, t, w, 1.0, fake((2, 3, 16), "float32")),
                 lambda: ml.embeddingForward(Ctx, t, fake((16,)), 1.0, y), lambda: ml.embeddingForward(Ctx, t, w, 1.0, fake(())), lambda: ml.embeddingForward(Ctx, fake((), "int32"), w, 1.0, y), lambda: ml.embeddingBackward(Ctx, t, fake((2, 3, 8)), 1.0, 0.0, w, space),
                 lambda: ml.embeddingBackward(Ctx, t, fake((2, 3, 16), "float32"), 1.0, 0.0, w, space), lambda: ml.embeddingBackward(Ctx, t, y, 1.0, 0.0, w, None)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ml.embeddingForward(Ctx, t, w, 1.0, y), lambda: ml.embeddingBackward(Ctx, t, y, 1.0, 0.0, w, space),
                 lambda: ml.embeddingForward(Ctx, fake((1,), "int32"), w, 1.0, fake((16,))), lambda: ml.embeddingBackward(Ctx, t, y, 1.0, 0.0, fake((90, 16), "float32"), space)):
        with pytest.raises(ValueError, match="null context"):
            call()


def policy_tensors(sequences=3, length=7):
    return [fake((sequences, length), "float32") for _ in range(3)] + [fake((sequences,), "float32"), fake((sequences, length), "int32")]


def test_policy_loss_refusals_of_the_library():
    names = ("nll", "old", "reference", "advantages", "targets")
    given = dict(zip(names, (t.desc() for t in policy_tensors())))
    loss, weights = fake((4,), "float32").desc(), fake((3,), "float32").desc()
    need = B.fn("policy_loss_get_workspace_size")(B.make_shape((3, 7)))

    def forward(clip=(0.2, 0.2), kl=0.1, average=0, loss=loss, weights=weights, space=0x7000, n=need, why=None, **other):
        refused("policy_loss_forward", *dict(given, **other).values(), 100, *clip, kl, average, loss, weights, space, n, why=why)

    def backward(clip=(0.2, 0.2), kl=0.1, weights=weights, dloss=NULL, dnll=fake((3, 7), "float32").desc(), why=None, **other):
        refused("policy_loss_backward", *dict(given, **other).values(), 100, *clip, kl, weights, dloss, 0.0, dnll, why=why)

    for call in (forward, backward):
        call(why="null context")
        call(reference=NULL, why="null context")
        call(advantages=fake((3, 7), "float32").desc(), why="null context")
        call(clip=(1.5, float("inf")), why="null context")
        for name in names:
            call(**{name: fake((3, 6), "float32").desc()})
            call(**{name: fake((3, 7), "float16").desc()})
        for name in ("nll", "old", "advantages", "targets"):
            call(**{name: NULL})
        call(nll=ml.Tensor((3, 7), "float32", _ptr=0x7002).desc())
        call(nll=fake((1, 3, 7), "float32").desc(), why=r"\[sequences, tokens\]")
        call(advantages=fake((7,), "float32").desc(), why="advantage")
        call(clip=(-0.1, 0.2), why="clip")
        call(clip=(0.2, float("nan")), why="clip")
        call(kl=float("inf"), why="weight must be finite")
        call(weights=fake((4,), "float32").desc())
        call(weights=fake((3,), "float16").desc())
    forward(average=2, why="average")
    forward(average=-1, why="average")
    forward(loss=fake((1,), "float32").desc())
    forward(loss=NULL)
    forward(loss=fake((4,)).desc())
    forward(weights=NULL)
    assert need == 0  # a few tokens need none
    many = dict(zip(names, (t.desc() for t in policy_tensors(300, 40))))
    of_many = dict(many, weights=fake((300,), "float32").desc())
    need = B.fn("policy_loss_get_workspace_size")(B.make_shape((300, 40)))
    forward(**of_many, space=None, why="workspace")
    forward(**of_many, space=0x7010, n=need, why="workspace")
    forward(**of_many, n=need - 1, why="workspace")
    forward(**of_many, n=need, why="null context")
    forward(loss=weights, weights=weights, why="4")
    forward(weights=given["advantages"], why="overlap")
    forward(**of_many, n=need, loss=ml.Tensor((4,), "float32", _ptr=0x7000).desc(), why="overlap")
    backward(dnll=fake((3, 8), "float32").desc())
    backward(dnll=NULL)
    backward(dnll=given["nll"], why="overlap")
    backward(dloss=fake((2,), "float32").desc(), why="single")
    backward(dloss=fake((1,)).desc(), why="single")
    with pytest.raises(ValueError, match="too many"):
        B.fn("policy_loss_get_workspace_size")(B.make_shape((1, 2 ** 28 + 1)))


def test_policy_loss_workspace_does_not_grow_with_the_tokens():
    for sequences, length in ((1, 2 ** 27), (500, 2 ** 20), (2 ** 20, 10), (4096, 4096)):
        assert B.fn("policy_loss_get_workspace_size")(B.make_shape((sequences, length))) <= 32 * 1024 + 256 + 4 * sequences


def test_policy_loss_refusals_of_the_mirror():
    tensors = policy_tensors()
    loss, weights, dnll = fake((4,), "float32"), fake((3,), "float32"), fake((3, 7), "float32")
    space = ml.Tensor((1 << 20,), "uint8", _ptr=1 << 50)

    def forward(clip=(0.2, 0.2), average="tokens", loss=loss, weights=weights, **other):
        ml.policyLossForward(Ctx, *(other.get(str(i), t) for i, t in enumerate(tensors)), 100, clip, 0.1, average, loss, weights, space)

    def backward(clip=(0.2, 0.2), weights=weights, dloss=None, dnll=dnll, **other):
        ml.policyLossBackward(Ctx, *(other.get(str(i), t) for i, t in enumerate(tensors)), 100, clip, 0.1, weights, dloss, 0.0, dnll)

    bad = [lambda: forward(average="words"), lambda: forward(loss=weights), lambda: forward(weights=loss), lambda: backward(weights=loss), lambda: backward(dloss=fake((2,), "float32")),
           lambda: backward(dnll=fake((7, 3), "float32"))]
    for call in (forward, backward):
        bad += [lambda call=call, i=i: call(**{str(i): fake((3, 5), "float32")}) for i in range(5)] + [lambda call=call: call(clip=(0.2,))]
    for call in bad:
        with pytest.raises(ValueError) as failure:
            call()
        assert "null context" not in str(failure.value)
    for call in (forward, backward, lambda: forward(**{"2": None}), lambda: backward(**{"2": None}, dloss=fake((1,), "float32"))):
        with pytest.raises(ValueError, match="null context"):
            call()


def test_distillation_refusals_of_the_library():
    x, w, b, named, taught, f, p = (fake(s, d).desc() for s, d in (((4, 16), "float16"), ((90, 16), "float16"), ((90,), "float16"), ((4, 8), "int32"), ((4, 8), "float16"), ((4,), "float32"), ((4, 8), "float32")))
    lse = fake((4,), "float32").desc()
    size = lambda backward, count=8: B.fn("linear_distillation_get_workspace_size")(B.make_shape((4, 16)), B.make_shape((90, 16)), count, B.DTYPE_FLOAT16, backward)
    assert size(True) >= size(False) > 0

    def forward(x=x, w=w, b=b, named=named, taught=taught, t=2.0, loss=f, lse=lse, p=p, space=0x7000, n=1 << 30, why=None):
        refused("linear_distillation_forward", x, w, b, named, taught, t, loss, lse, p, space, n, why=why)

    dx, dw, db, g = fake((4, 16)).desc(), fake((90, 16)).desc(), fake((90,)).desc(), fake((4,), "float32").desc()

    def backward(x=x, w=w, b=b, named=named, taught=taught, t=2.0, lse=lse, p=p, dloss=g, dx=dx, dw=dw, db=db, space=0x7000, n=1 << 30, why=None):
        refused("linear_distillation_backward", x, w, b, named, taught, t, lse, p, dloss, 0.0, dx, 0.0, dw, db, space, n, why=why)

    for call in (forward, backward):
        call(x=fake((4, 15)).desc())
        call(x=fake((4, 16), "int8").desc(), why="data type")
        call(w=fake((2, 90, 16)).desc())
        call(w=fake((0, 16)).desc())
        call(w=fake((90, 16), "float32").desc())
        call(b=fake((89,)).desc(), why="bias")
        call(named=fake((4, 8), "float32").desc(), why="int32")
        call(named=fake((3, 8), "int32").desc())
        call(named=fake((4, 0), "int32").desc(), why="1 to 1024")
        call(named=fake((4, 1025), "int32").desc(), taught=fake((4, 1025)).desc(), why="1 to 1024")
        call(named=NULL)
        call(taught=fake((4, 7)).desc(), why="logit")
        call(taught=fake((4, 8), "int32").desc(), why="logit")
        call(taught=NULL, why="logit")
        for t in (0.0, -1.0, float("nan"), float("inf"), 1e-45):
            call(t=t, why="temperature")
        call(lse=fake((5,), "float32").desc())
        call(lse=fake((4,)).desc())
        call(p=fake((4, 8)).desc(), why="log probabilities")
        call(p=fake((4, 9), "float32").desc(), why="log probabilities")
        call(p=NULL, why="log probabilities")
        call(x=ml.Tensor((4, 16), "float16", _ptr=0x7008).desc(), why="aligned")
        call(w=ml.Tensor((90, 16), "float16", _ptr=0x7002).desc(), why="aligned")
        call(space=None, why="workspace")
        call(space=0x7080, why="workspace")
        call(why="null context")
        call(b=NULL, taught=fake((4, 8), "float32").desc(), why="null context")
    # logits of half the type of an fp32 layer
    wide = dict(x=fake((4, 16), "float32").desc(), w=fake((90, 16), "float32").desc(), b=NULL)
    forward(**wide, why="logit")
    forward(n=size(False) - 1, why="workspace")
    forward(loss=fake((4, 2), "float32").desc())
    forward(loss=lse, why="overlap")
    forward(p=taught, why="log probabilities")
    backward(n=size(True) - 1, why="workspace")
    backward(dloss=fake((4,)).desc())
    backward(dx=fake((4, 17)).desc())
    backward(dx=fake((4, 16), "float32").desc())
    backward(dw=fake((91, 16)).desc())
    backward(dw=fake((90, 16), "int32").desc())
    backward(db=fake((91,)).desc())
    backward(dx=x, why="overlap")
    backward(dw=w, why="overlap")
    backward(dx=ml.Tensor((4, 16), "float16", _ptr=0x7000).desc(), why="overlap")
    B.fn("linear_distillation_backward")(None, x, w, b, named, taught, 1.0, lse, p, g, 0.0, NULL, 0.0, NULL, NULL, None, 0)  # nothing asked for
    for count in (0, -1, 1025):
        with pytest.raises(ValueError, match="1 to 1024"):
            size(True, count)


def test_distillation_workspace_does_not_grow_with_rows_times_classes():
    """What the cross entropy's backward pass holds, 16 bytes for every place and 2 for every row of every tile; for few rows their logits or gradients of them, 2 bytes of every 32 classes, and up to 512 sums of dx."""
    for dtype in (B.DTYPE_FLOAT16, B.DTYPE_FLOAT32):
        for rows, features, classes, count in ((4096, 2048, 65536, 64), (5000, 64, 200000, 1024), (7, 2048, 65536, 16), (64, 64, 1000, 3)):
            shapes = B.make_shape((rows, features)), B.make_shape((classes, features))
            size = B.fn("linear_distillation_get_workspace_size")(*shapes, count, dtype, True)
            other = B.fn("linear_cross_entropy_get_workspace_size")(*shapes, dtype, True)
            assert size <= other + rows * (16 * count + 2 * (classes // 128 + 2) + 8) + (5 * rows * classes if rows <= 64 else 0) + (512 * 4 * rows * features if rows <= 16 else 0) + 4096


def test_distillation_refusals_of_the_mirror():
    x, w, b, named, taught, f, p = fake((2, 3, 16)), fake((90, 16)), fake((90,)), fake((2, 3, 8), "int32"), fake((2, 3, 8)), fake((2, 3), "float32"), fake((2, 3, 8), "float32")
    space = ml.Tensor((1 << 24,), "uint8", _ptr=1 << 50)

    def forward(x=x, w=w, b=b, named=named, taught=taught, loss=f, lse=fake((2, 3), "float32"), p=p):
        ml.linearDistillationForward(Ctx, x, w, b, named, taught, 2.0, loss, lse, p, space)

    def backward(x=x, w=w, b=b, named=named, taught=taught, lse=f, p=p, g=fake((2, 3), "float32"), dx=fake((2, 3, 16)), dw=fake((90, 16), "float32"), db=fake((90,))):
        ml.linearDistillationBackward(Ctx, x, w, b, named, taught, 2.0, lse, p, g, 0.0, dx, 0.0, dw, db, space)

    bad = [lambda: forward(loss=fake((6,), "float32")), lambda: backward(g=fake((2, 3))), lambda: backward(dx=fake((6, 16))), lambda: backward(dw=fake((90, 15))), lambda: backward(db=fake((90,), "int32"))]
    for call in (forward, backward):
        bad += [lambda call=call, kw=kw: call(**kw) for kw in (dict(w=fake((90, 8))), dict(b=fake((91,))), dict(named=fake((6, 8), "int32")), dict(named=fake((2, 3, 8), "float32")), dict(taught=fake((2, 3, 7))),
                                                             dict(taught=fake((2, 3, 8), "int8")), dict(p=fake((2, 3, 8))), dict(p=fake((2, 3, 1), "float32")), dict(lse=fake((3, 2), "float32")))]
    for call in bad:
        with pytest.raises(ValueError) as failure:
            call()
        assert "null context" not in str(failure.value)
    one = dict(x=fake((16,)), named=fake((8,), "int32"), taught=fake((8,)), p=fake((8,), "float32"), lse=fake((1,), "float32"))
    for call in (forward, backward, lambda: backward(dx=None, db=None, b=None), lambda: forward(**one, loss=fake((1,), "float32")), lambda: backward(**one, g=fake((1,), "float32"), dx=fake((16,)))):
        with pytest.raises(ValueError, match="null context"):
            call()


def test_distillation_workspace_of_odd_widths_holds_the_padded_rows():
    """Rows that are no multiple of 16 bytes are copied before tiles read them, in the forward pass of more than 16 rows (in fp32 32) of large weights, where the cross entropy goes without, and in the
    backward pass of more than 8 (16)."""
    for dtype, element in ((B.DTYPE_FLOAT16, 2), (B.DTYPE_FLOAT32, 4)):
        for rows, features, classes in ((17, 1021, 32000), (24, 2047, 65536), (32, 1021, 20000), (33, 1021, 32000), (100, 1021, 200000), (4096, 2047, 65536), (7, 2045, 65536), (40, 30, 500)):
            piece = 16 // element
            whole = -(-features // piece) * piece
            for backward in (False, True):
                size = B.fn("linear_distillation_get_workspace_size")(B.make_shape((rows, features)), B.make_shape((classes, features)), 16, dtype, backward)
                tiles = rows > (16 if element == 2 else 32) and (rows > 64 or classes * features * element > 1 << 24)
                least = (rows + classes) * whole * element if tiles or (backward and rows > (8 if element == 2 else 16)) else rows * classes * 4
                assert size >= least + rows * 16 * (16 if tiles else 0)


def between(shape, dtype="float32"):
    """A tensor that begins between two elements, at an address of its own."""
    t = fake(shape, dtype).desc()
    t.data += 1 if dtype == "float16" else 2
    return t


def test_policy_loss_refuses_tensors_between_elements():
    names = ("nll", "old", "reference", "advantages", "targets")
    given = dict(zip(names, (t.desc() for t in policy_tensors())))
    results = dict(loss=fake((4,), "float32").desc(), weights=fake((3,), "float32").desc())
    of_gradient = dict(weights=results["weights"], dloss=fake((1,), "float32").desc(), dnll=fake((3, 7), "float32").desc())

    def forward(why=None, **other):
        tensors, out = dict(given, **{k: v for k, v in other.items() if k in given}), dict(results, **{k: v for k, v in other.items() if k in results})
        refused("policy_loss_forward", *tensors.values(), 100, 0.2, 0.2, 0.1, 0, out["loss"], out["weights"], 0x7000, 1 << 20, why=why)

    def backward(why=None, **other):
        tensors, out = dict(given, **{k: v for k, v in other.items() if k in given}), dict(of_gradient, **{k: v for k, v in other.items() if k in of_gradient})
        refused("policy_loss_backward", *tensors.values(), 100, 0.2, 0.2, 0.1, out["weights"], out["dloss"], 0.0, out["dnll"], why=why)

    for call, mine in ((forward, results), (backward, of_gradient)):
        call(why="null context")
        for name, t in dict(given, **mine).items():
            shape = tuple(t.dim[:t.rank])
            call(**{name: between(shape, "int32" if name == "targets" else "float32")}, why="^(?!.*null context)")


def test_distillation_refuses_tensors_between_elements():
    shapes = dict(b=((90,), "float16"), named=((4, 8), "int32"), taught=((4, 8), "float16"), loss=((4,), "float32"), lse=((4,), "float32"), p=((4, 8), "float32"), dloss=((4,), "float32"), dx=((4, 16), "float16"), dw=((90, 16), "float32"),
                  db=((90,), "float16"))
    x, w, whole = fake((4, 16)).desc(), fake((90, 16)).desc(), {k: fake(*v).desc() for k, v in shapes.items()}

    def forward(t, why):
        refused("linear_distillation_forward", x, w, t["b"], t["named"], t["taught"], 2.0, t["loss"], t["lse"], t["p"], 0x7000, 1 << 30, why=why)

    def backward(t, why):
        refused("linear_distillation_backward", x, w, t["b"], t["named"], t["taught"], 2.0, t["lse"], t["p"], t["dloss"], 0.0, t["dx"], 0.0, t["dw"], t["db"], 0x7000, 1 << 30, why=why)

    for call, names in ((forward, ("b", "named", "taught", "loss", "lse", "p")), (backward, ("b", "named", "taught", "lse", "p", "dloss", "dx", "dw", "db"))):
        call(whole, "null context")
        call(dict(whole, taught=fake((4, 8), "float32").desc()), "null context")
        for name in names:
            call(dict(whole, **{name: between(*shapes[name])}), "^(?!.*null context)")
        call(dict(whole, taught=between((4, 8))), "logit")


def test_embedding_refuses_tensors_between_elements():
    size = B.fn("embedding_get_workspace_size")(fake((40,), "int32").shape_desc(), fake((90, 16)).shape_desc(), B.DTYPE_FLOAT32)
    for dtype in ("float16", "float32"):
        tokens, table, rows = ((40,), "int32"), ((90, 16), dtype), ((40, 16), dtype)
        forward = lambda why, t=fake(*tokens).desc(), w=fake(*table).desc(), y=fake(*rows).desc(): refused("embedding_forward", t, w, 1.0, y, why=why)
        backward = lambda why, t=fake(*tokens).desc(), dw=fake(*table).desc(), y=fake(*rows).desc(): refused("embedding_backward", t, y, 1.0, 0.0, dw, 0x7000, size, why=why)
        for call, gradient in ((forward, {}), (backward, dict(dw=between(*table)))):
            call("null context")
            for name, t in dict(dict(t=between(*tokens), y=between(*rows)), **(gradient or dict(w=between(*table)))).items():
                call("^(?!.*null context)", **{name: t})
