"""No-GPU checks of the operators with a backward pass: what the library and the mirror refuse, before anything reaches a device."""
import numpy as np
import pytest

from minml_amd import backend as B
from minml_amd import core as ml


_next = [1 << 40]


def fake(shape, dtype="float16"):
    """A tensor at an address of its own, which no call of these tests reaches."""
    _next[0] += 1 << 24
    return ml.Tensor(shape, dtype, _ptr=_next[0])


NULL = B.make_tensor(None, B.DTYPE_UNKNOWN, ())


def refused(name, *args, why=None):
    with pytest.raises(ValueError, match=why):
        B.fn(name)(None, *args)


def test_layer_norm_refusals_of_the_library():
    x, w = fake((4, 16)).desc(), fake((16,)).desc()
    forward = lambda x, w, b, y, eps=1e-5: refused("layer_norm_forward", x, w, b, y, eps)
    forward(x, w, w, fake((4, 15)).desc())
    forward(x, w, w, fake((4, 16), "float32").desc())
    forward(x, fake((15,)).desc(), w, x)
    forward(x, w, fake((16,), "float32").desc(), x)
    forward(fake((4, 16), "int32").desc(), w, w, fake((4, 16), "int32").desc())
    forward(x, w, w, x, -1.0)
    forward(x, w, w, x, float("nan"))
    refused("layer_norm_forward", x, w, w, x, 1e-5, why="null context")  # all is well but the context
    backward = lambda x, w, dy, dx, dw, db, space=0x7000, size=1 << 30: refused("layer_norm_backward", x, w, dy, 0.0, dx, 0.0, dw, db, space, size, 1e-5)
    need = B.fn("layer_norm_get_workspace_size")(fake((4, 16)).shape_desc(), B.DTYPE_FLOAT16)
    assert need >= 2 * 16 * 4
    backward(x, w, fake((4, 17)).desc(), x, w, w)
    backward(x, w, x, fake((3, 16)).desc(), w, w)
    backward(x, w, x, x, fake((17,)).desc(), w)
    backward(x, w, x, x, w, fake((16,), "int32").desc())
    backward(x, w, x, x, w, w, None, 0)
    backward(x, w, x, x, w, w, 0x7000, need - 1)
    backward(x, w, x, x, w, w, 0x7004, need)
    backward(fake((4, 16), "float32").desc(), fake((16,), "float32").desc(), fake((4, 16), "float32").desc(), NULL, w, NULL)  # fp16 sums of fp32 tensors
    B.fn("layer_norm_backward")(None, x, w, x, 0.0, NULL, 0.0, NULL, NULL, None, 0, 1e-5)  # nothing asked for
    B.fn("layer_norm_forward")(None, fake((0, 16)).desc(), w, w, fake((0, 16)).desc(), 1e-5)


@pytest.mark.parametrize("columns", [2 ** 28 + 1, 2 ** 31 - 1])
def test_layer_norm_refuses_rows_that_its_counters_do_not_reach(columns):
    x, y, dy, w = (ml.Tensor(s, "float16", _ptr=(k + 1) << 44).desc() for k, s in enumerate([(2, columns)] * 3 + [(columns,)]))
    refused("layer_norm_forward", x, w, NULL, y, 1e-5, why="too long")
    refused("layer_norm_backward", x, w, dy, 0.0, y, 0.0, NULL, NULL, 0x7000, 1 << 50, 1e-5, why="too long")
    with pytest.raises(ValueError, match="too long"):
        B.fn("layer_norm_get_workspace_size")(B.make_shape((2, columns)), B.DTYPE_FLOAT16)
    refused("layer_norm_forward", *(ml.Tensor(s, "float16", _ptr=(k + 1) << 44).desc() for k, s in enumerate([(2, 2 ** 28)] + [(2 ** 28,)] * 2 + [(2, 2 ** 28)])), 1e-5, why="null context")


def test_layer_norm_refusals_of_the_mirror():
    class Ctx:
        handle = None

    x, w, f = fake((4, 16)), fake((16,)), fake((16,), "float32")
    for call in (lambda: ml.layerNormForward(Ctx, x, w, w, fake((4, 8))), lambda: ml.layerNormForward(Ctx, x, f, w, x), lambda: ml.layerNormForward(Ctx, x, w, fake((8,)), x),
                 lambda: ml.layerNormBackward(Ctx, x, w, fake((4, 8)), 0.0, x, 0.0, w, w, None), lambda: ml.layerNormBackward(Ctx, x, w, x, 0.0, fake((4, 16), "float32"), 0.0, w, w, None),
                 lambda: ml.layerNormBackward(Ctx, x, w, x, 0.0, x, 0.0, fake((8,)), w, None), lambda: ml.layerNormBackward(Ctx, x, w, x, 0.0, x, 0.0, fake((16,), "int32"), w, None),
                 lambda: ml.layerNormBackward(Ctx, x, w, x, 0.0, x, 0.0, f, f, None)):
        with pytest.raises(ValueError):
            call()


def test_gated_dense_refusals_of_the_library():
    x, w, b, y, p = (fake(s).desc() for s in ((4, 16), (2, 24, 16), (2, 24), (4, 24), (4, 2, 24)))
    size = lambda backward: B.fn("gated_dense_get_workspace_size")(fake((4, 16)).shape_desc(), fake((2, 24, 16)).shape_desc(), B.DTYPE_FLOAT16, backward)
    assert size(True) > 4 * 48 * 2
    forward = lambda x=x, w=w, b=b, y=y, p=p, gate=B.GATE_SILU, space=0x7000, n=1 << 30: refused("gated_dense_forward", x, w, b, y, p, gate, space, n)
    forward(x=fake((4, 15)).desc())
    forward(x=fake((4, 16), "int8").desc())
    forward(w=fake((3, 24, 16)).desc())
    forward(w=fake((48, 16)).desc())
    forward(w=fake((2, 24, 16), "float32").desc())
    forward(b=fake((24,)).desc())
    forward(y=fake((4, 25)).desc())
    forward(y=fake((3, 24)).desc())
    forward(p=fake((4, 24, 2)).desc())
    forward(gate=4)
    forward(gate=-1)
    forward(x=ml.Tensor((4, 16), "float16", _ptr=0x7008).desc())
    forward(w=ml.Tensor((2, 24, 16), "float16", _ptr=0x7002).desc())
    forward()  # all is well but the context
    odd = dict(x=fake((100, 15)).desc(), w=fake((2, 24, 15)).desc(), y=fake((100, 24)).desc(), p=NULL)  # rows that end between pieces need room
    forward(**odd, space=None, n=0)
    forward(**odd, n=100)
    dx, dw, db = (fake(s).desc() for s in ((4, 16), (2, 24, 16), (2, 24)))
    backward = lambda x=x, w=w, p=p, dy=y, dx=dx, dw=dw, db=db, space=0x7000, n=1 << 30: refused("gated_dense_backward", x, w, p, dy, 0.0, dx, 0.0, dw, db, B.GATE_SILU, space, n)
    backward(dy=fake((4, 16)).desc())
    backward(p=NULL)
    backward(p=fake((4, 2, 12)).desc())
    backward(dx=fake((4, 17)).desc())
    backward(dx=fake((4, 16), "float32").desc())
    backward(dw=fake((2, 24, 15)).desc())
    backward(dw=fake((2, 24, 16), "int32").desc())
    backward(db=fake((24,)).desc())
    backward(space=None)
    backward(space=0x7010)
    backward(n=size(True) - 1)
    backward()  # all is well but the context


def test_gated_dense_refusals_of_the_mirror():
    class Ctx:
        handle = None

    x, w, b, y, p = (fake(s) for s in ((4, 16), (2, 24, 16), (2, 24), (4, 24), (4, 2, 24)))
    for call in (lambda: ml.gatedDenseForward(Ctx, x, w, b, y, p, "swish", None), lambda: ml.gatedDenseForward(Ctx, x, fake((2, 24, 8)), b, y, p, "silu", None),
                 lambda: ml.gatedDenseForward(Ctx, x, w, b, fake((4, 8)), p, "silu", None), lambda: ml.gatedDenseForward(Ctx, x, w, fake((24,)), y, p, "silu", None),
                 lambda: ml.gatedDenseForward(Ctx, x, w, b, y, y, "silu", None), lambda: ml.gatedDenseBackward(Ctx, x, w, p, x, 0.0, x, 0.0, w, b, "silu", None),
                 lambda: ml.gatedDenseBackward(Ctx, x, w, p, y, 0.0, y, 0.0, w, b, "silu", None), lambda: ml.gatedDenseBackward(Ctx, x, w, p, y, 0.0, x, 0.0, b, b, "silu", None),
                 lambda: ml.gatedDenseBackward(Ctx, x, w, p, y, 0.0, x, 0.0, w, w, "silu", None)):
        with pytest.raises(ValueError):
            call()


def test_cross_entropy_refusals_of_the_library():
    x, w, b, t, f = fake((4, 16)).desc(), fake((90, 16)).desc(), fake((90,)).desc(), fake((4,), "int32").desc(), fake((4,), "float32").desc()
    size = lambda backward: B.fn("linear_cross_entropy_get_workspace_size")(fake((4, 16)).shape_desc(), fake((90, 16)).shape_desc(), B.DTYPE_FLOAT16, backward)
    assert size(True) >= size(False) > 0
    forward = lambda x=x, w=w, b=b, t=t, loss=f, lse=f, space=0x7000, n=1 << 30: refused("linear_cross_entropy_forward", x, w, b, t, loss, lse, space, n)
    forward(x=fake((4, 15)).desc())
    forward(x=fake((4, 16), "int8").desc())
    forward(w=fake((2, 90, 16)).desc())
    forward(w=fake((0, 16)).desc())
    forward(w=fake((90, 16), "float32").desc())
    forward(b=fake((89,)).desc())
    forward(t=fake((4,), "float32").desc())
    forward(t=fake((3,), "int32").desc())
    forward(t=NULL)
    forward(loss=fake((4,)).desc())
    forward(lse=fake((5,), "float32").desc())
    forward(x=ml.Tensor((4, 16), "float16", _ptr=0x7008).desc())
    forward(w=ml.Tensor((90, 16), "float16", _ptr=0x7002).desc())
    forward(space=None)
    forward(space=0x7080)
    forward(n=size(False) - 1)
    forward()  # all is well but the context
    dx, dw, db = fake((4, 16)).desc(), fake((90, 16)).desc(), fake((90,)).desc()
    backward = lambda x=x, w=w, b=b, t=t, lse=f, dloss=f, dx=dx, dw=dw, db=db, space=0x7000, n=1 << 30: refused("linear_cross_entropy_backward", x, w, b, t, lse, dloss, 0.0, dx, 0.0, dw, db, space, n)
    backward(lse=fake((4,)).desc())
    backward(dloss=fake((4, 2), "float32").desc())
    backward(dx=fake((4, 17)).desc())
    backward(dx=fake((4, 16), "float32").desc())
    backward(dw=fake((91, 16)).desc())
    backward(dw=fake((90, 16), "int32").desc())
    backward(db=fake((91,)).desc())
    backward(n=size(True) - 1)
    backward(space=None)
    backward()
    B.fn("linear_cross_entropy_backward")(None, x, w, b, t, f, f, 0.0, NULL, 0.0, NULL, NULL, None, 0)  # nothing asked for


def test_cross_entropy_workspace_does_not_grow_with_the_vocabulary():
    """256 MB of d at most, and what goes with it, whatever the number of classes; never the logits."""
    for dtype, element in ((B.DTYPE_FLOAT16, 2), (B.DTYPE_FLOAT32, 4)):
        for rows, features in ((1000, 64), (4096, 2048), (65536, 1024)):
            sizes = [B.fn("linear_cross_entropy_get_workspace_size")(B.make_shape((rows, features)), B.make_shape((classes, features)), dtype, True) for classes in (200000, 2000000)]
            # besides d: sums over rows, two floats a tile of logits and row, the fp32 sums of dx and of one piece of dw, each in parts of at most 512 tiles together
            assert all(s <= (1 << 28) + rows * 20 + 8 * rows * classes / 128 + 2 * 4 * rows * features * 8 + (1 << 26) + 4 * 2000000 * (rows / 128 + 1) for s, classes in zip(sizes, (200000, 2000000)))
            assert sizes[1] < rows * 2000000 * element / 2


def test_cross_entropy_workspace_of_odd_widths_holds_the_padded_rows():
    """Where rows are no multiple of 16 bytes a copy of x and of all of w is on top of what the next multiple needs, and nothing else."""
    for dtype, element in ((B.DTYPE_FLOAT16, 2), (B.DTYPE_FLOAT32, 4)):
        for rows, features, classes in ((4096, 2047, 65536), (100, 1021, 2000000), (7, 2045, 65536)):
            piece = 16 // element
            whole = -(-features // piece) * piece
            for backward in (False, True):
                odd, even = (B.fn("linear_cross_entropy_get_workspace_size")(B.make_shape((rows, f)), B.make_shape((classes, f)), dtype, backward) for f in (features, whole))
                copies = (rows + classes) * whole * element if backward or rows > 64 else 0
                # dx in fp32 and its parts are a little narrower
                assert copies - 16 * 4 * rows * piece <= odd - even <= copies + 1024


def test_results_over_inputs_are_refused():
    """Where a call does not say that a result may lie over an input, it may not; and never in part."""
    whole = fake((64, 16))
    part = lambda shape, offset: whole.view(shape, offset).desc()
    x, w, b = fake((4, 16)).desc(), fake((16,)).desc(), fake((16,)).desc()
    overlaps = "overlap"
    refused("layer_norm_forward", part((4, 16), 0), w, b, part((4, 16), 16), 1e-5, why=overlaps)
    refused("layer_norm_forward", x, part((16,), 0), b, part((4, 16), 0), 1e-5, why=overlaps)
    refused("layer_norm_forward", x, w, b, x, 1e-5, why="null context")  # in place is allowed
    space, n = 0x7000, 1 << 20
    refused("layer_norm_backward", x, w, part((4, 16), 0), 0.0, part((4, 16), 8), 0.0, w, b, space, n, 1e-5, why=overlaps)
    refused("layer_norm_backward", x, w, fake((4, 16)).desc(), 0.0, x, 0.0, b, b, space, n, 1e-5, why=overlaps)
    refused("layer_norm_backward", x, w, fake((4, 16)).desc(), 0.0, x, 0.0, w, b, space, n, 1e-5, why=overlaps)
    refused("layer_norm_backward", x, w, x, 0.0, x, 0.0, fake((16,)).desc(), b, space, n, 1e-5, why="null context")
    w2, y, p = fake((2, 24, 16)).desc(), fake((4, 24)).desc(), fake((4, 2, 24)).desc()
    refused("gated_dense_forward", part((4, 16), 0), w2, NULL, part((4, 24), 32), p, B.GATE_SILU, None, 0, why=overlaps)
    refused("gated_dense_forward", x, w2, NULL, part((4, 24), 0), part((4, 2, 24), 0), B.GATE_SILU, None, 0, why=overlaps)
    refused("gated_dense_forward", x, w2, NULL, y, p, B.GATE_SILU, None, 0, why="null context")
    refused("gated_dense_backward", x, w2, p, y, 0.0, x, 0.0, NULL, NULL, B.GATE_SILU, space, n, why=overlaps)
    refused("gated_dense_backward", x, w2, p, y, 0.0, fake((4, 16)).desc(), 0.0, w2, NULL, B.GATE_SILU, space, n, why=overlaps)
    refused("gated_dense_backward", ml.Tensor((4, 16), "float16", _ptr=space + 256).desc(), w2, p, y, 0.0, fake((4, 16)).desc(), 0.0, NULL, NULL, B.GATE_SILU, space, n, why=overlaps)
    wc, t, f, g = fake((90, 16)).desc(), fake((4,), "int32").desc(), fake((4,), "float32").desc(), fake((4,), "float32").desc()
    refused("linear_cross_entropy_forward", x, wc, NULL, t, f, f, space, n, why=overlaps)
    refused("linear_cross_entropy_forward", x, wc, NULL, t, f, g, space, n, why="null context")
    refused("linear_cross_entropy_backward", x, wc, NULL, t, f, g, 0.0, x, 0.0, NULL, NULL, space, n, why=overlaps)
    refused("linear_cross_entropy_backward", x, wc, NULL, t, f, g, 0.0, NULL, 0.0, wc, NULL, space, n, why=overlaps)


def test_a_single_row_without_leading_dimensions_is_taken():
    class Ctx:
        handle = None

    x, w, wc = fake((16,)), fake((2, 24, 16)), fake((90, 16))
    t, loss, lse, g = fake((1,), "int32"), *(fake((1,), "float32") for _ in range(3))
    space = ml.Tensor((1 << 22,), "uint8", _ptr=1 << 50)
    for call in (lambda: ml.layerNormForward(Ctx, x, None, None, fake((16,))), lambda: ml.gatedDenseForward(Ctx, x, w, None, fake((24,)), fake((2, 24)), "silu", space),
                 lambda: ml.gatedDenseBackward(Ctx, x, w, fake((2, 24)), fake((24,)), 0.0, fake((16,)), 0.0, None, None, "silu", space),
                 lambda: ml.linearCrossEntropyForward(Ctx, x, wc, None, t, loss, lse, space),
                 lambda: ml.linearCrossEntropyBackward(Ctx, x, wc, None, t, lse, g, 0.0, fake((16,)), 0.0, None, None, space)):
        with pytest.raises(ValueError, match="null context"):
            call()
    with pytest.raises(ValueError, match="one int32 target per row"):
        ml.linearCrossEntropyForward(Ctx, x, wc, None, fake((2,), "int32"), loss, lse, space)


def test_layer_norm_may_overwrite_its_rows_but_not_its_weights():
    """Of a single row the weights have the row's size; only the input and the gradient may be where dx is."""
    x, dy, w, b = (fake((1, 16)).desc() for _ in range(4))
    backward = lambda dx, dw, why: refused("layer_norm_backward", x, w, dy, 0.0, dx, 0.0, dw, NULL, 0x7000, 1 << 20, 1e-5, why=why)
    backward(w, NULL, "overlap")
    backward(NULL, x, "overlap")
    backward(fake((1, 16)).desc(), dy, "overlap")
    backward(x, NULL, "null context")
    backward(dy, b, "null context")
    refused("layer_norm_forward", x, w, b, w, 1e-5, why="overlap")
    refused("layer_norm_forward", x, w, b, b, 1e-5, why="overlap")
    refused("layer_norm_forward", x, x, b, x, 1e-5, why="overlap")
    refused("layer_norm_forward", x, w, b, x, 1e-5, why="null context")
