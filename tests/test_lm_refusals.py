"""What the sequence and layer operators refuse.  Every refusal comes before anything is allocated or launched, so these run
without a GPU: the arrays borrow an address that nothing reads."""
import pytest

import cumo_b200 as xp
from cumo_b200 import linalg
from cumo_b200.narray import ShapeError


def arr(*shape, T=xp.SFloat):
    return T.from_device_pointer(1 << 20, shape)


def test_gated_cumsum_refuses():
    x = arr(2, 5, 3)
    for bad in [dict(axis=3), dict(axis=-4)]:
        with pytest.raises(ValueError):
            x.gated_cumsum(arr(2, 5, 3), **bad)
    for bad in [None, 1.0, True, (0, 1)]:
        with pytest.raises(TypeError):
            x.gated_cumsum(arr(2, 5, 3), axis=bad)
    for gate in [arr(5, 2), arr(1, 2, 5, 3), arr(4, 1, 1)]:
        with pytest.raises(ShapeError):
            x.gated_cumsum(gate, axis=1)
    with pytest.raises(ShapeError):
        x.gated_cumsum(arr(2, 5, 3), axis=1, initial=arr(2, 5))
    with pytest.raises(ShapeError):
        x.gated_cumsum(arr(2, 5, 3), axis=1, initial=arr(1, 2, 3))
    with pytest.raises(TypeError):
        x.gated_cumsum(arr(2, 5, 3, T=xp.DFloat), axis=1)
    with pytest.raises(TypeError):
        x.gated_cumsum(arr(2, 5, 3), axis=1, initial=arr(2, 3, T=xp.DFloat))
    with pytest.raises(TypeError):
        arr(4, T=xp.Int32).gated_cumsum(arr(4, T=xp.Int32))
    with pytest.raises(TypeError):
        x.gated_cumsum(None, axis=1)
    with pytest.raises(TypeError):
        x.gated_cumsum("gate", axis=1)


def test_gated_cumsum_grad_refuses():
    g = arr(2, 5, 3)
    with pytest.raises(ShapeError):
        g.gated_cumsum_grad(arr(2, 5, 3), arr(2, 5, 1), axis=1)
    with pytest.raises(TypeError):
        g.gated_cumsum_grad(arr(2, 5, 3), arr(2, 5, 3, T=xp.DFloat), axis=1)
    with pytest.raises(TypeError):
        g.gated_cumsum_grad(arr(2, 5, 3), None, axis=1)
    with pytest.raises(ShapeError):
        g.gated_cumsum_grad(arr(2, 4, 3), arr(2, 5, 3), axis=1)


def test_linear_refuses():
    x, w = arr(4, 8), arr(8, 6)
    for kw in [dict(x=arr(4, 7)), dict(w=arr(8)), dict(w=arr(1, 8, 6)), dict(bias=arr(5)), dict(bias=arr(1, 6)), dict(residual=arr(5, 6)),
               dict(residual=arr(1, 1, 4, 6)), dict(x=arr(4, 0), w=arr(0, 6))]:
        with pytest.raises(ShapeError):
            linalg.linear(**{"x": x, "w": w, **kw})
    for kw in [dict(w=arr(8, 6, T=xp.DFloat)), dict(bias=arr(6, T=xp.DFloat)), dict(x=arr(4, 8, T=xp.Int32), w=arr(8, 6, T=xp.Int32)), dict(residual=1.0)]:
        with pytest.raises(TypeError):
            linalg.linear(**{"x": x, "w": w, **kw})
    for name in ["softmax", "ReLU", 1, True]:
        with pytest.raises(ValueError):
            linalg.linear(x, w, activation=name)


def test_linear_grad_refuses():
    g, x, w = arr(4, 6), arr(4, 8), arr(8, 6)
    for kw in [dict(grad=arr(5, 6)), dict(grad=arr(4, 5)), dict(w=arr(6, 8)), dict(activation="silu", pre=arr(4, 5)), dict(activation="silu", pre=arr(24))]:
        with pytest.raises(ShapeError):
            linalg.linear_grad(**{"grad": g, "x": x, "w": w, **kw})
    for kw in [dict(activation="silu"), dict(want=()), dict(want=("x", "x")), dict(want=("y",)), dict(activation="swish")]:
        with pytest.raises(ValueError):
            linalg.linear_grad(g, x, w, **kw)
    with pytest.raises(TypeError):
        linalg.linear_grad(g, arr(4, 8, T=xp.DFloat), w)


def test_orthogonalize_refuses():
    with pytest.raises(ShapeError):
        linalg.orthogonalize(arr(5))
    with pytest.raises(TypeError):
        linalg.orthogonalize(arr(5, 5, T=xp.Int64))
    for kw in [dict(steps=-1), dict(steps=2.5), dict(coefs=(1.0, 2.0)), dict(steps=2, coefs=[(1.5, -0.5, 0.0)]), dict(eps=-1.0), dict(eps=float("nan"))]:
        with pytest.raises(ValueError):
            linalg.orthogonalize(arr(5, 5), **kw)
