"""gated_cumsum (h[t] = gate[t] * h[t-1] + x[t]) and its gradients against the recurrence in 64 bits: layouts, views,
repeated gates, states, lengths from one step to many, and what an infinity or a NaN reaches."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu

#        shape, axis, gate shape (None: full), initial
CASES = [((1,), 0, None, False), ((1,), 0, None, True), ((5,), 0, None, True), ((3, 1, 40), 1, None, True), ((2, 7, 33), 1, None, False),
         ((2, 64, 128), 1, None, True), ((3, 65, 130), 1, None, False), ((1, 1000, 96), 1, None, True), ((1, 4099, 64), 1, None, False),
         ((2, 500, 4, 64), 1, (2, 500, 4, 1), True), ((2, 130, 3, 16), 1, (2, 130, 3, 1), False), ((1, 300, 2, 128), 1, (1, 300, 2, 1), True),
         ((2, 90, 2, 6), 1, (2, 90, 2, 1), True), ((1, 70, 2, 256), 1, (1, 70, 2, 1), False), ((4, 50, 8), 1, (8,), True), ((4, 50, 8), 1, (50, 1), False),
         ((4, 50, 8), 1, (1,), True), ((300, 17), 0, None, False), ((6, 2049), 1, None, True), ((3, 4, 600), 2, None, False), ((5, 31), 1, None, True),
         ((70, 255), 1, None, False), ((2, 20000), 1, None, True), ((1, 70001), 1, None, False), ((9, 33, 4), 0, None, True), ((40000, 3), 0, None, False),
         ((3000, 2), 1, None, False), ((2, 9, 5, 3, 4), 2, None, True)]


def make(shape, axis, gate_shape, initial, dt, seed=0):
    rng = np.random.default_rng(seed + sum(shape) + axis)
    x = rng.standard_normal(shape).astype(dt)
    gate = (1 / (1 + np.exp(-rng.standard_normal(gate_shape or shape) - 2))).astype(dt)
    state = tuple(n for d, n in enumerate(shape) if d != axis)
    init = rng.standard_normal(state).astype(dt) if initial else None
    return x, gate, init


def arrays(xp, dt):
    return {np.float32: xp.SFloat, np.float64: xp.DFloat}[dt]


def opt(T, x):
    return None if x is None else T.from_numpy(x)


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("shape,axis,gate_shape,initial", CASES)
def test_forward(shape, axis, gate_shape, initial, dt):
    import cumo_b200 as xp

    T = arrays(xp, dt)
    x, gate, init = make(shape, axis, gate_shape, initial, dt)
    got = T.from_numpy(x).gated_cumsum(T.from_numpy(gate), axis=axis, initial=opt(T, init))
    want, mag = ref.gated(x, gate, axis, init)
    assert type(got) is T and got.shape == shape
    full = np.broadcast_to(gate, shape)
    assert np.all(np.abs(got.to_numpy() - want) <= ref.gated_bound(mag, full, axis, ref.U[np.dtype(dt)]))


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("shape,axis,gate_shape,initial", CASES)
def test_gradients(shape, axis, gate_shape, initial, dt):
    import cumo_b200 as xp

    T = arrays(xp, dt)
    u = ref.U[np.dtype(dt)]
    x, gate, init = make(shape, axis, gate_shape, initial, dt, seed=1)
    grad = np.random.default_rng(7).standard_normal(shape).astype(dt)
    h = ref.gated(x, gate, axis, init)[0].astype(dt)
    got = T.from_numpy(grad).gated_cumsum_grad(T.from_numpy(gate), T.from_numpy(h), axis=axis, initial=opt(T, init))
    assert len(got) == (3 if initial else 2)
    full = np.broadcast_to(gate, shape)
    dx, dgate, dinit, mag, before, later = ref.gated_grad(grad, full, h, axis, init)
    bound = np.flip(ref.gated_bound(np.flip(mag, axis), np.flip(later, axis), axis, u), axis)
    assert np.all(np.abs(got[0].to_numpy() - dx) <= bound)
    # one product per element, then a sum of `many` of them (a rounding each at most)
    many = max(1, dgate.size // gate.size)
    each = bound * np.abs(before) + (many + 2) * u * mag * np.abs(before)
    assert got[1].shape == gate.shape
    assert np.all(np.abs(got[1].to_numpy() - ref.sum_to(dgate, gate.shape)) <= ref.sum_to(each, gate.shape))
    if initial:
        first = np.take(full, 0, axis).astype(np.float64)
        assert np.all(np.abs(got[2].to_numpy() - dinit) <= first * (np.take(bound, 0, axis) + 2 * u * np.take(mag, 0, axis)))


def test_gradients_against_differences():
    import cumo_b200 as xp

    rng = np.random.default_rng(3)
    x, gate, init = rng.standard_normal((2, 9, 6)), rng.uniform(0.3, 0.99, (2, 9, 1)), rng.standard_normal((6,))
    weight = rng.standard_normal((2, 9, 6))

    def loss(x, gate, init):
        return float((xp.DFloat.from_numpy(x).gated_cumsum(xp.DFloat.from_numpy(gate), axis=1, initial=xp.DFloat.from_numpy(init)).to_numpy() * weight).sum())

    h = xp.DFloat.from_numpy(x).gated_cumsum(xp.DFloat.from_numpy(gate), axis=1, initial=xp.DFloat.from_numpy(init))
    got = xp.DFloat.from_numpy(weight).gated_cumsum_grad(xp.DFloat.from_numpy(gate), h, axis=1, initial=xp.DFloat.from_numpy(init))
    step = 1e-5                                             # truncation ~ step^2, cancellation ~ 2^-53 * |loss| / step: both below 1e-8
    for which, a in enumerate((x, gate, init)):
        for at in [(0,) * a.ndim, tuple(n - 1 for n in a.shape), tuple(n // 2 for n in a.shape)]:
            up, down = a.copy(), a.copy()
            up[at] += step
            down[at] -= step
            args = [[x, gate, init], [x, gate, init]]
            args[0][which], args[1][which] = up, down
            assert abs((loss(*args[0]) - loss(*args[1])) / (2 * step) - got[which].to_numpy()[at]) < 1e-6


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_views_and_strides(dt):
    import cumo_b200 as xp

    T = arrays(xp, dt)
    u = ref.U[np.dtype(dt)]
    rng = np.random.default_rng(5)
    base, gbase = rng.standard_normal((6, 90, 70)).astype(dt), rng.uniform(0.5, 1, (70, 90, 6)).astype(dt)
    views = [(lambda a: a[1:5, ::2, 3:68], lambda g: g.transpose(2, 1, 0)[1:5, ::2, 3:68]),
             (lambda a: a[::-1, ::-1, ::-3], lambda g: g.transpose(2, 1, 0)[:, :, :24]),
             (lambda a: a.transpose(1, 0, 2), lambda g: g.transpose(1, 2, 0)), (lambda a: a.transpose(2, 0, 1), lambda g: g.transpose(0, 2, 1))]
    for vx, vg in views:
        x, gate = vx(T.from_numpy(base)), vg(T.from_numpy(gbase))
        hx, hg = vx(base), vg(gbase)
        for axis in range(3):
            h = x.gated_cumsum(gate, axis=axis - 3)
            want, mag = ref.gated(hx, hg, axis)
            assert np.all(np.abs(h.to_numpy() - want) <= ref.gated_bound(mag, hg, axis, u))
            dx, dgate, _, gmag, before, later = ref.gated_grad(hx, hg, h.to_numpy(), axis)
            got = x.gated_cumsum_grad(gate, h, axis=axis)
            bound = np.flip(ref.gated_bound(np.flip(gmag, axis), np.flip(later, axis), axis, u), axis)
            assert np.all(np.abs(got[0].to_numpy() - dx) <= bound)
            assert np.all(np.abs(got[1].to_numpy() - dgate) <= (bound + 3 * u * gmag) * np.abs(before))


@pytest.mark.parametrize("shape,axis", [((2, 700, 64), 1), ((2, 3000), 1), ((3, 40, 5), 1), ((1, 9000, 4), 1)])
def test_what_is_not_finite_reaches_what_the_recurrence_says(shape, axis):
    import cumo_b200 as xp

    x, gate, init = make(shape, axis, None, True, np.float32)
    n = shape[axis]
    xs, gs = np.moveaxis(x, axis, -1), np.moveaxis(gate, axis, -1)
    xs.reshape(-1, n)[0, n // 3] = np.inf            # stays infinite: gates are positive
    xs.reshape(-1, n)[1, n // 2] = np.nan
    gs.reshape(-1, n)[-1, n // 4] = np.inf
    init.reshape(-1)[-1] = 0
    xs.reshape(-1, n)[-1, : n // 4 + 1] = 0           # inf * 0 is NaN in the recurrence
    with np.errstate(invalid="ignore"):
        want, _ = ref.gated(x, gate, axis, init)
    got = xp.SFloat.from_numpy(x).gated_cumsum(xp.SFloat.from_numpy(gate), axis=axis, initial=xp.SFloat.from_numpy(init)).to_numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    assert np.allclose(got[fine], want[fine], rtol=1e-4, atol=1e-4)
    # without a state the first gate is not used, whatever it holds, and the first element is kept bit for bit
    g2 = gate.copy()
    np.moveaxis(g2, axis, 0)[0] = np.nan
    np.moveaxis(x, axis, 0)[0] = -0.0
    first = np.moveaxis(xp.SFloat.from_numpy(x).gated_cumsum(xp.SFloat.from_numpy(g2), axis=axis).to_numpy(), axis, 0)[0]
    assert np.all(first == 0) and np.all(np.signbit(first))


@pytest.mark.parametrize("shape,axis", [((1, 5000, 32), 1), ((2, 6000), 1)])
def test_gates_that_stop_or_grow(shape, axis):
    """A gate of zero starts a sequence anew; products of growing gates leave the range of the type while the sums do not."""
    import cumo_b200 as xp

    rng = np.random.default_rng(2)
    x = rng.standard_normal(shape).astype(np.float32)
    gate = rng.uniform(0.9, 1, shape).astype(np.float32)
    np.moveaxis(gate, axis, 0)[::611] = 0
    want, mag = ref.gated(x, gate, axis)
    got = xp.SFloat.from_numpy(x).gated_cumsum(xp.SFloat.from_numpy(gate), axis=axis).to_numpy()
    assert np.all(np.abs(got - want) <= ref.gated_bound(mag, gate, axis, 2.0 ** -24))
    quiet, big = np.zeros(shape, np.float32), np.full(shape, 1e6, np.float32)
    np.moveaxis(quiet, axis, 0)[-1] = 3
    got = xp.SFloat.from_numpy(quiet).gated_cumsum(xp.SFloat.from_numpy(big), axis=axis).to_numpy()
    assert np.array_equal(got, quiet)                        # 1e6 * 0 stays 0, however many steps


@pytest.mark.parametrize("shape,axis", [((1, 3000, 32), 1), ((2, 5000), 1), ((1, 700, 5), 1)])
def test_products_of_gates_that_nearly_vanish_and_return(shape, axis):
    """Two gates that multiply to less than the type's normal range, then one that brings the product back: the state passes
    through them without having been that small itself."""
    import cumo_b200 as xp

    n = shape[axis]
    x, gate = np.zeros(shape, np.float32), np.full(shape, 0.5, np.float32)
    xs, gs = np.moveaxis(x, axis, -1), np.moveaxis(gate, axis, -1)
    for at in range(20, n - 40, 37):
        xs[..., at] = 2.0 ** 90
        gs[..., at + 1:at + 5] = [2.0 ** -70, 2.0 ** -75, 2.0 ** 80, 2.0 ** 60]       # state 2^90 -> 2^20 -> 2^-55 -> 2^25 -> 2^85
        gs[..., at + 6] = 0
    want, mag = ref.gated(x, gate, axis)
    got = xp.SFloat.from_numpy(x).gated_cumsum(xp.SFloat.from_numpy(gate), axis=axis).to_numpy()
    assert np.all(np.abs(got - want) <= ref.gated_bound(mag, gate, axis, 2.0 ** -24))


def test_empty_and_token_by_token():
    import cumo_b200 as xp

    assert xp.SFloat(3, 0, 4).gated_cumsum(xp.SFloat(3, 0, 4), axis=1).shape == (3, 0, 4)
    assert xp.SFloat(0, 5).gated_cumsum(xp.SFloat(0, 5), axis=1).shape == (0, 5)
    dx, dgate, dinit = xp.SFloat(2, 0, 3).gated_cumsum_grad(xp.SFloat(2, 0, 1), xp.SFloat(2, 0, 3), axis=1, initial=xp.SFloat.ones(2, 3))
    assert dx.shape == (2, 0, 3) and dgate.shape == (2, 0, 1) and np.array_equal(dinit.to_numpy(), np.zeros((2, 3)))
    rng = np.random.default_rng(0)
    x, gate = (rng.standard_normal((5, 12, 40)).astype(np.float32), rng.uniform(0.5, 1, (5, 12, 40)).astype(np.float32))
    X, G = xp.SFloat.from_numpy(x), xp.SFloat.from_numpy(gate)
    whole = X.gated_cumsum(G, axis=1).to_numpy()
    state = None
    for t in range(12):                                      # one token at a time, the state carried by the caller
        h = X[True, t:t + 1, True].gated_cumsum(G[True, t:t + 1, True], axis=1, initial=state)
        state = h[True, 0, True]
        assert np.array_equal(state.to_numpy(), whole[:, t])


def test_ones_are_cumsum_and_repeated_calls_agree():
    import cumo_b200 as xp

    x = np.random.default_rng(1).integers(-8, 9, (3, 5000)).astype(np.float32)
    X = xp.SFloat.from_numpy(x)
    assert np.array_equal(X.gated_cumsum(1.0, axis=1).to_numpy(), np.cumsum(x, axis=1, dtype=np.float64).astype(np.float32))
    gate = xp.SFloat.from_numpy(np.random.default_rng(2).uniform(0.8, 1, (3, 5000)).astype(np.float32))
    a, b = X.gated_cumsum(gate, axis=1), X.gated_cumsum(gate, axis=1)
    assert np.array_equal(a.to_numpy(), b.to_numpy())

@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("head", [16, 64, 128, 6])
@pytest.mark.parametrize("where", ["heads", "time", "batch"])
def test_gate_of_the_full_shape_with_steps_of_zero(head, where, dt):
    """An expanded tensor is a gate of its own in every place: its gradient has the full shape, nothing summed, whichever
    dimension the steps of 0 run along -- heads that a warp could sum included -- and owns every element it shows."""
    import torch

    import cumo_b200 as xp

    T, u = arrays(xp, dt), ref.U[np.dtype(dt)]
    shape = (2, 40, 3, head)
    short = {"heads": (2, 40, 3, 1), "time": (2, 1, 3, head), "batch": (1, 40, 3, head)}[where]
    rng = np.random.default_rng(head)
    small = rng.uniform(0.5, 1, short).astype(dt)
    x, grad = rng.standard_normal(shape).astype(dt), rng.standard_normal(shape).astype(dt)
    wide = torch.from_numpy(small).cuda().expand(*shape)
    assert 0 in wide.stride()
    h = T.from_numpy(x).gated_cumsum(T.from_torch(wide), axis=1)
    dx, dgate = T.from_numpy(grad).gated_cumsum_grad(T.from_torch(wide), h, axis=1)
    full = np.broadcast_to(small, shape)
    want, want_gate, _, mag, before, later = ref.gated_grad(grad, full, h.to_numpy(), 1)
    bound = np.flip(ref.gated_bound(np.flip(mag, 1), np.flip(later, 1), 1, u), 1)
    assert dgate.shape == shape
    assert np.all(np.abs(dx.to_numpy() - want) <= bound)
    assert np.all(np.abs(dgate.to_numpy() - want_gate) <= (bound + 3 * u * mag) * np.abs(before))


@pytest.mark.parametrize("gate_shape,state_shape", [((2, 1, 3, 16), None), ((1, 40, 3, 16), None), ((2, 40, 3, 1), (16,)), ((16,), (2, 3, 16)), ((2, 40, 1, 1), None)])
def test_a_capture_refuses_sums_before_anything_is_recorded(gate_shape, state_shape):
    """Gradients that need a temporary array are refused in a capture with nothing launched: the graph that is finished
    afterwards leaves the memory alone that the refused call had held."""
    import torch

    import cumo_b200 as xp
    from cumo_b200 import _lib

    lib = _lib.load()
    S = xp.SFloat.from_torch
    shape = (2, 40, 3, 16)
    x, grad = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")
    gate, own_gate = torch.rand(gate_shape, device="cuda"), torch.rand(shape, device="cuda")
    state = None if state_shape is None else torch.randn(state_shape, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        lib.cb200_set_stream(stream.cuda_stream)
        try:
            init = None if state is None else S(state)
            h = S(x).gated_cumsum(S(gate), axis=1, initial=init)
            want = [g.to_numpy() for g in S(grad).gated_cumsum_grad(S(gate), h, axis=1, initial=init)]
            S(grad).gated_cumsum_grad(S(own_gate), h, axis=1)       # fills the stream's pool: a capture may not allocate
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                before = _lib.launch_count()
                with pytest.raises(xp.CudaError):
                    S(grad).gated_cumsum_grad(S(gate), h, axis=1, initial=init)
                assert _lib.launch_count() == before
                kept = S(grad).gated_cumsum_grad(S(own_gate), h, axis=1)
            others = [xp.SFloat.zeros(*shape) for _ in range(8)]    # whatever the refused call gave back is among these
            graph.replay()
            stream.synchronize()
            assert not any(o.to_numpy().any() for o in others)
            again = S(grad).gated_cumsum_grad(S(gate), h, axis=1, initial=init)
            assert all(np.array_equal(a.to_numpy(), b) for a, b in zip(again, want))
            eager = S(grad).gated_cumsum_grad(S(own_gate), h, axis=1)
            assert all(np.array_equal(a.to_numpy(), b.to_numpy()) for a, b in zip(kept, eager))
        finally:
            lib.cb200_set_stream(None)


@pytest.mark.parametrize("shape,axis", [((1, 3000, 32), 1), ((1, 700, 5), 1), ((2, 5000), 1), ((3, 300), 1), ((2, 100, 2400), 1), ((4, 33, 6), 1), ((2, 16, 3), 1)])
def test_sums_that_leave_the_range_from_zero_but_not_from_their_state(shape, axis):
    """A state of -3e38 and a few steps of +2e38: the state stays inside the range of the type, while the same steps summed
    from zero, as a stretch is before the state in front of it is known, do not."""
    import cumo_b200 as xp

    n = shape[axis]
    x, gate = np.zeros(shape, np.float32), np.ones(shape, np.float32)
    xs = np.moveaxis(x, axis, 0)
    xs[0] = -3e38
    for at in range(2, n - 3, 23):
        xs[at], xs[at + 1] = 2e38, 2e38                      # -3e38 -> -1e38 -> 1e38 -> (back below) ...
        xs[at + 2] = -4 / 3 * 3e38 * 0.75                    # -> -2e38, then
        xs[at + 3] = -1e38                                   # -> -3e38
    want, mag = ref.gated(x, gate, axis)
    assert np.abs(want).max() < 3.2e38
    X, G = xp.SFloat.from_numpy(x), xp.SFloat.from_numpy(gate)
    got = X.gated_cumsum(G, axis=axis)
    assert np.all(np.abs(got.to_numpy() - want) <= ref.gated_bound(mag, gate, axis, 2.0 ** -24))
    back = xp.SFloat.from_numpy(np.ascontiguousarray(np.flip(x, axis)))       # the gradient runs the other way
    dx = back.gated_cumsum_grad(G, xp.SFloat.zeros(*shape), axis=axis)[0].to_numpy()
    assert np.all(np.abs(np.flip(dx, axis) - want) <= ref.gated_bound(mag, gate, axis, 2.0 ** -24))
