"""linalg.linear (act(x . w + bias) + residual) and linear_grad against 64 bits."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid", "tanh"]
SIZES = [(1, 1, 1), (1, 33, 70), (1, 512, 1000), (2, 64, 64), (3, 1000, 4), (5, 7, 300), (8, 256, 130), (17, 31, 33), (31, 100, 257), (64, 64, 64),
         (65, 129, 63), (100, 1, 100), (128, 128, 256), (129, 300, 257), (200, 1030, 90), (256, 64, 512), (300, 17, 300), (513, 255, 129), (700, 40, 24)]


def data(m, k, n, dt, seed=0):
    rng = np.random.default_rng(seed + m + 3 * k + 7 * n)
    return (rng.standard_normal((m, k)).astype(dt), (rng.standard_normal((k, n)) / np.sqrt(k)).astype(dt), rng.standard_normal(n).astype(dt),
            rng.standard_normal((m, n)).astype(dt), rng)


def T_of(xp, dt):
    return xp.SFloat if dt is np.float32 else xp.DFloat


def d(a):
    return a.astype(np.float64)


def forward_bounds(x, w, bias, name, res, u):
    """z and y in 64 bits with the errors allowed: the product's, a rounding for the bias; a slope of at most 1.2 carries
    it through the activation, whose own value is good to 8 roundings (of z where values cancel); a rounding for the residual."""
    z = d(x) @ d(w) + (0 if bias is None else d(bias))
    ez = ref.product_bound(d(x), d(w), u) + u * np.abs(z)
    y0 = ref.act(z, name)
    ey = 1.2 * ez + (0 if name is None else 8 * u * (np.abs(y0) + np.minimum(1, np.abs(z))))
    y = y0 if res is None else y0 + d(res)
    return z, ez, y, ey + u * np.abs(y)


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward_sizes(m, k, n, dt):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    T, u = T_of(xp, dt), ref.U[np.dtype(dt)]
    x, w, bias, res, _ = data(m, k, n, dt)
    for name, b, r in [(None, None, None), ("silu", bias, res), ("gelu", bias, None), (None, None, res)]:
        got, pre = linalg.linear(T.from_numpy(x), T.from_numpy(w), bias=None if b is None else T.from_numpy(b), activation=name,
                                 residual=None if r is None else T.from_numpy(r), keep=True)
        z, ez, y, ey = forward_bounds(x, w, b, name, r, u)
        assert type(got) is T and got.shape == (m, n) and pre.shape == (m, n)
        assert np.all(np.abs(pre.to_numpy() - z) <= ez)
        assert np.all(np.abs(got.to_numpy() - y) <= ey)


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("name", ACTS)
def test_activations_and_their_slopes(name, dt):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    T, u = T_of(xp, dt), ref.U[np.dtype(dt)]
    z = np.concatenate([np.linspace(-12, 12, 4001), np.linspace(-88, 88, 333), [0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4, 1e15, -1e15]]).astype(dt)[None]
    one = np.ones((1, 1), dt)
    got = linalg.linear(T.from_numpy(one), T.from_numpy(z), activation=name).to_numpy()
    with np.errstate(over="ignore"):
        want, slope = ref.act(d(z), name), ref.slope(np.clip(d(z), -1e100, 1e100), name)
    # arguments inside the functions are rounded: an error of |z| u in z, times a slope of at most 1.2 that has died out by |z| = 30
    near = np.minimum(np.abs(d(z)), 30)
    assert np.all(np.abs(got - want) <= 8 * u * (np.abs(want) + near) + (1e-38 if dt is np.float32 else 1e-300))
    got = linalg.linear_grad(T.from_numpy(np.ones_like(z)), T.from_numpy(one), T.from_numpy(z), activation=name, pre=T.from_numpy(z), want="bias")[0].to_numpy()
    ok = np.abs(got - slope[0]) <= 16 * u * (np.abs(slope[0]) + near[0] * (1 + near[0]))
    assert np.all(ok), z[0][~ok][:5]


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gradients(m, k, n, dt):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    T, u = T_of(xp, dt), ref.U[np.dtype(dt)]
    x, w, bias, grad, _ = data(m, k, n, dt, seed=5)
    X, W, G = T.from_numpy(x), T.from_numpy(w), T.from_numpy(grad)
    for name in (None, "gelu_tanh"):
        pre = (d(x) @ d(w) + d(bias)).astype(dt)
        dx, dw, db = linalg.linear_grad(G, X, W, activation=name, pre=T.from_numpy(pre) if name else None)
        s = ref.slope(d(pre), name)
        dz = d(grad) * s
        # dz: the slope good to 16 roundings of what it is made of, one more for the product
        edz = 0 if name is None else np.abs(d(grad)) * 16 * u * (1 + np.minimum(np.abs(d(pre)), 6) ** 2)
        for got, want, bound in ((dx, dz @ d(w).T, ref.product_bound(dz, d(w).T, u) + edz @ np.abs(d(w).T) if name else ref.product_bound(dz, d(w).T, u)),
                                 (dw, d(x).T @ dz, ref.product_bound(d(x).T, dz, u) + (np.abs(d(x)).T @ edz if name else 0)),
                                 (db, dz.sum(0), (m + 2) * u * np.abs(dz).sum(0) + (edz.sum(0) if name else 0))):
            assert got.shape == want.shape
            assert np.all(np.abs(got.to_numpy() - want) <= bound)
        again = linalg.linear_grad(G, X, W, activation=name, pre=T.from_numpy(pre) if name else None)
        assert all(np.array_equal(a.to_numpy(), b.to_numpy()) for a, b in zip((dx, dw, db), again))


def test_gradients_against_differences():
    import cumo_b200 as xp
    from cumo_b200 import linalg

    D = xp.DFloat.from_numpy
    rng = np.random.default_rng(11)
    x, w, b, weight = rng.standard_normal((5, 7)), rng.standard_normal((7, 6)) / 3, rng.standard_normal(6), rng.standard_normal((5, 6))
    for name in ACTS[2:]:
        def loss(x, w, b):
            return float((linalg.linear(D(x), D(w), bias=D(b), activation=name).to_numpy() * weight).sum())
        _, pre = linalg.linear(D(x), D(w), bias=D(b), activation=name, keep=True)
        got = linalg.linear_grad(D(weight), D(x), D(w), activation=name, pre=pre)
        for which, a in enumerate((x, w, b)):
            at = tuple(n // 2 for n in a.shape)
            up, down = a.copy(), a.copy()
            up[at] += 1e-5
            down[at] -= 1e-5
            pair = [[x, w, b], [x, w, b]]
            pair[0][which], pair[1][which] = up, down
            assert abs((loss(*pair[0]) - loss(*pair[1])) / 2e-5 - got[which].to_numpy()[at]) < 1e-6


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_layouts(dt):
    """Leading axes, transposed and sliced operands, repeated residual, one wanted gradient."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    T, u = T_of(xp, dt), ref.U[np.dtype(dt)]
    rng = np.random.default_rng(1)
    for m, k, n in ((30, 41, 50), (260, 200, 130), (6, 300, 520)):
        big, wide = rng.standard_normal((2 * m, 3, k + 5)).astype(dt), rng.standard_normal((n + 3, 2 * k)).astype(dt)
        X, W = T.from_numpy(big)[::2, 1, 2:2 + k], T.from_numpy(wide)[3:, ::2].transpose()
        x, w = big[::2, 1, 2:2 + k], wide[3:, ::2].T
        res = rng.standard_normal(n).astype(dt)
        y = linalg.linear(X, W, residual=T.from_numpy(res))
        z, ez, want, ey = forward_bounds(x, w, None, None, np.broadcast_to(res, (m, n)), u)
        assert np.all(np.abs(y.to_numpy() - want) <= ey)
        Xr = X[::-1, True]
        assert np.array_equal(linalg.linear(Xr, W, residual=T.from_numpy(res)).to_numpy(), y.to_numpy()[::-1])
        grad = rng.standard_normal((n, m)).astype(dt)
        dw, = linalg.linear_grad(T.from_numpy(grad).transpose(), X, W, want="w")
        assert np.all(np.abs(dw.to_numpy() - d(x).T @ d(grad).T) <= ref.product_bound(d(x).T, d(grad).T, u))
    x3, w = rng.standard_normal((3, 4, 5, 20)).astype(dt), rng.standard_normal((20, 9)).astype(dt)
    for X, x in ((T.from_numpy(x3), x3), (T.from_numpy(x3)[True, ::2, True, True], x3[:, ::2]), (T.from_numpy(x3).transpose(1, 0, 2, 3), x3.transpose(1, 0, 2, 3)),
                 (T.from_numpy(x3)[1, 2, 3, True], x3[1, 2, 3])):
        y = linalg.linear(X, T.from_numpy(w))
        assert y.shape == x.shape[:-1] + (9,)
        assert np.all(np.abs(y.to_numpy() - d(x) @ d(w)) <= ref.product_bound(d(x), d(w), u))
    assert linalg.linear(T(0, 20), T.from_numpy(w)).shape == (0, 9)
    dx, dw, db = linalg.linear_grad(T(0, 9), T(0, 20), T.from_numpy(w))
    assert dx.shape == (0, 20) and not dw.to_numpy().any() and not db.to_numpy().any()
    assert linalg.linear(T.from_numpy(x3), T(20, 0)).shape == (3, 4, 5, 0)
    dx, dw, db = linalg.linear_grad(T(0, 9), T(0, 20), T.from_numpy(w), activation="silu", pre=T(0, 9))
    assert dx.shape == (0, 20) and not dw.to_numpy().any() and not db.to_numpy().any()
    dx, dw, db = linalg.linear_grad(T(5, 0), T.ones(5, 20), T(20, 0), activation="silu", pre=T(5, 0))
    assert not dx.to_numpy().any() and dw.shape == (20, 0) and db.shape == (0,)


@pytest.mark.parametrize("m,k,n", [(4, 300, 500), (300, 257, 260), (512, 512, 512)])
def test_what_is_not_finite_and_what_is_far_apart(m, k, n):
    """Infinities and NaN reach the rows and columns they belong to and no others; large and tiny values keep their digits."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    x, w, bias, res, rng = data(m, k, n, np.float32, seed=2)
    base = linalg.linear(xp.SFloat.from_numpy(x), xp.SFloat.from_numpy(w), bias=xp.SFloat.from_numpy(bias)).to_numpy()
    xb, wb = x.copy(), w.copy()
    xb[1, 3], xb[2, 5], wb[7, n - 2], xb[m - 1, 9] = np.inf, np.nan, -np.inf, 3.3e38
    w9 = np.float32(0.125)
    wb[9] = w9
    got = linalg.linear(xp.SFloat.from_numpy(xb), xp.SFloat.from_numpy(wb), bias=xp.SFloat.from_numpy(bias)).to_numpy()
    with np.errstate(invalid="ignore"):
        want = d(xb) @ d(wb) + d(bias)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(np.sign(got[np.isinf(got)]), np.sign(want[np.isinf(want)]))
    fine = np.isfinite(want)
    with np.errstate(invalid="ignore"):
        bound = ref.product_bound(np.where(np.isfinite(xb), d(xb), 0), np.where(np.isfinite(wb), d(wb), 0), 2.0 ** -24) + 2.0 ** -23 * np.abs(want) + 1e-6
    assert np.all(np.abs(got - want)[fine] <= bound[fine])
    assert np.isfinite(base).all()
    # columns of x from 2^-60 to 2^60 against rows of w the other way: every product has the same weight
    scale = 2.0 ** rng.integers(-60, 61, k)
    xs, ws = (x * scale).astype(np.float32), (w / scale[:, None]).astype(np.float32)
    got = linalg.linear(xp.SFloat.from_numpy(xs), xp.SFloat.from_numpy(ws)).to_numpy()
    assert np.all(np.abs(got - d(xs) @ d(ws)) <= ref.product_bound(d(xs), d(ws), 2.0 ** -24))
    # one huge column that meets zeros
    xh, wh = x.copy(), w.copy()
    xh[:, 0], wh[0] = 1e30, 0
    got = linalg.linear(xp.SFloat.from_numpy(xh), xp.SFloat.from_numpy(wh)).to_numpy()
    assert np.all(np.abs(got - d(xh[:, 1:]) @ d(wh[1:])) <= ref.product_bound(d(xh[:, 1:]), d(wh[1:]), 2.0 ** -24))


def test_long_sums_do_not_drift():
    """Products that are all positive: additions that truncate would lean one way by their number."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    rng = np.random.default_rng(4)
    for m, k, n in ((256, 8192, 256), (1, 8192, 640), (40, 8192, 512)):
        x, w = rng.random((m, k)).astype(np.float32), rng.random((k, n)).astype(np.float32)
        got = linalg.linear(xp.SFloat.from_numpy(x), xp.SFloat.from_numpy(w)).to_numpy()
        want = d(x) @ d(w)
        # rounding to nearest: the k-th partial sum s k / K is rounded by an error uniform within u s k / K, so the sum's error
        # has a standard deviation of at most u s sqrt(K / 3) / sqrt(3) = u s sqrt(K) / 3; six of them are 2 sqrt(K) u s.
        # K additions that truncate would be off by about K / 2 u s.
        assert np.abs(got / want - 1).max() <= 2 * np.sqrt(k) * 2.0 ** -24
