"""linalg.orthogonalize against Newton-Schulz in 64 bits."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu

MUON = (3.4445, -4.7750, 2.0315)
SHAPES = [(1, 1), (1, 9), (9, 1), (5, 5), (16, 64), (64, 16), (33, 100), (100, 33), (3, 40, 60), (2, 3, 60, 40), (130, 257), (257, 130), (128, 128), (2, 256, 300)]


def bound(x, steps, coefs, u, n):
    """An error e in X becomes at most (a + 3 |b| r^2 + 5 |c| r^4) e in a step for singular values up to r, but at most max
    |p'| on the singular values themselves; each step adds three products whose random roundings are below sqrt(n) * 8 u of
    what they are made of.  In the Frobenius norm."""
    a, b, c = coefs
    t = np.linspace(0, 1.3, 500)
    slope = max(1.0, np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4)[t <= 1.21].max())
    made = abs(a) + abs(b) * 1.5 + abs(c) * 2.2
    return sum(slope ** i for i in range(steps)) * made * 8 * u * np.sqrt(n) * np.sqrt((x * x).sum((-2, -1)).max() + 1)


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("shape", SHAPES)
def test_steps(shape, dt):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    T, u = (xp.SFloat, 2.0 ** -24) if dt is np.float32 else (xp.DFloat, 2.0 ** -53)
    g = np.random.default_rng(sum(shape)).standard_normal(shape).astype(dt)
    for steps in (0, 1, 2, 5):
        got = linalg.orthogonalize(T.from_numpy(g), steps=steps)
        want = ref.ortho(g.astype(np.float64), steps, MUON, 1e-7)
        assert type(got) is T and got.shape == shape
        err = np.sqrt(((got.to_numpy() - want) ** 2).sum((-2, -1)).max())
        assert err <= (bound(want, steps, MUON, u, max(shape[-2:])) if steps else 4 * u)


@pytest.mark.parametrize("shape", [(40, 70), (300, 200), (256, 256)])
def test_rows_become_orthonormal(shape):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    rng = np.random.default_rng(0)
    q1, _ = np.linalg.qr(rng.standard_normal((shape[0], min(shape))))
    q2, _ = np.linalg.qr(rng.standard_normal((shape[1], min(shape))))
    g = ((q1 * rng.uniform(0.2, 1, min(shape))) @ q2.T).astype(np.float32)
    x = linalg.orthogonalize(xp.SFloat.from_numpy(g)).to_numpy().astype(np.float64)
    s = np.linalg.svd(x, compute_uv=False)
    assert s.min() > 0.6 and s.max() < 1.25
    # the convergent cubic, to the end: the polar factor itself
    x = linalg.orthogonalize(xp.SFloat.from_numpy(g), steps=25, coefs=(1.5, -0.5, 0.0)).to_numpy()
    # every singular value has stopped at 1 and its slope there is 0: what is left is the last step's own rounding
    assert np.linalg.norm(x - q1 @ q2.T) <= 64 * 2.0 ** -24 * np.sqrt(max(shape) * min(shape))


def test_views_batches_and_schedules():
    import cumo_b200 as xp
    from cumo_b200 import linalg

    g = np.random.default_rng(8).standard_normal((4, 3, 50, 41)).astype(np.float32)
    G = xp.SFloat.from_numpy(g)
    for V, v in ((G[::2, True, True, True], g[::2]), (G.transpose(0, 1, 3, 2), g.transpose(0, 1, 3, 2)), (G.transpose(1, 0, 2, 3), g.transpose(1, 0, 2, 3)),
                 (G[1, 2, ::-1, 3:], g[1, 2, ::-1, 3:])):
        got = linalg.orthogonalize(V, steps=3).to_numpy()
        assert np.array_equal(got, linalg.orthogonalize(xp.SFloat.from_numpy(np.ascontiguousarray(v)), steps=3).to_numpy())
    coefs = [(4.0, -6.0, 3.0), (3.0, -3.5, 1.3), (1.875, -1.25, 0.375)]
    got = linalg.orthogonalize(G, steps=3, coefs=coefs).to_numpy()
    want = ref.ortho(g.astype(np.float64), 3, coefs, 1e-7)
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want) * 4.0 * 3.0 * 1.875     # 2^-24 * sqrt(50) * 8 is 3e-6
    assert linalg.orthogonalize(xp.SFloat(3, 0, 4)).shape == (3, 0, 4)


def test_sizes_of_values():
    """Zero, tiny, huge and non-finite matrices; each matrix of a batch stands for itself."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    g = np.random.default_rng(9).standard_normal((5, 40, 60)).astype(np.float32)
    plain = linalg.orthogonalize(xp.SFloat.from_numpy(g), eps=0.0).to_numpy()
    h = g.copy()
    h[1] *= 2.0 ** 100
    h[2] *= 2.0 ** -100
    h[3] = 0
    h[4, 5, 6] = np.inf
    got = linalg.orthogonalize(xp.SFloat.from_numpy(h), eps=1e-40).to_numpy()
    assert np.array_equal(got[:3], plain[:3])                     # powers of two leave every digit alone
    assert not got[3].any() and np.isnan(got[4]).all()


@pytest.mark.parametrize("shape", [(40, 60), (60, 40), (2, 3, 17, 30)])
def test_sizes_of_values_in_double_precision(shape):
    """Norms whose squares are beyond 64 bits, above and below, and matrices that hold both."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    D = xp.DFloat.from_numpy
    g = np.random.default_rng(12).standard_normal(shape)
    plain = linalg.orthogonalize(D(g), eps=0.0).to_numpy()
    for power in (600, 1015, -600, -1000):                       # powers of two leave every digit alone
        assert np.array_equal(linalg.orthogonalize(D(np.ldexp(g, power)), eps=0.0).to_numpy(), plain)
    tol = 64 * 2.0 ** -53 * 3.4445 ** 5 * np.abs(plain).max()     # the norm's sum in another order: a few roundings, carried through five steps
    for power in (500, 501, -500, -499):
        assert np.abs(linalg.orthogonalize(D(np.ldexp(g, power)), eps=0.0).to_numpy() - plain).max() <= tol
    # eps counts at any size: g / (|g| + |g|) is half of g / |g|
    norm = np.sqrt((g * g).sum((-2, -1))).max()
    for power in (0, 700, -700):
        got = linalg.orthogonalize(D(np.ldexp(g, power)), steps=0, eps=float(np.ldexp(norm, power))).to_numpy()
        n = np.sqrt((g * g).sum((-2, -1), keepdims=True))
        assert np.abs(got - g / (n + norm)).max() <= 16 * 2.0 ** -53
    # far below eps: g / eps
    got = linalg.orthogonalize(D(np.ldexp(g, -700)), steps=0, eps=2.0 ** -100).to_numpy()
    assert np.abs(got - np.ldexp(g, -600)).max() <= 16 * 2.0 ** -53 * 2.0 ** -600 * np.abs(g).max()
    # one entry above everything else by more than the type's own range of squares; zero stays zero
    h = g.copy()
    h[..., 3, 5] = 2.0 ** 800
    got = linalg.orthogonalize(D(h), steps=0, eps=0.0).to_numpy()
    assert np.all(got[..., 3, 5] == 1)
    got[..., 3, 5] = 0
    want = np.ldexp(g, -800)
    want[..., 3, 5] = 0
    assert np.abs(got - want).max() <= 16 * 2.0 ** -53 * 2.0 ** -800 * np.abs(g).max()
    h[...] = 0
    assert not linalg.orthogonalize(D(h), eps=1e-300).to_numpy().any()
    h[..., 0, 0] = np.inf
    assert np.isnan(linalg.orthogonalize(D(h), eps=1e-300).to_numpy()).all()
