"""The tensor-core product behind linear, linear_grad and orthogonalize at sizes that take each of its tiles (the tile is
chosen from the sizes; every test checks which one ran), and the recurrence at the sizes of its widest kernels."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
MUON = (3.4445, -4.7750, 2.0315)


def counts():
    from cumo_b200 import _lib

    return {(tile, sym): _lib.load().cb200_split_product_launches(tile, sym) for tile in (256, 128, 64) for sym in (0, 1)}


class Ran:
    """Which tiles were launched inside the block."""

    def __enter__(self):
        self.before = counts()
        return self

    def __exit__(self, *_):
        self.tiles = {k for k, v in counts().items() if v > self.before[k]}


def data(m, k, n, seed=0):
    rng = np.random.default_rng(seed + m + 3 * k + 7 * n)
    f = np.float32
    return (rng.standard_normal((m, k)).astype(f), (rng.standard_normal((k, n)) / np.sqrt(k)).astype(f), rng.standard_normal(n).astype(f),
            rng.standard_normal((m, n)).astype(f))


def d(a):
    return a.astype(np.float64)


# more tiles than SM pairs with remainders on every side; rows of whole packets and rows of odd lengths; K in pieces; one tile
@pytest.mark.parametrize("m,k,n,tile", [(2100, 1030, 2310, 256), (2048, 128, 2560, 256), (515, 2047, 515, 256), (1300, 200, 1100, 128), (1500, 257, 1283, 128),
                                        (900, 260, 1000, 64), (2100, 130, 2310, 256), (640, 33, 2000, 128)])
def test_linear_tiles(m, k, n, tile):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    S = xp.SFloat.from_numpy
    x, w, bias, res = data(m, k, n)
    z = d(x) @ d(w)
    ez = ref.product_bound(d(x), d(w), U)
    with Ran() as ran:
        plain = linalg.linear(S(x), S(w))
    assert ran.tiles == {(tile, 0)}
    assert np.all(np.abs(plain.to_numpy() - z) <= ez)
    for X, W in ((S(x), S(w)), (S(np.ascontiguousarray(x.T)).transpose(), S(np.ascontiguousarray(w.T)).transpose())):
        with Ran() as ran:
            y, pre = linalg.linear(X, W, bias=S(bias), activation="silu", residual=S(res), keep=True)
        assert ran.tiles == {(tile, 0)}
        zb = z + d(bias)
        eb = ez + U * np.abs(zb)
        a = ref.act(zb, "silu")
        want = a + d(res)
        assert np.all(np.abs(pre.to_numpy() - zb) <= eb)
        # the slope of silu is at most 1.2; its value is good to 8 roundings
        assert np.all(np.abs(y.to_numpy() - want) <= 1.2 * eb + 8 * U * (np.abs(a) + np.minimum(1, np.abs(zb))) + U * np.abs(want))


@pytest.mark.parametrize("m,k,n,tiles", [(2100, 130, 2310, {256}), (2049, 65, 1025, {128, 64}), (1300, 200, 1100, {128}), (1500, 257, 1283, {256}), (640, 33, 2000, {64, 128})])
def test_linear_grad_tiles(m, k, n, tiles):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    S = xp.SFloat.from_numpy
    x, w, bias, grad = data(m, k, n, seed=5)
    for name in (None, "gelu_tanh"):
        pre = (d(x) @ d(w) + d(bias)).astype(np.float32)
        args = dict(activation=name, pre=S(pre) if name else None)
        with Ran() as ran:
            dx, dw, db = linalg.linear_grad(S(grad), S(x), S(w), **args)
        assert ran.tiles == {(t, 0) for t in tiles}
        dz = d(grad) * ref.slope(d(pre), name)
        # dz: the slope good to 16 roundings of what it is made of, one more for the product
        edz = np.zeros_like(dz) if name is None else np.abs(d(grad)) * 16 * U * (1 + np.minimum(np.abs(d(pre)), 6) ** 2)
        for got, want, bound in ((dx, dz @ d(w).T, ref.product_bound(dz, d(w).T, U) + edz @ np.abs(d(w).T)),
                                 (dw, d(x).T @ dz, ref.product_bound(d(x).T, dz, U) + np.abs(d(x)).T @ edz),
                                 (db, dz.sum(0), (m + 2) * U * np.abs(dz).sum(0) + edz.sum(0))):
            assert got.shape == want.shape
            assert np.all(np.abs(got.to_numpy() - want) <= bound)
        turned = linalg.linear_grad(S(np.ascontiguousarray(grad.T)).transpose(), S(np.ascontiguousarray(x.T)).transpose(),
                                    S(np.ascontiguousarray(w.T)).transpose(), **args)
        for got, want, bound in ((turned[0], dz @ d(w).T, ref.product_bound(dz, d(w).T, U) + edz @ np.abs(d(w).T)),
                                 (turned[1], d(x).T @ dz, ref.product_bound(d(x).T, dz, U) + np.abs(d(x)).T @ edz)):
            assert np.all(np.abs(got.to_numpy() - want) <= bound)


@pytest.mark.parametrize("m,k,n", [(300, 257, 260), (1300, 200, 1100)])
@pytest.mark.parametrize("name", [None, "relu"])
def test_gradients_of_what_is_not_finite(m, k, n, name):
    """Infinities and NaN in grad, x and w reach the gradients that they belong to and no others."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    S = xp.SFloat.from_numpy
    x, w, _, grad = data(m, k, n, seed=9)
    pre = np.abs(data(m, k, n, seed=3)[3]) + np.float32(0.5)               # relu's slope is 1 everywhere but where this is turned
    pre[5, :] *= -1
    grad[1, 3], grad[2, n - 1], x[7, 4], x[m - 1, k - 1], w[6, 9], w[k - 2, 11] = np.inf, np.nan, -np.inf, np.nan, np.inf, np.nan
    grad[5, 8] = 3.0                                                       # a row of dz that relu makes zero: 0 * inf is NaN
    with Ran() as ran:
        dx, dw, db = linalg.linear_grad(S(grad), S(x), S(w), activation=name, pre=S(pre) if name else None)
    assert ran.tiles
    with np.errstate(invalid="ignore"):
        dz = d(grad) * (1.0 if name is None else (d(pre) > 0))
        wants = dz @ d(w).T, d(x).T @ dz, dz.sum(0)
        fine = [np.where(np.isfinite(a), a, 0) for a in (dz, d(x), d(w))]
        bounds = (ref.product_bound(fine[0], fine[2].T, U), ref.product_bound(fine[1].T, fine[0], U), (m + 2) * U * np.abs(fine[0]).sum(0))
    for got, want, bound in zip((dx, dw, db), wants, bounds):
        got = got.to_numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        inf = np.isinf(want)
        assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf].astype(np.float32))
        ok = np.isfinite(want)
        assert np.all(np.abs(got[ok] - want[ok]) <= bound[ok])


def in_64_bits(g, steps, coefs, eps=1e-7):
    """Newton-Schulz in 64 bits, and the same iteration in plain 32-bit arithmetic: its error is the measure below."""
    import torch

    out = []
    for dt in (torch.float64, torch.float32):
        x = torch.tensor(g, dtype=dt, device="cuda")
        x = x / (torch.sqrt((x.double() ** 2).sum((-2, -1), keepdim=True)) + eps).to(dt)
        wide = g.shape[-2] <= g.shape[-1]
        for s in range(steps):
            a, b, c = coefs
            p = x @ x.mT if wide else x.mT @ x
            q = b * p + c * (p @ p)
            x = a * x + (q @ x if wide else x @ q)
        out.append(x.double().cpu().numpy())
    return out


# the symmetric products take one side of the diagonal with square tiles; batches and tall matrices too
@pytest.mark.parametrize("shape,tiles", [((2100, 2300), {(256, 0), (256, 1)}), ((1030, 1500), {(128, 0), (128, 1)}), ((1501, 1030), {(128, 0), (128, 1)}),
                                         ((12, 384, 385), {(128, 0), (128, 1)}), ((3, 300, 500), {(64, 0)}), ((1030, 2710), {(128, 1), (256, 0)}),
                                         ((1023, 2731), {(64, 0), (256, 0)})])
def test_orthogonalize_tiles(shape, tiles):
    import torch

    import cumo_b200 as xp
    from cumo_b200 import linalg

    torch.backends.cuda.matmul.allow_tf32 = False
    g = np.random.default_rng(sum(shape)).standard_normal(shape).astype(np.float32)
    for steps in (1, 2, 5):
        want, plain = in_64_bits(g, steps, MUON)
        with Ran() as ran:
            got = linalg.orthogonalize(xp.SFloat.from_numpy(g), steps=steps).to_numpy()
        assert ran.tiles == tiles
        # numbers held to 22 to 24 bits and sums that drift no more than 32-bit ones: within four times what plain 32-bit
        # arithmetic is off by, matrix by matrix
        off, most = (np.sqrt(((a - want) ** 2).sum((-2, -1))) for a in (got, plain))
        assert np.all(off <= 4 * most)


#        shape, axis, gate shape: runs in 16-byte packets over several warps' stretches; more runs than a launch holds at once
WIDE = [((2, 100, 2400), 1, None), ((1, 70, 40, 64), 1, (1, 70, 40, 1)), ((1, 50, 40, 64), 1, None), ((1, 90, 10, 256), 1, (1, 90, 10, 1)),
        ((5000, 100), 1, None), ((5000, 300), 1, None), ((1300, 700), 1, None), ((700, 2500), 1, None)]


@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("shape,axis,gate_shape", WIDE)
def test_wide_recurrences(shape, axis, gate_shape, initial):
    import cumo_b200 as xp

    S = xp.SFloat.from_numpy
    rng = np.random.default_rng(sum(shape))
    x, grad = rng.standard_normal(shape).astype(np.float32), rng.standard_normal(shape).astype(np.float32)
    gate = rng.uniform(0.3, 1, gate_shape or shape).astype(np.float32)
    init = rng.standard_normal(shape[:axis] + shape[axis + 1:]).astype(np.float32) if initial else None
    I = S(init) if initial else None
    full = np.broadcast_to(gate, shape)
    h = S(x).gated_cumsum(S(gate), axis=axis, initial=I)
    want, mag = ref.gated(x, full, axis, init)
    assert np.all(np.abs(h.to_numpy() - want) <= ref.gated_bound(mag, full, axis, U))
    got = S(grad).gated_cumsum_grad(S(gate), h, axis=axis, initial=I)
    dx, dgate, dinit, mag, before, later = ref.gated_grad(grad, full, h.to_numpy(), axis, init)
    bound = np.flip(ref.gated_bound(np.flip(mag, axis), np.flip(later, axis), axis, U), axis)
    assert np.all(np.abs(got[0].to_numpy() - dx) <= bound)
    many = max(1, dgate.size // gate.size)
    each = bound * np.abs(before) + (many + 2) * U * mag * np.abs(before)
    assert np.all(np.abs(got[1].to_numpy() - ref.sum_to(dgate, gate.shape)) <= ref.sum_to(each, gate.shape))
    if initial:
        first = np.take(full, 0, axis).astype(np.float64)
        assert np.all(np.abs(got[2].to_numpy() - dinit) <= first * (np.take(bound, 0, axis) + 2 * U * np.take(mag, 0, axis)))


@pytest.mark.parametrize("m,k,n", [(300, 257, 260), (1300, 200, 1100), (2100, 130, 2310)])
def test_products_beyond_the_range(m, k, n):
    """Finite operands whose products leave the range of the type give infinities, not NaN, and products just inside it stay
    finite: an output is what 32-bit arithmetic makes of its operands, whatever their parts' products do on the way."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    S = xp.SFloat.from_numpy
    rng = np.random.default_rng(m)
    x, w, bias, _ = data(m, k, n, seed=4)
    sx, sw = rng.choice([-1.0, 1.0], m), rng.choice([-1.0, 1.0], n)
    big_rows, big_cols = rng.permutation(m)[: m // 3], rng.permutation(n)[: n // 4]
    x[:, 17], w[17] = 0, 0
    x[big_rows, 17] = (sx * rng.uniform(1, 2, m) * 1e30)[big_rows]
    w[17, big_cols] = (sw * rng.uniform(1, 2, n) * 1e30)[big_cols]
    huge = np.zeros((m, n), bool)
    huge[np.ix_(big_rows, big_cols)] = True
    for name in (None, "relu", "sigmoid", "tanh"):
        with Ran() as ran:
            y, pre = linalg.linear(S(x), S(w), bias=S(bias), activation=name, keep=True)
        assert ran.tiles
        pre, y = pre.to_numpy(), y.to_numpy()
        sign = np.outer(sx, sw)
        assert np.array_equal(pre[huge], np.where(sign[huge] > 0, np.inf, -np.inf))
        z = d(x) @ d(w) + d(bias)
        assert np.all(np.abs(pre - z)[~huge] <= (ref.product_bound(d(x), d(w), U) + U * np.abs(z))[~huge])
        ends = {None: (np.inf, -np.inf), "relu": (np.inf, 0), "sigmoid": (1, 0), "tanh": (1, -1)}[name]
        assert np.array_equal(y[huge], np.where(sign[huge] > 0, *ends))
    # the largest products that are still finite: 8 and fewer leading bits of their operands, rounded up, are not
    edge = np.sqrt(np.finfo(np.float32).max.astype(np.float64))
    x[big_rows, 17] = (sx * edge * (1 - rng.uniform(2.0 ** -20, 2.0 ** -8, m)))[big_rows]
    w[17, big_cols] = (sw * edge * (1 - rng.uniform(2.0 ** -20, 2.0 ** -8, n)))[big_cols]
    got = linalg.linear(S(x), S(w)).to_numpy()
    z = d(x) @ d(w)
    assert np.all(np.abs(z) < np.finfo(np.float32).max)
    assert np.all(np.abs(got - z) <= ref.product_bound(d(x), d(w), U))


@pytest.mark.parametrize("m,k,n", [(300, 257, 260), (2100, 130, 2310)])
def test_gradients_beyond_the_range(m, k, n):
    import cumo_b200 as xp
    from cumo_b200 import linalg

    S = xp.SFloat.from_numpy
    rng = np.random.default_rng(n)
    x, w, _, grad = data(m, k, n, seed=6)
    grad[:, 5], w[:, 5], x[:, 9] = 0, 0, 0
    rows, cols = rng.permutation(m)[:40], rng.permutation(k)[:30]
    rows, cols = rows[rows != 3], cols[cols != 9]
    sr, sc = rng.choice([-1.0, 1.0], m), rng.choice([-1.0, 1.0], k)
    grad[rows, 5] = (sr * rng.uniform(1, 2, m) * 1e30)[rows]
    w[cols, 5] = (sc * rng.uniform(1, 2, k) * 1e30)[cols]
    x[3, 9], grad[3] = 1e30, (rng.choice([-1.0, 1.0], n) * rng.uniform(1, 2, n) * 1e30).astype(np.float32)
    grad[3, 5] = 0
    dx, dw = linalg.linear_grad(S(grad), S(x), S(w), want=("x", "w"))
    dx, dw = dx.to_numpy(), dw.to_numpy()
    zx, zw = d(grad) @ d(w).T, d(x).T @ d(grad)
    top = np.finfo(np.float32).max
    for got, z, bound in ((dx, zx, ref.product_bound(d(grad), d(w).T, U)), (dw, zw, ref.product_bound(d(x).T, d(grad), U))):
        far = np.abs(z) > 2 * float(top)
        assert far.any() and np.array_equal(got[far], np.sign(z[far]) * np.inf)
        assert np.all(np.abs(got - z)[~far] <= bound[~far])


# kinds of matrices whose entries differ in size: what 32-bit arithmetic keeps of the small ones is kept
def uneven(kind, shape, rng):
    g = rng.standard_normal(shape).astype(np.float32)
    rows, cols = np.ones(shape[-2]), np.ones(shape[-1])
    rows[1::2], cols[::3] = 2.0 ** -17, 2.0 ** -20                   # about 1e-5 and 1e-6 of the others
    if kind == "rows":
        return (g * rows[:, None]).astype(np.float32), rows[:, None] < 1
    if kind == "columns":
        return (g * cols).astype(np.float32), np.broadcast_to(cols < 1, g.shape[-2:])
    apart = (rows[:, None] < 1) != (cols < 1)                        # two blocks that hardly touch
    return np.where(apart, g * np.float32(2.0 ** -24), g), apart


@pytest.mark.parametrize("steps", [1, 5, 15])
@pytest.mark.parametrize("shape", [(256, 512), (512, 256), (1030, 1500), (2100, 2300), (3, 300, 500)])
@pytest.mark.parametrize("kind", ["rows", "columns", "blocks"])
def test_entries_of_different_sizes(kind, shape, steps):
    """Rows, columns or blocks that are 1e-5 to 1e-7 of the rest, as dead units and rare tokens leave them: each group's error
    relative to the group itself is what plain 32-bit arithmetic's is, within the factor that roundings of another order take."""
    import torch

    import cumo_b200 as xp
    from cumo_b200 import linalg

    torch.backends.cuda.matmul.allow_tf32 = False
    g, small = uneven(kind, shape, np.random.default_rng(3 + sum(shape)))
    want, plain = in_64_bits(g, steps, MUON)
    got = linalg.orthogonalize(xp.SFloat.from_numpy(g), steps=steps).to_numpy()
    for group in (small, ~small):
        mask = np.broadcast_to(group, g.shape[-2:])
        off, most, size = (np.sqrt((a[..., mask] ** 2).sum(-1)) for a in (got - want, plain - want, want))
        assert np.all(off <= 4 * most)
        if steps == 5 and kind == "rows":
            assert np.all(off <= 2e-6 * size)


@pytest.mark.parametrize("norm", [1e-5, 1e-9, 1e-12, 1e-14, 1e-17, 1e-22])
@pytest.mark.parametrize("shape", [(200, 300), (300, 200), (40, 60)])
def test_matrices_far_below_eps(shape, norm):
    """g / (|g| + eps) is about g / eps then, however small: its digits stay."""
    import torch

    import cumo_b200 as xp
    from cumo_b200 import linalg

    torch.backends.cuda.matmul.allow_tf32 = False
    g = np.random.default_rng(7).standard_normal(shape)
    g = (g / np.linalg.norm(g) * norm).astype(np.float32)
    for steps in (1, 5):
        want, plain = in_64_bits(g, steps, MUON)
        got = linalg.orthogonalize(xp.SFloat.from_numpy(g), steps=steps).to_numpy()
        assert np.linalg.norm(got - want) <= 4 * np.linalg.norm(plain - want)


def test_more_steps_and_larger_coefficients_than_usual():
    import torch

    import cumo_b200 as xp
    from cumo_b200 import linalg

    torch.backends.cuda.matmul.allow_tf32 = False
    g = np.random.default_rng(11).standard_normal((200, 300)).astype(np.float32)
    for steps, coefs in ((70, (1.5, -0.5, 0.0)), (2, (3e6, -1e7, 8e6))):
        want, plain = in_64_bits(g, steps, coefs)
        with Ran() as ran:
            got = linalg.orthogonalize(xp.SFloat.from_numpy(g), steps=steps, coefs=coefs).to_numpy()
        assert ran.tiles == {(64, 0)}
        assert np.linalg.norm(got - want) <= 4 * np.linalg.norm(plain - want)
    # a last step close to the end of the range
    got = linalg.orthogonalize(xp.SFloat.from_numpy(g), steps=2, coefs=[(1.0, 0.0, 0.0), (3e38, 0.0, 0.0)]).to_numpy()
    x = g.astype(np.float64) / (np.linalg.norm(g.astype(np.float64)) + 1e-7)
    assert np.all(np.abs(got - 3e38 * x) <= 1e-5 * np.abs(3e38 * x))


@pytest.mark.parametrize("shape,on_planes", [((15, 300), False), ((16, 144), False), ((16, 143), True), ((143, 16), True), ((128, 1151), True), ((128, 1152), False), ((1152, 128), False),
                                             ((4, 128, 1152), False), ((5, 128, 1152), True), ((129, 2000), True), ((64, 64), True), ((40, 17, 33), True)])
def test_orthogonalize_few_rows(shape, on_planes):
    """Both sides of the rule that sends matrices of few rows and long sums to the row products."""
    import torch

    import cumo_b200 as xp
    from cumo_b200 import linalg

    torch.backends.cuda.matmul.allow_tf32 = False
    g = np.random.default_rng(sum(shape)).standard_normal(shape).astype(np.float32)
    want, plain = in_64_bits(g, 5, MUON)
    with Ran() as ran:
        got = linalg.orthogonalize(xp.SFloat.from_numpy(g)).to_numpy()
    assert bool(ran.tiles) == on_planes
    # one matrix' error varies with its values: four times 32-bit arithmetic's over the whole batch, and never above the
    # few roundings (64) that five steps' slopes of up to 3.4445 carry on from the first
    off, most = np.sqrt(((got - want) ** 2).sum()), np.sqrt(((plain - want) ** 2).sum())
    assert off <= 4 * most + 64 * U * np.sqrt((want ** 2).sum())
