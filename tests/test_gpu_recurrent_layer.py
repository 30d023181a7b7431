"""The operators as one layer uses them: a gated recurrence between two linear layers, its training step, decoding token by
token, and the ways a program runs it -- streams, threads, captured graphs, arrays beyond 2^32 bytes."""
import threading

import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu


def layer(xp, linalg, X, p):
    """x -> silu linear -> gated sums (gates from another linear, one per head) -> linear + x; everything the backward needs."""
    b, t, d = X.shape
    heads, width = p["heads"], p["width"]
    u, upre = linalg.linear(X, p["wu"], bias=p["bu"], activation="silu", keep=True)
    a, apre = linalg.linear(X, p["wa"], bias=p["ba"], activation="sigmoid", keep=True)
    h = u.reshape(b, t, heads, width).gated_cumsum(a.reshape(b, t, heads, 1), axis=1, initial=p["state"])
    y = linalg.linear(h.reshape(b, t, heads * width), p["wo"], residual=X)
    return y, (u, upre, a, apre, h)


def layer_grad(xp, linalg, G, X, p, saved):
    b, t, d = X.shape
    heads, width = p["heads"], p["width"]
    u, upre, a, apre, h = saved
    dh, dwo = linalg.linear_grad(G, h.reshape(b, t, heads * width), p["wo"], want=("x", "w"))
    du, da, dstate = dh.reshape(b, t, heads, width).gated_cumsum_grad(a.reshape(b, t, heads, 1), h, axis=1, initial=p["state"])
    dx1, dwu, dbu = linalg.linear_grad(du.reshape(b, t, heads * width), X, p["wu"], activation="silu", pre=upre)
    dx2, dwa, dba = linalg.linear_grad(da.reshape(b, t, heads), X, p["wa"], activation="sigmoid", pre=apre)
    return {"x": dx1 + dx2 + G, "wu": dwu, "bu": dbu, "wa": dwa, "ba": dba, "wo": dwo, "state": dstate}


def params(rng, d, heads, width, dt):
    e = heads * width
    return {"wu": (rng.standard_normal((d, e)) / np.sqrt(d)).astype(dt), "bu": rng.standard_normal(e).astype(dt),
            "wa": (rng.standard_normal((d, heads)) / np.sqrt(d)).astype(dt), "ba": (rng.standard_normal(heads) + 2).astype(dt),
            "wo": (rng.standard_normal((e, d)) / np.sqrt(e)).astype(dt), "state": rng.standard_normal((heads, width)).astype(dt)}


@pytest.mark.parametrize("b,t,d,heads,width", [(2, 37, 24, 3, 8), (1, 300, 96, 4, 64), (3, 129, 130, 2, 33)])
@pytest.mark.parametrize("dt", [np.float64, np.float32])
def test_training_step(b, t, d, heads, width, dt):
    """Every gradient of the layer against automatic differentiation in 64 bits, then the orthogonalised update."""
    import torch

    import cumo_b200 as xp
    from cumo_b200 import linalg

    rng = np.random.default_rng(b + t)
    T = xp.SFloat if dt is np.float32 else xp.DFloat
    x, host = rng.standard_normal((b, t, d)).astype(dt), params(rng, d, heads, width, dt)
    grad = rng.standard_normal((b, t, d)).astype(dt)
    p = {k: T.from_numpy(v) for k, v in host.items()}
    p.update(heads=heads, width=width)
    X, G = T.from_numpy(x), T.from_numpy(grad)
    y, saved = layer(xp, linalg, X, p)
    got = layer_grad(xp, linalg, G, X, p, saved)

    q = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in {**host, "x": x}.items()}
    u = torch.nn.functional.silu(q["x"] @ q["wu"] + q["bu"]).reshape(b, t, heads, width)
    a = torch.sigmoid(q["x"] @ q["wa"] + q["ba"]).reshape(b, t, heads, 1)
    h, steps = q["state"].expand(b, heads, width), []
    for i in range(t):
        h = a[:, i] * h + u[:, i]
        steps.append(h)
    want = torch.stack(steps, 1).reshape(b, t, heads * width) @ q["wo"] + q["x"]
    want.backward(torch.tensor(grad, dtype=torch.float64))
    # Sums of up to b * t (or a product's K) terms behind sums of up to t steps: relative to the norms, roundings of random sign
    # grow as the square root of their number, below u * sqrt(2000) per stage, five stages, and a factor of ten between a norm and
    # what it is made of.
    tol = 10 * 5 * 45 * ref.U[np.dtype(dt)]

    def near(g, w):
        return np.linalg.norm(g.to_numpy() - w) <= tol * np.linalg.norm(w)

    assert near(y, want.detach().numpy())
    for name, g in got.items():
        w = q[name].grad.numpy()
        assert g.shape == w.shape and near(g, w), name
    for name in ("wu", "wo"):
        step = linalg.orthogonalize(got[name], steps=3)
        exact = ref.ortho(got[name].to_numpy().astype(np.float64), 3, (3.4445, -4.7750, 2.0315), 1e-7)
        assert np.linalg.norm(step.to_numpy() - exact) <= 40 * tol * np.linalg.norm(exact)      # slopes of up to 3.4445 in each step
        moved = p[name] - step * 0.02
        assert np.isfinite(moved.to_numpy()).all()


def test_decoding_follows_the_whole_sequence():
    """Token by token with the state carried, against the prompt in one pass."""
    import cumo_b200 as xp
    from cumo_b200 import linalg

    rng = np.random.default_rng(5)
    b, t, d, heads, width = 3, 21, 64, 2, 32
    host = params(rng, d, heads, width, np.float32)
    p = {k: xp.SFloat.from_numpy(v) for k, v in host.items()}
    p.update(heads=heads, width=width)
    x = rng.standard_normal((b, t, d)).astype(np.float32)
    X = xp.SFloat.from_numpy(x)
    whole = layer(xp, linalg, X, p)[0].to_numpy()
    for i in range(t):
        y, saved = layer(xp, linalg, X[True, i:i + 1, True], p)
        p["state"] = saved[-1][True, 0, True, True]
        assert np.abs(y.to_numpy()[:, 0] - whole[:, i]).max() <= 64 * 2.0 ** -24 * np.abs(whole).max() * 8   # sums of 64 in another order


def test_graphs_and_streams():
    """Captured once, replayed on new inputs; two graphs of one call replayed at the same time keep their scratch apart."""
    import torch

    import cumo_b200 as xp
    from cumo_b200 import _lib, linalg

    lib = _lib.load()
    S = xp.SFloat.from_torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    sets, graphs, outs = [], [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(2):
        v = {"x": r(300, 260), "w": r(260, 514) / 16, "gate": torch.sigmoid(r(2, 150, 514)), "g": r(2, 96, 200), "grad": r(300, 514), "pre": r(300, 514)}
        sets.append(v)
        torch.cuda.synchronize()

        def work(v=v):
            y = linalg.linear(S(v["x"]), S(v["w"]), activation="gelu")
            h = y.reshape(2, 150, 514).gated_cumsum(S(v["gate"]), axis=1)
            return [y, h, *linalg.linear_grad(S(v["grad"]), S(v["x"]), S(v["w"]), activation="silu", pre=S(v["pre"])), linalg.orthogonalize(S(v["g"]))]

        with torch.cuda.stream(streams[k]):
            lib.cb200_set_stream(streams[k].cuda_stream)
            try:
                for _ in range(2):
                    work()                                     # fills the stream's pool: a capture may not allocate
                streams[k].synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=streams[k]):
                    outs.append(work())
                graphs.append(graph)
            finally:
                lib.cb200_set_stream(None)
    for turn in range(3):
        for v in sets:
            for t in v.values():
                t.copy_(torch.sigmoid(r(*t.shape)) if t is v["gate"] else r(*t.shape) / 4)
        torch.cuda.synchronize()
        for _ in range(4):
            for k in range(2):
                with torch.cuda.stream(streams[k]):
                    graphs[k].replay()
        torch.cuda.synchronize()
        for k, v in enumerate(sets):
            y = linalg.linear(S(v["x"]), S(v["w"]), activation="gelu")
            want = [y, y.reshape(2, 150, 514).gated_cumsum(S(v["gate"]), axis=1),
                    *linalg.linear_grad(S(v["grad"]), S(v["x"]), S(v["w"]), activation="silu", pre=S(v["pre"])), linalg.orthogonalize(S(v["g"]))]
            for a, b in zip(outs[k], want):
                assert np.array_equal(a.to_numpy(), b.to_numpy())
    assert lib.cb200_product_status() == 0


def test_a_capture_refuses_temporaries():
    import torch

    import cumo_b200 as xp
    from cumo_b200 import _lib, linalg

    lib = _lib.load()
    x, w = torch.randn(4, 5, 6, 32, device="cuda"), torch.randn(32, 16, device="cuda")
    X, W = xp.SFloat.from_torch(x).transpose(1, 0, 2, 3), xp.SFloat.from_torch(w)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        lib.cb200_set_stream(stream.cuda_stream)
        try:
            assert linalg.linear(X, W).shape == (5, 4, 6, 16)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                with pytest.raises(xp.CudaError):
                    linalg.linear(X, W)
                kept = linalg.linear(xp.SFloat.from_torch(x), W)
            graph.replay()
            stream.synchronize()
        finally:
            lib.cb200_set_stream(None)
    assert np.allclose(kept.to_numpy(), (x.double() @ w.double()).cpu().numpy(), atol=1e-4)


def test_threads_on_their_own_streams():
    import torch

    import cumo_b200 as xp
    from cumo_b200 import _lib, linalg

    lib = _lib.load()
    rng = np.random.default_rng(0)
    x, w, g = rng.standard_normal((200, 300)).astype(np.float32), rng.standard_normal((300, 400)).astype(np.float32), rng.standard_normal((100, 160)).astype(np.float32)
    X, W, G = (xp.SFloat.from_numpy(a) for a in (x, w, g))
    want = [linalg.linear(X, W, activation="tanh").to_numpy(), linalg.orthogonalize(G).to_numpy(), X.gated_cumsum(0.5, axis=0).to_numpy()]
    errors = []

    def body():
        stream = torch.cuda.Stream()
        lib.cb200_set_stream(stream.cuda_stream)
        try:
            for _ in range(20):
                got = [linalg.linear(X, W, activation="tanh"), linalg.orthogonalize(G), X.gated_cumsum(xp.SFloat.ones(1) * 0.5, axis=0)]
                stream.synchronize()
                for a, b in zip(got, want):
                    if not np.array_equal(a.to_numpy(), b):
                        errors.append("differs")
        except Exception as e:                                  # noqa: BLE001 -- a thread's exception must reach the test
            errors.append(repr(e))
        finally:
            lib.cb200_set_stream(None)

    threads = [threading.Thread(target=body) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


def test_beyond_32_bits():
    """Sums over an array of more than 2^32 bytes: the last steps agree with those taken from the state in front of them."""
    import torch

    import cumo_b200 as xp

    t, c = 1_100_003, 1024
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(1, t, c, device="cuda", generator=gen)
    gate = torch.rand(1, t, c, device="cuda", generator=gen)
    X, G = xp.SFloat.from_torch(x), xp.SFloat.from_torch(gate)
    h = torch.as_tensor(X.gated_cumsum(G, axis=1), device="cuda")
    tail = 777
    again = torch.as_tensor(xp.SFloat.from_torch(x[:, -tail:]).gated_cumsum(xp.SFloat.from_torch(gate[:, -tail:]), axis=1,
                                                                            initial=xp.SFloat.from_torch(h[:, -tail - 1])), device="cuda")
    scale = float(h[:, -tail:].abs().max())
    assert float((again - h[:, -tail:]).abs().max()) <= 16 * 2.0 ** -24 * scale
    state, want = h[0, t // 2 - 1].double(), []
    for i in range(5):
        state = gate[0, t // 2 + i].double() * state + x[0, t // 2 + i].double()
        want.append(state)
    assert float((torch.stack(want) - h[0, t // 2:t // 2 + 5].double()).abs().max()) <= 16 * 2.0 ** -24 * scale


def test_a_wait_that_ran_out_is_reported_by_every_operator():
    """Once the word is up, whatever its size and plan, each operator refuses until the status has been asked for."""
    import cumo_b200 as xp
    from cumo_b200 import _lib, linalg

    lib = _lib.load()
    f32 = lambda *s: xp.SFloat.ones(*s)
    f64 = lambda *s: xp.DFloat.ones(*s)
    calls = [lambda: f32(2, 3).gated_cumsum(0.5, axis=1), lambda: f32(1, 5000, 32).gated_cumsum(f32(1, 5000, 32), axis=1),
             lambda: f64(4, 900).gated_cumsum_grad(f64(4, 900), f64(4, 900), axis=1), lambda: linalg.linear(f32(1, 64), f32(64, 8)),
             lambda: linalg.linear(f32(300, 300), f32(300, 300)), lambda: linalg.linear(f64(9, 10), f64(10, 11)),
             lambda: linalg.linear_grad(f32(3, 5), f32(3, 4), f32(4, 5)), lambda: linalg.linear_grad(f32(3, 5), f32(3, 4), f32(4, 5), want="bias"),
             lambda: linalg.orthogonalize(f32(5, 7)), lambda: linalg.orthogonalize(f32(200, 300)), lambda: linalg.orthogonalize(f64(5, 7))]
    assert lib.cb200_product_status() == 0
    for call in calls:
        call()
        assert lib.cb200_product_status_set() == 0
        for _ in range(2):
            with pytest.raises(xp.CudaError, match="bounded wait"):
                call()
        assert lib.cb200_product_status() == 1 and lib.cb200_product_status() == 0
        call()
    assert (f32(2, 2) + f32(2, 2)).to_numpy().sum() == 8          # nothing is latched for what comes next
