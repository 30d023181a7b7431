"""What the sequence and layer operators cost: gated running sums along an axis (`gated_cumsum` and its gradients), the
linear layer with its epilogue (`linalg.linear` and its gradients) and the orthogonalised update
(`linalg.orthogonalize`), each as a program that trains or serves such a layer calls it.

`own` picks between the plain form in elementary torch operations (False) and this package's operators (True); both take
the torch tensors that `prepare` makes and return torch tensors."""
import math

import torch

own = False

SFLOAT, DFLOAT = "sfloat", "dfloat"
TYPES = {SFLOAT: torch.float32, DFLOAT: torch.float64}
MUON = (3.4445, -4.7750, 2.0315)          # the quintic whose five steps send singular values in (0, 1] near 1


# ---- the cases ---------------------------------------------------------------------------------------------------------
def _gated(batch, time, channels, head=0, **more):
    """`head`: channels that share one gate (0: every channel has its own).  `time_last`: the layout (batch, channels, time)."""
    return {"op": "gated", "batch": batch, "time": time, "channels": channels, "head": head, "time_last": False,
            "initial": True, "grad": False, "type": SFLOAT, **more}


def _linear(rows, inputs, outputs, **more):
    return {"op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "activation": "none", "bias": True,
            "residual": False, "grad": False, "w_transposed": False, "type": SFLOAT, **more}


def _ortho(batch, rows, columns, **more):
    return {"op": "ortho", "batch": batch, "rows": rows, "columns": columns, "steps": 5, **more}


def listed():
    return [
        # one new token for each of 128 sequences: the state goes one step on
        {"name": "gated_token", **_gated(128, 1, 2048)},
        # a long document through a layer of 2048 channels, too few sequences to fill a GPU without cutting time
        {"name": "gated_long", **_gated(1, 50000, 2048, initial=False)},
        # a signal bank in double precision with time as the contiguous axis and an odd length
        {"name": "gated_signal_f64", **_gated(257, 10007, 1, time_last=True, type=DFLOAT)},
        # the backward pass of a training batch whose channels each have a gate
        {"name": "gated_grad", **_gated(8, 4096, 1024, initial=False, grad=True)},
        # the same where 64 channels of a head share one gate and a carried state has a gradient too
        {"name": "gated_grad_heads", **_gated(4, 4096, 2048, head=64, grad=True)},
        # one token through a layer's output product: the weights are read once, the rest is latency
        {"name": "linear_token", **_linear(1, 4096, 4096, activation="silu", residual=True)},
        # a small prompt with odd sizes
        {"name": "linear_prompt", **_linear(251, 2047, 2731, activation="gelu")},
        # a training batch, forward
        {"name": "linear_batch", **_linear(8192, 4096, 4096, activation="gelu_tanh", residual=True)},
        # a training batch, backward: gradients of the inputs, the weights and the bias
        {"name": "linear_grad", **_linear(4096, 2048, 4096, activation="silu", grad=True)},
        # the update of eight small projections at once
        {"name": "ortho_heads", **_ortho(8, 256, 1024)},
        # a tall weight of odd sizes
        {"name": "ortho_tall", **_ortho(1, 2731, 1023)},
        # a square weight of a wide layer
        {"name": "ortho_square", **_ortho(1, 4096, 4096)},
    ]


def _spread(rng, low, high):
    """A size whose logarithm is uniform; two of three are left as they fall, odd or even, one is a multiple of 64 where it can be."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n >= 128 and rng.random() < 0.34:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["gated", "gated", "linear", "linear", "ortho"])
    if op == "gated":
        head = rng.choice([0, 0, 16, 64, 128])
        time_last = rng.random() < 0.3
        time = _spread(rng, 1, 50000)
        batch, channels = _spread(rng, 1, 256), _spread(rng, 1, 4096)
        if head and not time_last:
            channels = max(1, channels // head) * head
        else:
            head = 0
        most = 1 << 25
        while batch * time * channels > most and batch > 1:
            batch = (batch + 1) // 2
        time = max(1, min(time, most // (batch * channels)))
        return _gated(batch, time, channels, head, time_last=time_last, initial=rng.random() < 0.5, grad=rng.random() < 0.5,
                      type=rng.choice([SFLOAT, SFLOAT, DFLOAT]))
    if op == "linear":
        rows, inputs, outputs = _spread(rng, 1, 8192), _spread(rng, 32, 4096), _spread(rng, 32, 4096)
        return _linear(rows, inputs, outputs, activation=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid", "tanh"]),
                       bias=rng.random() < 0.7, residual=rng.random() < 0.5, grad=rng.random() < 0.4, w_transposed=rng.random() < 0.3)
    rows, columns = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
    batch = _spread(rng, 1, 16) if rows * columns < 1 << 19 else 1
    return _ortho(batch, rows, columns)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, dtype=dtype, generator=gen)

    s = {"case": dict(case)}
    if case["op"] == "gated":
        dt = TYPES[case["type"]]
        b, t, c, h = case["batch"], case["time"], case["channels"], case["head"]
        if h:
            shape, gate_shape, state_shape = (b, t, c // h, h), (b, t, c // h, 1), (b, c // h, h)
        elif case["time_last"]:
            shape, gate_shape, state_shape = (b, c, t), (b, c, t), (b, c)
        else:
            shape, gate_shape, state_shape = (b, t, c), (b, t, c), (b, c)
        s["axis"] = 2 if case["time_last"] and not h else 1
        s["x"] = normal(*shape, dtype=dt)
        s["gate"] = torch.sigmoid(normal(*gate_shape, dtype=dt) + 3.0)       # decays of about 0.7 to 0.995
        s["initial"] = normal(*state_shape, dtype=dt) if case["initial"] else None
        if case["grad"]:
            s["h"] = _gated_plain(s["x"], s["gate"], s["initial"], s["axis"])  # what the forward pass left
            s["grad"] = normal(*shape, dtype=dt)
    elif case["op"] == "linear":
        dt = TYPES[case["type"]]
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        s["x"] = normal(m, k, dtype=dt)
        w = normal(n, k, dtype=dt).t() if case["w_transposed"] else normal(k, n, dtype=dt)
        s["w"] = w.mul_(1.0 / math.sqrt(k))
        s["bias"] = normal(n, dtype=dt) * 0.1 if case["bias"] else None
        s["residual"] = normal(m, n, dtype=dt) if case["residual"] and not case["grad"] else None
        if case["grad"]:
            s["grad"] = normal(m, n, dtype=dt)
            s["pre"] = s["x"] @ s["w"] if s["bias"] is None else s["x"] @ s["w"] + s["bias"]
    else:
        # an update as momentum leaves it: a few strong directions over noise
        b, m, n = case["batch"], case["rows"], case["columns"]
        r = min(8, m, n)
        s["g"] = normal(b, m, n) * 0.02 + (normal(b, m, r) @ normal(b, r, n)) * 0.02
    return s


# ---- the plain form ----------------------------------------------------------------------------------------------------
def _gated_plain(x, gate, initial, axis):
    """h[t] = gate[t] * h[t-1] + x[t], by doubling: after the step of distance d every element covers 2d inputs."""
    h = x.movedim(axis, 0).clone()
    a = gate.movedim(axis, 0).expand_as(h).clone()
    if initial is not None:
        h[0] += a[0] * initial
    d = 1
    while d < h.shape[0]:
        h[d:] = h[d:] + a[d:] * h[:-d]
        a[d:] = a[d:] * a[:-d]
        d *= 2
    return h.movedim(0, axis).contiguous()


def _gated_grad_plain(grad, gate, h, initial, axis):
    g, a, y = grad.movedim(axis, 0), gate.movedim(axis, 0), h.movedim(axis, 0)
    later = torch.cat([a[1:], torch.zeros_like(a[:1])])                       # dh[t] = grad[t] + gate[t+1] * dh[t+1]
    dh = _gated_plain(g.flip(0), later.flip(0), None, 0).flip(0)
    first = torch.zeros_like(y[:1]) if initial is None else initial[None]
    dgate = dh * torch.cat([first, y[:-1]])
    if a.shape != y.shape:
        dgate = dgate.sum(-1, keepdim=True)
    out = [dh.movedim(0, axis).contiguous(), dgate.movedim(0, axis).contiguous()]
    if initial is not None:
        out.append(a[0] * dh[0])
    return out


def _activate(z, name):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if name == "tanh":
        return torch.tanh(z)
    return z


def _slope(z, name):
    """The activation's derivative."""
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 - p)
    if name == "tanh":
        t = torch.tanh(z)
        return 1 - t * t
    return torch.ones_like(z)


def _linear_plain(x, w, bias, activation, residual):
    z = x @ w
    if bias is not None:
        z = z + bias
    y = _activate(z, activation)
    return y if residual is None else y + residual


def _linear_grad_plain(grad, x, w, pre, activation, with_bias):
    dz = grad * _slope(pre, activation)
    out = [dz @ w.t(), x.t() @ dz]
    if with_bias:
        out.append(dz.sum(0))
    return out


def _ortho_plain(g, steps, coefs, eps):
    x = g.transpose(-1, -2) if g.shape[-2] > g.shape[-1] else g
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + eps)
    a, b, c = coefs
    for _ in range(steps):
        p = x @ x.transpose(-1, -2)
        x = a * x + (b * p + c * (p @ p)) @ x
    return (x.transpose(-1, -2) if g.shape[-2] > g.shape[-1] else x).contiguous()


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "gated":
        if c["grad"]:
            return _gated_grad_plain(s["grad"], s["gate"], s["h"], s["initial"], s["axis"])
        return _gated_plain(s["x"], s["gate"], s["initial"], s["axis"])
    if c["op"] == "linear":
        if c["grad"]:
            return _linear_grad_plain(s["grad"], s["x"], s["w"], s["pre"], c["activation"], c["bias"])
        return _linear_plain(s["x"], s["w"], s["bias"], c["activation"], s["residual"])
    return _ortho_plain(s["g"], c["steps"], MUON, 1e-7)


def _run_own(s, c):
    from cumo_b200 import DFloat, SFloat, linalg

    T = DFloat if c.get("type") == DFLOAT else SFloat

    def arr(t):
        return None if t is None else T.from_torch(t)

    def back(a):
        return torch.as_tensor(a, device="cuda")

    if c["op"] == "gated":
        if c["grad"]:
            got = arr(s["grad"]).gated_cumsum_grad(arr(s["gate"]), arr(s["h"]), axis=s["axis"], initial=arr(s["initial"]))
            return [back(a) for a in got]
        return back(arr(s["x"]).gated_cumsum(arr(s["gate"]), axis=s["axis"], initial=arr(s["initial"])))
    activation = None if c.get("activation") == "none" else c.get("activation")
    if c["op"] == "linear":
        if c["grad"]:
            want = ("x", "w", "bias") if c["bias"] else ("x", "w")
            got = linalg.linear_grad(arr(s["grad"]), arr(s["x"]), arr(s["w"]), activation=activation,
                                     pre=arr(s["pre"]) if activation else None, want=want)
            return [back(a) for a in got]
        return back(linalg.linear(arr(s["x"]), arr(s["w"]), bias=arr(s["bias"]), activation=activation, residual=arr(s["residual"])))
    return back(linalg.orthogonalize(arr(s["g"]), steps=c["steps"], coefs=MUON, eps=1e-7))


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "gated":
        size = 8 if case["type"] == DFLOAT else 4
        n = case["batch"] * case["time"] * case["channels"]
        gates = n // case["head"] if case["head"] else n
        state = case["batch"] * case["channels"] if case["initial"] else 0
        if case["grad"]:        # reads grad, gate, h (and initial), writes dx, dgate (and dinitial)
            return {"bytes": size * (3 * n + 2 * gates + 2 * state), "flops": 3 * n}
        return {"bytes": size * (2 * n + gates + state), "flops": 2 * n}
    if case["op"] == "linear":
        size = 8 if case["type"] == DFLOAT else 4
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        if case["grad"]:        # reads grad, x, w (and pre), writes dx, dw (and dbias)
            pre = 0 if case["activation"] == "none" else m * n
            return {"bytes": size * (m * n + pre + 2 * m * k + 2 * k * n + (n if case["bias"] else 0)), "flops": 4 * m * k * n}
        return {"bytes": size * (m * k + k * n + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)), "flops": 2 * m * k * n}
    b, m, n = case["batch"], min(case["rows"], case["columns"]), max(case["rows"], case["columns"])
    # per step x.x^T and p.p, both symmetric (half the products), and one full product with x
    return {"bytes": 8 * b * m * n, "flops": b * case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if torch.is_tensor(v) else v for k, v in s.items()}
    if case["op"] == "gated":
        axis, t = s["axis"], case["time"]
        if t > 100000:
            return None
        gate = d["gate"]
        if not case["grad"]:
            x = d["x"]
            out = torch.empty_like(x)
            state = d["initial"]
            for i in range(t):                              # the definition, one step after the other
                step = x.select(axis, i)
                state = step if state is None else gate.select(axis, i) * state + step
                out.select(axis, i).copy_(state)
            return out
        grad, h = d["grad"], d["h"]
        dx, dgate = torch.empty_like(grad), torch.empty_like(gate)
        carried = None
        for i in range(t - 1, -1, -1):
            step = grad.select(axis, i)
            dh = step if carried is None else carried + step
            dx.select(axis, i).copy_(dh)
            before = h.select(axis, i - 1) if i else d["initial"]
            product = torch.zeros_like(dh) if before is None else dh * before
            dgate.select(axis, i).copy_(product.sum(-1, keepdim=True) if case["head"] else product)
            carried = gate.select(axis, i) * dh
        return [dx, dgate] if d["initial"] is None else [dx, dgate, carried]
    if case["op"] == "linear":
        name = case["activation"]
        if not case["grad"]:
            z = d["x"].matmul(d["w"])
            z = z if d["bias"] is None else z.add(d["bias"])
            y = z if name == "none" else _defined(z, name)
            return y if d["residual"] is None else y.add(d["residual"])
        if name == "none":
            dz = d["grad"]
        else:
            z = d["pre"].requires_grad_(True)
            dz, = torch.autograd.grad(_defined(z, name), z, d["grad"])
        got = [torch.einsum("mn,kn->mk", dz, d["w"]), torch.einsum("mk,mn->kn", d["x"], dz)]
        return got + [dz.sum(dim=0)] if case["bias"] else got
    g = d["g"]
    x = g / (torch.linalg.matrix_norm(g, keepdim=True) + 1e-7)
    wide = g.shape[-2] <= g.shape[-1]
    for _ in range(case["steps"]):
        p = torch.matmul(x, x.mT) if wide else torch.matmul(x.mT, x)
        q = MUON[1] * p + MUON[2] * torch.matmul(p, p)
        x = MUON[0] * x + (torch.matmul(q, x) if wide else torch.matmul(x, q))
    return x


def _defined(z, name):
    return {"relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v), "sigmoid": torch.sigmoid, "tanh": torch.tanh,
            "gelu": lambda v: v * torch.special.ndtr(v),
            "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}[name](z)
