"""Plain 64-bit forms of the sequence and layer operators, in numpy, and the error bounds the tests compare with.

u is half a step of the type (2^-24 / 2^-53): the largest relative error of one rounding."""
import math

import numpy as np

U = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float64): 2.0 ** -53}


def gated(x, gate, axis, initial=None):
    """h, and the same recurrence over magnitudes (what the bounds scale with)."""
    x = np.moveaxis(np.asarray(x, np.float64), axis, 0)
    if np.ndim(gate) == 0 or gate.ndim < x.ndim:
        gate = np.reshape(gate, (1,) * (x.ndim - np.ndim(gate)) + np.shape(gate))
    a = np.moveaxis(np.broadcast_to(np.asarray(gate, np.float64), np.moveaxis(x, 0, axis).shape), axis, 0)
    h, mag = np.empty_like(x), np.empty_like(x)
    state = None if initial is None else np.broadcast_to(np.asarray(initial, np.float64), x.shape[1:])
    m = None if state is None else np.abs(state)
    for t in range(x.shape[0]):
        state = x[t] if state is None else a[t] * state + x[t]
        m = np.abs(x[t]) if m is None else np.abs(a[t]) * m + np.abs(x[t])
        h[t], mag[t] = state, m
    return np.moveaxis(h, 0, axis), np.moveaxis(mag, 0, axis)


def gated_bound(mag, gate, axis, u):
    """Every step rounds once, and the state in front of a stretch is rounded, composed from a product and a sum: at most
    four roundings per step relative to the magnitudes, carried on by the gates."""
    return gated(4 * u * mag, np.abs(np.asarray(gate, np.float64)), axis)[0]


def gated_grad(grad, gate, h, axis, initial=None):
    """(dx, dgate over the full shape, dinitial or None) and the magnitudes of dx."""
    g = np.flip(np.asarray(grad, np.float64), axis)
    full = np.broadcast_to(np.asarray(gate, np.float64), g.shape)
    later = np.concatenate([np.take(full, range(1, full.shape[axis]), axis), np.zeros_like(np.take(full, [0], axis))], axis)
    dx, mag = gated(g, np.flip(later, axis), axis)
    dx, mag = np.flip(dx, axis), np.flip(mag, axis)
    first = np.zeros_like(np.take(dx, [0], axis)) if initial is None else np.expand_dims(np.broadcast_to(np.asarray(initial, np.float64), np.take(dx, 0, axis).shape), axis)
    before = np.concatenate([first, np.take(np.asarray(h, np.float64), range(0, dx.shape[axis] - 1), axis)], axis)
    return dx, dx * before, (None if initial is None else np.take(full, 0, axis) * np.take(dx, 0, axis)), mag, before, later


def sum_to(a, shape):
    while a.ndim > len(shape):
        a = a.sum(0)
    for d, n in enumerate(shape):
        if n == 1 and a.shape[d] != 1:
            a = a.sum(d, keepdims=True)
    return a


def erfc(x):
    return np.vectorize(math.erfc, otypes=[np.float64])(x)


def logistic(z):
    return np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))


ROOT = 2 * math.sqrt(2 / math.pi)


def act(z, name):
    return {None: lambda: z, "relu": lambda: np.maximum(z, 0), "silu": lambda: z * logistic(z), "gelu": lambda: 0.5 * z * erfc(-z / math.sqrt(2)),
            "gelu_tanh": lambda: z * logistic(ROOT * (z + 0.044715 * z ** 3)), "sigmoid": lambda: logistic(z), "tanh": lambda: np.tanh(z)}[name]()


def slope(z, name):
    def tanh_form():
        p = logistic(ROOT * (z + 0.044715 * z ** 3))
        return p + z * p * (1 - p) * ROOT * (1 + 3 * 0.044715 * z * z)
    return {None: lambda: np.ones_like(z), "relu": lambda: (z > 0) * 1.0, "silu": lambda: logistic(z) * (1 + z * (1 - logistic(z))),
            "gelu": lambda: 0.5 * erfc(-z / math.sqrt(2)) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), "gelu_tanh": tanh_form,
            "sigmoid": lambda: logistic(z) * (1 - logistic(z)), "tanh": lambda: 1 - np.tanh(z) ** 2}[name]()


def product_bound(a, b, u):
    """|error| of an element of a . b: K products and K additions, each rounded (or, on the tensor cores, 6 K / 16 additions
    that truncate, twice the error each, and operands held to at least 2 u in their parts)."""
    k = a.shape[-1]
    return (k + 16) * u * (np.abs(a) @ np.abs(b))


def ortho(g, steps, coefs, eps):
    x = g / (np.sqrt((g * g).sum((-2, -1), keepdims=True)) + eps)
    wide = g.shape[-2] <= g.shape[-1]
    for s in range(steps):
        a, b, c = coefs[s] if hasattr(coefs[0], "__len__") else coefs
        p = x @ np.swapaxes(x, -1, -2) if wide else np.swapaxes(x, -1, -2) @ x
        q = b * p + c * (p @ p)
        x = a * x + (q @ x if wide else x @ q)
    return x
