"""Matrix products: SFloat on the tensor cores, DFloat and the batched / transposed / alpha-beta forms through
`cb200_{s,d}gemm_strided_batched` (the argument list of the cuBLAS call in the reference's gemm.c:277-296).

`dot(a, b)` is the reference's `a.dot(b)` on float matrices (ext/cumo/narray/gen/tmpl/gemm.c:252-297 hands it to
cuBLAS).  `gemm_nt` calls `cb200_sgemm_nt_tc` directly: a tcgen05 kernel that keeps fp32-grade accuracy by splitting
every operand into two TF32 numbers and wants both operands with K contiguous.
"""
from __future__ import annotations

from ctypes import byref, c_char_p, c_double, c_int, c_int64, c_size_t, c_void_p, create_string_buffer

from . import _lib
from .narray import CumoError, DFloat, SFloat, ShapeError, _raise_last


def gemm_nt(a: SFloat, bt: SFloat) -> SFloat:
    """a (M, K) . bt (N, K)^T -> (M, N).  Rows must be contiguous (the row steps may be larger than K)."""
    if not (isinstance(a, SFloat) and isinstance(bt, SFloat) and a.ndim == 2 and bt.ndim == 2 and a.shape[1] == bt.shape[1]):
        raise TypeError("gemm_nt needs SFloat a (M, K) and bt (N, K)")
    if not a.contiguous():
        a = a.dup()
    if not bt.contiguous():
        bt = bt.dup()
    m, k = a.shape
    n = bt.shape[0]
    out = SFloat(m, n)
    fn = _lib.load().cb200_sgemm_nt_tc
    fn.restype = c_int
    fn.argtypes = [c_int64, c_int64, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_char_p, c_size_t]
    err = create_string_buffer(256)
    if fn(m, n, k, a.data_ptr, k, bt.data_ptr, k, out.data_ptr, n, err, len(err)):
        raise CumoError(err.value.decode())
    return out


def gemm(a, b, alpha=1.0, beta=0.0, c=None):
    """The reference's `Cumo::NArray#gemm` for SFloat / DFloat operands (row-major, the last two axes are the
    matrices, leading axes are batches; either operand may be a transposed view; an operand that holds one matrix is
    used for every batch of the other): alpha * a . b + beta * c.
    It hands cuBLAS's column-major bookkeeping to the library exactly as gemm.c does: c^T = b^T . a^T."""
    from ctypes import c_float, c_longlong

    T = type(a)
    if T not in (SFloat, DFloat) or type(b) is not T or a.ndim < 2 or b.ndim < 2:
        raise TypeError("gemm needs two SFloat or two DFloat arrays of two or more dimensions")
    m, k = a.shape[-2:]
    k2, n = b.shape[-2:]
    if k != k2:
        raise ShapeError(f"shape mismatch: {a.shape} . {b.shape}")
    if 0 in (m, n, k):
        raise ShapeError("gemm of an empty operand")
    batch_a, batch_b = a.shape[:-2], b.shape[:-2]
    if batch_a and batch_b and batch_a != batch_b:
        raise ShapeError(f"batch dimensions differ: {batch_a} and {batch_b}")
    batch_shape = batch_a or batch_b                       # (gemm.c takes them from whichever operand has them)
    es = 4 if T is SFloat else 8

    def layout(x):
        """(array usable as it is or a contiguous copy, trans flag, leading dimension, batch stride in elements)"""
        st = x.steps
        rows, cols = x.shape[-2:]
        batch_ok = all(st[d] == (x.shape[d + 1] * st[d + 1] if d + 1 < x.ndim - 2 else rows * cols * es) for d in range(x.ndim - 2))
        stride = rows * cols if x.ndim > 2 else 0          # one matrix serves every batch
        if batch_ok and st[-1] == es and st[-2] >= cols * es and st[-2] % es == 0 and (x.ndim == 2 or st[-2] == cols * es):
            return x, 0, st[-2] // es, stride               # row-major: column-major of its transpose, no flag
        if batch_ok and st[-2] == es and st[-1] >= rows * es and st[-1] % es == 0 and (x.ndim == 2 or st[-1] == rows * es):
            return x, 1, st[-1] // es, stride               # a transposed view: flag T
        y = x.dup()
        return y, 0, cols, stride
    a2, ta, lda, sa = layout(a)
    b2, tb, ldb, sb = layout(b)
    batch = 1
    for d in batch_shape:
        batch *= d
    if c is not None and tuple(c.shape) != tuple(batch_shape) + (m, n):
        raise ShapeError(f"c has shape {c.shape}, the product {tuple(batch_shape) + (m, n)}")
    out = T(*batch_shape, m, n) if c is None or beta == 0.0 else c.dup()
    lib = _lib.load()
    fn = lib.cb200_sgemm_strided_batched if T is SFloat else lib.cb200_dgemm_strided_batched
    fn.restype = c_int
    fn.argtypes = None
    cT = c_float if T is SFloat else c_double
    rc = fn(c_int(tb), c_int(ta), c_int(n), c_int(m), c_int(k), byref(cT(alpha)), c_void_p(b2.data_ptr), c_int(ldb), c_longlong(sb),
            c_void_p(a2.data_ptr), c_int(lda), c_longlong(sa), byref(cT(beta)), c_void_p(out.data_ptr), c_int(n), c_longlong(m * n), c_int(batch))
    if rc:
        raise CumoError(f"gemm failed with status {rc}")
    return out


def dot(a, b):
    """a (M, K) . b (K, N) -> (M, N); a 1-D second operand gives (M,).  Both SFloat or both DFloat: the reference's
    `dot` on float matrices is `gemm` (lib/cumo/narray/extra.rb:1145-1196).  Large single-precision products run on the
    tensor cores, the rest on the CUDA-core kernel."""
    if not ((isinstance(a, SFloat) and isinstance(b, SFloat)) or (isinstance(a, DFloat) and isinstance(b, DFloat))):
        raise TypeError("dot is built for two SFloat or two DFloat operands (NArray#dot takes the other types)")
    return a.dot(b)


# ---- the linear layer --------------------------------------------------------------------------------------------------
ACTIVATIONS = (None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid", "tanh")     # their numbers in the library


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}, not {name!r}")
    return ACTIVATIONS.index(name)


def _check_types(T, **operands):
    if T not in (SFloat, DFloat):
        raise TypeError("the operands must be SFloat or DFloat arrays")
    for name, x in operands.items():
        if x is not None and type(x) is not T:
            raise TypeError(f"{name} is {type(x).__name__}, the other operands are {T.__name__}")


def _handle(x):
    return None if x is None else x._h


def linear(x, w, bias=None, activation=None, residual=None, keep=False):
    """act(x . w + bias) + residual in one pass: x (..., K), w (K, N) -> (..., N), all SFloat or all DFloat, every operand
    an array or any view of one (a transposed `w` is not copied).  `bias` (N,) and `residual` (repeated to the result's
    shape) may be left out; `activation` is None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid" or "tanh".  With `keep`
    also returns the value in front of the activation, which linear_grad needs."""
    _check_types(type(x), w=w, bias=bias, residual=residual)
    if w is None:
        raise TypeError("linear needs w")
    act = _activation(activation)
    pre = c_void_p()
    y = type(x)._from_handle(_lib.load().cb200_na_linear(x._h, w._h, _handle(bias), act, _handle(residual), byref(pre) if keep else None))
    return (y, type(x)._from_handle(pre.value)) if keep else y


def linear_grad(grad, x, w, activation=None, pre=None, want=("x", "w", "bias")):
    """The gradients of `y, pre = linear(x, w, bias, activation, residual, keep=True)` for grad = dL/dy (..., N): a tuple of
    those that `want` names, in its order -- "x" in x's shape, "w" in w's, "bias" (N,).  (The residual's gradient is grad.)
    `pre` may be left out when there is no activation.  Sums run in a fixed order: the same operands give the same bits."""
    _check_types(type(grad), x=x, w=w, pre=pre)
    if x is None or w is None:
        raise TypeError("linear_grad needs x and w")
    act = _activation(activation)
    want = (want,) if isinstance(want, str) else tuple(want)
    if not want or len(set(want)) != len(want) or not set(want) <= {"x", "w", "bias"}:
        raise ValueError('want names some of "x", "w" and "bias", each once')
    out = {name: c_void_p() for name in want}
    if _lib.load().cb200_na_linear_grad(grad._h, x._h, w._h, act, _handle(pre), *(byref(out[name]) if name in out else None for name in ("x", "w", "bias"))):
        _raise_last()
    return tuple(type(grad)._from_handle(out[name].value) for name in want)


def orthogonalize(g, steps=5, coefs=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """Every matrix of the last two axes taken towards the nearest matrix with orthonormal rows (columns, if it has fewer):
    X = g / (|g|_F + eps), then `steps` times X <- a X + (b P + c P P) X with P = X X^T, the smaller of the two products
    being taken.  `coefs` is one triple (a, b, c) for every step or a list of one triple per step.  With the default triple,
    which is quick but does not converge, five steps bring singular values above some thousandths of the norm to between 0.7
    and 1.2."""
    _check_types(type(g))
    if g.ndim < 2:
        raise ShapeError("orthogonalize needs an array of two or more dimensions")
    if not isinstance(steps, int) or isinstance(steps, bool) or steps < 0:
        raise ValueError("steps must be a number of steps")
    coefs = list(coefs)
    triples = [tuple(float(c) for c in t) for t in (coefs if not coefs or hasattr(coefs[0], "__len__") else [coefs] * steps)]
    if len(triples) != steps or any(len(t) != 3 for t in triples):
        raise ValueError("coefs must be three numbers, or three numbers for each step")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    flat = [c for t in triples for c in t]
    return type(g)._from_handle(_lib.load().cb200_na_orthogonalize(g._h, steps, (c_double * max(1, len(flat)))(*flat), eps))
