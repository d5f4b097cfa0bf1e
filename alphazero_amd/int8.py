"""Evaluation of layers in 8-bit integers: rows quantised with one scale each, products with a scale for each row and each
output channel.  Torch tensors in, torch tensors out, on the current stream of the tensors' device; everything is computed by
the HIP kernels of csrc/az_int8.hip (include/azamd.h: az_i8_*).  Inference only: no backward pass.
"""
import torch

from . import _abi
from ._abi import AzError, check, lib
from ._tensors import DTYPES, no_grad, rows_of, same_device, stream_of, vector, workspace, written

MAX_K = 131071   # the longest sum of products of two 8-bit integers that int32 holds


def quantize_rows(x, index=None):
    """(q int8 [rows, cols], scale float32 [rows]): scale = max|x| * (1/127), q = x / scale to the nearest integer.

    x: [rows, cols] float32 / float16 / bfloat16 with contiguous rows.  index: int32 [rows, taps] -- row r of q is then
    x[index[r, 0]], x[index[r, 1]], ... one after the other under one scale; an index outside x stands for zeros."""
    dtype = DTYPES.get(x.dtype)
    if dtype is None:
        raise AzError("quantize_rows: x must be float32, float16 or bfloat16")
    no_grad("quantize_rows", x)
    n_src, cols, ld = rows_of(x, "quantize_rows", "x")
    dev = same_device("quantize_rows", x, index)
    if cols < 1:
        raise AzError("quantize_rows: x has no columns")
    if index is None:
        rows, taps, where = n_src, 1, None
    else:
        if index.dtype is not torch.int32 or index.dim() != 2 or not index.is_contiguous() or index.shape[1] < 1:
            raise AzError("quantize_rows: index must be a contiguous int32 [rows, taps]")
        (rows, taps), where = index.shape, index.data_ptr()
    q = torch.empty((rows, taps * cols), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib().az_i8_quantize_dev(dev, dtype, rows, cols, x.data_ptr(), ld, n_src, where, taps, q.data_ptr(), taps * cols,
                                   scale.data_ptr(), stream_of(dev)))
    return q, scale


def _layer(what, m, k, w, w_scale, bias, residual, act, dtype, out):
    """the arguments that matmul and linear share, checked: n, the output, and the tail of the C call up to ld_y"""
    if w.dtype is not torch.int8:
        raise AzError("%s: w must be int8" % what)
    n, k_w, ld_w = rows_of(w, what, "w")
    if k_w != k:
        raise AzError("%s: x has %d columns, w has %d" % (what, k, k_w))
    if not 1 <= k <= MAX_K:
        raise AzError("%s: between 1 and %d columns" % (what, MAX_K))
    code, fn = DTYPES.get(dtype), _abi.ACTS.get(act)
    if code is None:
        raise AzError("%s: dtype must be float32, float16 or bfloat16" % what)
    if fn is None:
        raise AzError("%s: act must be one of %s" % (what, ", ".join(sorted(_abi.ACTS))))
    ws = vector(w_scale, n, what, "w_scale")
    b = None if bias is None else vector(bias, n, what, "bias")
    res, ld_res = None, 0
    if residual is not None:
        r_m, r_n, ld_res = rows_of(residual, what, "residual")
        if residual.dtype is not dtype or r_m != m or r_n != n:
            raise AzError("%s: residual must be [%d, %d] of the output's dtype" % (what, m, n))
        res = residual.data_ptr()
    if out is None:
        out, ld_y = torch.empty((m, n), dtype=dtype, device=w.device), n
    else:
        o_m, o_n, ld_y = rows_of(out, what, "out")
        if out.dtype is not dtype or o_m != m or o_n != n:
            raise AzError("%s: out must be [%d, %d] of the output's dtype" % (what, m, n))
    return n, w.data_ptr(), ld_w, out, (ws, b, res, ld_res, fn, code, out.data_ptr(), ld_y)


def matmul(q, scale, w, w_scale, bias=None, residual=None, act="none", dtype=torch.float32, out=None):
    """act(scale[m] * w_scale[n] * (q @ w.T)[m, n] + bias[n] + residual[m, n]) of `dtype` [m, n].

    q int8 [m, k], w int8 [n, k] with contiguous rows; scale [m], w_scale [n], bias [n] float32; residual [m, n] of `dtype`
    (may be `out` itself; `out` overlaps nothing else); act: "none", "relu" or "silu".  Integer sums are exact, the rest is float32, rounded once."""
    if q.dtype is not torch.int8:
        raise AzError("matmul: q must be int8")
    m, k, ld_q = rows_of(q, "matmul", "q")
    no_grad("matmul", scale, w_scale, bias, residual, out)
    dev = same_device("matmul", q, scale, w, w_scale, bias, residual, out)
    s = vector(scale, m, "matmul", "scale")
    given = out is not None
    n, wp, ld_w, out, tail = _layer("matmul", m, k, w, w_scale, bias, residual, act, dtype, out)
    L, qp = lib(), q.data_ptr()
    nws = L.az_i8_matmul_ws(m, n, k, qp, ld_q, wp, ld_w)
    ws, wsp = workspace(nws, q)
    check(L.az_i8_matmul_dev(dev, m, n, k, qp, ld_q, s, wp, ld_w, *tail, wsp, nws, stream_of(dev)))
    if given:
        written(out)
    return out


def linear(x, w, w_scale, bias=None, residual=None, act="none", out=None):
    """quantize_rows(x), then matmul with the result; the output has x's dtype."""
    if x.dtype not in DTYPES:
        raise AzError("linear: x must be float32, float16 or bfloat16")
    m, k, ld_x = rows_of(x, "linear", "x")
    no_grad("linear", x, w_scale, bias, residual, out)
    dev = same_device("linear", x, w, w_scale, bias, residual, out)
    given = out is not None
    n, wp, ld_w, out, tail = _layer("linear", m, k, w, w_scale, bias, residual, act, x.dtype, out)
    L, xp = lib(), x.data_ptr()
    nws = L.az_i8_linear_ws(m, n, k, wp, ld_w)
    ws, wsp = workspace(nws, x)
    check(L.az_i8_linear_dev(dev, m, n, k, xp, ld_x, wp, ld_w, *tail, wsp, nws, stream_of(dev)))
    if given:
        written(out)
    return out
