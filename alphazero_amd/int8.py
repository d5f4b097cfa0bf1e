"""Evaluation of layers in 8-bit integers: rows quantised with one scale each, products with a scale for each row and each
output channel.  Torch tensors in, torch tensors out, on the current stream of the tensors' device; everything is computed by
the HIP kernels of csrc/az_int8.hip (include/azamd.h: az_i8_*).  Inference only: no backward pass.
"""
import torch

from . import _abi
from ._abi import AzError, check, lib
from ._tensors import DTYPES, address, need, no_grad, rows_of, same_device, stream_of, workspace

MAX_K = 131071   # the longest sum of products of two 8-bit integers that int32 holds


def quantize_rows(x, index=None):
    """(q int8 [rows, cols], scale float32 [rows]): scale = max|x| * (1/127), q = x / scale to the nearest integer.

    x: [rows, cols] float32 / float16 / bfloat16 with contiguous rows.  index: int32 [rows, taps] -- row r of q is then
    x[index[r, 0]], x[index[r, 1]], ... one after the other under one scale; an index outside x stands for zeros."""
    need(x.dtype in DTYPES, "quantize_rows: x must be float32, float16 or bfloat16")
    no_grad("quantize_rows", x)
    ld = rows_of(x, "quantize_rows: x")
    dev = same_device("quantize_rows", x, index)
    n_src, cols = x.shape
    need(cols >= 1, "quantize_rows: x has no columns")
    rows, taps = n_src, 1
    if index is not None:
        need(index.dtype == torch.int32 and index.dim() == 2 and index.is_contiguous() and index.shape[1] >= 1,
             "quantize_rows: index must be a contiguous int32 [rows, taps]")
        rows, taps = index.shape
    q = torch.empty((rows, taps * cols), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib().az_i8_quantize_dev(dev, DTYPES[x.dtype], rows, cols, address(x), ld, n_src, address(index), taps, address(q),
                                   taps * cols, address(scale), stream_of(dev)))
    return q, scale


def _layer(what, m, k, w, w_scale, bias, residual, act, dtype, out):
    need(w.dtype == torch.int8, "%s: w must be int8" % what)
    ld_w = rows_of(w, "%s: w" % what)
    n = w.shape[0]
    need(w.shape[1] == k, "%s: x has %d columns, w has %d" % (what, k, w.shape[1]))
    need(1 <= k <= MAX_K, "%s: between 1 and %d columns" % (what, MAX_K))
    need(dtype in DTYPES, "%s: dtype must be float32, float16 or bfloat16" % what)
    need(act in _abi.ACTS, "%s: act must be one of %s" % (what, ", ".join(sorted(_abi.ACTS))))
    for t, size, name in ((w_scale, n, "w_scale"), (bias, n, "bias")):
        need(t is None or (t.dtype == torch.float32 and tuple(t.shape) == (size,) and t.is_contiguous()),
             "%s: %s must be a contiguous float32 [%d]" % (what, name, size))
    ld_res = 0
    if residual is not None:
        need(residual.dtype == dtype and tuple(residual.shape) == (m, n), "%s: residual must be [%d, %d] of the output's dtype"
             % (what, m, n))
        ld_res = rows_of(residual, "%s: residual" % what)
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=w.device)
    need(out.dtype == dtype and tuple(out.shape) == (m, n), "%s: out must be [%d, %d] of the output's dtype" % (what, m, n))
    return n, ld_w, ld_res, out, rows_of(out, "%s: out" % what)


def matmul(q, scale, w, w_scale, bias=None, residual=None, act="none", dtype=torch.float32, out=None):
    """act(scale[m] * w_scale[n] * (q @ w.T)[m, n] + bias[n] + residual[m, n]) of `dtype` [m, n].

    q int8 [m, k], w int8 [n, k] with contiguous rows; scale [m], w_scale [n], bias [n] float32; residual [m, n] of `dtype`
    (may be `out` itself); act: "none", "relu" or "silu".  Integer sums are exact, the rest is float32, rounded once."""
    need(q.dtype == torch.int8, "matmul: q must be int8")
    ld_q = rows_of(q, "matmul: q")
    m, k = q.shape
    need(scale.dtype == torch.float32 and tuple(scale.shape) == (m,) and scale.is_contiguous(),
         "matmul: scale must be a contiguous float32 [%d]" % m)
    no_grad("matmul", scale, w_scale, bias, residual)
    dev = same_device("matmul", q, scale, w, w_scale, bias, residual, out)
    n, ld_w, ld_res, out, ld_y = _layer("matmul", m, k, w, w_scale, bias, residual, act, dtype, out)
    L = lib()
    nws = L.az_i8_matmul_ws(m, n, k)
    ws = workspace(nws, q.device)
    check(L.az_i8_matmul_dev(dev, m, n, k, address(q), ld_q, address(scale), address(w), ld_w, address(w_scale), address(bias),
                             address(residual), ld_res, _abi.ACTS[act], DTYPES[dtype], address(out), ld_y, address(ws),
                             ws.numel(), stream_of(dev)))
    return out


def linear(x, w, w_scale, bias=None, residual=None, act="none", out=None):
    """quantize_rows(x), then matmul with the result; the output has x's dtype."""
    need(x.dtype in DTYPES, "linear: x must be float32, float16 or bfloat16")
    no_grad("linear", x, w_scale, bias, residual)
    ld_x = rows_of(x, "linear: x")
    m, k = x.shape
    dev = same_device("linear", x, w, w_scale, bias, residual, out)
    n, ld_w, ld_res, out, ld_y = _layer("linear", m, k, w, w_scale, bias, residual, act, x.dtype, out)
    need(out.data_ptr() != x.data_ptr() or m * n == 0, "linear: out must not be x")
    L = lib()
    ws = workspace(L.az_i8_linear_ws(m, n, k), x.device)
    check(L.az_i8_linear_dev(dev, m, n, k, address(x), ld_x, address(w), ld_w, address(w_scale), address(bias),
                             address(residual), ld_res, _abi.ACTS[act], DTYPES[x.dtype], address(out), ld_y, address(ws),
                             ws.numel(), stream_of(dev)))
    return out
