"""Orthogonalised updates of weight matrices (csrc/az_ortho.hip; include/azamd.h: az_orthogonalize_dev, az_muon_step_dev), for
the training step between ReplayBuffer.dataloader and CNN.sync_from.
"""
import ctypes as C

import torch

from . import _abi
from ._abi import AzError, check, lib
from ._tensors import DTYPES, address, need, no_grad, same_device, stream_of, workspace

COEFFS = (3.4445, -4.7750, 2.0315)


def _coeffs(coeffs):
    need(len(coeffs) == 3, "coeffs must be (a, b, c)")
    return (C.c_double * 3)(*[float(c) for c in coeffs])


def orthogonalize(g, steps=5, coeffs=COEFFS, eps=1e-7, out=None):
    """The orthogonalisation of every matrix g[..., rows, cols] by `steps` Newton-Schulz products (float32-accurate):
    X = G / (||G||_F + eps), X <- a X + (b A + c A^2) X with A = X X^T.  out: a contiguous tensor like g (may be g)."""
    need(g.dtype in DTYPES, "orthogonalize: g must be float32, float16 or bfloat16")
    need(g.dim() >= 2, "orthogonalize: g must have at least two dimensions")
    no_grad("orthogonalize", g)
    dev = same_device("orthogonalize", g, out)
    rows, cols = g.shape[-2:]
    batch = 1
    for d in g.shape[:-2]:
        batch *= d
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    need(out.dtype == g.dtype and out.shape == g.shape and out.is_contiguous(),
         "orthogonalize: out must be contiguous, of g's shape and dtype")
    if batch * rows * cols == 0:
        return out
    g = g.contiguous()
    L = lib()
    ws = workspace(L.az_orthogonalize_ws(batch, rows, cols), g.device)
    check(L.az_orthogonalize_dev(dev, DTYPES[g.dtype], batch, rows, cols, address(g), address(out), int(steps), _coeffs(coeffs),
                                 float(eps), address(ws), ws.numel(), stream_of(dev)))
    return out


def muon_step(weights, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coeffs=COEFFS, eps=1e-7):
    """One update, in place, of weight matrices by orthogonalised momentum; for each of them

        m <- momentum m + (1 - momentum) g;   u = momentum m + (1 - momentum) g if nesterov else m
        w <- (1 - lr weight_decay) w - lr sqrt(max(1, rows / cols)) orthogonalize(u)

    weights, grads: lists of contiguous tensors [rows, ...] of one dtype, seen as [rows, rest]; momenta: float32 of the same
    shapes.  No tensor may appear twice among weights and momenta."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    need(len(weights) == len(grads) == len(momenta), "muon_step: as many gradients and momenta as weights")
    if not weights:
        return
    dt = weights[0].dtype
    need(dt in DTYPES, "muon_step: weights must be float32, float16 or bfloat16")
    dev = same_device("muon_step", *weights, *grads, *momenta)
    items = (_abi.az_muon_item * len(weights))()
    for it, w, g, m in zip(items, weights, grads, momenta):
        need(w.dim() >= 2 and w.numel() > 0, "muon_step: weights must have at least two dimensions and no empty one")
        need(w.dtype == dt and g.dtype == dt and m.dtype == torch.float32,
             "muon_step: weights and gradients of one dtype, momenta of float32")
        need(w.shape == g.shape == m.shape, "muon_step: weights, gradients and momenta must have the same shapes")
        need(w.is_contiguous() and g.is_contiguous() and m.is_contiguous(), "muon_step: tensors must be contiguous")
        it.w_dev, it.g_dev, it.m_dev = address(w), address(g), address(m)
        it.rows, it.cols = w.shape[0], w.numel() // w.shape[0]
    L = lib()
    ws = workspace(L.az_muon_step_ws(items, len(weights)), weights[0].device)
    check(L.az_muon_step_dev(dev, DTYPES[dt], items, len(weights), float(lr), float(momentum), 1 if nesterov else 0,
                             float(weight_decay), int(steps), _coeffs(coeffs), float(eps), address(ws), ws.numel(),
                             stream_of(dev)))
