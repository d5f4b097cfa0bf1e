"""Orthogonalised updates of weight matrices (csrc/az_ortho.hip; include/azamd.h: az_orthogonalize_dev, az_muon_step_dev), for
the training step between ReplayBuffer.dataloader and CNN.sync_from.  The method, momentum orthogonalised by a quintic Newton-Schulz
iteration with these coefficients, was published as Muon (K. Jordan and others, 2024).
"""
import ctypes as C

import torch

from . import _abi
from ._abi import AzError, check, lib
from ._tensors import DTYPES, no_grad, same_device, stream_of, workspace, written

COEFFS = (3.4445, -4.7750, 2.0315)
MAX_DIM = 32768   # of a matrix


def _coeffs(coeffs):
    if len(coeffs) != 3:
        raise AzError("coeffs must be (a, b, c)")
    return (C.c_double * 3)(*coeffs)


def orthogonalize(g, steps=5, coeffs=COEFFS, eps=1e-7, out=None):
    """The orthogonalisation of every matrix g[..., rows, cols] by `steps` Newton-Schulz products (float32-accurate):
    X = G / (||G||_F + eps), X <- a X + (b A + c A^2) X with A = X X^T.  out: a contiguous tensor like g (may be g).
    Values of X are held to 2^-39 at best: of a matrix whose norm is 10^-4 of eps or less, fewer bits than float32's remain."""
    if g.dtype not in DTYPES or g.dim() < 2:
        raise AzError("orthogonalize: g must be float32, float16 or bfloat16 of at least two dimensions")
    no_grad("orthogonalize", g, out)
    dev = same_device("orthogonalize", g, out)
    rows, cols = g.shape[-2:]
    if out is None:
        out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    elif out.dtype is not g.dtype or out.shape != g.shape or not out.is_contiguous():
        raise AzError("orthogonalize: out must be contiguous, of g's shape and dtype")
    if g.numel() == 0:
        return out
    batch = g.numel() // (rows * cols)
    g = g.contiguous()
    L = lib()
    nws = L.az_orthogonalize_ws(batch, rows, cols)
    ws, wsp = workspace(nws, g)
    check(L.az_orthogonalize_dev(dev, DTYPES[g.dtype], batch, rows, cols, g.data_ptr(), out.data_ptr(), steps, _coeffs(coeffs),
                                 eps, wsp, nws, stream_of(dev)))
    written(out)
    return out


def _items(weights, grads, momenta):
    """the tensors of a muon_step call, checked: (device, dtype code, items)"""
    n = len(weights)
    if len(grads) != n or len(momenta) != n:
        raise AzError("muon_step: as many gradients and momenta as weights")
    if n == 0:
        return None, None, None
    dt = weights[0].dtype
    if dt not in DTYPES:
        raise AzError("muon_step: weights must be float32, float16 or bfloat16")
    dev = same_device("muon_step", *weights, *grads, *momenta)
    items = (_abi.az_muon_item * n)()
    for it, w, g, m in zip(items, weights, grads, momenta):
        if w.dim() < 2 or w.numel() == 0:
            raise AzError("muon_step: weights must have at least two dimensions and no empty one")
        if w.dtype is not dt or g.dtype is not dt or m.dtype is not torch.float32:
            raise AzError("muon_step: weights and gradients of one dtype, momenta of float32")
        if w.shape != g.shape or w.shape != m.shape:
            raise AzError("muon_step: weights, gradients and momenta must have the same shapes")
        if not (w.is_contiguous() and g.is_contiguous() and m.is_contiguous()):
            raise AzError("muon_step: tensors must be contiguous")
        it.w_dev, it.g_dev, it.m_dev = w.data_ptr(), g.data_ptr(), m.data_ptr()
        it.rows = rows = w.shape[0]
        it.cols = w.numel() // rows
    return dev, DTYPES[dt], items


def _update(dev, code, items, weights, momenta, lr, momentum, nesterov, weight_decay, steps, coeffs, eps):
    L, n = lib(), len(weights)
    nws = L.az_muon_step_ws(items, n)
    ws, wsp = workspace(nws, weights[0])
    check(L.az_muon_step_dev(dev, code, items, n, lr, momentum, 1 if nesterov else 0, weight_decay, steps, _coeffs(coeffs),
                             eps, wsp, nws, stream_of(dev)))
    written(*weights, *momenta)


def muon_step(weights, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coeffs=COEFFS, eps=1e-7):
    """One update, in place, of weight matrices by orthogonalised momentum; for each of them

        m <- momentum m + (1 - momentum) g;   u = momentum m + (1 - momentum) g if nesterov else m
        w <- (1 - lr weight_decay) w - lr sqrt(max(1, rows / cols)) orthogonalize(u)

    weights, grads: lists of contiguous tensors [rows, ...] of one dtype, seen as [rows, rest]; momenta: float32 of the same
    shapes.  No weight or momentum may overlap another one or a gradient.  Float32 weights come out the same, bit for bit, whatever else
    is in the lists; 16-bit ones may differ in their last bits (several steps at once, where the lists as a whole gain by it)."""
    dev, code, items = _items(weights, grads, momenta)
    if items is not None:
        _update(dev, code, items, weights, momenta, lr, momentum, nesterov, weight_decay, steps, coeffs, eps)


class Muon(torch.optim.Optimizer):
    """torch optimiser around muon_step, for the matrices and convolutions of a network that is trained beside the engine (the
    reference's Base.train_step calls self.opt, NetworkBase.py:26-62): weights of at least two dimensions in any memory format, seen as
    [out, rest], both up to 32768.  Biases and norms belong to another optimiser (`matrices_of` tells them apart).  Momenta are float32."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coeffs=COEFFS, eps=1e-7):
        if not lr >= 0.0:
            raise ValueError("Muon: bad lr %r" % (lr,))
        if not 0.0 <= momentum < 1.0:
            raise ValueError("Muon: bad momentum %r" % (momentum,))
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coeffs=tuple(coeffs), eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2 or p.dtype not in DTYPES or max(p.shape[0], p[:1].numel()) > MAX_DIM:
                del self.param_groups[-1]
                raise ValueError("Muon takes float32, float16 or bfloat16 weights of at least two dimensions, [out, rest] up to %d, not %s %s"
                                 % (MAX_DIM, tuple(p.shape), p.dtype))

    @torch.no_grad()
    def step(self, closure=None):
        """All weights that have a gradient, or, where one is refused, none of them."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = []   # one for the weights of a group, device and dtype
        for group in self.param_groups:
            lists = {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                if p.grad.is_sparse:
                    raise AzError("Muon: sparse gradients are not supported")
                m = self.state[p].get("momentum") if p in self.state else None
                if m is None:
                    m = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                at = lists.setdefault((p.device, p.dtype), ([], [], [], []))
                at[0].append(p)
                at[1].append(p.detach().contiguous())     # itself, but of one in another memory format
                at[2].append(p.grad.detach().to(p.dtype).contiguous())
                at[3].append(m)
            hyper = {k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "coeffs", "eps")}
            calls += [(at, _items(*at[1:]), hyper) for at in lists.values()]
        if len(calls) > 1:   # a single call is refused whole by itself
            for _, (_, code, items), h in calls:
                check(lib().az_muon_step_check(code, items, len(items), h["lr"], h["momentum"], h["weight_decay"], h["steps"],
                                               _coeffs(h["coeffs"]), h["eps"]))
        for (params, weights, _, momenta), (dev, code, items), hyper in calls:
            _update(dev, code, items, weights, momenta, **hyper)
            for p, w, m in zip(params, weights, momenta):
                self.state[p]["momentum"] = m
                if w.data_ptr() != p.data_ptr():
                    p.copy_(w)
        return loss

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)   # casts a state to its parameter's dtype; the momenta stay float32
        saved = state_dict["state"]
        order = [p for group in self.param_groups for p in group["params"]]
        names = [i for group in state_dict["param_groups"] for i in group["params"]]
        for p, i in zip(order, names):
            if i in saved and "momentum" in saved[i]:
                self.state[p]["momentum"] = saved[i]["momentum"].detach().to(device=p.device, dtype=torch.float32, copy=True)


def matrices_of(module):
    """(weights for Muon, the other parameters) of a module: of at least two dimensions, or not"""
    params = [p for p in module.parameters() if p.requires_grad]
    return [p for p in params if p.dim() >= 2], [p for p in params if p.dim() < 2]
