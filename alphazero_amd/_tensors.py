"""What the operators on torch tensors share: which tensors they take, and where and on which stream a call runs."""
import torch

from . import _abi
from ._abi import AzError

DTYPES = {torch.float32: _abi.F32, torch.float16: _abi.F16, torch.bfloat16: _abi.BF16}


def need(cond, what):
    if not cond:
        raise AzError(what)


def same_device(what, first, *rest):
    """every tensor on one GPU; returns its ordinal.  There is no CPU path."""
    need(first.device.type == "cuda", "%s: tensors must be on the GPU (no CPU path)" % what)
    for t in rest:
        need(t is None or t.device == first.device, "%s: tensors on different devices" % what)
    return first.device.index


def no_grad(what, *tensors):
    need(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)),
         "%s has no backward pass: call it under torch.no_grad() or detach its inputs" % what)


def stream_of(device):
    """the stream torch would run on there now; the caller's tensors are ordered by it"""
    return torch.cuda.current_stream(device).cuda_stream


def workspace(n, device):
    """scratch of this call alone (torch's allocator hands it on in stream order, and keeps a graph's inside its pool)"""
    return torch.empty(max(int(n), 1), dtype=torch.uint8, device=device)


def rows_of(t, what):
    """a 2-D tensor whose rows are contiguous -> distance between them in elements"""
    need(t.dim() == 2, "%s must have two dimensions" % what)
    need(t.shape[1] <= 1 or t.stride(1) == 1, "%s must have contiguous rows" % what)
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    need(ld >= t.shape[1], "%s: rows overlap" % what)
    return ld


def address(t):
    return None if t is None else t.data_ptr()
