"""What the operators on torch tensors share: which tensors they take, and where and on which stream a call runs."""
import torch

from . import _abi
from ._abi import AzError

DTYPES = {torch.float32: _abi.F32, torch.float16: _abi.F16, torch.bfloat16: _abi.BF16}
# the stream torch would run on now on a device of that ordinal, as an address: the caller's tensors are ordered by it
stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def same_device(what, first, *rest):
    """every tensor on one GPU; returns its ordinal.  There is no CPU path."""
    if not first.is_cuda:
        raise AzError("%s: tensors must be on the GPU (no CPU path)" % what)
    dev = first.get_device()
    for t in rest:
        if t is not None and not (t.is_cuda and t.get_device() == dev):
            raise AzError("%s: tensors on different devices" % what)
    return dev


def no_grad(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise AzError("%s has no backward pass: call it under torch.no_grad() or detach its inputs" % what)


def workspace(n, like):
    """scratch of this call alone (torch's allocator hands it on in stream order, and keeps a graph's inside its pool) and its
    address"""
    if n == 0:
        return None, None
    t = torch.empty(n, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr()


def rows_of(t, what, name):
    """a 2-D tensor whose rows are contiguous -> (rows, columns, distance between rows in elements)"""
    if t.dim() != 2:
        raise AzError("%s: %s must have two dimensions" % (what, name))
    r, c = t.shape
    if t.is_contiguous():
        return r, c, c
    ld, inner = t.stride()
    if c > 1 and inner != 1:
        raise AzError("%s: %s must have contiguous rows" % (what, name))
    if r <= 1:
        ld = c
    if ld < c:
        raise AzError("%s: rows of %s overlap" % (what, name))
    return r, c, ld


def vector(t, n, what, name):
    """address of a contiguous float32 [n]"""
    if t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise AzError("%s: %s must be a contiguous float32 [%d]" % (what, name, n))
    return t.data_ptr()
