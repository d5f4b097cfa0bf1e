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
    dev = first.get_device()   # -1: not on a device
    if dev < 0 or not first.is_cuda:
        raise AzError("%s: tensors must be on the GPU (no CPU path)" % what)
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise AzError("%s: tensors on different devices" % what)
    return dev


def no_grad(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise AzError("%s has no backward pass: call it under torch.no_grad() or detach its inputs" % what)


def written(*tensors):
    """tells autograd that a kernel wrote these in place: a backward pass that had saved one then says so"""
    torch.autograd.graph.increment_version(tensors)


def workspace(n, like):
    """scratch of this call alone (torch's allocator hands it on in stream order, and keeps a graph's inside its pool) and its
    address"""
    if n == 0:
        return None, None
    t = torch.empty(n, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr()


def rows_of(t, what, name):
    """a 2-D tensor whose rows are contiguous -> (rows, columns, distance between rows in elements)"""
    shape = t.shape
    if len(shape) != 2:
        raise AzError("%s: %s must have two dimensions" % (what, name))
    r, c = shape
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
    if t.dtype is not torch.float32 or t.shape != (n,) or not t.is_contiguous():
        raise AzError("%s: %s must be a contiguous float32 [%d]" % (what, name, n))
    return t.data_ptr()
