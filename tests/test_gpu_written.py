"""Outputs given to a call: autograd hears of those that were written, and of no others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_versions_of_outputs():
    from alphazero_amd import int8, optim
    from alphazero_amd._abi import AzError
    w, s = torch.ones(6, 8, dtype=torch.int8).cuda(), torch.ones(6).cuda()
    x, out = torch.randn(6, 8).cuda(), torch.zeros(6, 6).cuda()
    at = out._version
    for call in (lambda: int8.matmul(w, s, w, s, out=out[:, :5]), lambda: int8.matmul(w, s, w, s, dtype=torch.float16, out=out),
                 lambda: int8.linear(x, w, s, out=out.view(2, 18)), lambda: int8.linear(x, w, s, act="gelu", out=out),
                 lambda: int8.matmul(w, s, w, out[0], out=out), lambda: optim.orthogonalize(x, out=out), lambda: optim.orthogonalize(out, steps=0, out=out)):
        with pytest.raises(AzError):
            call()
        assert out._version == at
    for call in (lambda: int8.matmul(w, s, w, s, out=out), lambda: int8.linear(x, w, s, out=out), lambda: optim.orthogonalize(out, out=out)):
        call()
        assert out._version > at
        at = out._version
    saved = torch.randn(6, 6, device="cuda", requires_grad=True)
    y = (saved * out).sum()
    int8.matmul(w, s, w, s, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
