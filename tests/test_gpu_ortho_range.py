"""The orthogonalisation's divisor, ||G||_F + eps, over all that float64 holds of it: short sides on both sides of 128."""
import pytest
import torch

from test_gpu_ortho import allowed, gradient, plain

pytestmark = pytest.mark.gpu
SHAPES = [(30, 50), (50, 30), (150, 140), (140, 400)]


@pytest.mark.parametrize("eps", [1e-30, 4e-35, 1e-38, 1e-45, 1e-100, 5e-324])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_zero_matrices_with_a_small_eps(rows, cols, eps):
    """0 / (0 + eps) is 0 for every eps that is accepted: the update of a layer without gradient and momentum"""
    from alphazero_amd import optim
    g = torch.stack([torch.zeros(rows, cols), gradient(rows, cols, 1)]).cuda()
    y = optim.orthogonalize(g, eps=eps).cpu()
    assert (y[0] == 0).all()
    want, tol = allowed(g[1].cpu(), torch.float32, eps=eps)
    assert float((y[1].double() - want).norm()) <= tol
    w = torch.randn(rows, cols).cuda()
    before, m = w.clone(), torch.zeros(rows, cols).cuda()
    optim.muon_step([w], [torch.zeros_like(w)], [m], lr=0.1, eps=eps)
    assert torch.equal(w, before) and (m == 0).all()


@pytest.mark.parametrize("norm,eps", [(1e-33, 1e-33), (1e-33, 5e-324), (1e-36, 1e-30 / 1e3), (1e-36, 1e-36), (1e-36, 1e-38), (1e-36, 5e-324),
                                      (1e-41, 1e-41), (1e-41, 1e-44), (1e-41, 5e-324)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_matrices_of_a_tiny_norm(rows, cols, norm, eps):
    """The iteration depends on G / (||G|| + eps) alone, so the tolerance is the one of G and eps divided by ||G||.  G itself is
    given in float32, so its own rounding (the smallest are multiples of 2^-149) is on both sides."""
    from alphazero_amd import optim
    g = gradient(rows, cols, 2)
    g = (g.double() * (norm / float(g.double().norm()))).float()
    n = float(g.double().norm())
    want = plain(g.double(), eps=eps)
    _, tol = allowed((g.double() / n).float(), torch.float32, eps=eps / n)
    y = optim.orthogonalize(g.cuda(), eps=eps).cpu()
    assert float((y.double() - want).norm()) <= tol


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_an_eps_above_everything(rows, cols):
    from alphazero_amd import optim
    y = optim.orthogonalize(gradient(rows, cols, 3).cuda(), eps=1e300)
    assert (y == 0).all()


@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6, 1e8])
@pytest.mark.parametrize("rows,cols", SHAPES + [(128, 1152), (1024, 1024)])
def test_an_eps_far_above_the_norm(rows, cols, ratio):
    """X is small, and its low halves end at 2^-24 / 2^14: a value is off by up to 2^-39 however small it is.  The steps then only
    multiply by a, and each adds as much again: (a^5 + a^4 + ...) 2^-39 <= a^5 / (1 - 1 / a) 2^-39 a value, beside the usual tolerance."""
    from alphazero_amd import optim
    g = gradient(rows, cols, 4)
    eps = ratio * float(g.norm())
    want, tol = allowed(g, torch.float32, eps=eps)
    a = optim.COEFFS[0]
    y = optim.orthogonalize(g.cuda(), eps=eps).cpu()
    assert float((y.double() - want).norm()) <= tol + a ** 5 / (1 - 1 / a) * 2.0 ** -39 * (rows * cols) ** 0.5
