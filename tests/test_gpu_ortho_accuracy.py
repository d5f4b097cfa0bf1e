"""Orthogonalisation: the error beside a plain float32 evaluation's, and that a matrix's result is its own alone."""
import pytest
import torch

from test_gpu_ortho import DT, gradient, plain

pytestmark = pytest.mark.gpu


def relative(y, want):
    return float((y.cpu().double() - want).norm() / want.norm())


def step_by_step(g, steps=5, coeffs=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """the definition, one step after the other, on the kernels' operands and sums: halves of 22 bits; of 16 values of the sum's index the
    small products first, eight at a time added to a float32, as the matrix pipe does (2^24 + 16 x 0.1275 gives 2^24 + 4: twice
    8 x 0.1275 = 1.02, above half of the 2 that float32 moves by there; 16 x 0.125, two ties, gives 2^24)"""
    def halves(x, k):
        hi = (x * 2.0 ** k).half()
        lo = (x * 2.0 ** k - hi.float()).half()
        return hi.double(), lo.double()

    def product(x, kx, y, ky):
        (xh, xl), (yh, yl) = halves(x, kx), halves(y, ky)
        acc = torch.zeros(x.shape[0], y.shape[0], dtype=torch.float64, device=x.device)
        for i in range(0, x.shape[1], 16):
            for p, q in ((xl, yh), (xh, yl), (xh, yh)):
                for eight in (slice(i, i + 8), slice(i + 8, i + 16)):
                    acc = (acc + torch.mm(p[:, eight], q[:, eight].t())).float().double()
        return (acc * 2.0 ** -(kx + ky)).float()

    a, b, c = coeffs
    x = g / (float((g.double() ** 2).sum()) ** 0.5 + eps)
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    one = torch.eye(x.shape[0], device=x.device)
    for _ in range(steps):
        A = product(x, 14, x, 14)
        x = product(a * one + b * A + c * product(A, 12, A, 12), 11, x.t().contiguous(), 14)
    return x.t() if flip else x


def strong(rows, cols, seed):
    """six strong directions over weak noise: singular values of very different sizes"""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, 6, generator=g) @ torch.randn(6, cols, generator=g) + 0.3 * torch.randn(rows, cols, generator=g)


# squares and rectangles, short and long ones
NARROW = [(16, 16), (32, 32), (64, 64), (128, 128), (27, 128), (128, 27), (128, 256), (128, 1152), (64, 1100), (1100, 64), (32, 4096), (128, 2100)]
WIDE = [(300, 300), (200, 300), (512, 512), (300, 600), (600, 300), (300, 1250), (300, 2000), (256, 2048)]


@pytest.mark.parametrize("kind", [gradient, strong])
@pytest.mark.parametrize("rows,cols", NARROW + WIDE)
def test_float32_loses_nothing_to_the_order_of_its_steps(rows, cols, kind):
    """However the steps are grouped: the mean error over seeds is at most a quarter above that of steps one by one on the same
    operands and sums, or of a plain float32 evaluation, if that is larger.  (The error varies by less than a quarter from seed to
    seed, so a mean over 8 is good to a tenth, the quotient of two such means to 1.15; a tenth more is left for the exact
    evaluation's own order of sums.)"""
    from alphazero_amd import optim
    here = one = floats = 0.0
    for seed in range(8):
        g = kind(rows, cols, seed)
        want = plain(g.double())
        here += relative(optim.orthogonalize(g.cuda()), want) / 8
        one += relative(step_by_step(g.cuda()), want) / 8
        floats += relative(plain(g), want) / 8
    assert here <= 1.25 * max(one, floats), (here, one, floats)


@pytest.mark.parametrize("dt,shapes", [
    ("f32", [(27, 128, 20), (128, 1152, 3), (100, 2500, 5), (333, 1027, 17), (512, 512, 6), (300, 2000, 7), (640, 1500, 3), (200, 200, 40)]),
    ("f16", [(27, 128, 20), (128, 1152, 3), (100, 2500, 5)]), ("bf16", [(27, 128, 20), (128, 1152, 3), (100, 2500, 5)])])
def test_a_matrix_does_not_depend_on_its_batch(dt, shapes):
    """the same bits alone and in a batch, which takes tiles of the other size"""
    from alphazero_amd import optim
    for rows, cols, n in shapes:
        g = torch.stack([gradient(rows, cols, i) for i in range(n)]).to(DT[dt]).cuda()
        y = optim.orthogonalize(g)
        for i in (0, n // 2, n - 1):
            assert torch.equal(optim.orthogonalize(g[i]), y[i]), (rows, cols, i)


def test_a_weight_does_not_depend_on_its_companions():
    """a float32 update of matrices of all forms in one call, in another order, and one by one"""
    from alphazero_amd import optim
    shapes = [(300, 300), (1500, 300), (128, 128), (128, 27), (512, 512), (100, 2500), (64, 576), (256, 1100), (700, 640), (20, 9),
              (1024, 300), (130, 130), (128, 1152), (2100, 64), (900, 1000), (150, 150), (150, 160), (260, 1500)]

    def fresh():
        return [(gradient(*s, 50 + i, scale=0.1).cuda(), gradient(*s, i).cuda(), gradient(*s, 100 + i).cuda()) for i, s in enumerate(shapes)]

    together, turned, alone = fresh(), fresh(), fresh()
    order = list(range(len(shapes)))[::-1]
    for _ in range(2):
        optim.muon_step([t[0] for t in together], [t[1] for t in together], [t[2] for t in together], lr=0.02)
        optim.muon_step([turned[i][0] for i in order], [turned[i][1] for i in order], [turned[i][2] for i in order], lr=0.02)
        for w, g, m in alone:
            optim.muon_step([w], [g], [m], lr=0.02)
    for s, a, b, c in zip(shapes, together, turned, alone):
        for k in (0, 2):
            assert torch.equal(a[k], b[k]) and torch.equal(a[k], c[k]), s
