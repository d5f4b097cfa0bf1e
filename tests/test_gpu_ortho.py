"""Orthogonalisation and the update around it (alphazero_amd.optim / az_orthogonalize, az_muon_step) against float64.

Tolerance of the orthogonalisation, in the Frobenius norm: its float32 products are sums of three fp16 products of halves that
hold 22 bits (operands off by 2^-23, dropped term 2^-22) where a plain float32 evaluation has operands exact to 2^-24:
(2 * 2^-23 + 2^-22) / 2^-24 = 8 times its error, both amplified alike by the iteration.  The plain float32 error is measured
on the CPU against float64; 64 * 2^-24 stands below it where a matrix is too small for an average; the rounding of a
16-bit output adds eps / 2."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def O():
    from alphazero_amd import optim
    return optim


def plain(g, steps=5, coeffs=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """the definition in g's own precision, one matrix"""
    a, b, c = coeffs
    x = g / (torch.sqrt((g.double() ** 2).sum()).to(g.dtype) + eps)
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    for _ in range(steps):
        A = x @ x.t()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.t() if flip else x


def allowed(g, dt, **kw):
    """(float64 result, allowed Frobenius error)"""
    want = plain(g.double(), **kw)
    e32 = (plain(g.float(), **kw).double() - want).norm()
    return want, float(8 * torch.maximum(e32, 64 * U * want.norm()) + torch.finfo(dt).eps / 2 * 1.01 * want.norm())


def gradient(rows, cols, seed, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    k = min(8, rows, cols)
    return (torch.randn(rows, k, generator=g) @ torch.randn(k, cols, generator=g) / k ** 0.5
            + 0.5 * torch.randn(rows, cols, generator=g)) * scale


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 5), (16, 16), (27, 128), (128, 27), (64, 64), (65, 63), (128, 128), (128, 1152), (129, 40),
          (1152, 128), (130, 131), (200, 333), (333, 200), (255, 1000), (1, 3000), (100, 5000), (384, 384), (640, 513),
          (130, 2000), (1100, 300), (256, 512)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize(O, rows, cols, dt):
    g = gradient(rows, cols, rows * 7 + cols).to(DT[dt])
    y = O.orthogonalize(g.cuda())
    assert y.dtype == g.dtype and y.shape == g.shape
    want, tol = allowed(g, DT[dt])
    assert float((y.cpu().double() - want).norm()) <= tol


@pytest.mark.parametrize("rows,cols", [(40, 70), (70, 40), (200, 300), (150, 900)])
@pytest.mark.parametrize("kw", [dict(steps=1), dict(steps=2, coeffs=(1.5, -0.5, 0.0)), dict(steps=12, coeffs=(1.5, -0.5, 0.0)),
                                dict(steps=16), dict(steps=3, eps=1e-3), dict(steps=3, coeffs=(2.0, -1.5, 0.5))])
def test_steps_and_coefficients(O, rows, cols, kw):
    g = gradient(rows, cols, 3)
    want, tol = allowed(g, torch.float32, **kw)
    assert float((O.orthogonalize(g.cuda(), **kw).cpu().double() - want).norm()) <= tol


@pytest.mark.parametrize("noise", [0.5, 1e-3, 0.0])
@pytest.mark.parametrize("steps", [2, 3, 4, 6, 8])
def test_wide_matrices_of_low_rank(O, steps, noise):
    """the steps taken on the short side's products alone, down to singular values of nothing"""
    gen = torch.Generator().manual_seed(steps)
    g = torch.randn(160, 6, generator=gen) @ torch.randn(6, 1500, generator=gen) + noise * torch.randn(160, 1500, generator=gen)
    for m in (g, g.t().contiguous()):
        y = O.orthogonalize(m.cuda(), steps=steps)
        want, tol = allowed(m, torch.float32, steps=steps)
        assert float((y.cpu().double() - want).norm()) <= tol


@pytest.mark.parametrize("coeffs", [(2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (3.0, -3.2, 1.2), (4.1, -6.9, 2.95), (-1.5, 0.5, 0.0)])
@pytest.mark.parametrize("steps", [3, 5, 9])
def test_wide_matrices_with_other_coefficients(O, coeffs, steps):
    g = gradient(140, 1200, steps)
    y = O.orthogonalize(g.cuda(), steps=steps, coeffs=coeffs)
    want, tol = allowed(g, torch.float32, steps=steps, coeffs=coeffs)
    assert float((y.cpu().double() - want).norm()) <= tol


def test_cubic_iteration_converges_to_the_polar_factor(O):
    g = torch.linalg.qr(torch.randn(90, 60, dtype=torch.float64, generator=torch.Generator().manual_seed(1)))[0]
    g = g @ torch.diag(torch.linspace(0.5, 1.0, 60, dtype=torch.float64)) @ torch.linalg.qr(torch.randn(60, 60, dtype=torch.float64))[0]
    y = O.orthogonalize(g.float().cuda(), steps=16, coeffs=(1.5, -0.5, 0.0)).cpu().double()
    u, _, vt = torch.linalg.svd(g, full_matrices=False)
    # sigma <= 1 / sqrt(60) grows by 1.5 a step to 1; the polar factor's own condition is 2 / (2 sigma_min)
    assert float((y.t() @ y - torch.eye(60, dtype=torch.float64)).norm()) < 1e-4
    assert float((y - u @ vt).norm()) < 1e-4


def test_batches_of_all_lengths_and_dimensions(O):
    g = torch.stack([gradient(20, 9, i, scale=10.0 ** (i % 7 - 3)) for i in range(37)])
    y = O.orthogonalize(g.cuda()).cpu()
    for i in range(37):
        want, tol = allowed(g[i], torch.float32)
        assert float((y[i].double() - want).norm()) <= tol
    assert torch.equal(O.orthogonalize(g[:36].reshape(4, 3, 3, 20, 9).cuda()).cpu().reshape(36, 20, 9), y[:36])
    assert torch.equal(O.orthogonalize(g[5].cuda()).cpu(), y[5])          # a matrix does not depend on its batch
    assert O.orthogonalize(g[:0].cuda()).shape == (0, 20, 9)


def test_zero_nan_tiny_and_huge_matrices(O):
    for rows, cols in ((30, 50), (150, 140), (700, 140)):
        g = torch.stack([gradient(rows, cols, i) for i in range(7)])
        g[0] = 0
        g[1, 3, 4] = float("nan")
        g[2, 5, 6] = float("-inf")
        g[3] *= 1e-30
        g[4] *= 1e38 / float(g[4].abs().max())      # a factor above float32's largest value: all infinities and NaN
        g[6] = g[6].double().div(g[6].abs().max()).mul(1e38).float()
        y = O.orthogonalize(g.cuda(), eps=1e-30).cpu()
        assert (y[0] == 0).all() and y[1].isnan().all() and y[2].isnan().all()
        assert not g[4].isfinite().any() and y[4].isnan().all()
        for i in (3, 5, 6):     # far outside fp16's range, and float32's for their squares
            scaled = (g[i].double() / g[i].double().norm()).float()
            want = plain(g[i].double(), eps=1e-30)
            _, tol = allowed(scaled, torch.float32, eps=1e-30)
            assert float((y[i].double() - want).norm()) <= tol


@pytest.mark.parametrize("rows,cols", [(17000, 32768), (32768, 17000)])
def test_offsets_past_32_bits(O, rows, cols):
    """one value in each row and column: the iteration of numbers, in 2.2 GB"""
    s, gen = min(rows, cols), torch.Generator().manual_seed(rows)
    i, j = torch.randperm(rows, generator=gen)[:s].cuda(), torch.randperm(cols, generator=gen)[:s].cuda()
    v = torch.randn(s, generator=gen).cuda()
    g = torch.zeros(rows, cols, device="cuda")
    g[i, j] = v
    y = O.orthogonalize(g, out=g)
    x = v.double() / (v.double().norm() + 1e-7)
    for _ in range(5):
        x = x * (3.4445 - 4.7750 * x ** 2 + 2.0315 * x ** 4)
    got = y[i, j].double()
    assert float((got - x).norm()) <= 8 * 64 * U * float(x.norm())
    y[i, j] = 0
    assert not y.any()


def test_in_place_strided_input_streams_and_graphs(O):
    base = torch.randn(3, 50, 80).cuda()
    g = base.transpose(1, 2)
    y = O.orthogonalize(g)
    assert torch.equal(y, O.orthogonalize(g.contiguous()))
    z = g.contiguous()
    assert O.orthogonalize(z, out=z).data_ptr() == z.data_ptr() and torch.equal(z, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t = O.orthogonalize(g)
    side.synchronize()
    assert torch.equal(t, y)
    # two graphs alive together, replayed in turn with eager calls between
    made = []
    for shape in ((2, 100, 300), (1, 150, 150)):
        x = torch.randn(shape).cuda()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = O.orthogonalize(x)
        made.append((gr, x, out))
    for _ in range(4):
        for gr, x, out in made:
            x.copy_(torch.randn(x.shape))
        for gr, x, out in made:
            gr.replay()
        torch.cuda.synchronize()
        for gr, x, out in made:
            assert torch.equal(out, O.orthogonalize(x))


def muon64(w, g, m, lr, mu, nesterov, wd, **kw):
    w64, g64, m64 = w.double(), g.double(), m.double()
    m1 = mu * m64 + (1 - mu) * g64
    u = mu * m1 + (1 - mu) * g64 if nesterov else m1
    flat = u.reshape(u.shape[0], -1)
    kappa = math.sqrt(max(1.0, flat.shape[0] / flat.shape[1]))
    o, tol = allowed(flat.float(), torch.float32, **kw)
    o = plain(flat, **kw).reshape(w.shape)
    m_tol = 5 * U * (mu * m64.abs() + (1 - mu) * g64.abs())      # two products, one sum, two constants of 24 bits
    # u moves by 5 u of its terms before it is orthogonalised: like float32 inputs, inside the factor 8 of `allowed`
    return (1 - lr * wd) * w64 - lr * kappa * o, m1, lr * kappa * tol, m_tol


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("nesterov,wd", [(True, 0.0), (False, 0.1)])
def test_muon_step(O, dt, nesterov, wd):
    t = DT[dt]
    shapes = [(128, 3, 3, 3), (128, 128, 3, 3), (128, 128, 1, 1), (7, 126), (300, 20), (1, 128), (40, 500), (5, 5), (200, 250)] + [(9, 11)] * 12
    ws = [(torch.randn(s, generator=torch.Generator().manual_seed(i)) / 8).to(t) for i, s in enumerate(shapes)]
    ms = [torch.zeros(s) for s in shapes]
    wd_, md = [w.cuda() for w in ws], [m.cuda() for m in ms]
    for step in range(3):
        gs = [gradient(s[0], int(np.prod(s[1:])), 100 * step + i).reshape(s).to(t) for i, s in enumerate(shapes)]
        w0, m0 = [w.cpu() for w in wd_], [m.cpu() for m in md]
        O.muon_step(wd_, [g.cuda() for g in gs], md, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=wd)
        for i in range(len(shapes)):
            w1, m1, w_tol, m_tol = muon64(w0[i], gs[i], m0[i], 0.05, 0.9, nesterov, wd)
            assert ((md[i].cpu().double() - m1).abs() <= m_tol + 1e-45).all()
            err = float((wd_[i].cpu().double() - w1).norm())
            # 4 u: two products, a sum and the constants; then the type's own rounding
            assert err <= w_tol + float((4 * U + torch.finfo(t).eps / 2 * 1.01) * (w0[i].double().norm() + w1.norm())), (i, step)


def test_muon_step_in_a_graph_beside_an_eager_one(O):
    shapes = [(60, 100), (150, 150)]

    def fresh(seed):
        g = torch.Generator().manual_seed(seed)
        return [[torch.randn(s, generator=g).cuda() for s in shapes] for _ in range(3)]

    w, g, m = fresh(1)
    we, ge, me = fresh(1)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        O.muon_step(w, g, m, lr=0.1)
    for t, s in zip(w + g + m, we + ge + me):
        assert torch.equal(t, s)             # capturing ran nothing
    for i in range(4):
        for a, b in zip(g, ge):
            a.copy_(torch.randn(a.shape))
            b.copy_(a)
        gr.replay()
        O.muon_step(we, ge, me, lr=0.1)
        torch.cuda.synchronize()
        for t, s in zip(w + m, we + me):
            assert torch.equal(t, s)


def test_refusals(O):
    from alphazero_amd._abi import AzError
    x, m = torch.ones(4, 6).cuda(), torch.zeros(4, 6).cuda()
    bad = [lambda: O.orthogonalize(x[0]), lambda: O.orthogonalize(x.double()), lambda: O.orthogonalize(x.clone().requires_grad_()),
           lambda: O.orthogonalize(x, steps=0), lambda: O.orthogonalize(x, eps=0.0), lambda: O.orthogonalize(x, coeffs=(1, 2)),
           lambda: O.orthogonalize(x, coeffs=(9.0, 0.0, 0.0)), lambda: O.orthogonalize(x, out=x[:2]),
           lambda: O.muon_step([x], [x.clone()], [m.half()], lr=0.1), lambda: O.muon_step([x], [x.clone()], [], lr=0.1),
           lambda: O.muon_step([x], [x], [m], lr=0.1), lambda: O.muon_step([x, x], [x.clone()] * 2, [m, m.clone()], lr=0.1),
           lambda: O.muon_step([x.t()], [x.t()], [m.t()], lr=0.1), lambda: O.muon_step([x[0]], [x[0].clone()], [m[0]], lr=0.1),
           lambda: O.muon_step([x], [x.clone().cpu()], [m], lr=0.1), lambda: O.muon_step([x], [x.clone()], [m], lr=0.1, momentum=1.0)]
    for call in bad:
        with pytest.raises(AzError):
            call()
    assert (x == 1).all() and (m == 0).all()
    O.muon_step([], [], [], lr=0.1)
    z = torch.randn(100).cuda()
    with pytest.raises(AzError):
        O.orthogonalize(z[:48].view(6, 8), out=z[8:56].view(6, 8))


def test_in_place_updates_are_seen_by_autograd(O):
    """a weight that a graph has saved and that is updated before its backward pass: an error, not a wrong gradient"""
    w = torch.nn.Parameter(torch.randn(6, 8).cuda())
    x = torch.randn(8, 3, requires_grad=True, device="cuda")
    y = (w @ x).sum()
    O.muon_step([w.detach()], [torch.ones(6, 8).cuda()], [torch.zeros(6, 8).cuda()], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_repeated_calls_give_the_same_bits(O):
    for shape in ((3, 128, 1152), (1, 300, 700), (2, 640, 640), (1, 1500, 1500)):
        g = torch.randn(shape).cuda()
        first = O.orthogonalize(g)
        for _ in range(3):
            assert torch.equal(O.orthogonalize(g), first)
