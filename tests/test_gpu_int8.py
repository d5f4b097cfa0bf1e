"""8-bit rows and products (alphazero_amd.int8 / az_i8_*) against float64 restatements of their definitions.

Tolerance of a product, for outputs of type t (derived, u = 2^-24): with p = acc s w_s, the kernel's float32 steps are acc to
float, two products, two additions: at most 3 u |p| + 2 u (|p| + |bias| + |res|) <= 5.1 u S with S = |p| + |bias| + |res|.  The
activations are Lipschitz by 1.1 and SiLU's own quotient adds 8 u |y| (expf 2 ulp, one addition, one division).  The last
rounding is eps(t) / 2 |y|; a subnormal result of 16 bits rounds by half its smallest step."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def I8():
    from alphazero_amd import int8
    return int8


def rows64(x, index=None):
    """definition, on the CPU: (q, scale)"""
    x = x.detach().cpu().float().numpy()
    if index is not None:
        idx = index.cpu().numpy()
        z = np.zeros((x.shape[0] + 1, x.shape[1]), np.float32)
        z[:-1] = x
        x = z[np.where((idx >= 0) & (idx < len(x)), idx, len(x))].reshape(len(idx), -1)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(x).all(1)
        amax = np.where(bad, np.float32(np.nan), np.abs(x).max(1) if x.shape[1] else 0).astype(np.float32)
        s = amax * (np.float32(1) / np.float32(127))
        q = np.rint(x.astype(np.float64) / s.astype(np.float64)[:, None])
        q = np.where((s > 0)[:, None], np.clip(q, -127, 127), 0)
    return q.astype(np.int8), s


def check_rows(I8, x, index=None):
    q, s = I8.quantize_rows(x, index=index)
    q64, s64 = rows64(x, index)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    np.testing.assert_array_equal(s.cpu().numpy(), s64)
    np.testing.assert_array_equal(q.cpu().numpy(), q64)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2), (3, 5), (5, 63), (7, 64), (64, 65), (130, 127), (33, 128), (9, 1000),
                                       (4, 1152), (3, 4096), (2, 4099), (1, 16384), (1, 40001), (70000, 3),
                                       (2, 700001), (9, 2048), (5, 8191)])
def test_rows(I8, dt, rows, cols):
    g = torch.Generator().manual_seed(rows * 131 + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-12, 13, (rows, 1), generator=g).float())
    check_rows(I8, x.to(DT[dt]).cuda())


def test_rows_ties_and_extremes(I8):
    f = np.float32
    rng = np.random.default_rng(3)
    rows = []
    for _ in range(300):   # ties (k + 1/2) s and their neighbours, at scales over the whole float32 range
        amax = f(np.exp2(rng.uniform(-148, 127.9)))
        s = f(amax * (f(1) / f(127)))
        tie = ((rng.integers(-127, 127, 40) + 0.5) * np.float64(s)).astype(f)
        r = np.concatenate([tie, np.nextafter(tie, f(np.inf)), np.nextafter(tie, f(-np.inf)), [amax]])
        rows.append(np.clip(r, -amax, amax))
    rows.append(np.zeros(121, f))
    for special in (np.nan, np.inf, -np.inf):
        r = rng.normal(size=121).astype(f)
        r[17] = special
        rows.append(r)
    rows.append(np.full(121, -np.finfo(f).max, f))
    rows.append(np.full(121, f(1e-45), f))
    rows.append(np.where(np.arange(121) == 120, f(-0.0), f(0.0)))
    check_rows(I8, torch.from_numpy(np.array(rows, f)).cuda())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("cols,taps,rows", [(1, 9, 5), (3, 9, 100), (28, 9, 90), (128, 9, 84), (130, 4, 17), (16, 1, 3), (64, 30, 11), (3000, 7, 5),
                                             (1, 300, 4), (9000, 3, 2)])
def test_rows_by_index(I8, dt, cols, taps, rows):
    g = torch.Generator().manual_seed(cols + taps)
    x = torch.randn(50, cols, generator=g).to(DT[dt]).cuda()
    index = torch.randint(-3, 53, (rows, taps), generator=g, dtype=torch.int32)
    index[0] = -1                                     # a row of zeros
    index[1] = torch.tensor([2 ** 31 - 1, -2 ** 31] * taps, dtype=torch.int64)[:taps].int()
    check_rows(I8, x, index.cuda())


def test_rows_strided_empty_and_no_source(I8):
    x = torch.randn(40, 300).cuda()
    check_rows(I8, x[::2, 7:207])
    check_rows(I8, x[3:3])
    check_rows(I8, x[3:4, 5:6])
    q, s = I8.quantize_rows(x[:0], index=torch.zeros(3, 2, dtype=torch.int32).cuda())
    assert q.shape == (3, 600) and not q.any() and not s.any()


def layer64(q, s, w, ws, bias, res, act):
    p = (q.cpu().double() @ w.cpu().double().t()) * s.cpu().double()[:, None] * ws.cpu().double()[None]
    size = p.abs()
    y = p
    for t in (None if bias is None else bias.cpu().double()[None], None if res is None else res.cpu().double()):
        if t is not None:
            y, size = y + t, size + t.abs()
    if act == "relu":
        y = torch.clamp(y, min=0)
    elif act == "silu":
        y = y * torch.sigmoid(y)
    return y, size


def check_layer(y, y64, size):
    u, t = 2.0 ** -24, y.dtype
    tol = 1.1 * 5.1 * u * size + 8 * u * y64.abs() + torch.finfo(t).eps / 2 * (y64.abs() + 6 * u * size)
    tol = tol + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    err = (y.cpu().double() - y64).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


def operands(m, n, k, seed, dt, bias=True, res=False, full=False):
    g = torch.Generator().manual_seed(seed)
    lim = 128 if full else 127
    q = torch.randint(-lim, 128, (m, k), generator=g, dtype=torch.int32).to(torch.int8)
    w = torch.randint(-lim, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8)
    s, ws = torch.rand(m, generator=g) * 0.02 + 0.001, (torch.rand(n, generator=g) + 0.1) / (50 * k ** 0.5)
    b = torch.randn(n, generator=g) if bias else None
    r = torch.randn(m, n, generator=g).to(DT[dt]) if res else None
    return [None if t is None else t.cuda() for t in (q, s, w, ws, b, r)]


SHAPES = [(1, 1, 1), (1, 1, 129), (1, 7, 126), (2, 3, 42), (1, 128, 1152), (1, 1003, 4096), (3, 129, 27), (5, 64, 4097), (16, 256, 512),
          (17, 31, 64), (31, 33, 128), (42, 128, 1152), (63, 65, 127), (64, 64, 16), (65, 1, 1000), (84, 128, 252),
          (127, 129, 144), (128, 128, 128), (129, 257, 272), (300, 500, 1031), (256, 256, 2048), (257, 511, 384),
          (700, 130, 1152), (1000, 7, 126), (513, 1024, 640), (65, 64, 8192), (128, 130, 4100), (90, 201, 5000),
          (24, 200, 8192), (48, 100, 4096), (16, 8200, 4224)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act,bias,res", [("none", False, False), ("relu", True, False), ("silu", True, True)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(I8, m, n, k, act, bias, res, dt):
    q, s, w, ws, b, r = operands(m, n, k, m + 3 * n + 7 * k, dt, bias, res)
    y = I8.matmul(q, s, w, ws, bias=b, residual=r, act=act, dtype=DT[dt])
    check_layer(y, *layer64(q, s, w, ws, b, r, act))


def test_matmul_largest_sums(I8):
    """-128 * -128 over the longest k: 2^31 - 2^14, the last sum that int32 holds"""
    for m, n in ((1, 3), (130, 140)):
        k = I8.MAX_K
        q = torch.full((m, k), -128, dtype=torch.int8).cuda()
        w = torch.full((n, k), -128, dtype=torch.int8).cuda()
        y = I8.matmul(q, torch.ones(m).cuda(), w, torch.ones(n).cuda())
        assert (y == float(k * 16384)).all()


@pytest.mark.parametrize("m,n,k", [(1, 200, 300), (70, 200, 304), (300, 300, 256), (20, 130, 1024)])
def test_matmul_strides_and_neighbours(I8, m, n, k):
    """rows further apart than they are long, at odd addresses; what lies between the rows of the output stays as it was"""
    g = torch.Generator().manual_seed(m)
    for off, pad in ((0, 0), (1, 3), (16, 16), (16, 0), (3, 13)):
        bq = torch.randint(-127, 128, (m, k + off + pad), generator=g, dtype=torch.int32).to(torch.int8).cuda()
        bw = torch.randint(-127, 128, (n, k + off + pad), generator=g, dtype=torch.int32).to(torch.int8).cuda()
        q, w = bq[:, off:off + k], bw[:, off:off + k]
        s, ws = torch.rand(m, generator=g).cuda(), torch.rand(n, generator=g).cuda() / k
        buf = torch.full((m + 2, n + 11), 7.0, dtype=torch.bfloat16).cuda()
        out = buf[1:-1, 5:5 + n]
        res = torch.randn(m, n + 1, generator=g).bfloat16().cuda()[:, 1:]
        y = I8.matmul(q, s, w, ws, residual=res, dtype=torch.bfloat16, out=out)
        assert y.data_ptr() == out.data_ptr()
        check_layer(y, *layer64(q, s, w, ws, None, res, "none"))
        buf[1:-1, 5:5 + n] = 7.0
        assert (buf == 7.0).all()


def test_matmul_residual_in_place_and_nan(I8):
    q, s, w, ws, b, r = operands(50, 70, 96, 1, "f32", True, True)
    want = layer64(q, s, w, ws, b, r, "silu")
    y = I8.matmul(q, s, w, ws, bias=b, residual=r, act="silu", out=r)
    assert y.data_ptr() == r.data_ptr()
    check_layer(y, *want)
    # a row whose scale is NaN, one whose scale is 0, an infinite and a NaN bias
    s[3], s[4] = float("nan"), 0.0
    b[0], b[1] = float("inf"), float("nan")
    for act in ("none", "relu", "silu"):
        y = I8.matmul(q, s, w, ws, bias=b, act=act)
        assert y[3].isnan().all() and y[:, 1].isnan().all() and (y[[0, 1, 2, 4], 0] == float("inf")).all()
        check_layer(y[4:5, 2:], *layer64(q[4:5], s[4:5], w[2:], ws[2:], b[2:], None, act))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 1000, 4096), (1, 257, 1031), (2, 64, 100), (3, 7, 42), (4, 300, 4096), (8, 128, 1152),
                                   (16, 100, 5000), (33, 65, 130), (200, 300, 1031), (1, 33, 131071),
                                   (2, 17, 32000), (3, 40, 21845), (4, 16, 16384), (4, 100, 63), (5, 9, 64), (1, 5, 65472), (1, 5, 65600)])
def test_linear_is_quantize_then_matmul(I8, dt, m, n, k):
    g = torch.Generator().manual_seed(m * 7 + n + k)
    x = torch.randn(m, k, generator=g).to(DT[dt]).cuda()
    _, _, w, ws, b, r = operands(m, n, k, 11, dt, True, True)
    y = I8.linear(x, w, ws, bias=b, residual=r, act="silu")
    q, s = I8.quantize_rows(x)
    assert torch.equal(y, I8.matmul(q, s, w, ws, bias=b, residual=r, act="silu", dtype=DT[dt]))
    q64, s64 = rows64(x)
    check_layer(y, *layer64(torch.from_numpy(q64), torch.from_numpy(s64), w, ws, b, r, "silu"))


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 40])
def test_linear_non_finite_rows(I8, m):
    x = torch.randn(m, 200).cuda()
    x[0, 13] = float("inf")
    if m > 1:
        x[1, 14] = float("nan")
    if m > 2:
        x[2] = 0
    _, _, w, ws, b, _ = operands(m, 50, 200, 3, "f32")
    y = I8.linear(x, w, ws, bias=b)
    assert y[:2].isnan().all() and y[2:].isfinite().all()
    if m > 2:
        assert torch.equal(y[2], b)


def test_columns_of_one_buffer(I8):
    """output beside input and residual in the rows of one buffer"""
    from alphazero_amd._abi import AzError
    buf = torch.randn(50, 200, generator=torch.Generator().manual_seed(3)).cuda()
    w = torch.randint(-127, 128, (40, 64), dtype=torch.int8, generator=torch.Generator().manual_seed(4)).cuda()
    s = torch.rand(40, generator=torch.Generator().manual_seed(5)).cuda()
    x, res, out = buf[:, :64], buf[:, 100:140], buf[:, 64:104 - 4]
    want = I8.linear(x.clone(), w[:36], s[:36], residual=res[:, :36].clone(), act="relu")
    kept = buf.clone()
    y = I8.linear(x, w[:36], s[:36], residual=res[:, :36], act="relu", out=out)
    assert torch.equal(y, want) and y.data_ptr() == out.data_ptr()
    kept[:, 64:100] = want
    assert torch.equal(buf, kept)
    with pytest.raises(AzError, match="overlap"):
        I8.linear(x, w[:36], s[:36], out=buf[:, 40:76])
    with pytest.raises(AzError, match="residual"):
        I8.linear(x, w[:36], s[:36], residual=buf[:, 80:116], out=out)


def test_offsets_past_32_bits(I8):
    """3 GB of 8-bit rows on either side, 5.6 GB of output"""
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(-127, 128, (50000, 60000), dtype=torch.int8, device="cuda", generator=gen)
    w = torch.randint(-127, 128, (70, 60000), dtype=torch.int8, device="cuda", generator=gen)
    one = torch.ones(70000, device="cuda")
    at = [0, 17000, 35791, 35792, 49999]
    want = (q[at].double().unsqueeze(1) * w.double()).sum(2)          # exact; a float32 result is its rounding
    assert torch.equal(I8.matmul(q, one[:50000], w, one[:70])[at], want.float())
    assert torch.equal(I8.matmul(w, one[:70], q, one[:50000])[:, at], want.float().t())
    del q, w
    x = torch.empty(40000, 60000, dtype=torch.float16, device="cuda").normal_(generator=gen)
    r, s = I8.quantize_rows(x, torch.tensor([[39999], [35792], [0], [40000]], dtype=torch.int32, device="cuda"))
    assert torch.equal(r[:3].double(), torch.round(x[[39999, 35792, 0]].double() / s[:3].double().unsqueeze(1)))
    assert (r[3] == 0).all() and s[3] == 0
    r, s = I8.quantize_rows(x)
    assert torch.equal(r[at[:4]].double(), torch.round(x[at[:4]].double() / s[at[:4]].double().unsqueeze(1)))
    del x, r
    a = torch.randint(-127, 128, (70000, 48), dtype=torch.int8, device="cuda", generator=gen)
    y = I8.matmul(a, one, a[:40000], one[:40000], dtype=torch.bfloat16)
    for i in (0, 53687, 69999):
        assert torch.equal(y[i], (a[i].double() * a[:40000].double()).sum(1).to(torch.bfloat16))


def test_empty_calls(I8):
    w, ws = torch.zeros(5, 8, dtype=torch.int8).cuda(), torch.ones(5).cuda()
    assert I8.matmul(w[:0], ws[:0], w, ws).shape == (0, 5)
    assert I8.matmul(w, ws, w[:0], ws[:0]).shape == (5, 0)
    assert I8.linear(torch.zeros(0, 8).cuda(), w, ws).shape == (0, 5)


def test_streams_and_graph_replays(I8):
    """on a side stream, and captured: every replay on new inputs equals the eager call"""
    x = torch.randn(37, 500).cuda()
    _, _, w, ws, b, _ = operands(37, 90, 500, 2, "f32")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = I8.linear(x, w, ws, bias=b, act="relu")
    side.synchronize()
    assert torch.equal(y, I8.linear(x, w, ws, bias=b, act="relu"))
    graphs, xs, ys = [], [], []
    for rows in (37, 1):       # two graphs, alive together
        xi = torch.randn(rows, 500).cuda()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            I8.linear(xi, w, ws, bias=b)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            yi = I8.linear(xi, w, ws, bias=b, act="silu")
        graphs.append(g), xs.append(xi), ys.append(yi)
    for i in range(4):
        for xi in xs:
            xi.copy_(torch.randn(xi.shape))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for xi, yi in zip(xs, ys):
            assert torch.equal(yi, I8.linear(xi, w, ws, bias=b, act="silu"))


def test_refusals(I8):
    from alphazero_amd._abi import AzError
    x = torch.zeros(4, 8).cuda()
    w, s = torch.zeros(6, 8, dtype=torch.int8).cuda(), torch.ones(6).cuda()
    bad = [lambda: I8.quantize_rows(x.double()), lambda: I8.quantize_rows(x.t()), lambda: I8.quantize_rows(x[0]),
           lambda: I8.quantize_rows(x[:, :0]), lambda: I8.quantize_rows(x, index=torch.zeros(3, 2).cuda()),
           lambda: I8.quantize_rows(x, index=torch.zeros(3, 2, dtype=torch.int32)),
           lambda: I8.quantize_rows(x.requires_grad_()), lambda: I8.linear(x[:, :7].detach(), w, s),
           lambda: I8.matmul(w, s, w, s[:5]), lambda: I8.matmul(w, s, w.float(), s), lambda: I8.matmul(w, s.half(), w, s),
           lambda: I8.matmul(w, s, w, s, act="gelu"), lambda: I8.matmul(w, s, w, s, dtype=torch.float64),
           lambda: I8.matmul(w, s, w, s, residual=x.detach()), lambda: I8.matmul(w, s, w.cpu(), s),
           lambda: I8.matmul(w, s, w, s, bias=torch.zeros(6, 1).cuda()), lambda: I8.matmul(w.t(), s, w, s)]
    for call in bad:
        with pytest.raises(AzError):
            call()
