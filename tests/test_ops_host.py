"""Refusals of the operators on device tensors (include/azamd.h: az_i8_*, az_orthogonalize, az_muon_step) that need no GPU:
the C entry points check every argument before they look for a device, the Python ones refuse CPU tensors."""
import ctypes as C

import numpy as np
import pytest
import torch

from alphazero_amd import _abi, int8, optim

P = C.c_void_p(256)   # stands for a device pointer: no refused call dereferences it
ARG, NO_DEVICE = -1, -2


def _refused(rc, text):
    assert rc == ARG
    assert text in _abi.lib().az_last_error().decode()


def _accepted(rc):
    """past the argument checks: without a GPU the call ends at the missing device"""
    assert rc == (NO_DEVICE if _abi.device_count() == 0 else rc)


def test_quantize_refuses():
    L = _abi.lib()

    def call(dtype=0, rows=4, cols=8, x=P, ld_x=8, n_src=4, index=None, taps=1, q=P, ld_q=8, scale=P):
        return L.az_i8_quantize_dev(0, dtype, rows, cols, x, ld_x, n_src, index, taps, q, ld_q, scale, None)

    _refused(call(dtype=3), "dtype")
    _refused(call(dtype=-1), "dtype")
    _refused(call(rows=-1), "shape")
    _refused(call(cols=0), "shape")
    _refused(call(ld_x=7), "row distance")
    _refused(call(n_src=5), "without an index")
    _refused(call(taps=2), "without an index")
    _refused(call(index=P, taps=0), "taps")
    _refused(call(index=P, taps=9, ld_q=71), "taps or ld_q")
    _refused(call(cols=1 << 20, ld_x=1 << 20, index=P, taps=1 << 12, ld_q=1 << 40), "taps or ld_q")
    for missing in ("x", "q", "scale"):
        _refused(call(**{missing: None}), "null")


def test_matmul_refuses():
    L = _abi.lib()

    def call(fn, m=4, n=6, k=8, ld_x=8, ld_w=8, res=None, ld_res=6, act=0, dtype=0, y=P, ld_y=6, x=P, w=P, ws=P, nws=1 << 20):
        if fn == "matmul":
            return L.az_i8_matmul_dev(0, m, n, k, x, ld_x, P, w, ld_w, P, None, res, ld_res, act, dtype, y, ld_y, ws, nws, None)
        return L.az_i8_linear_dev(0, m, n, k, x, ld_x, w, ld_w, P, None, res, ld_res, act, dtype, y, ld_y, ws, nws, None)

    for fn in ("matmul", "linear"):
        _refused(call(fn, dtype=3), "dtype")
        _refused(call(fn, m=-1), "shape")
        _refused(call(fn, k=0), "shape")
        _refused(call(fn, k=131072, ld_x=131072, ld_w=131072), "131071")
        _refused(call(fn, ld_x=7), "row distance")
        _refused(call(fn, ld_w=7), "row distance")
        _refused(call(fn, ld_y=5), "row distance")
        _refused(call(fn, ld_x=1 << 62), "row distance")
        _refused(call(fn, ld_y=1 << 62), "row distance")
        _refused(call(fn, res=P, ld_res=5), "row distance")
        _refused(call(fn, act=3), "activation")
        _refused(call(fn, x=None), "null")
        _refused(call(fn, w=None), "null")
        _refused(call(fn, y=None), "null")
    _refused(call("linear", m=40, nws=16), "workspace")
    _refused(call("linear", m=40, ws=C.c_void_p(264)), "workspace")
    _refused(call("matmul", m=100, k=7, nws=16), "workspace")          # rows that have to be aligned first
    _refused(call("matmul", m=100, k=7, ws=C.c_void_p(264)), "workspace")
    assert L.az_i8_linear_ws(4, 6, 0, P, 8) == 0 and L.az_i8_matmul_ws(4, 6, 8, P, 8, P, 8) == 0


def test_int8_outputs_overlap_nothing():
    L = _abi.lib()
    at = {"x": 0x100000, "xs": 0x200000, "w": 0x300000, "ws": 0x400000, "bias": 0x500000, "res": 0x600000, "y": 0x700000}

    def call(fn, m=4, n=6, k=8, ld_x=8, ld_w=8, ld_res=6, ld_y=6, **over):
        a = {name: C.c_void_p(p) for name, p in {**at, **over}.items()}
        if fn == "matmul":
            return L.az_i8_matmul_dev(0, m, n, k, a["x"], ld_x, a["xs"], a["w"], ld_w, a["ws"], a["bias"], a["res"], ld_res, 0, 0,
                                      a["y"], ld_y, P, 1 << 20, None)
        return L.az_i8_linear_dev(0, m, n, k, a["x"], ld_x, a["w"], ld_w, a["ws"], a["bias"], a["res"], ld_res, 0, 0, a["y"], ld_y,
                                  P, 1 << 20, None)

    for fn in ("matmul", "linear"):
        for name in ("x", "w", "ws", "bias") + (("xs",) if fn == "matmul" else ()):
            _refused(call(fn, y=at[name]), "overlap")
            _refused(call(fn, y=at[name] - 92), "overlap")              # y is 96 bytes
        _refused(call(fn, res=at["y"] + 4), "residual")
        _refused(call(fn, res=at["y"], ld_res=12), "residual")
        _refused(call(fn, res=at["y"] + 20, ld_y=12, ld_res=12), "residual")     # columns 5..10 beside 0..5
        _refused(call(fn, res=at["y"] + 28, ld_y=12, ld_res=12), "residual")     # columns 7..12: into the next row
        if _abi.device_count() == 0:
            for kw in (dict(), dict(res=at["y"]), dict(y=at["x"] - 96), dict(res=at["y"] + 24, ld_y=12, ld_res=12),
                       dict(res=at["y"] - 24, ld_y=12, ld_res=12), dict(m=1, res=at["y"], ld_res=99)):
                assert call(fn, **kw) == NO_DEVICE
    def quantize(x=0x1000, q=0x8000, s=0x9000, index=0xa000):
        return L.az_i8_quantize_dev(0, 0, 4, 8, C.c_void_p(x), 8, 5, C.c_void_p(index), 2, C.c_void_p(q), 16, C.c_void_p(s), None)

    assert L.az_i8_quantize_dev(0, 0, 1 << 60, 8, C.c_void_p(0x10000), 1 << 40, 1 << 60, None, 1, C.c_void_p(0x1000), 8,
                                C.c_void_p(0x9000), None) == ARG     # 2^100 bytes: counted without overflow
    for kw in (dict(q=0x1000), dict(q=0x1000 + 156), dict(s=0x1000), dict(s=0x8004), dict(index=0x8000), dict(index=0x9008)):
        _refused(quantize(**kw), "overlap")
    if _abi.device_count() == 0:
        assert quantize() == NO_DEVICE and quantize(q=0x1000 + 160) == NO_DEVICE


def test_ortho_refuses():
    L = _abi.lib()
    good = (3.4445, -4.7750, 2.0315)

    def call(dtype=0, batch=2, rows=5, cols=7, g=P, out=P, steps=5, coeffs=good, eps=1e-7, ws=P, nws=None):
        co = None if coeffs is None else (C.c_double * 3)(*coeffs)
        n = L.az_orthogonalize_ws(max(batch, 0), rows, cols) if nws is None else nws
        return L.az_orthogonalize_dev(0, dtype, batch, rows, cols, g, out, steps, co, eps, ws, n, None)

    _refused(call(dtype=3), "dtype")
    _refused(call(batch=-1), "shape")
    _refused(call(rows=0), "shape")
    _refused(call(cols=32769), "shape")
    _refused(call(steps=0), "steps")
    _refused(call(steps=17), "steps")
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        _refused(call(eps=eps), "eps")
    _refused(call(coeffs=None), "coefficients")
    _refused(call(coeffs=(float("nan"), 0, 0)), "coefficients")
    _refused(call(coeffs=(4.0, 0.0, 0.0)), "coefficients")          # grows without bound
    _refused(call(coeffs=(1.0, -40.0, 39.5)), "coefficients")
    _refused(call(nws=L.az_orthogonalize_ws(2, 5, 7) - 1), "workspace")
    _refused(call(ws=C.c_void_p(128)), "workspace")
    _refused(call(g=None), "null")
    _accepted(call() if _abi.device_count() == 0 else NO_DEVICE)
    _accepted(call(coeffs=(1.5, -0.5, 0.0)) if _abi.device_count() == 0 else NO_DEVICE)


def test_muon_refuses():
    L = _abi.lib()

    def call(items, dtype=0, lr=0.1, momentum=0.9, wd=0.0, nws=None):
        arr = (_abi.az_muon_item * max(len(items), 1))()
        for a, (w, g, m, r, c) in zip(arr, items):
            a.w_dev, a.g_dev, a.m_dev, a.rows, a.cols = w, g, m, r, c
        co = (C.c_double * 3)(*optim.COEFFS)
        n = L.az_muon_step_ws(arr, len(items)) if nws is None else nws
        return L.az_muon_step_dev(0, dtype, arr, len(items), lr, momentum, 1, wd, 5, co, 1e-7, P, n, None)

    one, two = (0x1000, 0x2000, 0x3000, 4, 4), (0x4000, 0x5000, 0x6000, 4, 4)
    _refused(call([one, (0x1000, 0x5000, 0x6000, 4, 4)]), "overlap")
    _refused(call([one, (0x1020, 0x5000, 0x6000, 4, 4)]), "overlap")       # 32 bytes into the first one's 64
    _refused(call([one, (0x4000, 0x5000, 0x3000, 4, 4)]), "overlap")
    _refused(call([(0x1000, 0x1000, 0x3000, 4, 4)]), "overlap")            # the gradient is the weight
    _refused(call([(0x1000, 0x2000, 0x1000, 4, 4)]), "overlap")            # so is the momentum
    _refused(call([one, (0x4000, 0x5000, 0x2000, 4, 4)]), "overlap")       # another item's gradient is the momentum
    many = [(0x10000 + 0x300 * i, 0x10100 + 0x300 * i, 0x10200 + 0x300 * i, 4, 4) for i in range(3000)]
    _refused(call(many + [(0x10000 + 0x300 * 1234 + 0x20, 0x900000, 0xa00000, 4, 4)]), "overlap")
    _refused(call([(0x10000, 0x20000, 0x30000, 64, 64), (0x100000, 0x10100, 0x200000, 4, 4)]), "overlap")   # inside a long one
    if _abi.device_count() == 0:
        assert call(many) == NO_DEVICE
    _refused(call([(0, 0x2000, 0x3000, 4, 4)]), "null")
    _refused(call([(0x1000, 0x2000, 0x3000, 0, 4)]), "shape")
    _refused(call([one], lr=float("nan")), "lr")
    _refused(call([one], momentum=1.0), "momentum")
    _refused(call([one], wd=float("inf")), "weight_decay")
    _refused(call([one], dtype=7), "dtype")
    _refused(call([one], nws=8), "workspace")
    if _abi.device_count() == 0:
        assert call([one, two]) == NO_DEVICE
        assert call([one, (0x4000, 0x2000, 0x6000, 4, 4)]) == NO_DEVICE    # one gradient for two weights is fine


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    w, s = torch.zeros(6, 8, dtype=torch.int8), torch.ones(6)
    for call in (lambda: int8.quantize_rows(x), lambda: int8.linear(x, w, s),
                 lambda: int8.matmul(w, s, w, s), lambda: optim.orthogonalize(x),
                 lambda: optim.muon_step([x], [x.clone()], [x.clone()], lr=0.1)):
        with pytest.raises(_abi.AzError, match="GPU"):
            call()


def test_quotients_are_the_exact_ones():
    """csrc/az_int8.hip quant1 in numpy float32, against the rational quotient: random rows and every tie and its neighbours"""
    f = np.float32
    rng = np.random.default_rng(5)

    def quant1(x, s):
        rs = f(1) / s
        t = np.rint(x * rs).astype(f)
        # x - t s with one rounding: exact in float64 (24 + 8 bits against 24), rounded to float32
        e = (x.astype(np.float64) - t.astype(np.float64) * s.astype(np.float64)).astype(f)
        half, odd = f(0.5) * s, (t.astype(np.int64) & 1) != 0
        up, dn = (e > half) | ((e == half) & odd), (e < -half) | ((e == -half) & odd)
        return np.clip(t + up - dn, -127, 127).astype(np.int64)

    for _ in range(200):
        amax = f(np.exp2(rng.uniform(-60, 60)) * rng.uniform(1, 2))
        s = amax * (f(1) / f(127))
        k = rng.integers(-127, 127, 400)
        tie = ((k + 0.5) * np.float64(s)).astype(f)
        x = np.concatenate([tie, np.nextafter(tie, f(np.inf)), np.nextafter(tie, f(-np.inf)),
                            (rng.uniform(-1, 1, 400) * amax).astype(f)])
        x = np.clip(x, -amax, amax)
        # exact: compare 2 x with (2 k + 1) s in integers of one unit
        mx, ex = np.frexp(x.astype(np.float64))
        unit = int(np.frexp(np.float64(s))[1]) - 200
        xi = [int(m * (1 << 53)) << max(int(e) - 53 - unit, 0) if m else 0 for m, e in zip(mx, ex)]
        ms, es = np.frexp(np.float64(s))
        si = int(ms * (1 << 53)) << (int(es) - 53 - unit)
        want = []
        for v in xi:
            qd, rem = divmod(abs(v), si)
            qd += 1 if 2 * rem > si or (2 * rem == si and qd & 1) else 0
            want.append(max(-127, min(127, qd if v >= 0 else -qd)))
        assert np.array_equal(quant1(x, np.full_like(x, s)), np.array(want))


def test_muon_check_alone():
    """az_muon_step_check: what az_muon_step_dev refuses, without a device and a workspace"""
    L = _abi.lib()

    def call(items, dtype=0, lr=0.1, momentum=0.9, wd=0.0, steps=5, coeffs=optim.COEFFS, eps=1e-7):
        arr = (_abi.az_muon_item * max(len(items), 1))()
        for a, (w, g, m, r, c) in zip(arr, items):
            a.w_dev, a.g_dev, a.m_dev, a.rows, a.cols = w, g, m, r, c
        return L.az_muon_step_check(dtype, arr, len(items), lr, momentum, wd, steps, (C.c_double * 3)(*coeffs), eps)

    one, two = (0x1000, 0x2000, 0x3000, 4, 4), (0x4000, 0x5000, 0x6000, 4, 4)
    assert call([]) == 0 and call([one, two]) == 0
    _refused(call([one, (0x1020, 0x5000, 0x6000, 4, 4)]), "overlap")
    _refused(call([(0x1000, 0x2000, 0x3000, 4, 32769)]), "shape")
    _refused(call([(0x1000, 0, 0x3000, 4, 4)]), "null")
    _refused(call([one], dtype=3), "dtype")
    _refused(call([one], lr=float("inf")), "lr")
    _refused(call([one], momentum=-0.1), "momentum")
    _refused(call([one], steps=0), "steps")
    _refused(call([one], eps=0.0), "eps")
    _refused(call([one], coeffs=(9.0, 0.0, 0.0)), "coefficients")


def test_a_refused_muon_step_leaves_no_state():
    a, b = [torch.nn.Parameter(torch.randn(3, 4)) for _ in range(2)]
    opt = optim.Muon([{"params": [a]}, {"params": [b]}])
    a.grad, b.grad = torch.ones(3, 4), torch.ones(3, 4)
    with pytest.raises(_abi.AzError, match="GPU"):
        opt.step()
    assert not opt.state


def test_outputs_that_autograd_follows_are_refused():
    """written by a kernel, they would keep the graph of what they held before"""
    w, s = torch.zeros(6, 8, dtype=torch.int8), torch.ones(6)
    for out in (torch.zeros(6, 6, requires_grad=True), torch.zeros(6, 6, requires_grad=True) * 2):
        for call in (lambda: int8.matmul(w, s, w, s, out=out), lambda: int8.linear(torch.zeros(6, 8), w, s, out=out),
                     lambda: optim.orthogonalize(torch.zeros(6, 6), out=out)):
            with pytest.raises(_abi.AzError, match="no backward"):
                call()
            with torch.no_grad(), pytest.raises(_abi.AzError, match="GPU"):
                call()
