"""The operators as they are used together: Int8CNN as a policy_value_fn of the search, Muon between a replay batch and the
reload of the weights."""
import os

import numpy as np
import pytest
import torch

from helpers import blob_to_state_dict

pytestmark = pytest.mark.gpu
G = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


class Net(torch.nn.Module):
    """the reference's architecture (environments/Connect4/Network.py:16-64) with its parameter names, at any width"""

    class Block(torch.nn.Module):
        def __init__(self, h):
            super().__init__()
            self.conv = torch.nn.Sequential(torch.nn.Conv2d(h, h, 3, padding=1, bias=False), torch.nn.BatchNorm2d(h), torch.nn.SiLU(),
                                            torch.nn.Identity(), torch.nn.Conv2d(h, h, 1, bias=False), torch.nn.BatchNorm2d(h))

        def forward(self, x):
            return torch.nn.functional.silu(x + self.conv(x))

    def __init__(self, in_dim=3, h=128, out_dim=7, board=(6, 7)):
        super().__init__()
        n = torch.nn
        cells = board[0] * board[1]
        self.hidden = n.Sequential(n.Conv2d(in_dim, h, 3, padding=1, bias=False), n.BatchNorm2d(h), n.SiLU(), n.Identity(),
                                   Net.Block(h), Net.Block(h), Net.Block(h))
        self.policy_head = n.Sequential(n.Conv2d(h, 3, 1, bias=False), n.BatchNorm2d(3), n.SiLU(), n.Flatten(), n.Linear(3 * cells, out_dim))
        self.value_head = n.Sequential(n.Conv2d(h, 1, 1, bias=False), n.BatchNorm2d(1), n.SiLU(), n.Flatten(), n.Linear(cells, 3))

    def forward(self, x):
        t = self.hidden(x)
        return torch.log_softmax(self.policy_head(t), 1), torch.log_softmax(self.value_head(t), 1)


def jitter(net, seed):
    g = torch.Generator().manual_seed(seed)
    for m in net.modules():
        if isinstance(m, torch.nn.BatchNorm2d):
            m.running_mean.copy_(torch.randn(m.num_features, generator=g) * 0.1)
            m.running_var.copy_(torch.rand(m.num_features, generator=g) + 0.5)
            m.weight.data.copy_(torch.rand(m.num_features, generator=g) + 0.5)
            m.bias.data.copy_(torch.randn(m.num_features, generator=g) * 0.1)
    return net.eval()


def positions(n, seed, in_dim=3, board=(6, 7)):
    g = torch.Generator().manual_seed(seed)
    p = (torch.rand(n, in_dim, *board, generator=g) < 0.3).float()
    p[:, -1] = torch.where(torch.rand(n, 1, 1, generator=g) < 0.5, 1.0, -1.0)
    return p


@pytest.mark.parametrize("in_dim,h,out_dim,board,boards", [(3, 128, 7, (6, 7), 5), (3, 256, 7, (6, 7), 64), (28, 96, 9, (3, 3), 33), (3, 40, 9, (3, 3), 1)])
def test_every_layer_within_its_quantisation(in_dim, h, out_dim, board, boards, monkeypatch):
    """Each layer on the very rows it was given, against the unquantised float64 layer.  Bound (arithmetic): a row's values are
    off by s / 2, a channel's weights by s_w / 2, so a sum over k is off by at most sum |x| s_w / 2 + sum |w| s / 2 + k s s_w / 4; SiLU
    is Lipschitz by 1.1; on top the product's own rounding, (2^-20 of the sum of magnitudes for its float32 steps)."""
    from alphazero_amd import int8
    from alphazero_amd.int8_net import Int8CNN
    net = jitter(Net(in_dim, h, out_dim, board), h)
    q = Int8CNN(net, board=board)
    exact = {k: (w, b) for k, (w, b) in q._read(net.state_dict()).items()}
    names = ["stem"] + [n for i in range(3) for n in ("conv%d" % i, "mix%d" % i)] + ["policy_conv", "policy_out", "value_conv", "value_out"]
    calls = []
    real_rows, real_mm, real_linear = int8.quantize_rows, int8.matmul, int8.linear
    rows = {}

    def rows_spy(x, index=None):
        out = real_rows(x, index=index)
        src = x.double().cpu()
        if index is not None:
            src = torch.cat((src, torch.zeros(1, src.shape[1], dtype=torch.float64)))[index.long().cpu()].reshape(index.shape[0], -1)
        rows["last"] = src
        return out

    def mm_spy(qx, s, w, ws, **kw):
        y = real_mm(qx, s, w, ws, **kw)
        calls.append((rows["last"], y, kw))
        return y

    def linear_spy(x, w, ws, **kw):
        y = real_linear(x, w, ws, **kw)
        calls.append((x.double().cpu(), y, kw))
        return y

    monkeypatch.setattr(int8, "quantize_rows", rows_spy)
    monkeypatch.setattr(int8, "matmul", mm_spy)
    monkeypatch.setattr(int8, "linear", linear_spy)
    state = positions(boards, 1, in_dim, board)
    q.forward_device(state)
    assert len(calls) == len(names)
    for name, (x, y, kw) in zip(names, calls):
        w, b = exact[name]
        s, sw = x.abs().amax(1, keepdim=True) / 127, w.abs().amax(1) / 127
        pre = x @ w.t() + b
        size = x.abs() @ w.abs().t() + b.abs()
        if kw.get("residual") is not None:
            res = kw["residual"].double().cpu()
            pre, size = pre + res, size + res.abs()
        bound = 0.5 * x.abs().sum(1, keepdim=True) * sw + 0.5 * s * w.abs().sum(1) + 0.25 * x.shape[1] * s * sw
        want = pre * torch.sigmoid(pre) if kw.get("act") == "silu" else pre
        assert ((y.double().cpu() - want).abs() <= 1.1 * (1.001 * bound + 2.0 ** -20 * size)).all(), name


def test_predict_and_reload():
    from alphazero_amd._abi import AzError
    from alphazero_amd.int8_net import Int8CNN
    net = jitter(Net(h=64), 3)
    q = Int8CNN(net)
    s = positions(9, 2)
    probs, value = q.predict(s)
    logp, logv = q.forward(s)
    assert probs.shape == (9, 7) and value.shape == (9, 1) and probs.dtype == value.dtype == np.float32
    np.testing.assert_allclose(np.exp(logp), probs, rtol=1e-5)
    v = np.exp(logv)
    np.testing.assert_allclose(value[:, 0], -s[:, 2, 0, 0].numpy() * 0.5 * v[:, 0] + v[:, 1] - v[:, 2], atol=1e-6)
    np.testing.assert_array_equal(q.predict(s[4:5])[0], probs[4:5])       # a position does not depend on its batch
    assert q.predict(s[:0])[0].shape == (0, 7)
    other = jitter(Net(h=64), 4)
    q.sync_from(other)
    np.testing.assert_array_equal(q.predict(s)[0], Int8CNN(other).predict(s)[0])
    kept = q.predict(s)[0]
    bad = other.state_dict()
    bad["hidden.0.weight"][0, 0, 0, 0] = float("nan")
    with pytest.raises(AzError):
        q.load_state_dict(bad)
    np.testing.assert_array_equal(q.predict(s)[0], kept)                  # still the accepted weights
    for call in (lambda: Int8CNN(net, device="cpu"), lambda: Int8CNN(net, board=(3, 3)), lambda: q.predict(s[:, :2]), lambda: Int8CNN({})):
        with pytest.raises(AzError):
            call()


def test_as_policy_value_fn_of_the_search_and_the_arena():
    """a network twice as wide as the fused kernel's, through MCTS_AZ (az_select / az_backup) and a batch of arena games"""
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "alphazero_amd", "dropin")
    sys.path.insert(0, path)
    try:
        from MCTS import MCTS_AZ
        from environments import load
        from alphazero_amd import arena
        from alphazero_amd.int8_net import Int8CNN
        q = Int8CNN(jitter(Net(h=256), 5), dtype=torch.float16)
        env = load("Connect4").Env()
        mcts = MCTS_AZ(q, c_init=1.25, n_playout=24)
        mcts.eval()
        actions, visits = mcts.get_action_visits(env)
        assert len(actions) == 7 and sum(visits) == 23
        winners, plies = arena.play_sides("Connect4", 6, 2, arena.NetworkSide(q, seed=1), arena.NetworkSide(q, deterministic=True))
        assert winners.shape == (6,) and set(winners.tolist()) <= {-1, 0, 1} and (plies >= 7).all()
    finally:
        sys.path.remove(path)


def test_train_step_reload_and_play():
    """replay batch -> gradients -> Muon -> the engine's weights and the 8-bit network's; the update is muon_step's own"""
    from alphazero_amd import optim
    from alphazero_amd.engine import SelfPlayEngine
    from alphazero_amd.int8_net import Int8CNN
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "alphazero_amd", "dropin")
    sys.path.insert(0, path)
    try:
        from environments.network import state_dict_to_blob
    finally:
        sys.path.remove(path)
    blob = np.fromfile(os.path.join(G, "weights", "AZ_Connect4_CNN_current.f32"), dtype="<f4")
    torch.manual_seed(0)
    net = Net().cuda()
    net.load_state_dict(blob_to_state_dict(blob))
    mats, rest = optim.matrices_of(net)
    assert len(mats) == 11 and all(p.dim() < 2 for p in rest)
    opt, other = optim.Muon(mats, lr=0.01, weight_decay=0.01), torch.optim.SGD(rest, lr=0.01)
    net.train()
    x = positions(64, 7).cuda()
    pi, z = torch.softmax(torch.randn(64, 7), 1).cuda(), torch.randint(0, 3, (64,)).cuda()
    mirror = [p.detach().clone() for p in mats]
    momenta = [torch.zeros_like(p) for p in mats]
    for _ in range(3):
        opt.zero_grad(), other.zero_grad()
        logp, logv = net(x)
        loss = -(pi * logp).sum(1).mean() + torch.nn.functional.nll_loss(logv, z)
        loss.backward()
        grads = [p.grad.clone() for p in mats]
        opt.step(), other.step()
        optim.muon_step(mirror, grads, momenta, lr=0.01, weight_decay=0.01)
        for p, m, buf in zip(mats, mirror, momenta):
            assert torch.equal(p.detach(), m) and torch.equal(opt.state[p]["momentum"], buf)
            assert p.isfinite().all()
    net.eval()
    new = state_dict_to_blob(net.state_dict())
    eng = SelfPlayEngine("Connect4", n_games=4, n_playout=8, evaluator="cnn")
    eng.load_net(new)
    eng.search(8)
    assert eng.root_children()["visits"].sum() == 4 * 7
    q = Int8CNN(net)
    states = np.zeros((1, 2), np.uint64)
    _, _, p8, v8 = q.net_forward(states)
    _, _, p32, v32 = eng.net_forward(states)
    assert p8.shape == p32.shape and v8.shape == v32.shape and np.isfinite(p8).all()
    eng.close()


def test_muon_optimizer_states_groups_and_refusals():
    from alphazero_amd import optim
    from alphazero_amd._abi import AzError
    a = torch.nn.Parameter(torch.randn(40, 30).cuda())
    b = torch.nn.Parameter(torch.randn(8, 4, 3, 3).bfloat16().cuda())
    c = torch.nn.Parameter(torch.randn(5, 6).cuda())              # never gets a gradient
    opt = optim.Muon([{"params": [a, c]}, {"params": [b], "lr": 0.1, "nesterov": False}], lr=0.02)
    for _ in range(2):
        a.grad = torch.randn(30, 40).cuda().t()                   # not contiguous
        b.grad = torch.randn_like(b)
        before = c.detach().clone()
        opt.step()
        assert torch.equal(c.detach(), before) and c not in opt.state
    sd = opt.state_dict()
    a2, b2, c2 = [torch.nn.Parameter(p.detach().clone()) for p in (a, b, c)]
    opt2 = optim.Muon([{"params": [a2, c2]}, {"params": [b2]}], lr=0.5)
    opt2.load_state_dict(sd)
    assert opt2.state[b2]["momentum"].dtype == torch.float32 and torch.equal(opt2.state[b2]["momentum"], opt.state[b]["momentum"])
    ga, gb = torch.randn(40, 30).cuda(), torch.randn_like(b)
    for o, x, y in ((opt, a, b), (opt2, a2, b2)):
        x.grad, y.grad = ga.clone(), gb.clone()
        o.step()
    assert torch.equal(a, a2) and torch.equal(b, b2)
    for bad in (lambda: optim.Muon([torch.nn.Parameter(torch.zeros(4))]), lambda: optim.Muon([a], lr=-1.0), lambda: optim.Muon([a], momentum=1.0),
                lambda: optim.Muon([torch.nn.Parameter(torch.zeros(2, 2, dtype=torch.float64))])):
        with pytest.raises(ValueError):
            bad()
    cpu = torch.nn.Parameter(torch.randn(3, 4))
    cpu.grad = torch.randn(3, 4)
    with pytest.raises(AzError):
        optim.Muon([cpu]).step()
