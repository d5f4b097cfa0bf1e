"""Int8CNN's bookkeeping and layout on the CPU: what it keeps on the device, with float forms in the place of the 8-bit calls."""
import sys
import threading

import pytest
import torch

from alphazero_amd import int8, int8_net
from alphazero_amd._abi import AzError
from alphazero_amd.int8_net import Int8CNN, neighbour_index
from test_gpu_quantnet import Net, jitter, positions


@pytest.fixture
def on_the_cpu(monkeypatch):
    """Int8CNN on the CPU in float64; says whether a stream is being captured as told"""
    said = {"capturing": False, "settled": 0, "idle": 0}

    def settle(device):
        said["settled"] += 1

    def idle(device):
        said["idle"] += 1

    def quantize_rows(x, index=None):
        rows = x.double()
        if index is not None:
            rows = torch.cat((rows, rows.new_zeros(1, x.shape[1])))[index.long()].reshape(index.shape[0], -1)
        return rows, torch.ones(rows.shape[0], dtype=torch.float64)

    def matmul(q, scale, w, w_scale, bias=None, residual=None, act="none", dtype=None, out=None):
        y = q @ w.t() + bias
        y = y if residual is None else y + residual
        return torch.nn.functional.silu(y) if act == "silu" else y

    monkeypatch.setattr(int8_net, "capturing", lambda device: said["capturing"])
    monkeypatch.setattr(int8_net, "settle", settle)
    monkeypatch.setattr(int8_net, "idle", idle)
    monkeypatch.setattr(int8, "quantize_rows", quantize_rows)
    monkeypatch.setattr(int8, "matmul", matmul)
    monkeypatch.setattr(int8, "linear", lambda x, w, ws, **kw: matmul(x.double(), None, w, ws, **kw))

    def make(net=None, board=(6, 7)):
        q = Int8CNN.__new__(Int8CNN)
        q.device, q.board, q.dtype, q.game, q.cells = torch.device("cpu"), board, torch.float64, "Connect4", board[0] * board[1]
        q._tables, q.layers, q._captured = (), {}, False
        if net is not None:
            q.load_state_dict(net.state_dict())
        return q

    return make, said


def test_a_table_that_was_handed_out_stays_what_it_is(on_the_cpu):
    """a captured graph and other streams hold its address"""
    make, said = on_the_cpu
    q = make()
    held = {b: q._neighbours(b) for b in (5, 64, 1, 65, 300)}
    places = {b: t.data_ptr() for b, t in held.items()}
    for b in range(1, 700, 13):
        assert torch.equal(q._neighbours(b), neighbour_index(6, 7, b, "cpu"))
    for b, t in held.items():
        assert q._neighbours(b).data_ptr() == places[b] and torch.equal(t, neighbour_index(6, 7, b, "cpu"))
    assert said["settled"] == len(q._tables) == 4           # of 64, 128, 512 and 1024 boards
    assert sum(t.shape[0] for t in q._tables) <= 2 * q._tables[-1].shape[0]


def test_a_table_is_not_made_inside_a_capture(on_the_cpu):
    make, said = on_the_cpu
    q = make()
    q._neighbours(64)
    said["capturing"] = True
    assert q._neighbours(3).shape == (126, 9)
    with pytest.raises(AzError, match="65 boards once before"):
        q._neighbours(65)
    assert len(q._tables) == 1


def test_threads_that_ask_for_many_batch_sizes(on_the_cpu):
    make, _ = on_the_cpu
    q = make(board=(3, 3))
    bad = []

    def ask(k):
        try:
            for i in range(400):
                b = 1 + (i * 37 + k * 211) % 900
                if q._neighbours(b).shape != (9 * b, 9):
                    bad.append(b)
        except Exception as e:
            bad.append(repr(e))

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=ask, args=(k,)) for k in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert bad == []


def layers_of(q):
    return {k: [t.clone() for t in v] for k, v in q.layers.items()}


def same_layers(a, b):
    return a.keys() == b.keys() and all(torch.equal(x, y) for k in a for x, y in zip(a[k], b[k]))


def test_a_reload_goes_into_the_same_memory(on_the_cpu):
    """a captured graph and calls on other streams hold its address"""
    make, said = on_the_cpu
    q = make(jitter(Net(h=16), 1))
    places = {k: [t.data_ptr() for t in v] for k, v in q.layers.items()}
    other = jitter(Net(h=16), 2)
    before = said["idle"]
    q.sync_from(other)
    assert said["idle"] == before + 1                      # what was launched before has read the old ones
    assert {k: [t.data_ptr() for t in v] for k, v in q.layers.items()} == places
    assert same_layers(q.layers, make(other).layers)


def test_a_reload_beside_a_capture(on_the_cpu):
    make, said = on_the_cpu
    net = jitter(Net(h=16), 1)
    q = make(net)
    s = positions(3, 1)
    q.forward_device(s)
    kept, want = layers_of(q), q.forward_device(s)
    said["capturing"] = True
    with pytest.raises(AzError, match="while a graph is captured"):
        q.sync_from(jitter(Net(h=16), 2))
    q.forward_device(s)
    said["capturing"] = False
    with pytest.raises(AzError, match="other shapes"):
        q.sync_from(jitter(Net(h=24), 2))                  # the graph reads the old ones
    assert same_layers(q.layers, kept) and (q.h_dim, q.in_dim, q.n_blocks, q.n_actions) == (16, 3, 3, 7)
    assert all(torch.equal(a, b) for a, b in zip(q.forward_device(s), want))
    free = make(net)
    free.sync_from(jitter(Net(in_dim=4, h=24, out_dim=9), 2))
    assert (free.h_dim, free.in_dim, free.n_actions) == (24, 4, 9)
    assert free.forward_device(positions(3, 1, in_dim=4))[0].shape == (3, 9)


def test_weights_loaded_in_inference_mode_can_be_reloaded_outside(on_the_cpu):
    make, _ = on_the_cpu
    with torch.inference_mode():
        q = make(jitter(Net(h=16), 1))
    other = jitter(Net(h=16), 2)
    q.sync_from(other)
    assert same_layers(q.layers, make(other).layers)


def test_what_cannot_be_evaluated_is_refused_whole(on_the_cpu):
    make, _ = on_the_cpu
    q = make(jitter(Net(h=16), 1))
    kept = layers_of(q)
    good = jitter(Net(h=16), 2).state_dict()
    conv, conv1, bn = torch.nn.Conv2d(16, 16, 3).weight.data, torch.nn.Conv2d(16, 16, 1).weight.data, good["hidden.5.conv.1.running_var"]
    for key, value in [("hidden.5.conv.0.weight", conv1), ("hidden.5.conv.4.weight", conv), ("hidden.0.weight", conv1[:, :3]),
                       ("hidden.5.conv.0.weight", conv[:, :8]), ("hidden.5.conv.4.weight", conv1[:8]), ("policy_head.0.weight", conv[:3]),
                       ("policy_head.0.weight", conv1[:2]), ("value_head.4.weight", good["value_head.4.weight"][:2]),
                       ("value_head.4.bias", torch.zeros(2)), ("policy_head.4.bias", torch.zeros(6)),
                       ("hidden.5.conv.1.running_var", torch.full_like(bn, -1.0)),                    # the fold's root of a negative
                       ("hidden.5.conv.1.weight", torch.full(bn.shape, 1e42, dtype=torch.float64))]:      # above float32
        bad = dict(good)
        bad[key] = value
        with pytest.raises((AzError, RuntimeError)):
            q.load_state_dict(bad)
        assert same_layers(q.layers, kept)
    q.load_state_dict(good)
    assert same_layers(q.layers, make(jitter_of(good)).layers)


def jitter_of(state):
    net = Net(h=16)
    net.load_state_dict(state)
    return net


@pytest.mark.parametrize("in_dim,h,out_dim,board,boards", [(3, 24, 7, (6, 7), 5), (5, 16, 11, (3, 5), 4), (3, 40, 9, (4, 3), 1), (28, 8, 4, (2, 9), 3),
                                                           (2, 12, 3, (1, 6), 7)])
def test_without_rounding_it_is_the_float_network(on_the_cpu, in_dim, h, out_dim, board, boards):
    """BatchNorm's fold, the taps' and the flattened cells' order: with exact layers the answers are the torch module's own.  (Its
    float64 sums of at most 9 * 40 terms through 9 layers: 9 * 360 * 2^-53 = 4e-13 of values of some units.)"""
    make, _ = on_the_cpu
    net = jitter(Net(in_dim, h, out_dim, board), h).double()
    q = make(board=board)
    q._quantize = lambda w, b: (w, torch.ones(w.shape[0], dtype=torch.float64), b)
    q.load_state_dict(net.state_dict())
    s = positions(boards, 4, in_dim, board).double()
    with torch.no_grad():
        logp, logv = net(s)
    p, v = q.forward(s)
    assert abs(p - logp.numpy()).max() <= 1e-11 and abs(v - logv.numpy()).max() <= 1e-11
    probs, value = q.predict(s)
    assert abs(probs - logp.exp().numpy()).max() <= 1e-11
    e = logv.exp()
    player = s[:, -1, 0, 0]
    want = -player * 0.5 * e[:, 0] + e[:, 1] - e[:, 2]
    # predict takes the player as float32 (it is 1 or -1); everything else stays in float64 here
    assert abs(value[:, 0] - want.numpy()).max() <= 1e-11
