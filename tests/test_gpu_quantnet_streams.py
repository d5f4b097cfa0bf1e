"""Int8CNN shared by streams and threads, captured into graphs, and reloaded meanwhile."""
import threading

import pytest
import torch

from test_gpu_quantnet import Net, jitter, positions

pytestmark = pytest.mark.gpu


def net(h=64, seed=3, board=(6, 7)):
    torch.manual_seed(seed)
    return jitter(Net(h=h, board=board), seed)


def make(h=64, seed=3, board=(6, 7)):
    """the same network for the same arguments"""
    from alphazero_amd.int8_net import Int8CNN
    return Int8CNN(net(h, seed, board), board=board)


def busy():
    """some milliseconds of work in front of what is launched next on the current stream"""
    a = torch.randn(4096, 4096, device="cuda")
    for _ in range(4):
        a = a @ a * 1e-3
    return a


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_second_stream_asks_for_the_same_batch_at_once():
    for boards in (9, 100, 1000):
        q = make()
        s = positions(boards, boards).cuda()
        want = make().forward_device(s)
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            kept = busy()
            a = q.forward_device(s)
        with torch.cuda.stream(two):
            b = q.forward_device(s)
        torch.cuda.synchronize()
        assert same(a, want) and same(b, want) and kept.shape == (4096, 4096)


def test_threads_on_streams_of_their_own():
    q = make(h=32)
    batches = {b: positions(b, b).cuda() for b in (1, 3, 17, 64, 65, 130, 257, 300, 511, 600, 777, 1025)}
    want = {b: make(h=32).forward_device(s) for b, s in batches.items()}
    torch.cuda.synchronize()
    bad = []

    def ask(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                order = sorted(batches, key=lambda b: (b * 7919 * (k + 1)) % 1009)
                for b in order * 3:
                    y = q.forward_device(batches[b])
                    torch.cuda.current_stream().synchronize()
                    if not same(y, want[b]):
                        bad.append(b)
        except Exception as e:
            bad.append(repr(e))

    threads = [threading.Thread(target=ask, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert bad == []


def test_a_graph_outlives_many_other_batch_sizes():
    q = make()
    s = positions(33, 1).cuda()
    q.forward_device(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = q.forward_device(s)
    for i in range(12):
        s.copy_(positions(33, 50 + i))
        graph.replay()
        other = positions(40 * i + 7, i).cuda()
        q.forward_device(other)                        # other sizes between the replays
        filler = torch.full((300000,), -1, dtype=torch.int32, device="cuda")      # takes what was freed, if anything was
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, q.forward_device(s)) and filler.numel()


def test_a_batch_that_has_no_table_yet_is_refused_inside_a_capture():
    from alphazero_amd._abi import AzError
    q = make()
    s = positions(20, 1).cuda()
    graph, said = torch.cuda.CUDAGraph(), []
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = s * 2
        try:
            q.forward_device(s)
        except AzError as e:
            said.append(str(e))
    graph.replay()
    torch.cuda.synchronize()
    assert len(said) == 1 and "once before" in said[0] and torch.equal(out, s * 2)
    assert same(q.forward_device(s), make().forward_device(s))


def test_a_graph_goes_on_with_reloaded_weights():
    from alphazero_amd._abi import AzError
    q = make()
    s = positions(33, 1).cuda()
    q.forward_device(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = q.forward_device(s)
    for seed in (3, 4, 5, 6, 7):
        q.sync_from(net(seed=seed))
        filler = torch.full((4 << 20,), 77, dtype=torch.int8, device="cuda")       # takes what was freed, if anything was
        s.copy_(positions(33, seed))
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, make(seed=seed).forward_device(s)) and same(out, q.forward_device(s)) and filler.numel()
    with pytest.raises(AzError, match="other shapes"):
        q.sync_from(net(h=32))


def test_a_reload_waits_for_the_calls_before_it():
    q, s = make(seed=3), positions(500, 2).cuda()
    old, new = make(seed=3).forward_device(s), make(seed=4).forward_device(s)
    q.forward_device(s)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        kept = busy()
        a = q.forward_device(s)
    q.sync_from(net(seed=4))
    b = q.forward_device(s)
    torch.cuda.synchronize()
    assert same(a, old) and same(b, new) and not same(old, new) and kept.shape == (4096, 4096)


def test_reloads_between_the_calls_of_other_threads():
    """every answer is the one of some accepted weights as a whole"""
    q, s = make(h=32, seed=3), positions(70, 2).cuda()
    allowed = [make(h=32, seed=i).forward_device(s) for i in (3, 4)]
    states = [net(h=32, seed=i).state_dict() for i in (3, 4)]
    q.forward_device(s)
    torch.cuda.synchronize()
    bad, done = [], threading.Event()

    def ask():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not done.is_set():
                    y = q.forward_device(s)
                    torch.cuda.current_stream().synchronize()
                    if not any(same(y, w) for w in allowed):
                        bad.append(y)
        except Exception as e:
            bad.append(repr(e))

    threads = [threading.Thread(target=ask) for _ in range(2)]
    for t in threads:
        t.start()
    for i in range(20):
        q.load_state_dict(states[(i + 1) % 2])
    done.set()
    for t in threads:
        t.join()
    assert bad == []
