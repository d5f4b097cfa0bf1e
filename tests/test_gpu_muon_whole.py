"""optim.Muon: a step is made whole or not at all, in any memory format."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def weight(*shape, seed=0, dtype=torch.float32, channels_last=False):
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(*shape, generator=g) / 4).to(dtype).cuda()
    return torch.nn.Parameter(t.to(memory_format=torch.channels_last) if channels_last else t)


def give(p, seed):
    p.grad = torch.randn(*p.shape, generator=torch.Generator().manual_seed(seed)).to(p.dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_channels_last_weights(dtype):
    """the same update as of the contiguous weight, whatever the gradient's and the weight's memory format"""
    from alphazero_amd import optim
    for shape in ((40, 16, 3, 3), (16, 40, 1, 1), (150, 20, 3, 3)):
        a, b = weight(*shape, dtype=dtype), weight(*shape, dtype=dtype, channels_last=True)
        assert torch.equal(a, b)
        oa, ob = optim.Muon([a], weight_decay=0.01), optim.Muon([b], weight_decay=0.01)
        for i in range(3):
            give(a, i)
            b.grad = a.grad.clone(memory_format=torch.channels_last if i else torch.contiguous_format)
            version = b._version
            oa.step(), ob.step()
            assert torch.equal(a, b) and torch.equal(oa.state[a]["momentum"], ob.state[b]["momentum"]) and b._version > version
        assert shape[2] == 1 or (b.is_contiguous(memory_format=torch.channels_last) and not b.is_contiguous())


def test_a_network_in_channels_last():
    from alphazero_amd import optim
    from test_gpu_quantnet import Net, positions
    torch.manual_seed(1)
    nets = [Net(h=32).cuda() for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    nets[1].to(memory_format=torch.channels_last)
    opts = [optim.Muon(optim.matrices_of(n)[0]) for n in nets]
    g = torch.Generator().manual_seed(2)
    for a, b in zip(*[list(n.parameters()) for n in nets]):
        grad = torch.randn(*a.shape, generator=g).cuda()
        a.grad, b.grad = grad, grad.clone()
    for o in opts:
        o.step()
    assert all(torch.equal(a, b) for a, b in zip(*[list(n.parameters()) for n in nets]))
    nets[1](positions(4, 1).cuda())[0].sum().backward()
    opts[1].step()
    assert all(p.isfinite().all() for p in nets[1].parameters())


@pytest.mark.parametrize("how", ["lr", "steps", "coeffs", "eps", "momentum", "cpu", "sparse", "overlap", "large"])
def test_a_refused_step_changes_nothing(how):
    """the second group is refused: the first one's weights, momenta and states are as they were"""
    from alphazero_amd import optim
    from alphazero_amd._abi import AzError
    a, b, c = weight(20, 30, seed=1), weight(10, 12, seed=2), weight(6, 7, seed=3, dtype=torch.bfloat16)
    opt = optim.Muon([{"params": [a]}, {"params": [b, c]}])
    give(a, 1), give(c, 3)
    opt.step()                                  # b has no state yet
    for p, s in ((a, 4), (b, 5), (c, 6)):
        give(p, s)
    group = opt.param_groups[1]
    if how in ("lr", "steps", "coeffs", "eps", "momentum"):
        group[how] = {"lr": float("nan"), "steps": 17, "coeffs": (9.0, 0.0, 0.0), "eps": 0.0, "momentum": 1.0}[how]
    elif how == "cpu":
        bad = torch.nn.Parameter(torch.randn(3, 4))
        bad.grad = torch.randn(3, 4)
        group["params"].append(bad)
    elif how == "sparse":
        b.grad = b.grad.to_sparse()
    elif how == "overlap":
        twin = torch.nn.Parameter(b.detach().view(12, 10))
        twin.grad = b.grad.view(12, 10).clone()
        group["params"].append(twin)
    else:
        b.data, b.grad = torch.zeros(2, 32769).cuda(), torch.zeros(2, 32769).cuda()
    before = [p.detach().clone() for p in (a, b, c)]
    momenta, versions = {p: opt.state[p]["momentum"].clone() for p in (a, c)}, [p._version for p in (a, b, c)]
    with pytest.raises(AzError):
        opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip((a, b, c), before)) and [p._version for p in (a, b, c)] == versions
    assert set(opt.state) == {a, c} and all(torch.equal(opt.state[p]["momentum"], m) for p, m in momenta.items())


def test_weights_that_are_too_long_are_refused_at_once():
    from alphazero_amd import optim
    for shape in ((32769, 2), (2, 32769), (1, 2, 128, 129)):
        with pytest.raises(ValueError, match="32768"):
            optim.Muon([torch.nn.Parameter(torch.zeros(*shape))])
    assert optim.Muon([torch.nn.Parameter(torch.zeros(0, 5)), torch.nn.Parameter(torch.zeros(5, 0)), torch.nn.Parameter(torch.zeros(3, 32768))])


def test_a_step_in_a_graph_with_a_channels_last_weight():
    from alphazero_amd import optim
    a, b = weight(24, 8, 3, 3, channels_last=True), weight(24, 8, 3, 3)
    oa, ob = optim.Muon([a]), optim.Muon([b])
    a.grad = torch.zeros_like(a)
    give(b, 1)
    a.grad.copy_(b.grad)
    oa.step(), ob.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        oa.step()
    for i in range(4):
        give(b, 10 + i)
        a.grad.copy_(b.grad)
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.equal(oa.state[a]["momentum"], ob.state[b]["momentum"])
