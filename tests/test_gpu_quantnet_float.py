"""Int8CNN's layers against the torch module's own: inputs and outputs recorded from the module, weights read from it."""
import pytest
import torch

from test_gpu_quantnet import Net, jitter, positions

pytestmark = pytest.mark.gpu


def rows_of(t):
    """[B, C, rows, cols] -> [B * cells, C]"""
    return t.permute(0, 2, 3, 1).reshape(-1, t.shape[1]).contiguous()


def bound(x, w, s=None, extra=0.0):
    """how far a layer's sums may be from the exact ones on rows x [m, k], weights w [n, k]: values off by half a step of their row
    (largest / 127), weights by half a step of their channel, and the float32 of scales and epilogue, 2^-20 of the magnitudes"""
    step, step_w = x.abs().amax(1, keepdim=True) / 127, w.abs().amax(1) / 127
    size = x.abs() @ w.abs().t() + extra
    return 1.001 * (0.5 * x.abs().sum(1, keepdim=True) * step_w + 0.5 * step * w.abs().sum(1) + 0.25 * x.shape[1] * step * step_w) + 2.0 ** -20 * size


@pytest.mark.parametrize("in_dim,h,out_dim,board,boards", [(3, 128, 7, (6, 7), 9), (3, 64, 7, (6, 7), 40), (5, 96, 11, (3, 5), 33), (4, 40, 9, (4, 3), 1)])
def test_layers_are_the_modules(in_dim, h, out_dim, board, boards):
    """SiLU is Lipschitz by 1.1.  The module's convolutions are read as they are, BatchNorm as the scale of a channel that it is in
    eval mode; the rows of a 3x3 convolution come from unfold, with the weight's own (channel, tap) order."""
    from alphazero_amd import int8
    from alphazero_amd.int8_net import Int8CNN
    torch.manual_seed(h)
    net = jitter(Net(in_dim, h, out_dim, board), h)
    q = Int8CNN(net, board=board)
    net = net.double()
    seen = {}
    for name, m in net.named_modules():
        m.register_forward_hook(lambda mod, args, out, name=name: seen.__setitem__(name, (args[0], out)))
    with torch.no_grad():
        net(positions(boards, 2, in_dim, board).double())

    def gpu(t):
        return t.float().cuda()

    def check(y, want, x, w, k, what, extra=0.0):
        """x, w: the exact layer's rows and weights; k: the norm's factor per channel"""
        allowed = 1.1 * bound(x, w * k.abs()[:, None], extra=extra)
        assert ((y.double().cpu() - want).abs() <= allowed).all(), what

    def factor(bn):
        m = net.get_submodule(bn)
        return (m.weight / torch.sqrt(m.running_var + m.eps)).detach()

    def conv3(name, conv, bn, act):
        c = net.get_submodule(conv)
        x = seen[conv][0]
        y = q._conv3(gpu(rows_of(x)), name, q._neighbours(boards))
        rows = torch.nn.functional.unfold(x, 3, padding=1).transpose(1, 2).reshape(boards * board[0] * board[1], -1)
        b = net.get_submodule(bn).bias.detach().abs() + (net.get_submodule(bn).running_mean * factor(bn)).abs()
        check(y, rows_of(seen[act][1]), rows, c.weight.detach().reshape(c.weight.shape[0], -1), factor(bn), name, b)

    conv3("stem", "hidden.0", "hidden.1", "hidden.2")
    for i in range(3):
        at = "hidden.%d" % (4 + i)
        conv3("conv%d" % i, at + ".conv.0", at + ".conv.1", at + ".conv.2")
        c, bn = net.get_submodule(at + ".conv.4"), at + ".conv.5"
        x, whole = rows_of(seen[at + ".conv.4"][0]), rows_of(seen[at][0])
        w, ws, b = q.layers["mix%d" % i]
        y = int8.linear(gpu(x), w, ws, bias=b, residual=gpu(whole), act="silu")
        extra = whole.abs() + net.get_submodule(bn).bias.detach().abs() + (net.get_submodule(bn).running_mean * factor(bn)).abs()
        check(y, rows_of(seen[at][1]), x, c.weight.detach()[:, :, 0, 0], factor(bn), "mix%d" % i, extra)
    for head in ("policy", "value"):
        conv, bn, out = [net.get_submodule("%s_head.%d" % (head, n)) for n in (0, 1, 4)]
        x = rows_of(seen[head + "_head.0"][0])
        w, ws, b = q.layers[head + "_conv"]
        y = int8.linear(gpu(x), w, ws, bias=b, act="silu")
        k = factor(head + "_head.1")
        check(y, rows_of(seen[head + "_head.2"][1]), x, conv.weight.detach()[:, :, 0, 0], k, head + "_conv",
              bn.bias.detach().abs() + (bn.running_mean * k).abs())
        flat = seen[head + "_head.4"][0]
        rows = rows_of(seen[head + "_head.2"][1]).reshape(boards, -1)          # a board's cells, each with its channels
        w, ws, b = q.layers[head + "_out"]
        qx, s = int8.quantize_rows(gpu(rows))
        y = int8.matmul(qx, s, w, ws, bias=b)
        want = seen[head + "_head.4"][1]
        assert ((y.double().cpu() - want).abs() <= bound(flat, out.weight.detach(), extra=out.bias.detach().abs())).all(), head
