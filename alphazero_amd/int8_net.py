"""The reference's policy/value CNN (environments/Connect4/Network.py:16-85) evaluated in 8-bit integers, at any width, depth,
number of planes and board: for networks that the fused kernel does not know (az_net_load takes h_dim 128 on the 6 x 7 board).

An object of this class is a policy_value_fn: MCTS_AZ / AlphaZeroPlayer call its predict between az_select and az_backup
(MCTS.py:145-146), arena.NetworkSide its net_forward.  Weights are quantised once, a scale for each output channel
(BatchNorm folded in float64); activations anew in every layer, a scale for each board cell (alphazero_amd.int8).
Each weight is off by at most half of 1/127 of its channel's largest, each activation by half of 1/127 of its row's.
"""
import re
import threading

import numpy as np
import torch

from . import int8
from ._abi import AzError

BN_EPS = 1e-5   # torch.nn.BatchNorm2d's
F32_MAX = torch.finfo(torch.float32).max
LOCK = threading.RLock()   # held while a network's tensors on the device change


def capturing(device):
    if torch.cuda.current_device() == device.index:      # as a rule; making it current takes 5 us
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def idle(device):
    """everything that was launched on the device is done"""
    torch.cuda.synchronize(device)


def settle(device):
    """what was launched on the current stream is done: any stream may read it from now on"""
    torch.cuda.current_stream(device).synchronize()


def neighbour_index(rows, cols, boards, device):
    """int32 [boards * rows * cols, 9]: where the taps of a 3x3 convolution with zero padding come from, -1 outside the board"""
    r, c = np.divmod(np.arange(rows * cols), cols)
    taps = []
    for dr in (-1, 0, 1):
        for dc in (-1, 0, 1):
            inside = (r + dr >= 0) & (r + dr < rows) & (c + dc >= 0) & (c + dc < cols)
            taps.append(np.where(inside, (r + dr) * cols + c + dc, -1))
    one = torch.from_numpy(np.stack(taps, 1).astype(np.int32)).to(device)
    base = torch.arange(boards, dtype=torch.int32, device=device).view(-1, 1, 1) * (rows * cols)
    return torch.where(one >= 0, one + base, one).reshape(-1, 9).contiguous()


class Int8CNN:
    def __init__(self, state_dict, board=(6, 7), device="cuda", dtype=torch.float32, game="Connect4"):
        """state_dict: of the reference's CNN (or a module that has one).  dtype: of the activations between layers; float32
        holds whatever a checkpoint does, float16 halves their traffic for networks whose activations stay below 65504.

        Threads and streams may share an object.  forward_device may be captured into a graph once it has been called with as
        many boards or more; the graph needs the object alive, and goes on with the weights that are loaded later."""
        if dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise AzError("Int8CNN: dtype must be float32, float16 or bfloat16")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise AzError("Int8CNN runs on the GPU only (no CPU path)")
        if self.device.index is None:      # this one, whichever is current at a call
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.board, self.dtype, self.game = (int(board[0]), int(board[1])), dtype, game
        self.cells = self.board[0] * self.board[1]
        self._tables, self.layers, self._captured = (), {}, False
        self.load_state_dict(state_dict.state_dict() if hasattr(state_dict, "state_dict") else state_dict)

    def name(self):
        return "Int8CNN"

    # the torch module switches (Network.py:67,79); BatchNorm is folded, there is only eval mode
    def eval(self):
        return self

    def train(self, mode=True):
        return self

    # ---- weights
    def load_state_dict(self, sd):
        """All of it or nothing.  Weights of the shapes that are there go into the same memory, after everything that was launched on the
        device before: no call computes with some of either, and a captured graph goes on with the new ones."""
        with torch.inference_mode(False), torch.no_grad():
            if capturing(self.device):
                raise AzError("Int8CNN: weights cannot be loaded while a graph is captured")
            layers = self._read(sd)
            new = {k: self._quantize(*v) for k, v in layers.items()}
            settle(self.device)
            with LOCK:
                old = self.layers
                alike = old.keys() == new.keys() and all(a.shape == b.shape for k in new for a, b in zip(old[k], new[k]))
                if old and not alike and self._captured:
                    raise AzError("Int8CNN: weights of other shapes than the captured graph's: make a new Int8CNN for them")
                if old:
                    idle(self.device)
                if alike:
                    for k in new:
                        for a, b in zip(old[k], new[k]):
                            a.copy_(b)
                    settle(self.device)
                else:
                    self.layers = new
                self.n_blocks = sum(k.startswith("mix") for k in new)
                self.h_dim, self.in_dim = sd["hidden.0.weight"].shape[:2]
                self.n_actions = new["policy_out"][0].shape[0]

    def sync_from(self, module):
        """the hot reload after a training step: module is the reference's torch CNN (or anything with state_dict())"""
        self.load_state_dict(module.state_dict())

    def _read(self, sd):
        """name -> (matrix [out, k] float64, bias [out] float64), BatchNorm folded, k in the order of our rows"""
        def get(key):
            if key not in sd:
                raise AzError("Int8CNN: the state_dict has no %s" % key)
            t = sd[key].detach().double().cpu()
            if not torch.isfinite(t).all():
                raise AzError("Int8CNN: %s holds a non-finite value" % key)
            return t

        def folded(conv, bn):
            w, g, b = get(conv + ".weight"), get(bn + ".weight"), get(bn + ".bias")
            mean, var = get(bn + ".running_mean"), get(bn + ".running_var")
            if w.dim() != 4 or w.shape[2] != w.shape[3] or w.shape[2] not in (1, 3):
                raise AzError("Int8CNN: %s is no 1x1 or 3x3 convolution" % conv)
            k = g / torch.sqrt(var + BN_EPS)
            w = w * k.view(-1, 1, 1, 1)
            return w.permute(0, 2, 3, 1).reshape(w.shape[0], -1), b - mean * k      # (tap, input channel)

        def fits(name, inputs, taps, outputs=None):
            w, bias = out[name]
            if w.shape[1] != inputs * taps or (outputs is not None and w.shape[0] != outputs) or bias.shape != (w.shape[0],):
                raise AzError("Int8CNN: %s does not fit the layers around it" % name)
            if not all(-F32_MAX <= lo and hi <= F32_MAX for lo, hi in (w.aminmax(), bias.aminmax())):      # nor a NaN, which is no bound
                raise AzError("Int8CNN: %s is not finite in float32 once its BatchNorm is folded in" % name)
            return w.shape[0]

        out = {"stem": folded("hidden.0", "hidden.1")}
        h = fits("stem", sd["hidden.0.weight"].shape[1], 9)
        blocks = sorted({int(m.group(1)) for m in (re.match(r"hidden\.(\d+)\.conv\.0\.weight$", k) for k in sd) if m})
        for i, b in enumerate(blocks):
            out["conv%d" % i] = folded("hidden.%d.conv.0" % b, "hidden.%d.conv.1" % b)
            out["mix%d" % i] = folded("hidden.%d.conv.4" % b, "hidden.%d.conv.5" % b)
            fits("mix%d" % i, fits("conv%d" % i, h, 9), 1, h)
        for head, classes in (("policy", None), ("value", 3)):
            out[head + "_conv"] = folded(head + "_head.0", head + "_head.1")
            c = fits(head + "_conv", h, 1)
            w = get(head + "_head.4.weight")
            if w.dim() != 2 or w.shape[1] != c * self.cells:
                raise AzError("Int8CNN: %s_head.4 takes %d values, the board gives %d" % (head, w.shape[-1], c * self.cells))
            w = w.view(-1, c, self.cells).permute(0, 2, 1).reshape(w.shape[0], -1)  # nn.Flatten's (channel, cell) -> (cell, channel)
            out[head + "_out"] = (w, get(head + "_head.4.bias"))
            fits(head + "_out", c * self.cells, 1, classes)
        return out

    def _quantize(self, w, b):
        q, s = int8.quantize_rows(w.float().to(self.device).contiguous())
        return q, s, b.float().to(self.device)

    # ---- inference
    def _neighbours(self, boards):
        """The first rows of a larger batch's table are a smaller one's.  Tables hold a power of two of boards; they are complete before
        any call sees them and live as long as the object, so that no stream, thread or captured graph is left with one that changes:
        at most twice the memory of the largest, 1.5 KB a board of 42 cells."""
        rows = boards * self.cells
        for t in self._tables:
            if t.shape[0] >= rows:
                return t[:rows]
        with LOCK:
            if self._tables and self._tables[-1].shape[0] >= rows:
                return self._tables[-1][:rows]
            if capturing(self.device):
                raise AzError("Int8CNN: call with %d boards once before capturing a graph of it" % boards)
            t = neighbour_index(*self.board, max(64, 1 << (boards - 1).bit_length()), self.device)
            settle(self.device)
            self._tables += (t,)
        return t[:rows]

    def _conv3(self, x, name, table):
        q, s = int8.quantize_rows(x, index=table)
        w, ws, b = self.layers[name]
        return int8.matmul(q, s, w, ws, bias=b, act="silu", dtype=self.dtype)

    def _logits(self, x, head, boards):
        w, ws, b = self.layers[head + "_conv"]
        t = int8.linear(x, w, ws, bias=b, act="silu")
        q, s = int8.quantize_rows(t.view(boards, -1))
        w, ws, b = self.layers[head + "_out"]
        return int8.matmul(q, s, w, ws, bias=b)

    @torch.no_grad()
    def forward_device(self, planes):
        """(logits [B, n_actions], value logits [B, 3]) float32 of planes [B, in_dim, rows, cols], all on the device"""
        with LOCK:      # a reload waits until all of a call has been launched
            if planes.dim() != 4 or tuple(planes.shape[1:]) != (self.in_dim,) + self.board:
                raise AzError("Int8CNN: planes must be [B, %d, %d, %d]" % ((self.in_dim,) + self.board))
            B = planes.shape[0]
            if B == 0:
                return (torch.empty(0, self.n_actions, device=self.device), torch.empty(0, self.layers["value_out"][0].shape[0], device=self.device))
            self._captured = self._captured or capturing(self.device)
            x = planes.to(self.device, self.dtype).permute(0, 2, 3, 1).reshape(B * self.cells, self.in_dim).contiguous()
            table = self._neighbours(B)
            x = self._conv3(x, "stem", table)
            for i in range(self.n_blocks):
                t = self._conv3(x, "conv%d" % i, table)
                w, ws, b = self.layers["mix%d" % i]
                x = int8.linear(t, w, ws, bias=b, residual=x, act="silu")
            return self._logits(x, "policy", B), self._logits(x, "value", B)

    def forward(self, state):
        """(log_prob (B, n_actions), value_log_prob (B, 3)) float32 numpy -- Network.py:60-64"""
        p, v = self.forward_device(torch.as_tensor(state))
        return torch.log_softmax(p, 1).cpu().numpy(), torch.log_softmax(v, 1).cpu().numpy()

    def predict(self, state, draw_factor=0.5):
        """(probs (B, n_actions), value (B, 1)) float32 numpy, Network.py:78-85: classes [draw, mover wins, mover loses], a draw
        worth -player * draw_factor (the last plane holds the player to move)"""
        state = torch.as_tensor(state)
        p, v = self.forward_device(state)
        v = torch.softmax(v, 1)
        player = state[:, -1, 0, 0].to(self.device, torch.float32)
        value = -player * draw_factor * v[:, 0] + v[:, 1] - v[:, 2]
        return torch.softmax(p, 1).cpu().numpy(), value.view(-1, 1).cpu().numpy()

    def policy(self, state):
        return self.predict(state)[0]

    def value(self, state):
        return np.exp(self.forward(state)[1])

    def net_forward(self, states):
        """SelfPlayEngine.net_forward's form, of packed positions: (logp, logv, probs, value)"""
        from .engine import env_planes_batch
        planes = torch.from_numpy(env_planes_batch(self.game, states, device=self.device.index))
        p, v = self.forward_device(planes)
        logp, logv = torch.log_softmax(p, 1), torch.log_softmax(v, 1)
        w = logv.exp()
        player = planes[:, -1, 0, 0].to(self.device)
        value = (-player * 0.5 * w[:, 0] + w[:, 1] - w[:, 2]).view(-1, 1)
        return logp.cpu().numpy(), logv.cpu().numpy(), logp.exp().cpu().numpy(), value.cpu().numpy()
