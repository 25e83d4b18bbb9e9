"""Event histories: a state space encoder over the events of each node.

The reference encodes a node by the neighbours it samples (TGAT) or by a memory
that its last mail updates (TGN's GRU, memorys.py:270-304; APAN's attention over
a mailbox, memorys.py:342-386).  This encoder reads a node's whole history, of
any length, in one pass over packed rows,

    rows of node a | rows of node b | ...,   starts = [0, len a, len a + len b, ...]

and is trained in parallel along it.  What a node's history leaves behind is a
state of fixed size, so that afterwards the encoder follows the stream event by
event from per-node tables (NodeStates), as the framework's memory modules do.
A block, with the state space scan between two products:

    y = LayerNorm(x);  [v | z] = y W_in^T;  u = silu(conv(v))
    [d | B | C] = u W_x^T;  delta = d W_dt^T
    h[t] = exp(dt A) h[t - 1] + dt u B,  dt = softplus(delta + b_dt),  s = (<C, h> + D u) silu(z)
    x' = x + dropout(s W_out^T)

Parameters are fp32 (as the framework's models carry them) and receive fp32
gradients; `dtype` is what the kernels compute in: torch.float32, or
torch.bfloat16 with fp32 states, decays and sums.

    python -m fast_b200.ranking --history     # trains it in front of the node-ranking head (one GPU)
"""
import math

import torch

from . import ops
from .first_order import first_order
from .ranking import LayerNormFunction, _rows


class ShortConvFunction(torch.autograd.Function):
    """(y, final) of packed rows x [rows, D]; w [D, K] and bias [D] in fp32.
    Without `final` only y is computed, None comes in the states' place."""

    @staticmethod
    def forward(ctx, x, w, bias, starts, init, act, final=True):
        x, w = _rows(x), w.contiguous()
        bias, init = (None if t is None else t.contiguous() for t in (bias, init))
        ctx.save_for_backward(x, w, bias, starts, init)
        ctx.act = act
        ctx.set_materialize_grads(False)
        out = ops.short_conv_fwd(x, w, bias, starts, init, act, final=final)
        return out if final else (out, None)

    @staticmethod
    @first_order
    def backward(ctx, dy, dfinal):
        x, w, bias, starts, init = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 7
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        dx, dw, dbias, dinit = ops.short_conv_bwd(dy, x, w, bias, starts, init, ctx.act,
                                                  None if dfinal is None else dfinal.contiguous())
        return dx, dw, dbias, None, dinit, None, None


class SelectiveScanFunction(torch.autograd.Function):
    """(y, final) of packed rows u, delta, z [rows, D]; A [D, N], D, delta_bias [D], init [seqs, D, N] in fp32.
    `graph`: whether the caller records one (torch.is_grad_enabled(), which a
    function's forward cannot see); without, nothing is kept for a backward.
    `final` as in ShortConvFunction."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, starts, init, softplus, graph=True, final=True):
        u, delta = _rows(u), _rows(delta)
        B, C = (t if t.stride(-1) == 1 else t.contiguous() for t in (B, C))
        z = None if z is None else _rows(z)
        A, D, delta_bias, init = (None if t is None else t.contiguous() for t in (A, D, delta_bias, init))
        y, carry, behind = ops.selective_scan_fwd(u, delta, A, B, C, D, z, delta_bias, starts, init, softplus, final=final,
                                                  keep=graph and any(ctx.needs_input_grad))
        ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, starts, init, carry)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, behind

    @staticmethod
    @first_order
    def backward(ctx, dy, dfinal):
        u, delta, A, B, C, D, z, delta_bias, starts, init, carry = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 13
        dy = torch.zeros_like(u) if dy is None else _rows(dy)
        du, dd, dA, dB, dC, dD, dz, db, dinit = ops.selective_scan_bwd(
            dy, u, delta, A, B, C, carry, D, z, delta_bias, starts, init, ctx.softplus,
            None if dfinal is None else dfinal.contiguous())
        return du, dd, dA, dB, dC, dD, dz, db, None, dinit, None, None, None


class DropoutFunction(torch.autograd.Function):
    """res + dropout(x) (res None: dropout(x)) of rows, from (seed, offset); the
    mask is drawn again in the backward.  offset_dev: a device int64 [1] added to
    the offset, which must keep its value until the backward (autograd refuses one
    that was changed)."""

    @staticmethod
    def forward(ctx, x, res, p, seed, offset, offset_dev=None):
        ctx.how = p, seed, offset
        ctx.has_res = res is not None
        ctx.save_for_backward(offset_dev if p else None)                # p = 0 draws nothing again
        return ops.dropout_fwd(_rows(x), p, seed, offset, None if res is None else _rows(res), offset_dev)

    @staticmethod
    @first_order
    def backward(ctx, dy):
        offset_dev, = ctx.saved_tensors
        dx = ops.dropout_bwd(_rows(dy), *ctx.how, offset_dev) if ctx.how[0] else dy      # p = 0 keeps all, unscaled
        return dx, dy if ctx.has_res else None, None, None, None, None


class NodeStates:
    """What every node's history has left behind, for one encoder: for each block
    the last K - 1 inputs of its convolution [nodes, K - 1, inner] (compute type)
    and the states of its scan [nodes, inner, N] (fp32)."""

    def __init__(self, encoder, nodes, device):
        self.conv, self.scan = [], []
        for b in encoder.blocks:
            self.conv.append(torch.zeros(nodes, b.taps - 1, b.inner, dtype=b.dtype, device=device))
            self.scan.append(torch.zeros(nodes, b.inner, b.states, dtype=torch.float32, device=device))

    def reset(self):
        for t in self.conv + self.scan:
            t.zero_()


class StateSpaceBlock(torch.nn.Module):
    """One block over packed rows [rows, dim] (see the module's docstring)."""

    def __init__(self, dim, inner=None, states=16, taps=4, rank=None, dropout=0.0, dtype=torch.float32, eps=1e-5):
        super().__init__()
        if not 1 <= states <= 64 or not 1 <= taps <= 8 or not 0.0 <= dropout < 1.0:
            raise ValueError("StateSpaceBlock: 1 to 64 states, 1 to 8 taps, dropout in [0, 1)")
        inner, rank = inner or 2 * dim, rank or max(1, dim // 16)
        self.inner, self.states, self.taps, self.rank = inner, states, taps, rank
        self.dropout, self.dtype, self.eps = dropout, dtype, eps
        self.norm = torch.nn.ParameterDict(dict(weight=torch.nn.Parameter(torch.ones(dim)),
                                                bias=torch.nn.Parameter(torch.zeros(dim))))
        self.w_in = torch.nn.Parameter(torch.randn(2 * inner, dim) * dim ** -0.5)
        self.w_conv = torch.nn.Parameter(torch.randn(inner, taps) * taps ** -0.5)
        self.b_conv = torch.nn.Parameter(torch.zeros(inner))
        self.w_x = torch.nn.Parameter(torch.randn(rank + 2 * states, inner) * inner ** -0.5)
        self.w_dt = torch.nn.Parameter(torch.randn(inner, rank) * rank ** -0.5)
        # dt log-uniform in [0.001, 0.1] at the start, decays of 1 .. N
        dt = torch.exp(torch.rand(inner) * math.log(100.0) + math.log(1e-3))
        self.b_dt = torch.nn.Parameter(torch.log(torch.expm1(dt)))
        self.log_decay = torch.nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32)).repeat(inner, 1))
        self.skip = torch.nn.Parameter(torch.ones(inner))
        self.w_out = torch.nn.Parameter(torch.randn(dim, inner) * inner ** -0.5)

    def _product(self, x, w):
        return torch.nn.functional.linear(x, w.to(self.dtype))

    def _inner(self, x):
        y = LayerNormFunction.apply(x, self.norm["weight"], self.norm["bias"], self.eps, None)
        return self._product(y, self.w_in).split(self.inner, dim=1)

    def _scan_inputs(self, u):
        d, b, c = self._product(u, self.w_x).split([self.rank, self.states, self.states], dim=1)
        return self._product(d, self.w_dt), -torch.exp(self.log_decay.float()), b, c

    def forward(self, x, starts=None, conv=None, scan=None, seed=0, offset=0, states=True, offset_dev=None):
        """Rows x [rows, dim] of packed histories -> (x', conv, scan): the rows
        behind the block and what each history leaves, which a call for the rows
        to come takes as `conv` and `scan` (None without `states`).  In training,
        dropout draws from (seed, offset + offset_dev), the latter a device int64
        [1] for graphs whose replays draw anew."""
        return self._run(x, starts, conv, scan, self.dropout if self.training else 0.0, seed, offset, states, offset_dev)

    def _run(self, x, starts, conv, scan, p, seed=0, offset=0, states=True, offset_dev=None):
        v, z = self._inner(x)
        u, conv = ShortConvFunction.apply(v, self.w_conv.float(), self.b_conv.float(), starts, conv, "silu", states)
        delta, A, b, c = self._scan_inputs(u)
        s, scan = SelectiveScanFunction.apply(u, delta, A, b, c, self.skip.float(), z, self.b_dt.float(), starts, scan, True,
                                              torch.is_grad_enabled(), states)
        return DropoutFunction.apply(self._product(s, self.w_out), x, p, seed, offset, offset_dev), conv, scan

    @torch.no_grad()
    def step(self, x, conv, scan, index=None):
        """One event a row: x [n, dim] of nodes index [n] (None: row r is node r)
        through the block, against the tables conv and scan, updated in place."""
        v, z = self._inner(x)
        u = ops.short_conv_step(_rows(v), conv, self.w_conv.float(), self.b_conv.float(), index)
        delta, A, b, c = self._scan_inputs(u)
        s = ops.selective_scan_step(u, delta, A, b, c, scan, self.skip.float(), _rows(z), self.b_dt.float(), index)
        return x + self._product(s, self.w_out)


class HistoryEncoder(torch.nn.Module):
    """Blocks over packed event rows.  forward: training and whole histories;
    follow: histories that continue the nodes' states, and leave theirs; step:
    single events."""

    def __init__(self, dim, blocks=2, inner=None, states=16, taps=4, dropout=0.0, dtype=torch.float32):
        super().__init__()
        self.dtype = dtype
        self.blocks = torch.nn.ModuleList(StateSpaceBlock(dim, inner, states, taps, None, dropout, dtype) for _ in range(blocks))

    def forward(self, x, starts=None, seed=0, offset=0, offset_dev=None):
        """Rows [rows, dim] -> encoded rows.  Rows of no history come out as they
        went in.  Block i draws its dropout from (seed + i, offset + offset_dev),
        counted in 64 bits; a captured training step advances the counter
        offset_dev (device int64 [1]) behind its backward, so that every replay
        draws anew."""
        x = x.to(self.dtype)
        for i, b in enumerate(self.blocks):
            x = b(x, starts, seed=(seed + i) % (1 << 64) if i else seed, offset=offset, states=False, offset_dev=offset_dev)[0]
        return x

    @staticmethod
    def last(rows, starts):
        """The last row of each history [seqs, dim]; zeros for an empty one."""
        if not rows.shape[0]:
            return rows.new_zeros(starts.shape[0] - 1, rows.shape[1])
        starts = starts.clamp(0, rows.shape[0])                      # as the operators do
        some = starts[1:] > starts[:-1]
        return torch.where(some.unsqueeze(1), rows[(starts[1:] - 1).clamp(min=0)], rows.new_zeros(()))

    @torch.no_grad()
    def follow(self, x, starts, tables, index):
        """Encodes packed histories that continue those of nodes index [seqs]
        (each node once; int64, 0 .. nodes - 1), whose states in `tables` are read
        and replaced.  As in step nothing drops out, in training mode either: the
        tables outlive the call."""
        x = x.to(self.dtype)
        for b, conv, scan in zip(self.blocks, tables.conv, tables.scan):
            x, c, s = b._run(x, starts, conv[index], scan[index], 0.0)
            conv[index], scan[index] = c, s
        return x

    def step(self, x, tables, index=None):
        """One event a row of nodes index [n], in chronological order (a node may
        come several times): encoded rows; `tables` is updated in place.  A
        negative index holds its row out."""
        x = x.to(self.dtype)
        for b, conv, scan in zip(self.blocks, tables.conv, tables.scan):
            x = b.step(x, conv, scan, index)
        return x
