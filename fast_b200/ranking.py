"""Node-ranking head: scores an embedding against every node.

The reference's EdgePredictor (layers.py:31-50) compares one positive and one
sampled negative per edge.  This head trains the same root embeddings on the
question a recommender asks -- which node comes next? -- with a softmax over
the whole node table, and answers it for single queries:

    s = x + r;  y = LayerNorm(s);  z = GatedFFN(y);  h = LayerNorm(s + z)
    loss_i = log sum_v exp(h_i . w_v) - h_i . w_target(i)

The logits [rows, nodes] are never kept.  The modules carry fp32 parameters
(as the framework's models do) and give them fp32 gradients; `dtype` is what
the kernels compute in: torch.float32, or torch.bfloat16 with fp32 accumulation
and statistics.  bf16 from fp32 parameters converts them at every call; a head
that only answers queries saves that as a bf16 module throughout
(NodeRankingHead(..., dtype=torch.bfloat16).to(torch.bfloat16)).

    python -m fast_b200.ranking            # trains it on a synthetic temporal graph (one GPU)
    python -m fast_b200.ranking --history  # the same, roots encoded from their own past events (history.py)
"""
import argparse
import math

import torch

from . import ops
from .first_order import first_order


def _rows(t):
    """t as rows the kernels take: unit column stride, no overlap."""
    if t.dim() == 2 and t.stride(1) == 1 and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _f32_or_none(w):
    """The type a weight's gradient is asked for: fp32 for fp32, else the rows'."""
    return torch.float32 if w.dtype == torch.float32 else None


class LayerNormFunction(torch.autograd.Function):
    """(y, s) of rows x [n, D] with the residual res (None: s is x itself)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, eps, res):
        x = _rows(x)
        if res is None:
            y, mean, rstd = ops.layer_norm_fwd(x, gamma, beta, eps)
            s = x
        else:
            y, s, mean, rstd = ops.layer_norm_fwd(x, gamma, beta, eps, _rows(res))
        ctx.save_for_backward(s, gamma, mean, rstd)
        ctx.flags = res is not None, beta is not None
        ctx.set_materialize_grads(False)
        if res is None:
            return y
        return y, s

    @staticmethod
    @first_order
    def backward(ctx, dy, ds=None):
        s, gamma, mean, rstd = ctx.saved_tensors
        has_res, has_beta = ctx.flags
        if dy is None:
            return ds, None, None, None, ds
        dx, dg, db = ops.layer_norm_bwd(_rows(dy), s, gamma, mean, rstd, None if ds is None else _rows(ds))
        return dx, dg, db if has_beta else None, None, dx if has_res else None


class GatedFfnFunction(torch.autograd.Function):
    """y = (act(x Wg^T) * (x Wu^T)) Wd^T; x and the weights in x's type are kept
    for the backward.  Weights of fp32 receive fp32 gradients whatever x's type."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        x, *w = (_rows(t.to(x.dtype)) for t in (x, w_gate, w_up, w_down))
        ctx.save_for_backward(x, *w)
        ctx.act, ctx.grad_dtype = act, _f32_or_none(w_gate)
        return ops.gated_ffn_fwd(x, *w, act)

    @staticmethod
    @first_order
    def backward(ctx, dy):
        x, *w = ctx.saved_tensors
        return (*ops.gated_ffn_bwd(_rows(dy), x, *w, ctx.act, grad_dtype=ctx.grad_dtype), None)


class SoftmaxXentFunction(torch.autograd.Function):
    """Per-row cross entropy (fp32 [n]) of softmax(h w^T), w in h's type.  A
    table of fp32 receives an fp32 gradient.  target: whole numbers of any type."""

    @staticmethod
    def forward(ctx, h, w, target):
        if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool:
            raise ValueError("softmax cross entropy: the targets must be node numbers")
        target = target.to(torch.int64).contiguous()
        ctx.grad_dtype = _f32_or_none(w)
        h, w = _rows(h), _rows(w.to(h.dtype))
        loss, lse = ops.softmax_xent_fwd(h, w, target)
        ctx.save_for_backward(h, w, target, lse)
        return loss

    @staticmethod
    @first_order
    def backward(ctx, dloss):
        h, w, target, lse = ctx.saved_tensors
        dh, dw = ops.softmax_xent_bwd(h, w, target, lse, dloss.contiguous(), grad_dtype=ctx.grad_dtype)
        return dh, dw, None


class GatedFeedForward(torch.nn.Module):
    """The gated feed-forward block with torch.nn.Linear's weight layout."""

    def __init__(self, dim, hidden, act="silu", dtype=torch.float32):
        super().__init__()
        if act not in ops.ACTS:
            raise ValueError("GatedFeedForward: act must be one of %s" % ", ".join(sorted(ops.ACTS)))
        self.act, self.dtype = act, dtype
        self.w_gate = torch.nn.Parameter(torch.randn(hidden, dim) * dim ** -0.5)
        self.w_up = torch.nn.Parameter(torch.randn(hidden, dim) * dim ** -0.5)
        self.w_down = torch.nn.Parameter(torch.randn(dim, hidden) * hidden ** -0.5)

    def forward(self, x):
        rows = x.to(self.dtype).reshape(-1, x.shape[-1])
        return GatedFfnFunction.apply(rows, self.w_gate, self.w_up, self.w_down, self.act).view(x.shape)


class NodeRankingHead(torch.nn.Module):
    """Residual, norm, gated block, norm, and the softmax over `nodes` nodes.
    forward(x, target, res) -> (mean loss over the rows whose target is not
    negative, per-row losses); embed(x, res) -> the rows that are compared with
    the node table.  x and res are [..., dim], target [...]."""

    def __init__(self, dim, nodes, hidden=None, act="silu", dtype=torch.float32, eps=1e-5):
        super().__init__()
        self.dtype, self.eps = dtype, eps
        self.norm1 = torch.nn.ParameterDict(dict(weight=torch.nn.Parameter(torch.ones(dim)),
                                                 bias=torch.nn.Parameter(torch.zeros(dim))))
        self.norm2 = torch.nn.ParameterDict(dict(weight=torch.nn.Parameter(torch.ones(dim)),
                                                 bias=torch.nn.Parameter(torch.zeros(dim))))
        self.ffn = GatedFeedForward(dim, hidden or 4 * dim, act, dtype)
        self.node_table = torch.nn.Parameter(torch.randn(nodes, dim) * dim ** -0.5)

    def embed(self, x, res=None):
        shape = x.shape
        x = x.to(self.dtype).reshape(-1, shape[-1])
        if res is None:
            s, y = x, LayerNormFunction.apply(x, self.norm1["weight"], self.norm1["bias"], self.eps, None)
        else:
            res = res.to(self.dtype).reshape(-1, shape[-1])
            y, s = LayerNormFunction.apply(x, self.norm1["weight"], self.norm1["bias"], self.eps, res)
        h, _ = LayerNormFunction.apply(self.ffn(y), self.norm2["weight"], self.norm2["bias"], self.eps, s)
        return h.view(shape)

    def forward(self, x, target, res=None):
        h = self.embed(x, res)
        rows = SoftmaxXentFunction.apply(h.view(-1, h.shape[-1]), self.node_table, target.reshape(-1)).view(target.shape)
        return rows.sum() / (target >= 0).sum().clamp(min=1), rows


def train_synthetic(steps=60, nodes=400, edges=20000, batch=200, dim=64, dtype=torch.bfloat16, lr=3e-3, seed=0,
                    log=None):
    """Trains a one-layer TGAT embedding and the head on a synthetic graph in
    which most nodes return to a node of their own; returns the losses."""
    import numpy as np

    from .ext import sampler_core
    from .model import DeviceBlock, GeneralModel
    rng = np.random.default_rng(seed)
    dev = torch.device("cuda")
    src = rng.integers(0, nodes, edges).astype(np.int32)
    dst = np.where(rng.random(edges) < 0.9, (src * 7 + 3) % nodes, rng.integers(0, nodes, edges)).astype(np.int32)
    t = np.sort(rng.random(edges) * 1e4).astype(np.float32)
    order = np.argsort(src, kind="stable")
    indptr = np.concatenate([[0], np.cumsum(np.bincount(src, minlength=nodes))]).astype(np.int32)
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    sampler = sampler_core.ParallelSampler(put(indptr), put(dst[order]), put(order.astype(np.int32)), put(t[order]), 1, 1, 1,
                                           [10], True, False, 1, 0.0)
    torch.manual_seed(seed)
    feats, edge_feats = torch.randn(nodes, 32, device=dev), torch.zeros(edges, 4, device=dev)
    model = GeneralModel(32, 4, dict(layer=1, neighbor=[10], strategy="recent", prop_time=False, history=1, duration=0),
                         dict(type="none", dim_out=0),
                         dict(arch="transformer_attention", layer=1, att_head=2, dim_time=16, dim_out=dim),
                         dict(lr=lr, dropout=0.0, att_dropout=0.0)).to(dev)
    head = NodeRankingHead(dim, nodes, dtype=dtype).to(dev)
    params = [p for n, p in model.named_parameters() if not n.startswith("edge_predictor")] + list(head.parameters())
    opt = torch.optim.Adam(params, lr=lr)
    losses, at = [], edges // 4
    for step in range(steps):
        if at + batch > edges:
            at = edges // 4
            sampler.reset()
        sampler.sample_device(put(src[at:at + batch]), put(t[at:at + batch]))
        blocks = [DeviceBlock(v, d) for v, d in zip(sampler.block_views(), sampler.dims())]
        loss, _ = head(model.embed(blocks, feats, edge_feats), put(dst[at:at + batch].astype(np.int64)))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        if log and step % 10 == 0:
            log("step %d: loss %.4f (uniform over %d nodes: %.4f)" % (step, losses[-1], nodes, math.log(nodes)))
        at += batch
    return losses


def train_histories(steps=60, nodes=400, edges=20000, batch=200, dim=64, longest=50, dropout=0.1, dtype=torch.bfloat16, lr=3e-3,
                    seed=0, log=None):
    """Trains a state space encoder of each root's own past events (up to
    `longest`; some roots have none) and the head on a synthetic graph in which
    the next node follows from the last one; returns the losses."""
    import numpy as np

    from .history import HistoryEncoder
    rng = np.random.default_rng(seed)
    dev = torch.device("cuda")
    src = rng.integers(0, nodes, edges)
    jump, last, past = rng.random(edges) < 0.1, rng.integers(0, nodes, nodes), [[] for _ in range(nodes)]
    dst, seen = np.empty(edges, np.int64), []
    for e, s in enumerate(src):
        dst[e] = rng.integers(0, nodes) if jump[e] else (last[s] * 7 + 3) % nodes
        seen.append(len(past[s]))
        last[s] = dst[e]
        past[s].append(dst[e])
    torch.manual_seed(seed)
    embedding = torch.nn.Embedding(nodes, dim).to(dev)
    encoder, head = HistoryEncoder(dim, 2, dropout=dropout, dtype=dtype).to(dev), NodeRankingHead(dim, nodes, dtype=dtype).to(dev)
    opt = torch.optim.Adam([*embedding.parameters(), *encoder.parameters(), *head.parameters()], lr=lr)
    losses, at = [], edges // 4
    for step in range(steps):
        if at + batch > edges:
            at = edges // 4
        rows, starts = [], [0]
        for e in range(at, at + batch):
            rows += past[src[e]][max(0, seen[e] - longest):seen[e]]
            starts.append(len(rows))
        starts = torch.tensor(starts, device=dev)
        x = encoder(embedding(torch.tensor(np.array(rows, dtype=np.int64), device=dev)), starts, seed=seed, offset=step)
        loss, _ = head(encoder.last(x, starts), torch.from_numpy(dst[at:at + batch]).to(dev))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        if log and step % 10 == 0:
            log("step %d: loss %.4f (uniform over %d nodes: %.4f)" % (step, losses[-1], nodes, math.log(nodes)))
        at += batch
    return losses


def main(argv=None):
    ap = argparse.ArgumentParser(description="Train the node-ranking head on a synthetic temporal graph (one GPU).")
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--nodes", type=int, default=400)
    ap.add_argument("--dtype", choices=("bf16", "fp32"), default="bf16")
    ap.add_argument("--history", action="store_true", help="encode roots from their own past events, not sampled neighbours")
    a = ap.parse_args(argv)
    losses = (train_histories if a.history else train_synthetic)(a.steps, a.nodes, dtype=torch.bfloat16 if a.dtype == "bf16" else torch.float32, log=print)
    print("first ten steps %.4f, last ten %.4f" % (sum(losses[:10]) / len(losses[:10]), sum(losses[-10:]) / len(losses[-10:])))


if __name__ == "__main__":
    main()
