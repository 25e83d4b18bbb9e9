"""CPU: differentiating a gradient of the framework's autograd functions is refused, not answered without their part.
The kernel calls are stood in for by torch code or by tensors of the right shape."""
from types import SimpleNamespace

import pytest
import torch


def _refused(y, x, loss_of=lambda g: (g * g).sum()):
    """First derivatives under create_graph come out; a loss of theirs and of x refuses its backward."""
    g, = torch.autograd.grad(y.sum() + (x ** 3).sum(), x, create_graph=True)
    assert g.isfinite().all()
    with pytest.raises(RuntimeError, match="second derivative"):
        (loss_of(g) + x.sum()).backward()


def _plain(y, x):
    y.sum().backward()
    assert x.grad.isfinite().all()


@pytest.fixture
def head(monkeypatch):
    from fast_b200 import ops, ranking

    def ln_fwd(x, gamma, beta=None, eps=1e-5, res=None):
        s = x if res is None else x + res
        mean, rstd = s.mean(1), (s.var(1, unbiased=False) + eps).rsqrt()
        y = (s - mean[:, None]) * rstd[:, None] * gamma
        return (y, mean, rstd) if res is None else (y, s, mean, rstd)
    monkeypatch.setattr(ops, "layer_norm_fwd", ln_fwd)
    monkeypatch.setattr(ops, "layer_norm_bwd", lambda dy, x, gamma, mean, rstd, ds=None: (dy * gamma, dy.sum(0), dy.sum(0)))
    monkeypatch.setattr(ops, "gated_ffn_fwd", lambda x, wg, wu, wd, act="silu": ((x @ wg.t()) * (x @ wu.t())) @ wd.t())
    monkeypatch.setattr(ops, "gated_ffn_bwd", lambda dy, x, wg, wu, wd, act="silu", **kw: (
        dy @ wd @ wg, wg.clone(), wu.clone(), wd.clone()))
    monkeypatch.setattr(ops, "softmax_xent_fwd", lambda h, w, t: (torch.ones(len(h)), torch.ones(len(h))))
    monkeypatch.setattr(ops, "softmax_xent_bwd", lambda h, w, t, lse, dl, **kw: (dl[:, None] * h, w.clone()))
    return ranking


@pytest.mark.parametrize("check", [_plain, _refused])
def test_ranking_functions(head, check):
    x = torch.randn(6, 8, requires_grad=True)
    check(head.LayerNormFunction.apply(x, torch.ones(8), torch.zeros(8), 1e-5, None), x)
    x = torch.randn(6, 8, requires_grad=True)
    check(sum(head.LayerNormFunction.apply(x, torch.ones(8, requires_grad=True), None, 1e-5, torch.randn(6, 8))), x)
    x = torch.randn(6, 8, requires_grad=True)
    check(head.GatedFfnFunction.apply(x, torch.randn(12, 8), torch.randn(12, 8), torch.randn(8, 12), "silu"), x)
    x = torch.randn(6, 8, requires_grad=True)
    check(head.SoftmaxXentFunction.apply(x, torch.randn(20, 8), torch.zeros(6, dtype=torch.int64)), x)


def test_a_gradient_penalty_on_the_weights_is_refused(head):
    """The rows need no gradient: the weights' part must not be dropped either."""
    w = [torch.randn(s, requires_grad=True) for s in ((12, 8), (12, 8), (8, 12))]
    y = head.GatedFfnFunction.apply(torch.randn(6, 8), *w, "silu")
    g = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (sum((p * p).sum() for p in g) + sum(p.sum() for p in w)).backward()


@pytest.mark.parametrize("check", [_plain, _refused])
def test_attention_core(monkeypatch, check):
    from fast_b200 import ops
    nd, E, D = 3, 5, 4
    monkeypatch.setattr(ops, "gather_time_encode", lambda n, **kw: torch.ones(n, 2))
    monkeypatch.setattr(ops, "gemm_nt", lambda A, B, bias=None, out=None, M_dev=None: (
        A @ B.t() if out is None else out.copy_(A @ B.t())))
    monkeypatch.setattr(ops, "gemm_tn", lambda A, B, M_dev=None: A.t() @ B)
    monkeypatch.setattr(ops, "colsum", lambda A, M_dev=None: A.sum(0))
    monkeypatch.setattr(ops, "attn_fwd", lambda *a, **kw: (torch.ones(nd, D), torch.ones(E)))
    monkeypatch.setattr(ops, "attn_bwd", lambda *a, **kw: (torch.ones(nd, D), torch.ones(E, 2 * D)))
    blk = SimpleNamespace(n_dst=nd, n_edges=E, n_dst_dev=None, n_edges_dev=None, static=False, src_nodes=None, dst_nodes=None,
                          eid=None, dt_edges=None, rptr=None)
    h = torch.randn(nd + E, 2, requires_grad=True)
    out = ops.AttentionCore.apply(h, None, None, torch.randn(D, 2), torch.randn(D), torch.randn(2 * D, 2), torch.randn(2 * D),
                                  blk, None, None, 1, 0.2, 0.0, 0, None)
    check(out, h)


@pytest.mark.parametrize("check", [_plain, _refused])
def test_fused_softmax_agg(monkeypatch, check):
    from fast_b200 import efficient_gop as eg
    monkeypatch.setattr(eg, "fastAgg", SimpleNamespace(
        forward_fused_softmax_agg=lambda q, k, v, rptr, *a: (q * 2, torch.ones(5)),
        backward_fused_softmax_agg=lambda q, k, v, rptr, att, d, *a: (d * 2, k.clone(), v.clone())))
    q = torch.randn(3, 4, requires_grad=True)
    check(eg.FusedSoftmaxAggTGAT.apply(q, torch.randn(5, 4), torch.randn(5, 4), torch.zeros(4, dtype=torch.int32), 1), q)
