"""GPU: the node-ranking head's modules -- gradients of the whole head against
fp64 autograd, the head's use on sampled blocks, and rows no target is left
for."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(head, x, res, target, dtype):
    """The head in plain torch at fp64 (parameters rounded to the compute type
    where the head rounds them), and the gradients of its mean loss."""
    F = torch.nn.functional
    p = {n: v.detach().double().requires_grad_(True) for n, v in head.named_parameters()}
    q = {n: (v.to(dtype).double() if n in ("ffn.w_gate", "ffn.w_up", "ffn.w_down", "node_table") else v) for n, v in p.items()}
    x, res = x.detach().double().requires_grad_(True), res.detach().double().requires_grad_(True)
    d = (x.shape[1],)
    s = x + res
    y = F.layer_norm(s, d, q["norm1.weight"], q["norm1.bias"], head.eps)
    z = F.linear(F.silu(F.linear(y, q["ffn.w_gate"])) * F.linear(y, q["ffn.w_up"]), q["ffn.w_down"])
    h = F.layer_norm(s + z, d, q["norm2.weight"], q["norm2.bias"], head.eps)
    loss = F.cross_entropy(F.linear(h, q["node_table"]), target, ignore_index=-1)
    loss.backward()
    return loss.detach(), dict(x=x.grad, res=res.grad, **{n: v.grad for n, v in p.items()})


# The head chains about ten roundings (rows, block input, hidden, gradients ...) of u = 2^-8 (bf16) or 2^-24, each
# relative to the tensor it rounds; the norms and the softmax pass relative errors on with a gain of a few.  In the
# 2-norm the roundings are independent: 10 u allowed for the loss, 16 u for a gradient, fp32 products adding theirs
# (2^-21 of the terms' size, K = 300 terms of random sign: 2^-21 sqrt(300) = 2^-17).
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2.0 ** -17), (torch.bfloat16, 16 * 2.0 ** -8)])
def test_head_gradients(cuda, dtype, tol):
    from fast_b200.ranking import NodeRankingHead
    torch.manual_seed(1)
    n, d, v = 150, 100, 700
    head = NodeRankingHead(d, v, dtype=dtype).to(cuda)
    x, res = torch.randn(n, d, device=cuda).to(dtype), torch.randn(n, d, device=cuda).to(dtype)
    target = torch.randint(0, v, (n,), device=cuda)
    target[::7] = -1
    want, grads = _reference(head, x, res, target, dtype)
    x.requires_grad_(True)
    res.requires_grad_(True)
    loss, rows = head(x, target, res)
    loss.backward()
    assert abs(float(loss.detach()) - float(want)) <= tol * float(want)
    assert bool((rows.detach()[::7] == 0).all())
    got = dict(x=x.grad, res=res.grad, **{k: p.grad for k, p in head.named_parameters()})
    assert set(got) == set(grads)
    for k, g in got.items():
        off = float((g.double() - grads[k]).norm() / grads[k].norm())
        assert off <= tol, (k, off)


def test_head_without_residual_and_with_nothing_to_learn(cuda):
    from fast_b200.ranking import NodeRankingHead
    head = NodeRankingHead(32, 90).to(cuda)
    x = torch.randn(8, 32, device=cuda, requires_grad=True)
    loss, rows = head(x, torch.full((8,), -1, device=cuda))
    loss.backward()
    assert float(loss.detach()) == 0 and bool((x.grad == 0).all())
    assert all(bool((p.grad == 0).all()) for p in head.parameters())
    # gradients that arrive as broadcast or transposed tensors
    rows = head(x, torch.arange(8, device=cuda))[1]
    rows.backward(torch.ones(1, device=cuda).expand(8))
    head.embed(x).backward(torch.randn(32, 8, device=cuda).t())
    # one query, no gradient
    with torch.no_grad():
        assert head.embed(x[:1]).shape == (1, 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_synthetic_training_learns_the_next_node(cuda, dtype):
    from fast_b200.ranking import train_synthetic
    losses = train_synthetic(steps=80, nodes=200, edges=8000, batch=100, dim=48, dtype=dtype, lr=5e-3)
    start, end = sum(losses[:5]) / 5, sum(losses[-10:]) / 10
    assert all(math.isfinite(v) for v in losses)
    assert abs(start - math.log(200)) < 1.5 and end < 0.7 * start, (start, end)


def test_operators_in_a_captured_graph(cuda):
    """The operators allocate and launch on the capture stream only."""
    from fast_b200 import ops
    torch.manual_seed(0)
    x, wg, wu = (torch.randn(s, device=cuda).bfloat16() for s in ((300, 64), (128, 64), (128, 64)))
    wd, w = torch.randn(64, 128, device=cuda).bfloat16(), torch.randn(500, 64, device=cuda).bfloat16()
    g, t = torch.ones(64, device=cuda), torch.randint(0, 500, (300,), device=cuda)
    dl = torch.ones(300, device=cuda)

    def step():
        y, mean, rstd = ops.layer_norm_fwd(x, g)
        z = ops.gated_ffn_fwd(y, wg, wu, wd)
        loss, lse = ops.softmax_xent_fwd(z, w, t)
        dz, dw = ops.softmax_xent_bwd(z, w, t, lse, dl)
        dy, *dws = ops.gated_ffn_bwd(dz, y, wg, wu, wd)
        return [loss, dw, *dws, *ops.layer_norm_bwd(dy, x, g, mean, rstd)]
    want = step()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.mul_(0.5)
    graph.replay()
    new = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, new))
    assert not torch.equal(out[0], want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_takes_the_layouts_that_torch_takes(cuda, dtype):
    """Strided and int32 targets, weights and tables that are transposes, rows under several leading dimensions: the
    results are those of contiguous int64 ones."""
    from fast_b200.ranking import GatedFeedForward, GatedFfnFunction, NodeRankingHead, SoftmaxXentFunction
    torch.manual_seed(5)
    x, w = torch.randn(24, 40, device=cuda).to(dtype), torch.randn(90, 40, device=cuda).to(dtype)
    t = torch.randint(0, 90, (24,), device=cuda)
    t[3] = -1
    wide = torch.stack([t, t + 1], 1)
    want = SoftmaxXentFunction.apply(x, w, t)
    for other in (wide[:, 0], t.int(), t.short(), wide.int()[:, 0]):
        assert torch.equal(SoftmaxXentFunction.apply(x, w, other), want)
    table = w.t().contiguous().requires_grad_(True)             # [D, V]; its transpose has no unit column stride
    got = SoftmaxXentFunction.apply(x, table.t(), t)
    assert torch.equal(got, want)
    got.sum().backward()
    assert table.grad.shape == table.shape and bool(table.grad.isfinite().all())
    ws = [torch.randn(s, device=cuda).to(dtype) for s in ((64, 40), (64, 40), (40, 64))]
    y = GatedFfnFunction.apply(x, *ws, "silu")
    turned = [p.t().contiguous().requires_grad_(True) for p in ws]
    y2 = GatedFfnFunction.apply(x, *(p.t() for p in turned), "silu")
    assert torch.equal(y, y2)
    y2.sum().backward()
    assert all(p.grad.shape == p.shape for p in turned)
    with pytest.raises(ValueError):
        SoftmaxXentFunction.apply(x, w, t.float())
    ffn = GatedFeedForward(40, 64, dtype=dtype).to(cuda)
    assert torch.equal(ffn(x.view(2, 3, 4, 40)), ffn(x).view(2, 3, 4, 40))
    head = NodeRankingHead(40, 90, dtype=dtype).to(cuda)
    xs = x.float().view(4, 6, 40).requires_grad_(True)
    loss, rows = head(xs, t.view(4, 6), x.view(4, 6, 40))
    flat, flat_rows = head(x, t, x)
    assert torch.equal(loss, flat) and torch.equal(rows, flat_rows.view(4, 6))
    assert head.embed(xs).shape == xs.shape
    loss.backward()
    assert xs.grad.shape == xs.shape
