"""GPU: the node-ranking head's operators where the caller, single values or rows are out of the ordinary, against fp64
restatements.  Bounds are test_head_gpu.py's: c = (K + 64) 2^-22 of the terms' sum for a product of K terms, 2^-8 for a
rounding to bf16."""
import math
import threading

import pytest
import torch

from test_head_gpu import _c, _check, _gen, _mat, test_gated_ffn as gated_ffn, test_softmax_xent as softmax_xent

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TYPES = [F32, BF]


# ---- threads ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("call", ["ffn_fwd", "ffn_bwd", "xent_fwd", "xent_bwd", "gemm"])
@pytest.mark.parametrize("dtype", TYPES)
def test_first_gpu_call_of_a_thread(cuda, call, dtype):
    """A thread that has no CUDA context yet (autograd's, in a first backward) gets the main thread's results."""
    from fast_b200 import ops
    g = _gen(cuda, 150, 64)
    x, dy = _mat(cuda, g, 300, 64, dtype), _mat(cuda, g, 300, 64, dtype)
    wg, wu, wd = _mat(cuda, g, 136, 64, dtype), _mat(cuda, g, 136, 64, dtype), _mat(cuda, g, 64, 136, dtype)
    t = torch.randint(0, 136, (300,), device=cuda, generator=g)
    lse, one = ops.softmax_xent_fwd(x, wg, t)[1], torch.ones(300, device=cuda)
    run = dict(ffn_fwd=lambda: [ops.gated_ffn_fwd(x, wg, wu, wd)], ffn_bwd=lambda: ops.gated_ffn_bwd(dy, x, wg, wu, wd),
               xent_fwd=lambda: ops.softmax_xent_fwd(x, wg, t), xent_bwd=lambda: ops.softmax_xent_bwd(x, wg, t, lse, one),
               gemm=lambda: [ops.gemm_nt_tc(x.float(), wg.float())])[call]
    want, again = run(), run()                                  # memory for a third run is at hand
    del again
    torch.cuda.synchronize()
    got = []

    def body():
        try:
            got.extend(run())
        except Exception as e:                                  # noqa: BLE001 (reported below)
            got.append(e)
    th = threading.Thread(target=body)
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert not isinstance(got[0], Exception), got[0]
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_block_alone_trains(cuda):
    """The block's backward is the first thing autograd's thread runs."""
    from fast_b200.ranking import GatedFeedForward
    torch.manual_seed(2)
    ffn = GatedFeedForward(64, 136, dtype=BF).to(cuda)
    x = torch.randn(150, 64, device=cuda).bfloat16()
    ffn(x).backward(torch.ones(150, 64, device=cuda, dtype=BF))
    assert all(bool(p.grad.isfinite().all()) for p in ffn.parameters())


# ---- infinities ------------------------------------------------------------------------------------------------------
# rows on both sides of every rule that picks a path: few rows, tiles, fp32 logits stored in split sums
@pytest.mark.parametrize("n,d,v", [(1, 40, 700), (8, 33, 700), (9, 33, 700), (300, 40, 3000), (60, 600, 500)])
@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_nodes_masked_by_an_infinite_bias(cuda, n, d, v, dtype):
    """h has a column of ones, the table -inf there for some nodes: they have probability 0."""
    from fast_b200 import ops
    g = _gen(cuda, n, d, v)
    h, w = _mat(cuda, g, n, d, dtype), _mat(cuda, g, v, d, dtype, 2 * d ** -0.5)
    h[:, 0] = 1
    masked = torch.arange(v, device=cuda) % 3 == 1
    w[masked, 0] = -math.inf
    t = torch.randint(0, v // 3, (n,), device=cuda, generator=g) * 3
    dl = torch.rand(n, device=cuda, generator=g) + 0.5
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    H, W = h.double(), w.double()[~masked]
    L = H @ W.t()
    Z = torch.logsumexp(L, 1)
    el = (_c(d) * (H.abs() @ W.abs().t())).max(1).values
    fn = 2.0 ** -20 * (1 + Z.abs() + L.abs().max(1).values)
    at = (t - (t + 1) // 3).unsqueeze(1)                       # t's place among the nodes left
    _check("lse", lse, Z, el + fn, F32)
    _check("loss", loss, Z - L.gather(1, at)[:, 0], 2 * el + fn, F32)
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, dl)
    P = torch.softmax(L, 1)
    G = P.clone()
    G.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float64))
    scale = dl.double().unsqueeze(1)
    eG = scale * (P * (2 * el + 2 * fn).unsqueeze(1) + 2.0 ** -22 * G.abs())
    G = G * scale
    eG = eG + (2.0 ** -8 if dtype == BF else 0.0) * (G.abs() + eG)
    assert bool((dw[masked] == 0).all())
    _check("dw", dw[~masked], G.t() @ H, eG.t() @ H.abs() + _c(n) * ((G.abs() + eG).t() @ H.abs()), dtype)
    # the bias column of dh is 0 times -inf; the others are sums over the nodes left
    _check("dh", dh[:, 1:], (G @ W)[:, 1:], (eG @ W.abs() + _c(v) * ((G.abs() + eG) @ W.abs()))[:, 1:], dtype)


@pytest.mark.parametrize("n", [1, 8, 9, 200])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_ffn_with_infinite_values(cuda, n, dtype):
    """An infinite weight makes infinities of its own column, an infinite row reaches no other row."""
    from fast_b200 import ops
    d, f = 40, 72
    g = _gen(cuda, n, d, f)
    x = _mat(cuda, g, n, d, dtype)
    wg, wu, wd = _mat(cuda, g, f, d, dtype, 0.2), _mat(cuda, g, f, d, dtype, 0.2), _mat(cuda, g, d, f, dtype, 0.2)
    plain = ops.gated_ffn_fwd(x, wg, wu, wd)
    G, U = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    H = G * torch.sigmoid(G) * U
    big = wd.clone()
    big[5, 7], big[6, 7] = math.inf, -math.inf
    y = ops.gated_ffn_fwd(x, wg, wu, big)
    sure = H[:, 7].abs() > 1e-2                                 # rows whose sign no rounding turns
    want = torch.where(H[:, 7] > 0, math.inf, -math.inf)
    assert bool((y[sure, 5].double() == want[sure]).all()) and bool((y[sure, 6].double() == -want[sure]).all())
    rest = [k for k in range(d) if k not in (5, 6)]
    assert torch.equal(y[:, rest], plain[:, rest])
    if n > 1:
        x2 = x.clone()
        x2[1, 3] = math.inf
        y = ops.gated_ffn_fwd(x2, wg, wu, wd)
        keep = torch.arange(n, device=cuda) != 1
        assert torch.equal(y[keep], plain[keep]) and not bool(torch.isfinite(y[1]).any())


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_fp32_products_of_infinities(cuda, value):
    """Logits of one node (lse is the logit itself) from one infinite element against ones, halves, short and long
    significands, zero and infinities."""
    from fast_b200 import ops
    n, d = 12, 40
    h = torch.full((n, d), 0.375, device=cuda)
    h[:, 5] = torch.tensor([1, -1, 0.5, 1 + 2.0 ** -10, 1 / 3, -1 / 3, 1e-20, 3e38, 0, math.inf, -math.inf, math.nan], device=cuda)
    w = torch.full((1, d), 0.25, device=cuda)
    w[0, 5] = value
    want = (h.double() @ w.double().t())[:, 0]
    # one logit: lse = max + log(1), but an infinite maximum has no finite distance to itself
    lse = ops.softmax_xent_fwd(h, w, torch.zeros(n, dtype=torch.int64, device=cuda))[1].double()
    low = want == -math.inf
    assert bool((lse[low] == -math.inf).all()) and not bool(torch.isfinite(lse).any())
    # the same through the gated block's last product: relu(1) * 1 in column 5, weights of the table's row
    x = torch.zeros(n, 16, device=cuda)
    x[:, 0] = 1
    x[:, 1:9] = torch.randn(n, 8, device=cuda)
    wg, wu, wd = torch.zeros(24, 16, device=cuda), torch.zeros(24, 16, device=cuda), torch.ones(16, 24, device=cuda)
    wg[:, 0] = 1
    wu[:, 0] = h[3, 5]
    wd[4, 5] = value
    y = ops.gated_ffn_fwd(x, wg, wu, wd, act="relu")
    ref = (x.double() @ wg.double().t()).relu() * (x.double() @ wu.double().t()) @ wd.double().t()
    assert torch.equal(y[:, 4].double().isnan(), ref[:, 4].isnan())
    if not math.isnan(value):
        assert bool((y[:, 4].double() == ref[:, 4]).all())
    other = [k for k in range(16) if k != 4]
    assert bool(torch.isfinite(y[:, other]).all())


# ---- rows held out of the loss ---------------------------------------------------------------------------------------
# few rows; tiles over aligned rows, read where they lie, and over copied ones; stored logits
@pytest.mark.parametrize("n,d,v,pad", [(2, 64, 17000, 0), (8, 33, 900, 0), (40, 64, 900, 0), (300, 64, 700, 8),
                                       (300, 33, 700, 1), (60, 600, 500, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_held_out_rows_reach_no_gradient(cuda, n, d, v, pad, dtype):
    """Whatever a row without a target holds, the gradients are those of a call in which it holds zeros."""
    from fast_b200 import ops
    g = _gen(cuda, n, d, v)
    h, w = _mat(cuda, g, n, d, dtype, 1.0, pad), _mat(cuda, g, v, d, dtype, d ** -0.5, pad)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    dl = torch.rand(n, device=cuda, generator=g) + 0.5
    out = [1] if n < 5 else [1, 3, n - 1]
    t[out] = -1
    if n >= 5:
        t[3] = v + 5                                            # no target in the table: no gradient either
    clean = h.clone()
    clean[out] = 0
    _, lse = ops.softmax_xent_fwd(clean, w, t)
    want = ops.softmax_xent_bwd(clean, w, t, lse, dl)
    h[1] = math.nan
    if n >= 5:
        h[3, ::2], h[n - 1, -1] = math.inf, -math.inf
    kept = h.clone()
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    assert bool((loss[t < 0] == 0).all()) and bool(loss[(t >= 0) & (t < v)].isfinite().all())
    dl[out] = math.nan                                          # nor does their gradient of the loss
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, dl)
    assert bool(dh.isfinite().all()) and bool(dw.isfinite().all())
    assert torch.equal(dh, want[0]) and torch.equal(dw, want[1])
    buf = torch.zeros(v, d, device=cuda)
    ops.softmax_xent_bwd(h, w, t, lse, dl, dw=buf)
    assert bool(buf.isfinite().all())
    same = torch.equal(h.view(torch.int16 if dtype == BF else torch.int32), kept.view(torch.int16 if dtype == BF else torch.int32))
    assert same                                                 # the caller's rows stay as they are


# ---- the tail of GELU ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 2, 8, 89])
@pytest.mark.parametrize("dtype", TYPES)
def test_gelu_of_negative_values_keeps_its_relative_accuracy(cuda, rows, dtype):
    """h = gelu(g) * 1 and dg = gelu'(g) for g in [-8, -3], where erf is nearly -1: an error that is small beside 1 is
    not small beside the result.  fp32: the normal distribution function to 5 ulp, the exponential to 2, both times a
    few products, whose sum in gelu' cancels by a factor of at most 1.3: below 2^-19.  bf16: 2^-8 for the rounding and
    2^-10 for what the fast exponential and the tail's polynomial leave."""
    from fast_b200 import ops
    g = torch.linspace(-8, -3, 89, device=cuda).bfloat16().to(dtype)[:, None]
    wg, wu, wd = (torch.zeros(16, 16, device=cuda, dtype=dtype) for _ in range(3))
    wg[0, 0], wu[0, 1], wd[0, 0] = 1, 1, 1
    x = torch.zeros(89, 16, device=cuda, dtype=dtype)
    x[:, :1], x[:, 1] = g, 1
    dy = torch.zeros_like(x)
    dy[:, 0] = 1
    y = torch.cat([ops.gated_ffn_fwd(p, wg, wu, wd, act="gelu") for p in x.split(rows)])[:, :1].double()
    dx = torch.cat([ops.gated_ffn_bwd(q, p, wg, wu, wd, act="gelu")[0] for p, q in zip(x.split(rows), dy.split(rows))])
    G = g.double()
    phi = 0.5 * torch.special.erfc(-G * 0.5 ** 0.5)
    tol = 2.0 ** -19 if dtype == F32 else 2.0 ** -8 + 2.0 ** -10
    want = G * phi
    assert float(((y - want) / want).abs().max()) <= tol
    want = phi + G * torch.exp(-G * G / 2) / math.sqrt(2 * math.pi)
    assert float(((dx[:, :1].double() - want) / want).abs().max()) <= tol


# ---- the module's gradients ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 150])
def test_bf16_head_gives_its_fp32_parameters_unrounded_gradients(cuda, n):
    """Weight gradients are fp32 sums; fp32 parameters receive them as they are, not rounded to bf16 on the way."""
    from fast_b200 import ops
    from fast_b200.ranking import GatedFeedForward, NodeRankingHead, SoftmaxXentFunction
    torch.manual_seed(2)
    ffn = GatedFeedForward(64, 136, dtype=BF).to(cuda)
    x, dy = torch.randn(n, 64, device=cuda).bfloat16(), torch.randn(n, 64, device=cuda).bfloat16()
    ffn(x).backward(dy)
    bufs = [torch.zeros(p.shape, device=cuda) for p in (ffn.w_gate, ffn.w_up, ffn.w_down)]
    ops.gated_ffn_bwd(dy, x, *(p.detach().bfloat16() for p in (ffn.w_gate, ffn.w_up, ffn.w_down)), grads=bufs)
    for p, b in zip((ffn.w_gate, ffn.w_up, ffn.w_down), bufs):
        assert p.grad.dtype == F32 and torch.equal(p.grad, b)
    table = torch.randn(300, 64, device=cuda, requires_grad=True)
    t = torch.randint(0, 300, (n,), device=cuda)
    SoftmaxXentFunction.apply(x, table, t).sum().backward()
    buf, w = torch.zeros(300, 64, device=cuda), table.detach().bfloat16()
    _, lse = ops.softmax_xent_fwd(x, w, t)
    ops.softmax_xent_bwd(x, w, t, lse, torch.ones(n, device=cuda), dw=buf)
    assert table.grad.dtype == F32 and torch.equal(table.grad, buf)
    # a module that is bf16 throughout: no fp32 parameters, no conversions of them, gradients of their type
    head = NodeRankingHead(64, 300, hidden=136, dtype=BF).to(cuda).to(BF)
    loss, _ = head(x, t)
    loss.backward()
    assert all(p.grad.dtype == BF and bool(p.grad.isfinite().all()) for p in head.parameters())
    assert torch.isfinite(loss)


# ---- counts ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d,f", [(0, 64, 128), (1, 64, 128), (40, 64, 128), (300, 413, 700), (5000, 64, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_launches_are_counted(cuda, n, d, f, dtype):
    """ops.LAUNCHES rises by the kernel nodes that the same call leaves in a captured graph."""
    from cuda.bindings import runtime
    from fast_b200 import ops
    g = _gen(cuda, n, d, f)
    x, dy, ln = _mat(cuda, g, n, d, dtype), _mat(cuda, g, n, d, dtype), torch.ones(d, device=cuda)
    wg, wu, wd = _mat(cuda, g, f, d, dtype), _mat(cuda, g, f, d, dtype), _mat(cuda, g, d, f, dtype)
    t, one = torch.zeros(n, dtype=torch.int64, device=cuda), torch.ones(n, device=cuda)
    for run in (lambda: ops.layer_norm_fwd(x, ln), lambda: ops.layer_norm_bwd(dy, x, ln, one, one),
                lambda: ops.gated_ffn_fwd(x, wg, wu, wd), lambda: ops.gated_ffn_bwd(dy, x, wg, wu, wd),
                lambda: ops.softmax_xent_fwd(x, wg, t), lambda: ops.softmax_xent_bwd(x, wg, t, one, one)):
        before = ops.LAUNCHES[0]
        run()
        counted = ops.LAUNCHES[0] - before
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            run()
        raw = runtime.cudaGraph_t(init_value=graph.raw_cuda_graph())
        err, _, count = runtime.cudaGraphGetNodes(raw)
        assert err == runtime.cudaError_t.cudaSuccess
        err, nodes, _ = runtime.cudaGraphGetNodes(raw, count)
        kinds = [runtime.cudaGraphNodeGetType(nd)[1] for nd in nodes[:count]]
        assert counted == kinds.count(runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel), (counted, kinds)


# ---- the smallest sizes ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d,f,pad", [(1, 1, 1, 0), (2, 1, 3, 0), (9, 1, 1, 0), (9, 2, 1, 1), (12, 3, 5, 0), (130, 7, 2, 5),
                                       (300, 1, 9, 0), (257, 8, 1, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_widths_below_sixteen(cuda, n, d, f, pad, dtype):
    gated_ffn(cuda, n, d, f, pad, dtype, "silu")
    softmax_xent(cuda, n, d, f, pad, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_in_a_wider_buffer_leave_the_rest_of_it_alone(cuda, dtype):
    """Not-a-numbers around every operand are not read into a result; buffers written with a pitch keep what lies between
    their rows."""
    from fast_b200 import ops
    g = _gen(cuda, 11, 3)

    def framed(rows, cols, off):
        buf = torch.full((rows + 2, cols + 7), math.nan, device=cuda, dtype=dtype)
        view = buf[1:-1, off:off + cols]
        view.copy_(torch.randn(rows, cols, device=cuda, generator=g))
        return view
    for n in (2, 70):
        for d, f, off in ((40, 72, 0), (33, 65, 3), (64, 128, 7)):
            x, dy, wg, wu, wd = (framed(*s, off) for s in ((n, d), (n, d), (f, d), (f, d), (d, f)))
            t = torch.randint(0, f, (n,), device=cuda, generator=g)
            lse = ops.softmax_xent_fwd(x, wg, t)[1]
            one = torch.ones(n, device=cuda)
            outs = [*ops.layer_norm_fwd(x, torch.ones(d, device=cuda)), ops.gated_ffn_fwd(x, wg, wu, wd), lse,
                    *ops.gated_ffn_bwd(dy, x, wg, wu, wd), *ops.softmax_xent_bwd(x, wg, t, lse, one),
                    *ops.layer_norm_bwd(dy, x, torch.ones(d, device=cuda), one, one)]
            assert all(bool(o.isfinite().all()) for o in outs)
            bufs = [torch.full((r, c + 5), 7.0, device=cuda) for r, c in ((f, d), (f, d), (d, f), (f, d))]
            views = [b[:, off % 4:off % 4 + c] for b, c in zip(bufs, (d, d, f, d))]
            ops.gated_ffn_bwd(dy, x, wg, wu, wd, grads=views[:3])
            ops.softmax_xent_bwd(x, wg, t, lse, one, dw=views[3])
            for b, c in zip(bufs, (d, d, f, d)):
                assert bool((b[:, :off % 4] == 7).all()) and bool((b[:, off % 4 + c:] == 7).all())
                assert bool(b.isfinite().all())
