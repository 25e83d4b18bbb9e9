"""GPU: the state space blocks and the encoder -- gradients against fp64
autograd, histories at once and event by event, captured graphs, streams,
training, and what a call leaves alone."""
import history_math as hm
import pytest
import torch

pytestmark = pytest.mark.gpu


def _block(dim=48, dropout=0.0, dtype=torch.float32, states=16, taps=4):
    from fast_b200.history import StateSpaceBlock
    torch.manual_seed(3)
    return StateSpaceBlock(dim, states=states, taps=taps, dropout=dropout, dtype=dtype).cuda()


def _reference(b, x, starts, scale, dtype):
    """The block in plain torch at fp64, products' weights rounded to the compute type; scale: dropout's."""
    p = {n: v.detach().double().requires_grad_(True) for n, v in b.named_parameters()}
    q = {n: p[n] + (p[n].detach().to(dtype).double() - p[n].detach()) if n in ("w_in", "w_x", "w_dt", "w_out") else p[n] for n in p}
    x = x.detach().double().requires_grad_(True)
    F = torch.nn.functional
    y = F.layer_norm(x, x.shape[1:], q["norm.weight"], q["norm.bias"], b.eps)
    v, z = (y @ q["w_in"].t()).split(b.inner, 1)
    u, _ = hm.short_conv(v, q["w_conv"], q["b_conv"], starts, None, "silu")
    d, B, C = (u @ q["w_x"].t()).split([b.rank, b.states, b.states], 1)
    s, _ = hm.selective_scan(u, d @ q["w_dt"].t(), -torch.exp(q["log_decay"]), B.unsqueeze(1), C.unsqueeze(1), q["skip"], z, q["b_dt"],
                             starts, None, True)
    return x + scale * (s @ q["w_out"].t()), x, p


# About a dozen roundings of u = 2^-9 on average (bf16: half a step is 2^-9 .. 2^-8 of a value) lie between x and a gradient,
# each relative to the tensor it rounds and independent of the others, with gains of a few through the norm, the gate and
# softplus: 24 * 2^-8 in the 2-norm.  fp32: products of torch (2^-24 sqrt(K) a term) and the scan's 2^-14 bound its rest.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2.0 ** -12), (torch.bfloat16, 24 * 2.0 ** -8)])
@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_block_gradients(cuda, dtype, tol, dropout):
    b = _block(dropout=dropout, dtype=dtype).train()
    starts = torch.tensor([0, 30, 30, 31, 95], device=cuda)
    x = torch.randn(99, 48, device=cuda).to(dtype)
    x[95:] = 0                                                      # rows of no history
    dy = torch.randn(99, 48, device=cuda).to(dtype)
    dy[95:] = 0
    scale = hm.keep_scale(99, 48, dropout, 5, 7).cuda()
    clean = x.clone()
    want, wx, wp = _reference(b, clean, starts, scale, dtype)
    want.backward(dy.double())
    clean.requires_grad_(True)
    y, conv, scan = b(clean, starts, seed=5, offset=7)
    y.backward(dy)
    assert conv.shape == (4, 3, 96) and scan.shape == (4, 96, 16)
    assert float((y[:95].double() - want[:95]).norm() / want[:95].norm()) <= tol
    got = dict(x=clean.grad, **{n: p.grad for n, p in b.named_parameters()})
    ref = dict(x=wx.grad, **{n: p.grad for n, p in wp.items()})
    for n, g in got.items():
        assert g.dtype == (dtype if n == "x" else torch.float32), n
        off = float((g.double() - ref[n]).norm() / ref[n].norm())
        assert off <= tol, (n, off)


def test_functions_pass_gradients_to_states(cuda):
    """A history cut in two calls, the first's states given to the second: the gradients of the whole."""
    from fast_b200.history import SelectiveScanFunction, ShortConvFunction
    g = torch.Generator().manual_seed(2)
    make = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    n, cut, d, N = 60, 23, 20, 16
    src = [make(n, d) for _ in range(3)] + [make(n, N) for _ in range(2)]
    w, A, D, bias = make(d, 4), -torch.rand(d, N, generator=g).cuda() * 4 - 0.5, make(d), make(d) * 0.3

    def run(parts):
        leaves = [t.clone().requires_grad_(True) for t in src + [w, A, D, bias]]
        x, delta, z, B, C, w_, A_, D_, b_ = leaves
        conv = scan = None
        out = []
        for s in parts:
            u, conv = ShortConvFunction.apply(x[s], w_, None, None, conv, "silu")
            y, scan = SelectiveScanFunction.apply(u, delta[s], A_, B[s], C[s], D_, z[s], b_, None, scan, True)
            out.append(y)
        y = torch.cat(out)
        return y, torch.autograd.grad((y * y.detach().cos()).sum(), leaves)
    whole, grads = run([slice(0, n)])
    split, parts = run([slice(0, cut), slice(cut, n)])
    for a, b in zip((whole, *grads), (split, *parts)):
        # the same sums in another order: a few 2^-24 of the terms, 2^-14 as for the operators
        assert float((a - b).norm()) <= 2.0 ** -14 * float(a.norm())


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2.0 ** -12), (torch.bfloat16, 48 * 2.0 ** -8)])
def test_histories_at_once_and_event_by_event(cuda, dtype, tol):
    """forward, follow in two parts, and step agree (bf16: two blocks' roundings fall differently)."""
    from fast_b200.history import HistoryEncoder, NodeStates
    torch.manual_seed(0)
    enc = HistoryEncoder(32, 2, dropout=0.3, dtype=dtype).cuda().eval()
    lengths, nodes = [12, 0, 5, 31], torch.tensor([6, 2, 0, 3], device=cuda)
    starts = torch.tensor([0, 12, 12, 17, 48], device=cuda)
    x = torch.randn(48, 32, device=cuda)
    with torch.no_grad():
        want = enc(x, starts)
    tables = NodeStates(enc, 8, cuda)
    first = [n // 2 for n in lengths]
    at = [torch.arange(int(s), int(s) + f) for s, f in zip(starts, first)]
    got = torch.zeros_like(want)
    rows = torch.cat(at).to(cuda)
    got[rows] = enc.follow(x[rows], torch.tensor([0, 6, 6, 8, 23], device=cuda), tables, nodes)
    # the rest as a chronological stream: several events of a node in one call
    rest = [(int(s) + j, int(v)) for s, f, n, v in zip(starts, first, lengths, nodes) for j in range(f, n)]
    for i in range(0, len(rest), 10):
        r = torch.tensor([e[0] for e in rest[i:i + 10]], device=cuda)
        got[r] = enc.step(x[r], tables, torch.tensor([e[1] for e in rest[i:i + 10]], device=cuda))
    assert float((got.double() - want.double()).norm()) <= tol * float(want.double().norm())
    before = [t.clone() for t in tables.conv + tables.scan]
    out = enc.step(x[:3], tables, torch.tensor([-1, -1, -1], device=cuda))
    assert all(torch.equal(a, b) for a, b in zip(before, tables.conv + tables.scan))
    assert bool(torch.isfinite(out).all())
    assert not any(bool(t[[1, 4, 5, 7]].any()) for t in tables.conv + tables.scan)       # nodes without events
    tables.reset()
    assert not any(bool(t.any()) for t in tables.conv + tables.scan)
    assert torch.equal(enc.last(want, starts)[1], torch.zeros(32, device=cuda, dtype=dtype))
    assert torch.equal(enc.last(want, starts)[3], want[47])
    assert enc.last(want[:0], torch.zeros(3, dtype=torch.int64, device=cuda)).shape == (2, 32)


def test_calls_in_captured_graphs(cuda):
    """Forward, backward and steps replay on new inputs; two graphs do not share what one of them needs."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(4)
    rows, d, n = 3000, 40, 16
    starts = torch.tensor([0, 700, 700, 2990], device=cuda)
    ins = [torch.randn(rows, c, generator=g).cuda() for c in (d, d, d, n, n, d)]
    u, delta, z, B, C, dy = ins
    A, w = -torch.rand(d, n, generator=g).cuda() - 0.1, torch.randn(d, 4, generator=g).cuda()
    table, index = torch.zeros(500, d, n, device=cuda), torch.randint(0, 500, (rows,), generator=g).cuda()
    count = torch.zeros(1, dtype=torch.int64, device=cuda)

    def scan():
        v = ops.short_conv_fwd(u, w, starts=starts)
        dx, dw, _, _ = ops.short_conv_bwd(dy, u, w, starts=starts)
        y, carry, final = ops.selective_scan_fwd(v, delta, A, B, C, z=z, starts=starts, final=True)
        return [v, dx, dw, y, final] + [t for t in ops.selective_scan_bwd(dy, v, delta, A, B, C, carry, z=z, starts=starts) if t is not None]

    def step():
        y = ops.selective_scan_step(u, delta, A, B, C, table, z=z, index=index)
        return [y, ops.dropout_fwd(y, 0.5, 9, 100, offset_dev=count)]
    scan(), step()
    table.zero_()
    graphs = []
    for f in (scan, step):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    for k in range(2):
        for t in ins:
            t.copy_(torch.randn(t.shape, generator=g).cuda())
        count.fill_(k)
        table.normal_()
        kept = table.clone()
        for graph, _ in graphs:
            graph.replay()
        got = [[t.clone() for t in out] for _, out in graphs]
        after = table.clone()
        table.copy_(kept)
        for a, b in zip(got[0], scan()):
            assert torch.equal(a, b)
        for a, b in zip(got[1], step()):
            assert torch.equal(a, b)
        assert torch.equal(table, after)
    del graphs


def test_another_stream(cuda):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(6)
    x, w = torch.randn(2000, 64, generator=g), torch.randn(64, 4, generator=g).cuda()
    A, side = -torch.rand(64, 16, generator=g).cuda(), torch.cuda.Stream()
    want = None
    for stream in (torch.cuda.current_stream(), side):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            v = x.cuda(non_blocking=True)
            for _ in range(3):                                       # pending work in front of the calls
                v = v + 1 - 1
            u = ops.short_conv_fwd(v, w)
            y, carry, _ = ops.selective_scan_fwd(u, v, A, v[:, :16], v[:, 16:32])
            out = [u, y, *ops.selective_scan_bwd(v, u, v, A, v[:, :16], v[:, 16:32], carry)[:5], ops.dropout_fwd(y, 0.1, 3)]
        stream.synchronize()
        if want is None:
            want = out
        else:
            assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_gradients_cannot_be_differentiated(cuda):
    from fast_b200.history import DropoutFunction, SelectiveScanFunction, ShortConvFunction
    x = torch.randn(20, 8, device=cuda, requires_grad=True)
    A, B = -torch.rand(8, 16, device=cuda), torch.randn(20, 16, device=cuda)
    for y in (ShortConvFunction.apply(x, torch.randn(8, 4, device=cuda), None, None, None, "silu")[0],
              SelectiveScanFunction.apply(x, x, A, B, B, None, None, None, None, None, True)[0], DropoutFunction.apply(x, None, 0.5, 1, 0)):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_layouts_of_the_modules(cuda):
    """Transposed and overlapping rows are laid out by the functions; without a graph nothing is kept."""
    from fast_b200.history import SelectiveScanFunction, ShortConvFunction
    x, w = torch.randn(16, 30, device=cuda), torch.randn(4, 16, device=cuda)
    a = ShortConvFunction.apply(x.t(), w.t(), None, None, None, None)[0]
    b = ShortConvFunction.apply(x.t().contiguous(), w.t().contiguous(), None, None, None, None)[0]
    assert torch.equal(a, b)
    one, A, B = torch.randn(1, 16, device=cuda).expand(30, 16), -torch.rand(16, 16, device=cuda).t(), torch.randn(16, 30, device=cuda).t()
    a = SelectiveScanFunction.apply(b, one, A, B, B, None, one, None, None, None, True)[0]
    b = SelectiveScanFunction.apply(b, one.contiguous(), A.contiguous(), B.contiguous(), B.contiguous(), None, one.contiguous(), None, None,
                                    None, True)[0]
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_runs(cuda, dtype):
    from fast_b200.ranking import train_histories
    losses = train_histories(steps=4, nodes=120, edges=4000, batch=80, dim=32, dtype=dtype)
    assert len(losses) == 4 and all(torch.isfinite(torch.tensor(losses)))
