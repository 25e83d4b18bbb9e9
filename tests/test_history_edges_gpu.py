"""GPU: event histories at the edges of what the calls document -- dropout and
training mode, what is kept, gates and decays of extreme values, tables of no
node, and the kernels that only large calls reach."""
import history_math as hm
import numpy as np
import pytest
import torch
from test_history_gpu import BF, F32, close, poison, rows_of, scan_case, starts_of

pytestmark = pytest.mark.gpu


def _encoder(dim=32, blocks=2, dropout=0.5, dtype=F32):
    from fast_b200.history import HistoryEncoder
    torch.manual_seed(0)
    return HistoryEncoder(dim, blocks, dropout=dropout, dtype=dtype).cuda()


def _histories(dim=32, seed=1):
    x = torch.randn(48, dim, generator=torch.Generator().manual_seed(seed)).cuda()
    return x, torch.tensor([0, 12, 12, 17, 48], device="cuda"), torch.tensor([6, 2, 0, 3], device="cuda")


# ---- modules -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
def test_following_the_stream_drops_nothing_out(cuda, dtype):
    """follow writes tables that step goes on from: in training mode, too, it computes what it computes in eval mode."""
    from fast_b200.history import NodeStates
    enc = _encoder(dtype=dtype)
    x, starts, nodes = _histories()
    tables = [NodeStates(enc, 8, cuda) for _ in range(2)]
    want = enc.eval().follow(x, starts, tables[0], nodes)
    got = enc.train().follow(x, starts, tables[1], nodes)
    assert torch.equal(got, want)
    for a, b in zip(tables[0].conv + tables[0].scan, tables[1].conv + tables[1].scan):
        assert torch.equal(a, b)
    assert torch.equal(enc.step(x[:4], tables[0], nodes), enc.step(x[:4], tables[1], nodes))


def _recorded(monkeypatch, name, argument):
    """Values of an argument of ops.`name` from here on."""
    import inspect
    from fast_b200 import ops
    call, seen = getattr(ops, name), []
    signature = inspect.signature(call)

    def run(*args, **kw):
        bound = signature.bind(*args, **kw)
        bound.apply_defaults()
        seen.append(bound.arguments[argument])
        return call(*args, **kw)
    monkeypatch.setattr(ops, name, run)
    return seen


def test_states_are_kept_for_a_backward_pass_only(cuda, monkeypatch):
    """Parameters require gradients under no_grad, too; the states in front of every 8th row are written only where
    there is a graph."""
    from fast_b200.history import NodeStates
    enc, (x, starts, nodes) = _encoder(), _histories()
    kept = _recorded(monkeypatch, "selective_scan_fwd", "keep")
    with torch.no_grad():
        enc(x, starts)
    enc.follow(x, starts, NodeStates(enc, 8, cuda), nodes)
    with torch.inference_mode():
        enc(x, starts)
    assert kept == [False] * 6
    del kept[:]
    enc(x, starts)
    assert kept == [True] * 2


def test_states_behind_histories_are_computed_where_they_are_asked_for(cuda, monkeypatch):
    from fast_b200.history import NodeStates
    enc, (x, starts, nodes) = _encoder(), _histories()
    asked = [_recorded(monkeypatch, n, "final") for n in ("short_conv_fwd", "selective_scan_fwd")]
    enc(x, starts)
    assert asked == [[False] * 2] * 2
    enc.follow(x, starts, NodeStates(enc, 8, cuda), nodes)
    assert asked == [[False] * 2 + [True] * 2] * 2
    y, conv, scan = enc.blocks[0](x, starts, states=False)
    assert conv is None and scan is None
    again, conv, scan = enc.blocks[0](x, starts)
    assert torch.equal(y, again) and conv.shape == (4, 3, 64) and scan.shape == (4, 64, 16)
    # the gradients are those of a call that asks for the states
    a = torch.autograd.grad(y.square().sum(), list(enc.blocks[0].parameters()))
    b = torch.autograd.grad(again.square().sum(), list(enc.blocks[0].parameters()))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_training_draws_anew(cuda):
    """A device counter added to the dropout's offset: a graph of a training step replays with the masks of its value, forward
    and backward."""
    enc = _encoder(dropout=0.4).train()
    x, starts, _ = _histories()
    params = list(enc.parameters())
    count = torch.zeros(1, dtype=torch.int64, device=cuda)

    def step(offset, counter):
        y = enc(x, starts, seed=5, offset=offset, offset_dev=counter)
        return [y, *torch.autograd.grad(y.square().sum(), params)]
    want = [[t.detach().clone() for t in step(k, None)] for k in range(3)]
    assert not torch.equal(want[0][0], want[1][0])
    count.fill_(2)
    assert all(torch.equal(a, b) for a, b in zip(step(0, count), want[2]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0, count)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(0, count)
    for k in (1, 0, 2):
        count.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


def test_a_counter_that_moves_before_the_backward_is_refused(cuda):
    """The backward draws the forward's words again: a counter advanced in between would give it others."""
    from fast_b200.history import DropoutFunction
    x, count = torch.ones(9, 8, device=cuda, requires_grad=True), torch.zeros(1, dtype=torch.int64, device=cuda)
    y = DropoutFunction.apply(x, None, 0.5, 1, 0, count)
    count += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_a_counter_may_move_where_nothing_drops_out(cuda):
    from fast_b200.history import DropoutFunction
    x, count = torch.ones(9, 8, device=cuda, requires_grad=True), torch.zeros(1, dtype=torch.int64, device=cuda)
    y = DropoutFunction.apply(x, None, 0.0, 1, 0, count)
    count += 1
    grad, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(grad, torch.ones_like(grad))


def test_no_dropout_hands_the_gradient_on(cuda):
    from fast_b200 import ops
    from fast_b200.history import DropoutFunction
    x, res = (torch.randn(9, 8, device=cuda, requires_grad=True) for _ in range(2))
    y = DropoutFunction.apply(x, res, 0.0, 1, 0)
    dy = torch.randn(9, 8, device=cuda)
    before = ops.LAUNCHES[0]
    gx, gr = torch.autograd.grad(y, (x, res), dy)
    assert ops.LAUNCHES[0] == before
    assert torch.equal(gx, dy) and torch.equal(gr, dy)


def test_seeds_up_to_64_bits(cuda):
    """Block i draws from seed + i, counted in 64 bits."""
    enc = _encoder().train()
    x, starts, _ = _histories()
    with torch.no_grad():
        y = enc.blocks[0](x, starts, seed=(1 << 64) - 1, offset=3)[0]
        want = enc.blocks[1](y, starts, seed=0, offset=3)[0]
        assert torch.equal(enc(x, starts, seed=(1 << 64) - 1, offset=3), want)


def test_seeds_beyond_64_bits_are_refused(cuda):
    """The encoder's count past 2^64 does not make a bad seed a good one."""
    enc = _encoder().train()
    x, starts, _ = _histories()
    for seed in (-1, 1 << 64, 1.0, True):
        with pytest.raises(ValueError, match="seed"):
            enc(x, starts, seed=seed)


# ---- gates -------------------------------------------------------------------------------------------
def _gate_calls(z, dtype=F32):
    """silu(z) and silu'(z) as every kernel that gates computes them: (name, values, slopes or None) with the factor 1."""
    from fast_b200 import ops
    n = z.numel()
    rows, one = z.to(dtype).reshape(-1, 8), torch.ones(n // 8, 8, device="cuda", dtype=dtype)
    w, r = torch.ones(8, 1, device="cuda"), n // 8
    yield "convolution", ops.short_conv_fwd(rows, w), ops.short_conv_bwd(one, rows, w)[0]
    # the gradient of the inputs in front of a sequence: w = (1, 0), one row a sequence
    two = torch.tensor([[1.0, 0.0]], device="cuda").repeat(8, 1)
    starts = torch.arange(r + 1, device="cuda")
    yield ("convolution, states in", ops.short_conv_fwd(one, two, starts=starts, init=rows.unsqueeze(1)),
           ops.short_conv_bwd(one, one, two, starts=starts, init=rows.unsqueeze(1))[3].squeeze(1))
    yield "convolution, event", ops.short_conv_step(rows, torch.zeros(r, 0, 8, device="cuda", dtype=dtype), w), None
    A, B, D = -torch.ones(8, 4, device="cuda"), torch.zeros(r, 4, device="cuda", dtype=dtype), torch.ones(8, device="cuda")
    y, carry, _ = ops.selective_scan_fwd(one, one, A, B, B, D, rows)
    yield "scan", y, ops.selective_scan_bwd(one, one, one, A, B, B, carry, D, rows)[6]
    yield "scan, event", ops.selective_scan_step(one, one, A, B, B, torch.zeros(r, 8, 4, device="cuda"), D, rows), None


def test_gates_of_large_positive_values(cuda):
    """silu'(z) is 1 + z (1 - sigmoid(z)) times sigmoid(z), which tends to 1.  The sigmoid is off by 2^-23 (its reciprocal)
    + 2^-24; 1 - sigmoid is that much off where it does not vanish (z <= 17): 17 * 1.5 * 2^-23 < 2^-18 of the result."""
    z = torch.cat([torch.linspace(1, 40, 400), torch.logspace(1.6, 30, 400)]).cuda()
    w = z.double().requires_grad_(True)
    y = torch.nn.functional.silu(w)
    slope, = torch.autograd.grad(y.sum(), w)
    w, y = w.detach(), y.detach()
    for name, got, dgot in _gate_calls(z):
        assert float(((got.reshape(-1).double() - y) / y).abs().amax()) <= 2.0 ** -18, name
        if dgot is not None:
            assert float(((dgot.reshape(-1).double() - slope) / slope).abs().amax()) <= 2.0 ** -18, name


def test_gates_of_bf16_rows(cuda):
    """One rounding to bf16 (8 bits of significand: half a step is up to 2^-8 of the value); in front of it at most |z| 2^-23
    (|z| <= 64 where it counts) = 2^-17."""
    z = torch.cat([torch.linspace(-60, 60, 800), torch.logspace(1.7, 38, 400)]).cuda().to(BF)
    w = z.double().requires_grad_(True)
    y = torch.nn.functional.silu(w)
    slope, = torch.autograd.grad(y.sum(), w)
    w, y = w.detach(), y.detach()
    near = (z < -2.5) | (z > 0)                                     # away from the slope's zero at -1.28
    for name, got, dgot in _gate_calls(z, BF):
        assert bool(((got.reshape(-1).double() - y).abs() <= (2.0 ** -8 + 2.0 ** -16) * y.abs()).all()), name
        if dgot is not None:
            off = (dgot.reshape(-1).double() - slope).abs()
            assert bool((off <= (2.0 ** -8 + 2.0 ** -16) * slope.abs())[near].all()), name


def test_gates_keep_their_relative_accuracy(cuda):
    """fp32.  e^-z: 2^-22 of the exponential unit and 2^-23 of its correction; 1 + e^-z, the reciprocal (2^-23) and the product
    with z: 2^-22 more.  The slope, away from its zero at -1.28, has the sigmoid's error and 1 + z (1 - sigmoid)'s: twice that."""
    z = torch.cat([torch.linspace(-86, -20, 400), torch.linspace(-20, 20, 800)]).cuda()
    w = z.double().requires_grad_(True)
    y = torch.nn.functional.silu(w)
    slope, = torch.autograd.grad(y.sum(), w)
    w, y = w.detach(), y.detach()
    far = (z < -2.5) | (z > 0)                                      # 1 + z (1 - sigmoid) does not cancel there
    for name, got, dgot in _gate_calls(z):
        assert float(((got.reshape(-1).double() - y) / y).abs().amax()) <= 2.5 * 2.0 ** -22, name
        if dgot is not None:
            assert float(((dgot.reshape(-1).double() - slope) / slope).abs()[far].amax()) <= 5 * 2.0 ** -22, name


@pytest.mark.parametrize("dtype", [F32, BF])
def test_gates_of_the_largest_values(cuda, dtype):
    """Neither end of the type overflows on the way: silu tends to 0 and z, its slope to 0 and 1; NaN stays."""
    top = torch.finfo(dtype).max
    z = torch.tensor([-top, -1e30, -200.0, -90.0, 0.0, 90.0, 1e30, top], device=cuda)
    for name, got, dgot in _gate_calls(z, dtype):
        want = torch.nn.functional.silu(z.to(dtype).double())
        assert float((got.reshape(-1).double() - want).abs()[:5].amax()) <= 1e-30, name
        assert torch.equal(got.reshape(-1)[5:], z.to(dtype)[5:]), name
        if dgot is not None:
            assert float(dgot.reshape(-1)[:4].abs().amax()) <= 1e-30, name
            assert torch.equal(dgot.reshape(-1)[4:].float(), torch.tensor([0.5, 1, 1, 1], device=cuda)), name
    for name, got, dgot in _gate_calls(torch.full((8,), float("nan"), device=cuda), dtype):
        assert bool(torch.isnan(got).all()) and (dgot is None or bool(torch.isnan(dgot).all())), name
    for name, got, _ in _gate_calls(torch.full((8,), float("inf"), device=cuda), dtype):
        assert bool((got == float("inf")).all()), name


# ---- decays ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("n", [5, 16, 64])
def test_events_decay_as_histories_do(cuda, softplus, n):
    """Rows of one chunk, at once and event by event: the same operations in the same order, so the same states."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(n)
    rows, d = 13, 40
    u, B, C = rows_of(g, rows, d, F32), rows_of(g, rows, n, F32), rows_of(g, rows, n, F32)
    delta = (torch.rand(rows, d, generator=g) * 0.01).cuda() - (4.0 if softplus else 0.0)
    A = -(torch.rand(d, n, generator=g) * 4 + 0.5).cuda()
    final = ops.selective_scan_fwd(u, delta, A, B, C, softplus=softplus, final=True)[2][0]
    state = torch.zeros(3, d, n, device="cuda")
    for r in range(rows):
        ops.selective_scan_step(u[r:r + 1], delta[r:r + 1], A, B[r:r + 1], C[r:r + 1], state, softplus=softplus,
                                index=torch.tensor([1], device="cuda"))
    assert torch.equal(state[1], final) and not bool(state[[0, 2]].any())


def test_events_with_decays_of_minus_infinity(cuda):
    """A state with A = -infinity keeps nothing of the event before, and a step of 0 leaves every state as it is, as in the scan."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(2)
    d, n = 24, 16
    u, B, C = rows_of(g, 6, d, F32), rows_of(g, 6, n, F32), rows_of(g, 6, n, F32)
    delta = rows_of(g, 6, d, F32, 0.5)
    delta[3] = -200.0                                               # softplus gives 0
    A = -(torch.rand(d, n, generator=g) + 0.5).cuda()
    A[:, 3] = float("-inf")
    y, _, final = ops.selective_scan_fwd(u, delta, A, B, C, final=True)
    state = torch.zeros(1, d, n, device="cuda")
    for r in range(6):
        close(ops.selective_scan_step(u[r:r + 1], delta[r:r + 1], A, B[r:r + 1], C[r:r + 1], state), y[r:r + 1], "row %d" % r)
    assert torch.equal(state, final)


def test_slow_decays_over_a_long_stream(cuda):
    """4,000 events of one node.  As for a history (a decay's mean error at most 1.3e-8 of itself, a thousand steps remembered):
    2^-16 of the state."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(8)
    rows, d, n = 4000, 32, 16
    u, B, C = rows_of(g, rows, d, F32).abs(), rows_of(g, rows, n, F32).abs(), rows_of(g, rows, n, F32)
    delta = (torch.rand(rows, d, generator=g) * 0.001 + 0.0005).cuda()
    A = -torch.arange(1, n + 1, dtype=torch.float32, device="cuda").repeat(d, 1)
    state = torch.zeros(2, d, n, device="cuda")
    y = ops.selective_scan_step(u, delta, A, B, C, state, index=torch.ones(rows, dtype=torch.int64, device="cuda"), softplus=False)
    wide = [t.double() for t in (u, delta, A, B.unsqueeze(1), C.unsqueeze(1))]
    wy, wf = hm.selective_scan(*wide, None, None, None, None, None, False)
    for got, ref in ((y, wy), (state[1], wf[0])):
        assert float((got.double() - ref).norm() / ref.norm()) <= 2.0 ** -16


def test_growth_over_chunks(cuda):
    """States that grow (A > 0): a chunk's factor beyond fp32 carries a 0 as 0 and a small state as the product it is, in both
    directions."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(4)
    rows, d, n = 64, 8, 8
    u, B, C, dy = (rows_of(g, rows, c, F32) for c in (d, n, n, d))
    u[:40], dy[24:] = 0, 0                                          # nothing until row 40; nothing wanted from row 24 on
    delta = torch.ones(rows, d, device="cuda")
    for rate in (1.0, 4.0, 7.0, 20.0):
        A = torch.full((d, n), rate, device="cuda") * torch.linspace(0.25, 1, n, device="cuda")
        v = u.clone()
        v[40:] = 0
        v[60:] = u[60:]
        y, carry, final = ops.selective_scan_fwd(v, delta, A, B, C, softplus=False, final=True)
        wide = [t.double().requires_grad_(True) for t in (v, delta, A, B, C)]
        wy, wf = hm.selective_scan(*wide[:3], wide[3].unsqueeze(1), wide[4].unsqueeze(1), None, None, None, None, None, False)
        assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(final).all()), rate
        assert float((final.double() - wf).norm() / wf.norm()) <= 2.0 ** -14, rate
        e = dy.clone()
        e[4:] = 0
        du = ops.selective_scan_bwd(e, v, delta, A, B, C, carry, softplus=False)[0]
        want, = torch.autograd.grad(wy, wide[0], e.double())
        assert bool(torch.isfinite(du).all()), rate
        assert float((du.double() - want).norm() / want.norm()) <= 2.0 ** -14, rate
    # a state of 2^-100 that a chunk of 16 rows lifts by e^112 = 2^161.6
    u = torch.zeros(rows, d, device="cuda")
    u[15], A = 2.0 ** -100, torch.full((d, n), 7.0, device="cuda")
    delta[32:] = 0
    B = torch.ones(rows, n, device="cuda")
    final = ops.selective_scan_fwd(u, delta, A, B, B, softplus=False, final=True)[2]
    want = 2.0 ** -100 * float(np.exp(112.0))
    # 161.6 = 16 * 7 * log2 e, off by 2^-17.3 where the steps' exponents or the chunk's are rounded, each way twice at most
    assert float((final.double() / want - 1).abs().amax()) <= 2.0 ** -15


# ---- tables ------------------------------------------------------------------------------------------
def test_tables_of_no_node(cuda):
    """Every index is beyond the table, or held out."""
    from fast_b200 import ops
    x, index = torch.randn(3, 8, device=cuda), torch.tensor([0, -1, 5], device=cuda)
    w, A, B = torch.randn(8, 4, device=cuda), -torch.rand(8, 16, device=cuda), torch.randn(3, 16, device=cuda)
    for y in (ops.short_conv_step(x, torch.zeros(0, 3, 8, device=cuda), w, index=index),
              ops.selective_scan_step(x, x, A, B, B, torch.zeros(0, 8, 16, device=cuda), index=index)):
        assert bool(torch.isnan(y[[0, 2]]).all()) and not bool(y[1].any())


# ---- kernels of large calls --------------------------------------------------------------------------
def conv_at_once(x, w, bias, starts, init, act):
    """(y, final) of hm.short_conv for many rows, by gathering."""
    rows, (d, k) = x.shape[0], w.shape
    seqs, t = starts.shape[0] - 1, torch.arange(rows, device=x.device)
    s = torch.searchsorted(starts, t, right=True) - 1
    some = (s >= 0) & (s < seqs)
    s = s.clamp(0, seqs - 1)
    pos = t - starts[s]

    def before(at, seq):                                            # input number `at` of a sequence, from -(k - 1) on
        v = x[(starts[seq] + at).clamp(0, rows - 1)]
        past = x.new_zeros(1, d) if init is None or k == 1 else init[seq, (at + k - 1).clamp(0, k - 2)]
        return torch.where((at >= 0).unsqueeze(1), v, past)
    p = sum(w[:, i] * before(pos - (k - 1 - i), s) for i in range(k))
    p = p if bias is None else p + bias
    y = torch.where(some.unsqueeze(1), p * torch.sigmoid(p) if act == "silu" else p, x.new_zeros(1))
    every = torch.arange(seqs, device=x.device)
    n = starts[1:] - starts[:-1]
    final = [before(n - (k - 1) + m, every) for m in range(k - 1)]
    return y, torch.stack(final, 1) if final else x.new_zeros(seqs, 0, d)


def test_convolution_at_once_is_the_restatement(cuda):
    g = torch.Generator().manual_seed(0)
    starts = starts_of([5, 0, 1, 9, 0, 2], 3)
    for k in (1, 2, 4, 7):
        x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64).cuda() for s in ((25, 6), (6, k), (6,)))
        i = torch.randn(6, k - 1, 6, generator=g, dtype=torch.float64).cuda()
        for a, c in zip(conv_at_once(x, w, b, starts, i, "silu"), hm.short_conv(x, w, b, starts, i, "silu")):
            assert torch.allclose(a, c, rtol=1e-13, atol=1e-13)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("whole", [True, False])
def test_conv_of_four_columns_a_thread(cuda, k, dtype, whole):
    """From 9,472 rows of width 512 on a thread has four columns (rows / 32 * (width / 128) >= 148 * 8)."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(k)
    lengths, d = [4000, 0, 1, 2, 3, 0, 2500, 64, 17] + [5] * 300 + [0, 1400, 7], 512
    starts = starts_of(lengths, 3)
    n = int(starts[-1]) + 70
    x, dy = rows_of(g, n, d, dtype, 1, 8), rows_of(g, n, d, dtype, 1, 4)
    w = (torch.randn(d, k, generator=g) * k ** -0.5).cuda()
    b, act = (torch.randn(d, generator=g).cuda() * 0.2, "silu") if whole else (None, None)
    i, df = ((torch.randn(len(lengths), k - 1, d, generator=g).to(dtype).cuda() if whole else None) for _ in range(2))
    poison(n, starts, x, dy)
    wide = [None if t is None else t.double().nan_to_num(0, 0, 0).requires_grad_(True) for t in (x, w, b, i)]
    y, final = conv_at_once(*wide[:3], starts, wide[3], act)
    got_y, got_final = ops.short_conv_fwd(x, w, b, starts, i, act, final=True)
    close(got_y, y, "y")
    assert torch.equal(got_final.double(), final.double())
    names = [m for m, t in zip(("dx", "dw", "dbias", "dinit"), wide) if t is not None]
    have = [t for t in wide if t is not None]
    outs, grads = [y], [dy.double().nan_to_num(0, 0, 0)]
    if whole:
        outs, grads = outs + [final + 0 * wide[0].sum()], grads + [df.double()]
    want = dict(zip(names, torch.autograd.grad(outs, have, grads, allow_unused=True)))
    got = dict(zip(("dx", "dw", "dbias", "dinit"), ops.short_conv_bwd(dy, x, w, b, starts, i, act, dfinal=df)))
    for m, v in got.items():
        if m in want:
            close(v, torch.zeros_like(v) if want[m] is None else want[m], m)
        else:
            assert v is None


# With so wide rows a chunk has as many rows as make two waves of warps forward (three of CTAs backward), if those are 48
# (64) or more, else those that make one less.
LONG = [400, 0, 1, 7, 64, 0, 0, 300, 3, 500]


@pytest.mark.parametrize("n,d,dtype,lengths", [
    (5, 8192, BF, LONG), (16, 4096, F32, LONG), (16, 4096, BF, LONG), (13, 4096, BF, LONG), (32, 2048, BF, LONG),   # 56 and 72 rows
    (16, 2048, F32, [700, 0, 1, 1100, 9, 111]),                                                                     # 80 and 80
    (64, 2048, F32, [310, 2, 0, 300, 9])])                                                                          # 56 and 80
def test_scan_of_long_chunks(cuda, n, d, dtype, lengths):
    """Chunks of many tiles of eight rows, sequences that begin inside them, several waves of chunks."""
    scan_case(lengths, d, n, dtype, init=True, front=30, tail=45)


def test_scan_of_long_chunks_in_groups(cuda):
    scan_case(LONG, 4096, 16, BF, groups=4, gate=False, skip=False, pad=3, front=5, tail=70)


def _event_case(g, n, nodes):
    """Indices of n events: nodes that come once or several times, anywhere; the last rows hold one that is held out and one
    beyond the table."""
    index = torch.randint(0, nodes, (n,), generator=g)
    index[-2], index[-5 if n > 5 else 0] = -1, nodes
    index[-1] = index[0]
    return index


@pytest.mark.parametrize("n", [64, 65, 4095, 4096, 4097, 8193, 9000])
@pytest.mark.parametrize("often", [1, 3, 700])
def test_events_that_meet_their_nodes_again(cuda, n, often):
    """Up to 64 rows the warps compare indices themselves; beyond, a kernel does, 4,096 rows at a time."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(n + often)
    nodes, d, k, s = max(2, n // often), 4, 3, 4
    index = _event_case(g, n, nodes)
    x, delta = torch.randn(n, d, generator=g), torch.randn(n, d, generator=g) * 0.5
    B, C = torch.randn(n, 1, s, generator=g), torch.randn(n, 1, s, generator=g)
    w, A = torch.randn(d, k, generator=g), -(0.5 + torch.rand(d, s, generator=g) * s)
    conv, scan = torch.randn(nodes, k - 1, d, generator=g), torch.randn(nodes, d, s, generator=g)
    at = index.cuda()
    c, h = conv.cuda(), scan.cuda()
    yc = ops.short_conv_step(x.cuda(), c, w.cuda(), None, at)
    ys = ops.selective_scan_step(x.cuda(), delta.cuda(), A.cuda(), B.cuda(), C.cuda(), h, index=at)
    dt = np.logaddexp(delta.double().numpy(), 0.0)
    x, B, C, w, A, conv, scan = (t.double().numpy() for t in (x, B, C, w, A, conv, scan))
    wc, wsc = np.zeros((n, d)), np.zeros((n, d))
    for r, i in enumerate(index.tolist()):
        if 0 <= i < nodes:
            win = np.concatenate([conv[i], x[r:r + 1]])
            p = (win * w.T).sum(0)
            wc[r], conv[i] = p / (1 + np.exp(-p)), win[1:]
            scan[i] = np.exp(dt[r][:, None] * A) * scan[i] + (dt[r] * x[r])[:, None] * B[r]
            wsc[r] = (C[r] * scan[i]).sum(1)
    beyond, held = index >= nodes, index < 0
    for got, want in ((yc, wc), (ys, wsc)):
        assert bool(torch.isnan(got[beyond.cuda()]).all()) and not bool(got[held.cuda()].any())
        got[beyond.cuda()] = 0
        close(got, torch.from_numpy(want).cuda(), "y")
    assert torch.equal(c.double().cpu(), torch.from_numpy(conv))
    close(h, torch.from_numpy(scan).cuda(), "state")


def philox_at_once(rows, cols, seed, offset):
    """hm.philox for many rows."""
    m = np.uint64(0xFFFFFFFF)
    c = [np.broadcast_to(np.arange((cols + 3) // 4, dtype=np.uint64), (rows, (cols + 3) // 4)),
         np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], (rows, (cols + 3) // 4)),
         np.uint64(offset & 0xFFFFFFFF), np.uint64(offset >> 32)]
    for r in range(10):
        k = [np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ k[0], p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ k[1], p0 & m]
        c = [np.broadcast_to(v, (rows, (cols + 3) // 4)) for v in c]
    return torch.from_numpy(np.stack(c, 2).reshape(rows, -1)[:, :cols].astype(np.int64))


@pytest.mark.parametrize("d,pad", [(1028, 0), (1026, 0), (2056, 8), (2056, 1)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_dropout_down_the_rows(cuda, d, pad, dtype):
    """Wide rows, more than CTAs down the grid: a thread draws for several rows."""
    from fast_b200 import ops
    assert torch.equal(philox_at_once(5, 11, 0x123456789ABCDEF0, (7 << 32) + 5), hm.philox(5, 11, 0x123456789ABCDEF0, (7 << 32) + 5))
    g = torch.Generator().manual_seed(1)
    n, p, seed, offset = 2900, 0.3, 0xFFFFFFFF00000001, (3 << 40) + 9
    x, res = (rows_of(g, n, d, dtype, pad=pad) for _ in range(2))
    kept = (philox_at_once(n, d, seed, offset).cuda() >> 8).double() * 2.0 ** -24 >= float(torch.tensor(p))
    scale = kept.double() / (1 - p)
    half = torch.finfo(dtype).eps / 2
    for got, want in ((ops.dropout_fwd(x, p, seed, offset), x.double() * scale),
                      (ops.dropout_fwd(x, p, seed, offset, res), res.double() + x.double() * scale)):
        # the scale, its product and the sum are rounded in fp32, the result once more
        room = half * want.abs() + 3 * 2.0 ** -24 * (x.double().abs().amax() / (1 - p) + res.double().abs())
        assert bool(((got.double() - want).abs() <= room).all())
