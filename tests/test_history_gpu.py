"""GPU: the event-history operators against fp64 restatements (history_math.py),
forward and backward, at the lengths, masks, layouts and types where they can go
wrong."""
import history_math as hm
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32

# Tolerance.  A result of type t is rounded once: eps(t) / 2 of itself.  Before that, fp32: the decay exp(dt A) of a
# step is off by 2^-22 (two units of the exponential) and as much again from its argument and the state's two roundings;
# steps that decay by e^-0.025 or more (dt >= 0.05, |A| >= 0.5 below) remember 40 of each other: 40 * 2^-21 < 2^-15.6.
# A gradient chains two such recursions, forward states and backward ones, and adds rows of one sign and the other:
# 2^-14 of the tensor's size.  Held row by row (last axis), against the row's norm and the tensor's mean row norm.
TAU = 2.0 ** -14


def close(got, want, name):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if not got.numel():
        return
    half = torch.finfo(got.dtype).eps / 2
    got, want = got.double().reshape(-1, got.shape[-1]), want.detach().double().reshape(-1, want.shape[-1])
    assert bool(torch.isfinite(got).all()), name
    off, size = (got - want).norm(dim=1), want.norm(dim=1)
    room = half * size + TAU * (size + size.square().mean().sqrt()) + 1e-30
    worst = int((off / room).argmax())
    assert float(off[worst]) <= float(room[worst]), (name, worst, float(off[worst]), float(room[worst]))


def rows_of(g, n, d, dtype, scale=1.0, pad=0, shift=0):
    """Rows in a buffer `pad` wider and `shift` elements into it."""
    t = (torch.randn(n, d + pad + shift, generator=g) * scale).to(dtype).cuda()
    return t[:, shift:shift + d]


LENGTHS = {
    "one row": [1],
    "one": [37],
    "ragged": [5, 0, 1, 64, 0, 0, 17, 130, 3, 0],
    "long": [700, 1, 333],
    "aligned": [64, 64, 128, 8, 8],
    "empty": [0, 0],
    "ones": [1] * 50,
    "many empty": [3] + [0] * 100 + [9] + [0] * 40,
}


def starts_of(lengths, front=0, dtype=torch.int64):
    s = [front]
    for n in lengths:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=dtype, device="cuda")


def poison(rows, starts, *tensors):
    """NaN and infinities in every row of no sequence."""
    for t in tensors:
        if t is not None:
            t[:int(starts[0])] = float("nan")
            t[int(starts[-1]):] = float("inf")


# ---- short convolution -------------------------------------------------------------------------------
def conv_case(lengths, d, k, dtype, bias=True, init=False, act="silu", front=0, tail=0, pad=0, shift=0, seed=0, ints=torch.int64):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(seed)
    starts = None if lengths is None else starts_of(lengths, front, ints)
    n = 37 if lengths is None else int(starts[-1]) + tail
    seqs = 1 if lengths is None else len(lengths)
    x, dy = rows_of(g, n, d, dtype, 1, pad, shift), rows_of(g, n, d, dtype, 1, pad, shift)
    w = torch.randn(d, k, generator=g).cuda() * k ** -0.5
    b = torch.randn(d, generator=g).cuda() * 0.2 if bias else None
    i = torch.randn(seqs, k - 1, d, generator=g).to(dtype).cuda() if init else None
    df = torch.randn(seqs, k - 1, d, generator=g).to(dtype).cuda() if init else None
    if starts is not None:
        poison(n, starts, x, dy)
    wide = [t.detach().double().requires_grad_(True) if t is not None else None for t in (x.nan_to_num(0, 0, 0), w, b, i)]
    y, final = hm.short_conv(wide[0], wide[1], wide[2], starts, wide[3], act)
    got_y, got_final = ops.short_conv_fwd(x, w, b, starts, i, act, final=True)
    close(got_y, y, "y")
    close(got_final, final, "final")
    assert torch.equal(got_final.double(), final.double())         # copies, nothing computed
    only = ops.short_conv_fwd(x, w, b, starts, i, act)
    assert torch.equal(only, got_y)
    clean = dy.double().nan_to_num(0, 0, 0)
    have = [t for t in wide if t is not None]
    none = sum(t.sum() for t in have) * 0                          # empty sequences leave y without a graph
    outs, grads = [y + none, final + none], [clean, None if df is None else df.double()]
    if df is None:
        outs, grads = outs[:1], grads[:1]
    want = dict(zip([m for m, t in zip(("dx", "dw", "dbias", "dinit"), wide) if t is not None],
                    torch.autograd.grad(outs, have, grads, allow_unused=True)))
    got = dict(zip(("dx", "dw", "dbias", "dinit"), ops.short_conv_bwd(dy, x, w, b, starts, i, act, dfinal=df)))
    for m, v in got.items():
        if m in want:
            close(v, torch.zeros_like(v) if want[m] is None else want[m], m)
        else:
            assert v is None
    again = ops.short_conv_bwd(dy, x, w, b, starts, i, act, dfinal=df)
    assert all(a is b2 or torch.equal(a, b2) for a, b2 in zip(got.values(), again))


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("init", [False, True])
def test_conv_lengths(cuda, lengths, dtype, init):
    conv_case(LENGTHS[lengths], 24, 4, dtype, init=init, front=3, tail=11)


@pytest.mark.parametrize("k", [1, 2, 3, 5, 7, 8])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_conv_taps(cuda, k, dtype):
    conv_case([9, 0, 1, 2, 3, 40, 6], 20, k, dtype, init=True, tail=2)
    conv_case([9, 0, 1, 2, 3, 40, 6], 20, k, dtype, bias=False, act=None, init=True)


@pytest.mark.parametrize("d,pad,shift", [(1, 0, 0), (3, 0, 0), (7, 2, 1), (100, 0, 0), (130, 2, 2), (1031, 1, 0), (2048, 8, 0)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_conv_widths(cuda, d, pad, shift, dtype):
    conv_case([30, 2, 0, 51], d, 4, dtype, pad=pad, shift=shift, tail=5)


def test_conv_one_sequence_and_int32(cuda):
    conv_case(None, 16, 4, F32, init=True)
    conv_case([40, 7, 0, 3], 16, 4, BF, init=True, ints=torch.int32)


def test_conv_many_rows(cuda):
    """Several CTAs along the rows, runs that end inside sequences."""
    conv_case([1500, 3, 0, 2200, 999], 8, 4, F32, init=True, tail=100)
    conv_case([4000], 260, 8, BF, init=True)


# ---- selective scan ----------------------------------------------------------------------------------
def scan_case(lengths, d, n, dtype, groups=1, skip=True, gate=True, bias=True, init=False, softplus=True, front=0, tail=0, pad=0,
              seed=0, ints=torch.int64, flat=False):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(seed)
    starts = None if lengths is None else starts_of(lengths, front, ints)
    rows = 37 if lengths is None else int(starts[-1]) + tail
    seqs = 1 if lengths is None else len(lengths)
    u, dy = rows_of(g, rows, d, dtype, 1, pad), rows_of(g, rows, d, dtype, 1, pad)
    z = rows_of(g, rows, d, dtype, 1, pad) if gate else None
    if softplus:
        delta = rows_of(g, rows, d, dtype, 0.7, pad)
        delta_bias = torch.randn(d, generator=g).cuda() * 0.3 - 0.5 if bias else None      # dt about 0.1 .. 2
    else:
        delta = (torch.rand(rows, d + pad, generator=g) * 0.6 + 0.05).to(dtype).cuda()[:, :d]
        delta_bias = torch.rand(d, generator=g).cuda() * 0.1 if bias else None
    A = -(0.5 + torch.rand(d, n, generator=g) * n).cuda()
    B, C = (rows_of(g, rows, groups * n, dtype, 1, pad).unflatten(1, (groups, n)) for _ in range(2))
    D = torch.randn(d, generator=g).cuda() if skip else None
    i = torch.randn(seqs, d, n, generator=g).cuda() if init else None
    df = torch.randn(seqs, d, n, generator=g).cuda() if init else None
    if starts is not None:
        poison(rows, starts, u, delta, z, B, C, dy)
    src = dict(u=u, delta=delta, A=A, B=B, C=C, D=D, z=z, delta_bias=delta_bias, init=i)
    wide = {m: None if t is None else t.detach().double().nan_to_num(0, 0, 0).requires_grad_(True) for m, t in src.items()}
    y, final = hm.selective_scan(**{k: wide[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")}, starts=starts,
                                 init=wide["init"], softplus=softplus)
    Bx, Cx = (B[:, 0], C[:, 0]) if flat else (B, C)
    kw = dict(D=D, z=z, delta_bias=delta_bias, starts=starts, init=i, softplus=softplus)
    got_y, carry, got_final = ops.selective_scan_fwd(u, delta, A, Bx, Cx, final=True, **kw)
    close(got_y, y, "y")
    close(got_final, final, "final")
    alone, nothing, none = ops.selective_scan_fwd(u, delta, A, Bx, Cx, keep=False, **kw)
    assert nothing is None and none is None and torch.equal(alone, got_y)
    names = [m for m in wide if wide[m] is not None]
    none = sum(wide[m].sum() for m in names) * 0
    outs, grads = [y + none], [dy.double().nan_to_num(0, 0, 0)]
    if df is not None:
        outs, grads = outs + [final + none], grads + [df.double()]
    want = dict(zip(names, torch.autograd.grad(outs, [wide[m] for m in names], grads, allow_unused=True)))
    order = "u", "delta", "A", "B", "C", "D", "z", "delta_bias", "init"
    got = dict(zip(order, ops.selective_scan_bwd(dy, u, delta, A, Bx, Cx, carry, dfinal=df, **kw)))
    for m, v in got.items():
        if src[m] is None:
            assert v is None
            continue
        if flat and m in "BC":
            assert v.shape == Bx.shape
            v = v.unsqueeze(1)
        close(v, torch.zeros_like(src[m]) if want[m] is None else want[m], "d" + m)
    again = ops.selective_scan_bwd(dy, u, delta, A, Bx, Cx, carry, dfinal=df, **kw)
    assert all((a is None and b2 is None) or torch.equal(a.reshape(-1), b2.reshape(-1)) for a, b2 in zip(got.values(), again))


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("init", [False, True])
def test_scan_lengths(cuda, lengths, dtype, init):
    scan_case(LENGTHS[lengths], 24, 16, dtype, init=init, front=3, tail=11)


@pytest.mark.parametrize("n", [1, 3, 4, 8, 9, 13, 16, 17, 32, 40, 64])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_scan_states(cuda, n, dtype):
    scan_case([70, 0, 2, 100], 20, n, dtype, init=True, tail=2)


@pytest.mark.parametrize("d,groups,pad", [(1, 1, 0), (5, 1, 3), (33, 1, 0), (64, 2, 0), (66, 2, 1), (100, 4, 0), (130, 1, 2), (257, 1, 0)])
@pytest.mark.parametrize("n", [8, 16, 32, 64])
def test_scan_widths(cuda, d, groups, pad, n):
    scan_case([90, 3], d, n, BF, groups=groups, pad=pad)


@pytest.mark.parametrize("skip,gate,bias,softplus", [(False, False, False, True), (True, False, True, False), (False, True, False, False),
                                                     (True, True, False, True)])
def test_scan_options(cuda, skip, gate, bias, softplus):
    scan_case([100, 0, 31], 40, 16, F32, skip=skip, gate=gate, bias=bias, softplus=softplus, init=True, flat=True)


def test_scan_one_sequence_and_int32(cuda):
    scan_case(None, 16, 16, F32, init=True)
    scan_case([40, 7, 0, 3], 16, 16, BF, init=True, ints=torch.int32)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_scan_many_chunks(cuda, dtype):
    """Chunks of no sequence, of one sequence and of several, over several CTAs and groups; states in and out."""
    scan_case([150, 0, 400, 1, 1, 60], 200, 16, dtype, groups=2, init=True, front=130, tail=300)
    scan_case([611], 300, 8, dtype, init=True, front=1, tail=1)
    scan_case([48, 48, 96, 0, 192], 70, 32, dtype, init=True, gate=False)


def test_no_sequences(cuda):
    """starts of one element: every row is of no sequence."""
    from fast_b200 import ops
    x = torch.full((100, 8), float("nan"), device="cuda")
    w, A, B = torch.randn(8, 4, device="cuda"), -torch.rand(8, 16, device="cuda"), torch.full((100, 16), float("inf"), device="cuda")
    starts = torch.zeros(1, dtype=torch.int64, device="cuda")
    y, final = ops.short_conv_fwd(x, w, starts=starts, final=True)
    assert not bool(y.any()) and final.shape == (0, 3, 8)
    assert not any(bool(t.any()) for t in ops.short_conv_bwd(x, x, w, starts=starts)[:2])
    y, carry, final = ops.selective_scan_fwd(x, x, A, B, B, starts=starts, final=True)
    assert not bool(y.any()) and final.shape == (0, 8, 16)
    assert not any(bool(t.any()) for t in ops.selective_scan_bwd(x, x, x, A, B, B, carry, starts=starts)[:5])


def test_scan_long_memory(cuda):
    """Slow decays over a long sequence.  A decay's mean error is at most 1.3e-8 after centring (measured without: 0.6 to
    2.4e-8), its rounding 2^-25 at random; a thousand steps remembered (dt 0.001, |A| 1) add up 1.3e-5 of the state at worst,
    2^-16, twice that for gradients, which chain two recursions."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(8)
    rows, d, n = 4000, 32, 16
    u, dy, B, C = rows_of(g, rows, d, F32), rows_of(g, rows, d, F32), rows_of(g, rows, n, F32), rows_of(g, rows, n, F32)
    delta = (torch.rand(rows, d, generator=g) * 0.001 + 0.0005).cuda()
    A = -torch.arange(1, n + 1, dtype=torch.float32, device="cuda").repeat(d, 1)
    y, carry, final = ops.selective_scan_fwd(u, delta, A, B, C, softplus=False, final=True)
    grads = ops.selective_scan_bwd(dy, u, delta, A, B, C, carry, softplus=False)
    wide = [t.double().requires_grad_(True) for t in (u, delta, A, B, C)]
    wy, wf = hm.selective_scan(*wide[:3], wide[3].unsqueeze(1), wide[4].unsqueeze(1), None, None, None, None, None, False)
    want = torch.autograd.grad(wy, wide, dy.double())
    for got, ref, tol in ((y, wy, 2.0 ** -16), (final, wf, 2.0 ** -16), *((a, b, 2.0 ** -15) for a, b in zip(grads, want))):
        assert float((got.double() - ref).norm() / ref.norm()) <= tol


def test_scan_decays_of_minus_infinity(cuda):
    """States with A = -infinity keep nothing of the row before; rows of no sequence in front change nothing."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(9)
    rows, d, n = 300, 8, 16
    u, delta, B, C = rows_of(g, rows, d, F32), rows_of(g, rows, d, F32), rows_of(g, rows, n, F32), rows_of(g, rows, n, F32)
    A = -torch.rand(d, n, generator=g).cuda() - 0.5
    A[:, 3] = float("-inf")
    starts = starts_of([100, 150], front=7)
    y, _, final = ops.selective_scan_fwd(u, delta, A, B, C, starts=starts, final=True)
    wide = [t.double() for t in (u, delta, A, B, C)]
    wy, wf = hm.selective_scan(*wide[:3], wide[3].unsqueeze(1), wide[4].unsqueeze(1), None, None, None, starts, None, True)
    close(y, wy, "y")
    close(final, wf, "final")


def test_scan_infinity_stays_in_its_sequence(cuda):
    """A sequence that overflows leaves its neighbours as they are."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(5)
    starts = starts_of([70, 70, 200, 60])
    rows, d, n = 400, 24, 16
    u, delta, dy = (rows_of(g, rows, d, F32) for _ in range(3))
    B, C = rows_of(g, rows, n, F32), rows_of(g, rows, n, F32)
    A = -(0.5 + torch.rand(d, n, generator=g) * n).cuda()
    y, carry, final = ops.selective_scan_fwd(u, delta, A, B, C, starts=starts, final=True)
    grads = ops.selective_scan_bwd(dy, u, delta, A, B, C, carry, starts=starts)
    for bad in (float("inf"), float("nan")):
        v = u.clone()
        v[100] = bad
        y2, carry2, final2 = ops.selective_scan_fwd(v, delta, A, B, C, starts=starts, final=True)
        assert not bool(torch.isfinite(y2[100:140]).any())
        grads2 = ops.selective_scan_bwd(dy, v, delta, A, B, C, carry2, starts=starts)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[70:140] = False
        assert torch.equal(y2[keep], y[keep])
        assert torch.equal(final2[[0, 2, 3]], final[[0, 2, 3]])
        for i in (0, 1, 3, 4):
            assert torch.equal(grads2[i][keep], grads[i][keep]), i


def test_scan_gradients_against_differences(cuda):
    """The sum over dy y moves as the gradients say (central differences in fp64 of the restatement's inputs would
    test the restatement; these are of the kernel itself, fp32: a step of 2^-6 loses 2^-24 / 2^-6 of the value)."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(7)
    starts = starts_of([40, 0, 33])
    rows, d, n = 73, 12, 16
    src = dict(u=rows_of(g, rows, d, F32), delta=rows_of(g, rows, d, F32, 0.7), A=-(0.5 + torch.rand(d, n, generator=g) * 4).cuda(),
               B=rows_of(g, rows, n, F32), C=rows_of(g, rows, n, F32), D=torch.randn(d, generator=g).cuda(),
               z=rows_of(g, rows, d, F32), delta_bias=torch.randn(d, generator=g).cuda() * 0.2, init=torch.randn(2, d, n, generator=g).cuda()[[0, 0, 1]])
    dy = rows_of(g, rows, d, F32)

    def run(**new):
        s = dict(src, **new)
        return ops.selective_scan_fwd(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                      starts=starts, init=s["init"])
    y, carry, _ = run()
    names = "u", "delta", "A", "B", "C", "D", "z", "delta_bias", "init"
    kw = dict(D=src["D"], z=src["z"], delta_bias=src["delta_bias"], starts=starts, init=src["init"])
    grads = dict(zip(names, ops.selective_scan_bwd(dy, *(src[m] for m in names[:5]), carry, **kw)))
    for m in names:
        # along the gradient itself, so the difference is large against its rounding
        way = grads[m] / grads[m].norm()
        e = 2.0 ** -6
        up, down = run(**{m: (src[m] + e * way).contiguous()})[0], run(**{m: (src[m] - e * way).contiguous()})[0]
        slope = float(((up.double() - down.double()) * dy.double()).sum()) / (2 * e)
        want = float(grads[m].double().norm())
        # third derivative times e^2 / 6 = 2^-14.6 of it, and 2^-22 |y . dy| / e of rounding
        assert abs(slope - want) <= 2.0 ** -9 * want + 2.0 ** -16 * float((y * dy).abs().sum()), (m, slope, want)


# ---- single events -----------------------------------------------------------------------------------
def turns(index, n):
    """Rows in order, with the node of each; None: the row is held out."""
    return [(r, r if index is None else int(index[r])) for r in range(n)]


@pytest.mark.parametrize("n,repeat", [(1, 1), (2, 2), (7, 1), (33, 3), (300, 7), (1000, 300)])
@pytest.mark.parametrize("d,k", [(24, 4), (9, 2), (40, 8), (6, 1), (18, 3)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_conv_step(cuda, n, repeat, d, k, dtype):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(n + d)
    nodes = n + 5
    index = torch.randperm(nodes, generator=g)[:n]
    index[torch.randperm(n, generator=g)[:repeat]] = index[0].clone()
    if n > 5:
        index[3], index[4] = -1, nodes
    x = rows_of(g, n, d, dtype, pad=3)
    w, b = torch.randn(d, k, generator=g).cuda() * k ** -0.5, torch.randn(d, generator=g).cuda()
    state = torch.randn(nodes, k - 1, d, generator=g).to(dtype).cuda()
    s = state.double().clone()
    want = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    for r, i in turns(index, n):
        if 0 <= i < nodes:
            win = torch.cat([s[i], x[r:r + 1].double()])
            p = (win * w.double().t()).sum(0) + b
            want[r], s[i] = p * torch.sigmoid(p), win[1:]
    y = ops.short_conv_step(x, state, w, b, index.cuda())
    if n > 5:
        assert bool(torch.isnan(y[4]).all()) and bool((y[3] == 0).all())
        y[4] = 0
    close(y, want, "y")
    assert torch.equal(state.double(), s)


@pytest.mark.parametrize("n,repeat", [(1, 1), (2, 2), (7, 1), (33, 3), (300, 7), (600, 200)])
@pytest.mark.parametrize("d,states,groups", [(24, 16, 1), (9, 4, 1), (40, 64, 4), (6, 1, 2), (18, 13, 1), (35, 30, 1)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_scan_step(cuda, n, repeat, d, states, groups, dtype):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(n + d)
    nodes = n + 5
    index = torch.randperm(nodes, generator=g)[:n]
    index[torch.randperm(n, generator=g)[:repeat]] = index[0].clone()
    if n > 5:
        index[3], index[4] = -1, nodes
    u, delta, z = (rows_of(g, n, d, dtype, pad=3) for _ in range(3))
    B, C = (rows_of(g, n, groups * states, dtype, pad=1).unflatten(1, (groups, states)) for _ in range(2))
    A = -(0.5 + torch.rand(d, states, generator=g) * states).cuda()
    D, bias = torch.randn(d, generator=g).cuda(), torch.randn(d, generator=g).cuda() * 0.3 - 0.5
    state = torch.randn(nodes, d, states, generator=g).cuda()
    s = state.double().clone()
    want = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    for r, i in turns(index, n):
        if 0 <= i < nodes:
            y, h = hm.selective_scan(*(t.double() for t in (u[r:r + 1], delta[r:r + 1], A, B[r:r + 1], C[r:r + 1], D, z[r:r + 1], bias)),
                                     None, s[i:i + 1], True)
            want[r], s[i] = y[0], h[0]
    y = ops.selective_scan_step(u, delta, A, B, C, state, D, z, bias, index.cuda())
    if n > 5:
        assert bool(torch.isnan(y[4]).all()) and bool((y[3] == 0).all())
        y[4] = 0
    close(y, want, "y")
    close(state, s, "state")


def test_steps_without_index(cuda):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(3)
    x, w = rows_of(g, 5, 12, F32), torch.randn(12, 4, generator=g).cuda()
    state = torch.randn(8, 3, 12, generator=g).cuda()
    other = state.clone()
    a = ops.short_conv_step(x, state, w)
    b = ops.short_conv_step(x, other, w, index=torch.arange(5, device="cuda"))
    assert torch.equal(a, b) and torch.equal(state, other)
    A, B, C = -torch.rand(12, 16, generator=g).cuda(), rows_of(g, 5, 16, F32), rows_of(g, 5, 16, F32)
    h = torch.randn(8, 12, 16, generator=g).cuda()
    k = h.clone()
    a = ops.selective_scan_step(x, x, A, B, C, h)
    b = ops.selective_scan_step(x, x, A, B, C, k, index=torch.arange(5, device="cuda"))
    assert torch.equal(a, b) and torch.equal(h, k) and torch.equal(h[5:], k[5:])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_histories_and_then_events(cuda, dtype):
    """A history at once, or its first part at once and the rest event by event: the same results and states."""
    from fast_b200 import ops
    g = torch.Generator().manual_seed(11)
    lengths, more, d, n, k = [20, 1, 0, 9], 6, 32, 16, 4
    seqs = len(lengths)
    w, b = torch.randn(d, k, generator=g).cuda() * 0.5, torch.randn(d, generator=g).cuda() * 0.1
    A, D, bias = -(0.5 + torch.rand(d, n, generator=g) * n).cuda(), torch.randn(d, generator=g).cuda(), torch.randn(d, generator=g).cuda() * 0.3 - 0.5
    total = sum(lengths) + seqs * more
    x, delta, z, B, C = (rows_of(g, total, c, dtype) for c in (d, d, d, n, n))
    full = starts_of([m + more for m in lengths])
    u = ops.short_conv_fwd(x, w, b, full)
    y, _, final = ops.selective_scan_fwd(u, delta, A, B, C, D, z, bias, full, final=True, keep=False)
    head = torch.cat([torch.arange(int(full[i]), int(full[i]) + m) for i, m in enumerate(lengths)]).cuda()
    starts = starts_of(lengths)
    u1, conv = ops.short_conv_fwd(x[head], w, b, starts, final=True)
    y1, _, scan = ops.selective_scan_fwd(u1, delta[head], A, B[head], C[head], D, z[head], bias, starts, final=True, keep=False)
    close(y1, y[head], "history")
    nodes = torch.tensor([4, 1, 3, 0], device="cuda")                       # the sequences' places in the tables
    ct, st = torch.zeros(6, k - 1, d, device="cuda", dtype=dtype), torch.zeros(6, d, n, device="cuda")
    ct[nodes], st[nodes] = conv, scan
    for j in range(more):
        at = torch.tensor([int(full[i]) + m + j for i, m in enumerate(lengths)], device="cuda")
        ue = ops.short_conv_step(x[at], ct, w, b, nodes)
        ye = ops.selective_scan_step(ue, delta[at], A, B[at], C[at], st, D, z[at], bias, nodes)
        close(ye, y[at], "event %d" % j)
    close(st[nodes], final, "final")


# ---- dropout -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d,pad,shift", [(1, 1, 0, 0), (5, 4, 0, 0), (33, 7, 0, 0), (20, 64, 4, 0), (20, 64, 3, 0), (9, 100, 0, 1)])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("p", [0.0, 0.3, 0.95])
def test_dropout(cuda, n, d, pad, shift, dtype, p):
    from fast_b200 import ops
    g = torch.Generator().manual_seed(1)
    x, res, dy = (rows_of(g, n, d, dtype, pad=pad, shift=shift) for _ in range(3))
    seed, offset = 0x123456789ABCDEF0, (7 << 32) + 5
    scale = hm.keep_scale(n, d, p, seed, offset).cuda()
    half = torch.finfo(dtype).eps / 2
    for got, want in ((ops.dropout_fwd(x, p, seed, offset), x.double() * scale),
                      (ops.dropout_fwd(x, p, seed, offset, res), res.double() + x.double() * scale),
                      (ops.dropout_bwd(dy, p, seed, offset), dy.double() * scale)):
        # the scale, its product and the sum are rounded in fp32, the result once more
        room = half * want.abs() + 3 * 2.0 ** -24 * (x.double().abs().amax() / (1 - p) + res.double().abs())
        assert bool(((got.double() - want).abs() <= room).all())
    plus = torch.tensor([4], device="cuda")
    assert torch.equal(ops.dropout_fwd(x, p, seed, offset - 4, offset_dev=plus), ops.dropout_fwd(x, p, seed, offset))


def test_dropout_keeps_its_share(cuda):
    """Of n elements n (1 - p) are kept, six standard deviations at most apart; other seeds, offsets and rows draw others."""
    from fast_b200 import ops
    x = torch.ones(4000, 250, device="cuda")
    runs = [ops.dropout_fwd(x, 0.25, s, o) > 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 40, 0), (1, 1 << 40))]
    n = x.numel()
    for k in runs:
        assert abs(int(k.sum()) - 0.75 * n) <= 6 * (n * 0.25 * 0.75) ** 0.5
    for i, a in enumerate(runs):
        for b in runs[:i]:
            assert abs(int((a == b).sum()) - 0.625 * n) <= 6 * (n * 0.625 * 0.375) ** 0.5
    assert bool((runs[0][0] != runs[0][1]).any())


# ---- calls of no rows, launches ----------------------------------------------------------------------
def test_no_rows(cuda):
    from fast_b200 import ops
    x, w = torch.zeros(0, 8, device="cuda"), torch.randn(8, 4, device="cuda")
    starts, init = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.randn(3, 3, 8, device="cuda")
    y, final = ops.short_conv_fwd(x, w, starts=starts, init=init, final=True)
    assert y.shape == (0, 8) and torch.equal(final, init)
    dx, dw, db, dinit = ops.short_conv_bwd(x, x, w, starts=starts, init=init, dfinal=init)
    assert dx.shape == (0, 8) and not bool(dw.any()) and torch.equal(dinit, init) and db is None
    A, B, h = -torch.rand(8, 16, device="cuda"), torch.zeros(0, 16, device="cuda"), torch.randn(3, 8, 16, device="cuda")
    y, carry, final = ops.selective_scan_fwd(x, x, A, B, B, starts=starts, init=h, final=True)
    assert y.shape == (0, 8) and torch.equal(final, h)
    out = ops.selective_scan_bwd(x, x, x, A, B, B, carry, starts=starts, init=h, dfinal=h, D=A[:, 0].contiguous())
    assert not bool(out[2].any()) and not bool(out[5].any()) and torch.equal(out[8], h)
    at = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.short_conv_step(x, init, w, index=at).shape == (0, 8)
    assert ops.selective_scan_step(x, x, A, B, B, h, index=at).shape == (0, 8)
    assert ops.dropout_fwd(x, 0.5, 1).shape == (0, 8)


def test_launches_are_counted(cuda):
    from fast_b200 import ops
    x, w = torch.randn(50, 16, device="cuda"), torch.randn(16, 4, device="cuda")
    before = ops.LAUNCHES[0]
    ops.dropout_fwd(x, 0.5, 1)
    ops.short_conv_fwd(x, w)
    assert ops.LAUNCHES[0] == before + 2
