"""GPU: the node-ranking head's operators (layer norm, gated feed-forward
block, softmax cross entropy over all nodes) against plain fp64 restatements.

Tolerances are error bounds, elementwise, computed beside the reference: with
c = (K + 64) 2^-22 for fp32 products of K terms accumulated in any order (the
3xTF32 split's 2^-21 included), an intermediate rounded to bf16 is off by 2^-8
of itself (bf16 keeps 8 significant bits), and a result by 2^-8 (bf16) or 2^-23
of itself.  Each bound sums
|terms| the way the error propagates; nothing is fitted."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TYPES = [F32, BF]


def _mat(cuda, g, rows, cols, dtype, scale=1.0, pad=0, off=0):
    """Rows in a buffer pad elements wider, off elements past its start."""
    buf = torch.empty(rows * (cols + pad) + off + 8, device=cuda, dtype=torch.float32).normal_(generator=g)
    buf = (buf * scale).to(dtype)
    return buf[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]


def _gen(cuda, *key):
    return torch.Generator(device=cuda).manual_seed(sum((i + 1) * len(str(k)) * 7919 + (k if isinstance(k, int) else len(k)) for i, k in
                                                        enumerate(key)) & 0xFFFF)


def _check(name, dev, ref, bound, dtype):
    dev, ref = dev.double(), ref.double()
    half = 2.0 ** (-8 if dtype == BF else -23)
    tol = bound + half * (ref.abs() + bound) + 1e-37
    bad = ~((dev - ref).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d outside; worst %.3e, allowed there %.3e" % (
        name, int(bad.sum()), bad.numel(), float(((dev - ref).abs() - tol).max()),
        float(tol.reshape(-1)[int(((dev - ref).abs() - tol).reshape(-1).argmax())]))


def _c(k):
    return (k + 64) * 2.0 ** -22


# ---- layer norm --------------------------------------------------------------------------------------------------
NORM = [(1, 1, 0, 0), (3, 7, 0, 0), (5, 100, 4, 0), (33, 413, 6, 1), (130, 64, 0, 0), (300, 128, 8, 0), (17, 500, 0, 2),
        (7, 1024, 0, 0), (9, 1027, 0, 0), (2, 2050, 0, 0), (5, 4096, 0, 0), (3, 5000, 0, 0), (3, 8200, 0, 0),
        (2, 16384, 0, 0), (40000, 16, 0, 0), (2, 6144, 0, 0), (2, 6144, 1, 0), (3, 5890, 1, 0), (33, 414, 0, 0), (700, 413, 0, 1),
        (5, 3, 0, 1), (301, 2047, 0, 0), (300, 4095, 2, 1), (3, 9001, 0, 1), (2, 16383, 0, 1)]


@pytest.mark.parametrize("n,d,pad,off", NORM)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("res", [False, True])
def test_layer_norm(cuda, n, d, pad, off, dtype, res):
    from fast_b200 import ops
    g = _gen(cuda, n, d, res)
    x = _mat(cuda, g, n, d, dtype, 1.5, pad, off)
    r = _mat(cuda, g, n, d, dtype, 0.7, pad) if res else None
    gamma = (1 + 0.3 * torch.randn(d, device=cuda, generator=g)).to(dtype)
    beta = (0.3 * torch.randn(d, device=cuda, generator=g)).to(dtype)
    dy = _mat(cuda, g, n, d, dtype, 1.0, pad, off)
    ds = _mat(cuda, g, n, d, dtype, 1.0, pad) if res else None
    out = ops.layer_norm_fwd(x, gamma, beta, res=r)
    y, s, mean, rstd = out if res else (out[0], x, out[1], out[2])
    if res:
        want = (x.double() + r.double()).to(dtype)
        assert torch.equal(s, want) or dtype == BF and bool(((s.double() - want.double()).abs() <=
                                                             2.0 ** -8 * want.double().abs()).all())
    S, G, B, DY = s.double(), gamma.double(), beta.double(), dy.double()
    mu = S.mean(1, keepdim=True)
    rs = 1 / torch.sqrt(((S - mu) ** 2).mean(1, keepdim=True) + 1e-5)
    xh = (S - mu) * rs
    c = _c(d)
    # mean is off by c mean|s|; xhat by that over the deviation, and by c of itself (variance and square root)
    exh = c * ((S.abs().mean(1, keepdim=True) + S.abs()) * rs + 2 * xh.abs() * (1 + S.abs().mean(1, keepdim=True) * rs))
    _check("mean", mean, mu[:, 0], c * S.abs().mean(1), F32)
    _check("rstd", rstd, rs[:, 0], 2 * c * rs[:, 0] * (1 + S.abs().mean(1) * rs[:, 0]), F32)
    _check("y", y, xh * G + B, exh * G.abs() + 2.0 ** -22 * (xh * G).abs(), dtype)
    dx, dg, db = ops.layer_norm_bwd(dy, s, gamma, mean, rstd, ds=ds)
    a = DY * G
    m1, m2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    A = a.abs()
    em1 = c * A.mean(1, keepdim=True)
    em2 = c * (A * xh.abs()).mean(1, keepdim=True) + (A * exh).mean(1, keepdim=True)
    ers = 2 * c * (1 + S.abs().mean(1, keepdim=True) * rs)
    want = rs * (a - m1 - xh * m2)
    mag = rs * (A + m1.abs() + (xh * m2).abs())
    edx = rs * (em1 + xh.abs() * em2 + exh * m2.abs()) + (ers + 2.0 ** -21) * mag
    if res:
        want = want + ds.double()
        edx = edx + 2.0 ** -22 * ds.double().abs()
    _check("dx", dx, want, edx, dtype)
    cn = _c(n)
    _check("dgamma", dg, (DY * xh).sum(0), (DY.abs() * exh).sum(0) + cn * (DY * xh).abs().sum(0), dtype)
    _check("dbeta", db, DY.sum(0), cn * DY.abs().sum(0), dtype)
    again = ops.layer_norm_bwd(dy, s, gamma, mean, rstd, ds=ds)
    assert all(torch.equal(p, q) for p, q in zip((dx, dg, db), again))


def test_layer_norm_fp32_parameters_accumulate_and_constant_rows(cuda):
    from fast_b200 import ops
    n, d = 70, 100
    x = torch.full((n, d), 3.0, device=cuda, dtype=BF)          # variance 0: y = beta, dx finite
    gamma, beta = torch.ones(d, device=cuda), torch.linspace(-1, 1, d, device=cuda)
    y, mean, rstd = ops.layer_norm_fwd(x, gamma, beta)
    assert torch.equal(y, beta.to(BF).expand(n, d)) and bool((mean == 3).all())
    dg, db = torch.full((d,), 2.0, device=cuda), torch.zeros(d, device=cuda)
    dy = torch.ones(n, d, device=cuda, dtype=BF)
    dx, dg2, db2 = ops.layer_norm_bwd(dy, x, gamma, mean, rstd, dgamma=dg, dbeta=db)
    assert dg2 is dg and bool((dg == 2).all()) and bool((db == n).all()) and bool((dx == 0).all())
    e = torch.empty(0, d, device=cuda, dtype=BF)
    y, mean, rstd = ops.layer_norm_fwd(e, gamma)
    dx, dg, db = ops.layer_norm_bwd(e, e, gamma, mean, rstd)
    assert y.shape == (0, d) and dx.shape == (0, d) and bool((dg == 0).all()) and bool((db == 0).all())


def test_layer_norm_keeps_nonfinite_rows_to_themselves(cuda):
    from fast_b200 import ops
    x = torch.randn(40, 96, device=cuda)
    x[3, 5], x[17, 0] = float("nan"), float("inf")
    gamma = torch.ones(96, device=cuda)
    y, _, _ = ops.layer_norm_fwd(x, gamma)
    rows = torch.isfinite(y).all(1)
    assert not bool(rows[3]) and not bool(rows[17]) and int(rows.sum()) == 38


# ---- gated feed-forward block ------------------------------------------------------------------------------------
FFN = [(1, 16, 16, 0), (1, 100, 37, 0), (2, 1024, 520, 0), (3, 413, 50, 3), (7, 64, 129, 0), (130, 100, 400, 4),
       (257, 72, 300, 0), (300, 264, 520, 8), (64, 33, 65, 1), (515, 130, 260, 0), (1000, 172, 688, 4), (1, 11900, 24, 0),
       (1, 12288, 16, 0), (8, 1500, 24, 1), (9, 100, 64, 0)]


def _act(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).double()


def _ffn_inputs(cuda, n, d, f, pad, dtype, act, off=0):
    g = _gen(cuda, n, d, f, act)
    x, dy = _mat(cuda, g, n, d, dtype, 1.0, pad, off), _mat(cuda, g, n, d, dtype, 1.0, pad)
    wg, wu = _mat(cuda, g, f, d, dtype, d ** -0.5, pad), _mat(cuda, g, f, d, dtype, d ** -0.5, pad, off)
    wd = _mat(cuda, g, d, f, dtype, f ** -0.5, pad)
    if act == "relu":       # multiples of 1/8: the pre-activation is exact, so the kink is met on the same side
        for t in (x, wg):
            t.copy_((t.float() * 8).round().clamp(-31, 31) / 8)
    return x, wg, wu, wd, dy


@pytest.mark.parametrize("n,d,f,pad", FFN)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_ffn(cuda, n, d, f, pad, dtype, act):
    from fast_b200 import ops
    x, wg, wu, wd, dy = _ffn_inputs(cuda, n, d, f, pad, dtype, act, off=pad & 1)
    X, WG, WU, WD, DY = (t.double() for t in (x, wg, wu, wd, dy))
    G, U = X @ WG.t(), X @ WU.t()
    A, DA = _act(act, G)
    H = A * U
    cd, cf, cn = _c(d), _c(f), _c(n)
    r = 2.0 ** -8 if dtype == BF else 0.0
    eg = 0 * G if act == "relu" else cd * (X.abs() @ WG.abs().t())
    eu = cd * (X.abs() @ WU.abs().t())
    fn = 2.0 ** -20                                  # exp / erf and the few products around them, of O(1) values
    eh = 1.2 * eg * U.abs() + A.abs() * eu + fn * (A.abs() + G.abs()) * U.abs()
    eh = eh + r * (H.abs() + eh)
    _check("y", ops.gated_ffn_fwd(x, wg, wu, wd, act=act), H @ WD.t(),
           eh @ WD.abs().t() + cf * ((H.abs() + eh) @ WD.abs().t()), dtype)
    DH = DY @ WD
    ed = cd * (DY.abs() @ WD.abs())
    DG, DU = DH * U * DA, DH * A
    edg = ed * (U * DA).abs() + DH.abs() * eu * DA.abs() + (DH * U).abs() * (1.2 * eg + fn * (1 + G.abs()))
    edu = ed * A.abs() + DH.abs() * (1.2 * eg + fn * (A.abs() + G.abs()))
    edg, edu = edg + r * (DG.abs() + edg), edu + r * (DU.abs() + edu)
    dx, dwg, dwu, dwd = ops.gated_ffn_bwd(dy, x, wg, wu, wd, act=act)
    _check("dx", dx, DG @ WG + DU @ WU,
           edg @ WG.abs() + edu @ WU.abs() + 2 * cf * ((DG.abs() + edg) @ WG.abs() + (DU.abs() + edu) @ WU.abs()), dtype)
    _check("dw_gate", dwg, DG.t() @ X, edg.t() @ X.abs() + cn * ((DG.abs() + edg).t() @ X.abs()), dtype)
    _check("dw_up", dwu, DU.t() @ X, edu.t() @ X.abs() + cn * ((DU.abs() + edu).t() @ X.abs()), dtype)
    _check("dw_down", dwd, DY.t() @ H, DY.abs().t() @ eh + cn * (DY.abs().t() @ (H.abs() + eh)), dtype)
    again = ops.gated_ffn_bwd(dy, x, wg, wu, wd, act=act)
    assert all(torch.equal(p, q) for p, q in zip((dx, dwg, dwu, dwd), again))
    # fp32 buffers accumulate; minus their start they are the gradients before the last rounding
    bufs = [torch.full(t.shape, 0.5, device=cuda) for t in (wg, wu, wd)]
    ops.gated_ffn_bwd(dy, x, wg, wu, wd, act=act, grads=bufs)
    for name, b, want, e in (("dw_gate", bufs[0], DG.t() @ X, edg.t() @ X.abs() + cn * ((DG.abs() + edg).t() @ X.abs())),
                             ("dw_up", bufs[1], DU.t() @ X, edu.t() @ X.abs() + cn * ((DU.abs() + edu).t() @ X.abs())),
                             ("dw_down", bufs[2], DY.t() @ H, DY.abs().t() @ eh + cn * (DY.abs().t() @ (H.abs() + eh)))):
        _check("accumulated " + name, b, want + 0.5, e, F32)


# few rows against weights of more than 2^20 elements: the path that reads them without tensor cores, both layouts
@pytest.mark.parametrize("n,d,f,pad", [(1, 520, 2056, 0), (2, 520, 2056, 8), (2, 519, 2051, 0), (1, 1100, 1000, 3),
                                       (3, 520, 2056, 0), (8, 519, 2051, 0), (8, 2056, 520, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_ffn_few_rows_of_large_weights(cuda, n, d, f, pad, dtype):
    test_gated_ffn(cuda, n, d, f, pad, dtype, "silu")


def test_gated_ffn_gradient_against_differences(cuda):
    """fp32: <dy, y(p + e v) - y(p - e v)> / 2e against <grad, v> for every input."""
    from fast_b200 import ops
    x, wg, wu, wd, dy = _ffn_inputs(cuda, 40, 48, 96, 0, F32, "silu")
    grads = ops.gated_ffn_bwd(dy, x, wg, wu, wd)
    g = _gen(cuda, 5)
    e = 2.0 ** -7
    for i, grad in enumerate(grads):
        p = [x, wg, wu, wd]
        v = torch.randn(p[i].shape, device=cuda, generator=g) * float(p[i].std())

        def y(sign):
            q = list(p)
            q[i] = q[i] + sign * e * v
            return ops.gated_ffn_fwd(*q).double()
        yp, ym = y(1), y(-1)
        diff = float((dy.double() * (yp - ym)).sum()) / (2 * e)
        # third-order remainder: e^2 times a third derivative of the order of |dy||y|; rounding: 2^-20 |dy||y| / e
        size = float((dy.double().abs() * torch.maximum(yp.abs(), ym.abs())).sum())
        assert abs(diff - float((grad.double() * v.double()).sum())) <= size * (4 * e * e + 2.0 ** -20 / e), i


def test_gated_ffn_without_rows(cuda):
    from fast_b200 import ops
    x, wg, wu, wd, _ = _ffn_inputs(cuda, 4, 24, 40, 0, BF, "silu")
    e = x[:0]
    assert ops.gated_ffn_fwd(e, wg, wu, wd).shape == (0, 24)
    out = ops.gated_ffn_bwd(e, e, wg, wu, wd)
    assert out[0].shape == (0, 24) and all(bool((t == 0).all()) for t in out[1:])


# ---- softmax cross entropy ---------------------------------------------------------------------------------------
XENT = [(1, 16, 10, 0), (1, 64, 1, 0), (1, 200, 5000, 0), (5, 100, 1000, 4), (130, 413, 777, 3), (300, 100, 5001, 0),
        (64, 33, 129, 1), (257, 512, 2000, 0), (3000, 32, 5000, 0), (700, 100, 260, 4)]


@pytest.mark.parametrize("n,d,v,pad", XENT)
@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent(cuda, n, d, v, pad, dtype):
    from fast_b200 import ops
    g = _gen(cuda, n, d, v)
    h, w = _mat(cuda, g, n, d, dtype, 1.0, pad, pad & 1), _mat(cuda, g, v, d, dtype, 3 * d ** -0.5, pad)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    t[torch.rand(n, device=cuda, generator=g) < 0.2] = -1
    t[0] = v - 1
    dl = torch.rand(n, device=cuda, generator=g) + 0.5
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    Hd, W = h.double(), w.double()
    L = Hd @ W.t()
    Z = torch.logsumexp(L, 1)
    keep = (t >= 0).double()
    at = t.clamp(min=0).unsqueeze(1)
    el = (_c(d) * (Hd.abs() @ W.abs().t())).max(1).values       # of a logit, and so of lse
    fn = 2.0 ** -20 * (1 + Z.abs() + L.abs().max(1).values)     # exp, log and the subtraction of the maximum
    _check("lse", lse, Z, el + fn, F32)
    _check("loss", loss, (Z - L.gather(1, at)[:, 0]) * keep, (2 * el + fn) * keep, F32)
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, dl)
    P = torch.softmax(L, 1)
    scale = (dl.double() * keep).unsqueeze(1)
    G = P.clone()
    G.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float64))
    eG = scale * (P * (2 * el + 2 * fn).unsqueeze(1) + 2.0 ** -22 * G.abs())
    G = G * scale
    eG = eG + (2.0 ** -8 if dtype == BF else 0.0) * (G.abs() + eG)
    _check("dh", dh, G @ W, eG @ W.abs() + _c(v) * ((G.abs() + eG) @ W.abs()), dtype)
    _check("dw", dw, G.t() @ Hd, eG.t() @ Hd.abs() + _c(n) * ((G.abs() + eG).t() @ Hd.abs()), dtype)
    buf = torch.full((v, d), 0.25, device=cuda)
    dh2, _ = ops.softmax_xent_bwd(h, w, t, lse, dl, dw=buf)
    assert torch.equal(dh, dh2)
    _check("accumulated dw", buf, G.t() @ Hd + 0.25, eG.t() @ Hd.abs() + _c(n) * ((G.abs() + eG).t() @ Hd.abs()), F32)


# few tiles of long sums: fp32 stores these logits, in parts of the sums
@pytest.mark.parametrize("n,d,v,pad", [(9, 513, 2048, 0), (300, 1030, 657, 3), (60, 2050, 1, 0), (256, 640, 130, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_few_tiles_of_long_sums(cuda, n, d, v, pad, dtype):
    test_softmax_xent(cuda, n, d, v, pad, dtype)


@pytest.mark.parametrize("n,d,v,pad", [(1, 130, 9001, 0), (2, 128, 9000, 0), (2, 127, 9003, 1), (2, 1030, 2000, 0),
                                       (3, 128, 9000, 8), (7, 1030, 2001, 0), (8, 127, 9003, 0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_few_rows_of_large_tables(cuda, n, d, v, pad, dtype):
    test_softmax_xent(cuda, n, d, v, pad, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_held_out_and_out_of_range_rows(cuda, dtype):
    from fast_b200 import ops
    n, d, v = 20, 40, 90
    h, w = torch.randn(n, d, device=cuda).to(dtype), torch.randn(v, d, device=cuda).to(dtype)
    dl = torch.ones(n, device=cuda)
    t = torch.full((n,), -1, device=cuda)
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, dl)
    assert bool((loss == 0).all()) and bool((dh == 0).all()) and bool((dw == 0).all()) and bool(lse.isfinite().all())
    t[3] = v
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    assert bool(loss[3].isnan()) and int(loss.isnan().sum()) == 1
    # a held-out row may hold anything: it reaches no gradient
    h[5, 0] = float("nan")
    t[3], t[4] = 0, 7
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, dl)
    assert float(loss[5]) == 0 and bool((dh[5] == 0).all())
    assert bool(torch.isfinite(dh).all()) and int(torch.isfinite(loss).sum()) == n


@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_large_logits(cuda, dtype):
    """Logits of +-2000: no overflow, the losses of a sharp softmax."""
    from fast_b200 import ops
    h = torch.zeros(3, 16, device=cuda, dtype=dtype)
    h[:, 0] = 1
    w = torch.zeros(500, 16, device=cuda, dtype=dtype)
    w[:, 0] = -2000
    w[7, 0], w[300, 0] = 2000, 2000
    t = torch.tensor([7, 300, 2], device=cuda)
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    want = torch.tensor([math.log(2), math.log(2), 4000 + math.log(2)], dtype=torch.float64, device=cuda)
    assert bool(((loss.double() - want).abs() <= 2.0 ** -20 * 4000).all())
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, torch.ones(3, device=cuda))
    assert bool(torch.isfinite(dh).all()) and bool(torch.isfinite(dw).all())


def test_softmax_xent_gradient_against_differences(cuda):
    from fast_b200 import ops
    g = _gen(cuda, 9)
    n, d, v = 30, 40, 200
    h, w = _mat(cuda, g, n, d, F32), _mat(cuda, g, v, d, F32, d ** -0.5)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    dl = torch.rand(n, device=cuda, generator=g) + 0.5
    _, lse = ops.softmax_xent_fwd(h, w, t)
    grads = ops.softmax_xent_bwd(h, w, t, lse, dl)
    e = 2.0 ** -7
    for i, grad in enumerate(grads):
        p = [h, w]
        dv = torch.randn(p[i].shape, device=cuda, generator=g) * float(p[i].std())

        def total(sign):
            q = list(p)
            q[i] = q[i] + sign * e * dv
            return float((dl.double() * ops.softmax_xent_fwd(*q, t)[0].double()).sum())
        diff = (total(1) - total(-1)) / (2 * e)
        size = float((dl.double() * lse.double().abs()).sum())
        assert abs(diff - float((grad.double() * dv.double()).sum())) <= size * (4 * e * e + 2.0 ** -20 / e), i


def test_softmax_xent_without_rows(cuda):
    from fast_b200 import ops
    h, w = torch.randn(0, 24, device=cuda), torch.randn(50, 24, device=cuda)
    t = torch.empty(0, dtype=torch.int64, device=cuda)
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    dh, dw = ops.softmax_xent_bwd(h, w, t, lse, loss)
    assert loss.shape == (0,) and dh.shape == (0, 24) and bool((dw == 0).all())


# ---- use -----------------------------------------------------------------------------------------------------------
def test_operators_run_on_the_current_stream(cuda):
    """Inputs made on a side stream, operators called there: every result
    equals the default stream's."""
    from fast_b200 import ops
    torch.manual_seed(0)
    base = [torch.randn(s, device=cuda) for s in ((200, 64), (128, 64), (128, 64), (64, 128), (300, 64))]
    t = torch.randint(0, 300, (200,), device=cuda)

    def run(x, wg, wu, wd, w):
        y, m, r = ops.layer_norm_fwd(x, torch.ones(64, device=cuda))
        z = ops.gated_ffn_fwd(y, wg, wu, wd)
        loss, lse = ops.softmax_xent_fwd(z, w, t)
        return [y, z, loss, *ops.softmax_xent_bwd(z, w, t, lse, torch.ones_like(loss))]
    for dt in TYPES:
        want = run(*[b.to(dt) for b in base])
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            torch.cuda._sleep(10_000_000)
            got = run(*[(b * 1).to(dt) for b in base])
        st.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))
