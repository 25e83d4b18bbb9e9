"""GPU: what only large calls of the node-ranking head's operators reach -- several pieces of the table, several slices
of the rows, more tiles than there are SM pairs -- and products of fp32 operands held to the accuracy of all their
planes."""
import ctypes
import math

import pytest
import torch

from test_head_gpu import _c, _check, _gen, _mat, test_gated_ffn as gated_ffn, test_softmax_xent as softmax_xent

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TYPES = [F32, BF]


# ---- pieces, slices, many tiles --------------------------------------------------------------------------------------
# G's pieces hold 512 MB: 10,880 nodes of 8,192 fp32 rows, 32,768 of as many bf16 ones; the last piece is ragged
@pytest.mark.parametrize("n,d,v,pad,dtype", [(8192, 32, 23001, 0, F32), (8192, 33, 12000, 1, F32), (8192, 32, 40001, 0, BF),
                                             (8190, 33, 40000, 1, BF)])
def test_softmax_xent_over_several_pieces_of_the_table(cuda, n, d, v, pad, dtype):
    softmax_xent(cuda, n, d, v, pad, dtype)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("v,dtype", [(12000, F32), (40000, BF)])
def test_softmax_xent_piece_by_piece_without_one_of_the_gradients(cuda, v, dtype):
    """The C entry takes NULL for dh or dw.  (What a launch holds decides how its sums are split, so the gradient left
    need not repeat the other call's bit for bit.)"""
    from fast_b200 import ops
    from fast_b200.capi import SoftmaxXent, call, lib, stream_ptr
    n, d = 8192, 32
    g = _gen(cuda, n, v)
    h, w = _mat(cuda, g, n, d, dtype), _mat(cuda, g, v, d, dtype)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    dl = torch.rand(n, device=cuda, generator=g)
    _, lse = ops.softmax_xent_fwd(h, w, t)
    H, W = h.double(), w.double()
    L = H @ W.t()
    Z = torch.logsumexp(L, 1, keepdim=True)
    e = 2 * _c(d) * (H.abs() @ W.abs().t()).max(1, keepdim=True).values + \
        2.0 ** -19 * (1 + Z.abs() + L.abs().max(1, keepdim=True).values)
    P = torch.exp(L - Z)
    G = P.clone()
    G.scatter_add_(1, t[:, None], torch.full_like(t[:, None], -1, dtype=torch.float64))
    scale = dl.double()[:, None]
    eG = scale * (P * e + 2.0 ** -22 * G.abs())
    G = G * scale
    eG = eG + (2.0 ** -8 if dtype == BF else 0.0) * (G.abs() + eG)
    for name, want, bound in (("dh", G @ W, eG @ W.abs() + _c(v) * ((G.abs() + eG) @ W.abs())),
                                 ("dw", G.t() @ H, eG.t() @ H.abs() + _c(n) * ((G.abs() + eG).t() @ H.abs()))):
        out = torch.empty(want.shape, device=cuda, dtype=dtype)
        a = SoftmaxXent()
        a.type = a.grad_type = int(dtype == BF)
        a.n, a.D, a.V, a.ldh, a.ldw, a.lddh, a.lddw = n, d, v, d, d, d, d
        a.h, a.w, a.target, a.lse, a.dloss = (p.data_ptr() for p in (h, w, t, lse, dl))
        setattr(a, name, out.data_ptr())
        nb = lib.fb_softmax_xent_ws_bytes(a, 1)
        ws = torch.empty(nb, dtype=torch.uint8, device=cuda)
        call("fb_softmax_xent_bwd", ctypes.byref(a), ws.data_ptr(), nb, stream_ptr())
        _check(name, out, want, bound, dtype)


# partial maxima and sums of one launch hold 256 MB: 15,104 fp32 or 30,464 bf16 rows against 140,000 nodes
@pytest.mark.parametrize("n,dtype", [(15400, F32), (30700, BF)])
def test_softmax_xent_forward_in_slices_of_the_rows(cuda, n, dtype):
    from fast_b200 import ops
    d, v = 20, 140000
    g = _gen(cuda, n, d, v)
    h, w = _mat(cuda, g, n, d, dtype, 1.0, 4), _mat(cuda, g, v, d, dtype, 3 * d ** -0.5, 4)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    t[::9] = -1
    loss, lse = ops.softmax_xent_fwd(h, w, t)
    W = w.double()
    for r in range(0, n, 1024):
        H, T = h[r:r + 1024].double(), t[r:r + 1024]
        L = H @ W.t()
        Z = torch.logsumexp(L, 1)
        keep = (T >= 0).double()
        el = (_c(d) * (H.abs() @ W.abs().t())).max(1).values
        fn = 2.0 ** -20 * (1 + Z.abs() + L.abs().max(1).values)
        _check("lse", lse[r:r + 1024], Z, el + fn, F32)
        _check("loss", loss[r:r + 1024], (Z - L.gather(1, T.clamp(min=0)[:, None])[:, 0]) * keep, (2 * el + fn) * keep, F32)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
def test_softmax_xent_many_tiles_of_long_sums(cuda, dtype):
    softmax_xent(cuda, 2600, 1100, 2300, 0, dtype)              # 99 tiles of more than 16 stages (bf16)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_ffn_more_tiles_than_sm_pairs(cuda, act, dtype):
    gated_ffn(cuda, 4200, 72, 1300, 0, dtype, act)              # 17 x 11 tiles: three for some pairs


# ---- the planes of fp32 operands -------------------------------------------------------------------------------------
# x = x0 + x1 + x2 of 8 significant bits each; the products 00, 01, 10, 02, 11, 20 are summed in slabs of 64 k.
def _with_third_planes(cuda, g, rows, pairs):
    """u in [1, 2) whose planes have fixed places (bits 2^-8 and 2^-16 .. 2^-23 set), as (u, -(u0 + u1)) side by side:
    leading planes cancel, and what is left of a pair is u2 = 2^-15 - 2^-23."""
    bits = torch.randint(0, 1 << 23, (rows, pairs), device=cuda, generator=g, dtype=torch.int32) | 0x3F800000 | 0x80FF
    u = bits.view(torch.float32)
    lead = (bits & ~0xFF).view(torch.float32)
    return torch.stack([u, -lead], 2).reshape(rows, 2 * pairs), 2.0 ** -15 - 2.0 ** -23


# Against v in [1, 2) the exact sum of m pairs is u2 sum(v).  Left out: u2 v1, below 2^-7 of it.  An MMA takes 8 pairs
# whose products, at most 4, cancel in it: 16 truncations of 2^-24 of 4 against 8 u2, below 2^-6 of it.
_TOL = 2.0 ** -5


@pytest.mark.parametrize("n,pairs", [(9, 8), (300, 100), (20, 260), (300, 300)])       # 260: stored logits, split sums
@pytest.mark.parametrize("side", [0, 1])
def test_third_planes_reach_the_logits(cuda, n, pairs, side):
    from fast_b200 import ops
    g = _gen(cuda, n, pairs, side)
    v = 1 + torch.rand(n if side else 1, pairs, device=cuda, generator=g)
    v = v.repeat_interleave(2, 1).contiguous()
    x, u2 = _with_third_planes(cuda, g, 1 if side else n, pairs)
    h, w = (v, x) if side else (x, v)
    want = (h.double() @ w.double().t())[:, 0]
    assert bool(((want / (u2 * v.double().sum(1) / 2) - 1).abs() < 1e-6).all())
    t = torch.zeros(n, dtype=torch.int64, device=cuda)
    lse = ops.softmax_xent_fwd(h, w, t)[1].double()             # of one node: its logit
    assert float((lse / want - 1).abs().max()) <= _TOL
    # and the backward's logits: two nodes, the other one's logit 0; dh = G0 w0 with G0 = p0 - 1
    s = 2.0 ** 15 / pairs                                       # logits of about 1.5
    w2 = torch.cat([w * s, torch.zeros_like(w)])
    logit = want * s
    _, lse = ops.softmax_xent_fwd(h, w2, t)
    dh, _ = ops.softmax_xent_bwd(h, w2, t, lse, torch.ones(n, device=cuda))
    G = dh.double() / w2[:1].double()
    want = torch.sigmoid(logit) - 1
    # d p0 = p0 (1 - p0) d l0, once from the logits and once from lse
    assert float((G - want[:, None]).abs().max()) <= 0.25 * 2 * _TOL * float(logit.max())
    assert float((G + 0.5).abs().min()) > 0.25 * 2 * _TOL * float(logit.max())         # logits of 0 would not pass


@pytest.mark.parametrize("n,d,f", [(9, 72, 136), (300, 264, 520), (1000, 520, 72), (40, 1100, 200)])
def test_products_of_the_gated_block_keep_all_planes(cuda, n, d, f):
    """A block whose gate is 1 throughout is a chain of plain products.  In the 2-norm a product is off by 2^-19.5 of
    itself at most: 2^-23 for the plane products left out (below 2^-21 and 2^-24.5 on average), six truncations of a
    slab's sum at 2^-23 each.  Without one of the six plane products it would be off by 2^-16.5 and more."""
    from fast_b200 import ops
    g = _gen(cuda, n, d, f)
    x, wu, wd = _mat(cuda, g, n, d, F32), _mat(cuda, g, f, d, F32, d ** -0.5), _mat(cuda, g, d, f, F32, f ** -0.5)
    dy = _mat(cuda, g, n, d, F32)
    x[:, 0] = 1
    wg = torch.zeros(f, d, device=cuda)
    wg[:, 0] = 1
    X, WU, WD, DY = (p.double() for p in (x, wu, wd, dy))
    U, DH = X @ WU.t(), DY @ WD
    out = (ops.gated_ffn_fwd(x, wg, wu, wd, act="relu"), *ops.gated_ffn_bwd(dy, x, wg, wu, wd, act="relu"))
    dx = DH @ WU
    dx[:, 0] += (DH * U).sum(1)
    for name, got, want, chain in (("y", out[0], U @ WD.t(), 2), ("dx", out[1], dx, 3),
                                   ("dw_gate", out[2], (DH * U).t() @ X, 3), ("dw_up", out[3], DH.t() @ X, 2),
                                   ("dw_down", out[4], DY.t() @ U, 2)):
        off = float((got.double() - want).norm() / want.norm())
        assert off <= chain * 2.0 ** -19.5, (name, math.log2(off))


# ---- long sums in front of a discontinuity ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,d,f", [(300, 1100, 700), (1500, 4096, 2000), (2000, 2306, 3000)])
def test_relu_gradients_of_wide_bf16_rows(cuda, n, d, f):
    """relu'(g) turns with the sign of g, so an error of g next to zero is one of the gradients: the products of g must
    be as good as fp32 sums.  A bf16 rounding is off by 2^-8 / sqrt(3) in the 2-norm at most, and the gradients carry two;
    fp32 sums turn few enough signs to add nothing that shows."""
    from fast_b200 import ops
    g = _gen(cuda, n, d, f)
    x, dy = _mat(cuda, g, n, d, BF), _mat(cuda, g, n, d, BF)
    wg, wu, wd = _mat(cuda, g, f, d, BF, d ** -0.5), _mat(cuda, g, f, d, BF, d ** -0.5), _mat(cuda, g, d, f, BF, f ** -0.5)
    X, DY, WG, WU, WD = (p.double() for p in (x, dy, wg, wu, wd))
    G, U, DH = X @ WG.t(), X @ WU.t(), DY @ WD
    A = G.clamp(min=0)
    DG, DU, H = DH * U * (G > 0), DH * A, A * U
    out = ops.gated_ffn_bwd(dy, x, wg, wu, wd, act="relu")
    for name, got, want in (("dx", out[0], DG @ WG + DU @ WU), ("dw_gate", out[1], DG.t() @ X), ("dw_up", out[2], DU.t() @ X),
                            ("dw_down", out[3], DY.t() @ H)):
        off = float((got.double() - want).norm() / want.norm())
        assert off <= 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5, (name, off)


@pytest.mark.parametrize("n,d,f", [(4, 2048, 1000), (300, 700, 900), (300, 2048, 500), (260, 4096, 3000)])
def test_relu_turns_where_an_fp32_sum_of_bf16_rows_would(cuda, n, d, f):
    """g = 1024 + (small terms) - 1024, in this order along the row: truncating every 16 terms beside the 1024 loses
    2^-14 each time, a hundred times and more; summing 256 terms at a time and these sums in fp32 is off by less than
    16 * 2^-14 + 2^-13 < 2^-9.  u = dh = 1, so dg = relu'(g), which columns of the unit matrix show in dw_gate."""
    from fast_b200 import ops
    g = _gen(cuda, n, d, f)
    x, wg = torch.zeros(n, d, device=cuda, dtype=BF), torch.zeros(f, d, device=cuda, dtype=BF)
    wu, wd, dy = torch.zeros_like(wg), torch.zeros(d, f, device=cuda, dtype=BF), torch.zeros_like(x)
    x[:, 0], wu[:, 0], wd[0], dy[:, 0] = 1, 1, 1, 1
    x[:, 1], wg[:, 1], x[:, d - 1], wg[:, d - 1] = 32, 32, 32, -32
    small = slice(256, d - 1 - n) if d > 1000 else slice(64, d - 1 - n)
    x[:, small] = _mat(cuda, g, n, small.stop - small.start, BF)
    wg[:, small] = _mat(cuda, g, f, small.stop - small.start, BF, 0.02 * (small.stop - small.start) ** -0.5)
    unit = slice(small.stop, small.stop + n)
    x[:, unit] = torch.eye(n, device=cuda, dtype=BF)
    dg = ops.gated_ffn_bwd(dy, x, wg, wu, wd, act="relu")[1][:, unit].t()
    G = x.double() @ wg.double().t()
    sure = G.abs() > 2.0 ** -9
    assert 0.5 < float(sure.double().mean()) < 1
    assert bool((dg[sure].double() == (G[sure] > 0).double()).all())


# ---- few rows in bf16 ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d,v,pad", [(2, 100, 600, 0), (3, 257, 895, 1), (7, 1670, 2207, 0), (17, 43, 58432, 3), (31, 64, 3000, 0),
                                       (70, 378, 3259, 0), (127, 100, 1001, 4), (128, 1127, 1664, 0)])
def test_few_bf16_rows_give_gradients_of_one_rounding(cuda, n, d, v, pad):
    """With few rows the gradients hang on few elements of G (the targets'), whose rounding would not average out.  dh and
    dw are then off by their own rounding alone: in the 2-norm 2^-8 / sqrt(3) at most, and 2^-12 for the rest."""
    from fast_b200 import ops
    for seed in range(4):
        g = torch.Generator(device=cuda).manual_seed(1000 * seed + n)
        h, w = _mat(cuda, g, n, d, BF, 1.0, pad), _mat(cuda, g, v, d, BF, 2 * d ** -0.5, pad)
        t = torch.randint(0, v, (n,), device=cuda, generator=g)
        if n > 2:
            t[1] = -1
            h[1] = math.nan
        dl = torch.rand(n, device=cuda, generator=g) + 0.5
        _, lse = ops.softmax_xent_fwd(h, w, t)
        dh, dw = ops.softmax_xent_bwd(h, w, t, lse, dl)
        H, W, keep = h.double().nan_to_num(0), w.double(), (t >= 0)
        G = torch.softmax(H @ W.t(), 1)
        G.scatter_add_(1, t.clamp(min=0)[:, None], torch.full((n, 1), -1.0, device=cuda, dtype=torch.float64))
        G = G * (dl.double() * keep)[:, None]
        for name, got, want in (("dh", dh, G @ W), ("dw", dw, G.t() @ H)):
            off = float((got.double() - want).norm() / want.norm())
            assert off <= 2.0 ** -8 / 3 ** 0.5 + 2.0 ** -12, (name, seed, off)
        buf = torch.zeros(v, d, device=cuda)
        dh2, _ = ops.softmax_xent_bwd(h, w, t, lse, dl, dw=buf)
        assert torch.equal(dh, dh2)
        off = float((buf.double() - G.t() @ H).norm() / (G.t() @ H).norm())
        assert off <= 2.0 ** -12, (seed, off)                   # fp32 sums of h and G's two parts


def test_few_bf16_rows_over_several_pieces_of_the_table(cuda):
    softmax_xent(cuda, 128, 16, 1_200_000, 0, BF)               # 1,048,576 nodes a piece
    torch.cuda.empty_cache()
