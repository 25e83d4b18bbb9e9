"""CPU: refusals of the event-history operators before any launch (the wrappers
raise ValueError, the C entries return FB_ERR_ARG (1) or FB_ERR_UNSUPPORTED (3)),
and the restatements the GPU tests compare with (history_math.py)."""
import ctypes

import history_math as hm
import pytest
import torch


def test_wrappers_refuse_bad_operands():
    from fast_b200 import ops
    x, w, v = torch.zeros(4, 8), torch.zeros(8, 4), torch.zeros(8)
    A, B, state = torch.zeros(8, 16), torch.zeros(4, 16), torch.zeros(4, 8, 16)
    for bad in (x.half(), x.double(), x):                       # type; not on a GPU
        with pytest.raises(ValueError):
            ops.short_conv_fwd(bad, w)
        with pytest.raises(ValueError):
            ops.short_conv_bwd(bad, bad, w)
        with pytest.raises(ValueError):
            ops.short_conv_step(bad, torch.zeros(4, 3, 8), w)
        with pytest.raises(ValueError):
            ops.selective_scan_fwd(bad, bad, A, B, B)
        with pytest.raises(ValueError):
            ops.selective_scan_bwd(bad, bad, bad, A, B, B, torch.zeros(1, 8, 16))
        with pytest.raises(ValueError):
            ops.selective_scan_step(bad, bad, A, B, B, state)
        with pytest.raises(ValueError):
            ops.dropout_fwd(bad, 0.5, 1)
    for act in ("gelu", 0, True, ["silu"]):
        with pytest.raises(ValueError):
            ops.short_conv_fwd(x, w, v, act=act)
    for seed, offset in ((-1, 0), (1 << 64, 0), (1.0, 0), (True, 0), (0, -1), (0, 1 << 64)):
        with pytest.raises(ValueError):
            ops.dropout_fwd(x, 0.5, seed, offset)


def test_blocks_refuse_bad_sizes():
    from fast_b200.history import StateSpaceBlock
    for bad in (dict(states=0), dict(states=65), dict(taps=9), dict(dropout=1.0), dict(dropout=-0.1)):
        with pytest.raises(ValueError):
            StateSpaceBlock(8, **bad)


def _addr():
    buf = ctypes.create_string_buffer(64)
    return buf, ctypes.addressof(buf)


def _set(s, **kw):
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_short_conv_entry_refuses():
    from fast_b200.capi import ShortConv, lib
    buf, p = _addr()

    def args(**kw):
        return _set(ShortConv(type=0, act=0, starts_type=1, D=8, K=4, rows=2, seqs=1, x=p, ldx=8, w=p, y=p, ldy=8, dy=p, lddy=8,
                              dx=p, lddx=8, dw=p, dbias=p), **kw)
    both = ((1, dict(type=2)), (1, dict(act=1)), (1, dict(D=0)), (1, dict(K=0)), (1, dict(rows=-1)), (1, dict(x=None)),
            (1, dict(w=None)), (1, dict(ldx=7)), (1, dict(seqs=2)), (1, dict(starts=p, starts_type=2)), (1, dict(x=p + 1)),
            (3, dict(K=9)), (3, dict(D=1 << 21, ldx=1 << 21)), (3, dict(seqs=1 << 31, starts=p)), (3, dict(ldx=1 << 29)))
    for rc, bad in both + ((1, dict(y=None)), (1, dict(ldy=7)), (1, dict(y=p + 2))):
        a = args(**bad)
        assert lib.fb_short_conv_fwd(ctypes.byref(a), p, 64, None) == rc, bad
    # {rows=10000}: no workspace, one that is too small, one that is not aligned
    for rc, bad, ws, nb in tuple((rc, bad, p, 64) for rc, bad in both) + (
            (1, dict(dy=None), p, 64), (1, dict(dx=None), p, 64), (1, dict(dw=None), p, 64), (1, dict(lddx=3), p, 64),
            (1, dict(dinit=p), p, 64), (1, dict(rows=10000), None, 0), (1, dict(rows=10000), p, 64), (1, dict(rows=10000), p + 4, 1 << 30)):
        a = args(**bad)
        assert lib.fb_short_conv_bwd(ctypes.byref(a), ws, nb, None) == rc, bad
    assert lib.fb_short_conv_fwd(None, None, 0, None) == 1
    a = args(rows=0)
    assert lib.fb_short_conv_fwd(ctypes.byref(a), None, 0, None) == 0
    assert lib.fb_short_conv_ws_bytes(ctypes.byref(args(rows=10000)), 1) >= 5 * 8 * 4
    assert lib.fb_short_conv_ws_bytes(ctypes.byref(args(rows=10000)), 0) == 0


def test_selective_scan_entry_refuses():
    from fast_b200.capi import SelectiveScan, lib
    buf, p = _addr()

    def args(**kw):
        return _set(SelectiveScan(type=0, starts_type=1, D=8, N=16, G=1, rows=2, seqs=1, u=p, ldu=8, delta=p, ld_delta=8, B=p, ldb=16,
                                  C=p, ldc=16, A=p, y=p, ldy=8, keep=p, dy=p, lddy=8, du=p, ddelta=p, dB=p, dC=p, dA=p, dD=p,
                                  ddelta_bias=p), **kw)
    both = ((1, dict(type=2)), (1, dict(D=0)), (1, dict(N=0)), (1, dict(G=3)), (1, dict(G=0)), (1, dict(rows=-1)), (1, dict(u=None)),
            (1, dict(A=None)), (1, dict(C=None)), (1, dict(ldu=7)), (1, dict(ld_delta=7)), (1, dict(z=p, ldz=7)), (1, dict(seqs=0)),
            (1, dict(starts=p, starts_type=5)), (3, dict(N=65)), (3, dict(D=1 << 21)), (3, dict(seqs=1 << 31, starts=p)))
    for rc, bad in both + ((1, dict(y=None)), (1, dict(ldy=7))):
        a = args(**bad)
        assert lib.fb_selective_scan_fwd(ctypes.byref(a), p, 64, None) == rc, bad
    for rc, bad in both + ((1, dict(dy=None)), (1, dict(keep=None)), (1, dict(du=None)), (1, dict(z=p, ldz=8)), (1, dict(dA=None)),
                           (1, dict(lddy=1))):
        a = args(**bad)
        assert lib.fb_selective_scan_bwd(ctypes.byref(a), p, 64, None) == rc, bad
    for entry in (lib.fb_selective_scan_fwd, lib.fb_selective_scan_bwd):
        for ws, nb in ((None, 0), (p, 64), (p + 4, 1 << 40)):    # many rows need a workspace
            a = args(rows=100000)
            assert entry(ctypes.byref(a), ws, nb, None) == 1
        assert entry(None, None, 0, None) == 1
    a = args(rows=0)
    assert lib.fb_selective_scan_fwd(ctypes.byref(a), None, 0, None) == 0
    assert lib.fb_selective_scan_ws_bytes(ctypes.byref(args()), 0) == 0
    assert lib.fb_selective_scan_ws_bytes(ctypes.byref(args(N=65)), 1) == 0


def test_single_event_entries_refuse():
    from fast_b200.capi import SelectiveScanEvent, lib
    buf, p = _addr()
    ok = dict(type=0, act=0, x=p, ldx=8, w=p, bias=None, state=p, states=4, index=p, y=p, ldy=8, n=2, D=8, K=4, ws=p, nb=64, stream=None)
    for rc, bad in ((1, dict(type=3)), (1, dict(act=2)), (1, dict(n=-1)), (1, dict(states=-1)), (1, dict(D=0)), (1, dict(K=0)),
                    (1, dict(x=None)), (1, dict(state=None)), (1, dict(w=None)), (1, dict(ldx=7)), (1, dict(ldy=1)), (1, dict(x=p + 2)),
                    (1, dict(index=None, n=5)), (1, dict(n=100)), (1, dict(n=100, ws=None)), (3, dict(K=9)), (3, dict(n=65537, states=1 << 20)),
                    (3, dict(states=1 << 31))):
        assert lib.fb_short_conv_step(*dict(ok, **bad).values()) == rc, bad
    assert lib.fb_short_conv_step(*dict(ok, n=0).values()) == 0

    def args(**kw):
        return _set(SelectiveScanEvent(type=0, D=8, N=16, G=1, n=2, states=4, index=p, u=p, ldu=8, delta=p, ld_delta=8, B=p, ldb=16, C=p,
                                       ldc=16, A=p, state=p, y=p, ldy=8), **kw)
    for rc, bad in ((1, dict(type=3)), (1, dict(n=-1)), (1, dict(N=0)), (1, dict(G=3)), (1, dict(u=None)), (1, dict(state=None)),
                    (1, dict(A=None)), (1, dict(ldu=7)), (1, dict(z=p)), (1, dict(index=None, n=5)), (1, dict(n=100)), (3, dict(N=65)),
                    (3, dict(n=65537)), (3, dict(states=1 << 31))):
        a = args(**bad)
        assert lib.fb_selective_scan_step(ctypes.byref(a), p, 64, None) == rc, bad
    assert lib.fb_selective_scan_step(None, None, 0, None) == 1
    assert lib.fb_event_step_ws_bytes(1) == 0 and lib.fb_event_step_ws_bytes(4000) == 32000


def test_dropout_entry_refuses():
    from fast_b200.capi import lib
    buf, p = _addr()
    ok = dict(type=1, x=p, ldx=8, res=None, ldr=0, y=p, ldy=8, rows=2, D=8, p=0.5, seed=1, offset=0, offset_dev=None, stream=None)
    for rc, bad in ((1, dict(type=2)), (1, dict(p=1.0)), (1, dict(p=-0.1)), (1, dict(p=float("nan"))), (1, dict(rows=-1)), (1, dict(D=0)),
                    (1, dict(x=None)), (1, dict(y=None)), (1, dict(ldx=7)), (1, dict(res=p, ldr=7)), (1, dict(x=p + 1)),
                    (3, dict(rows=1 << 32))):
        assert lib.fb_dropout(*dict(ok, **bad).values()) == rc, bad
    assert lib.fb_dropout(*dict(ok, rows=0).values()) == 0


def test_philox_restatement_gives_the_published_words():
    """Known answers of Philox4x32-10 published with the generator."""
    assert [hex(v) for v in hm.philox(1, 4, 0, 0)[0].tolist()] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def test_convolution_restatement_is_torchs():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((12, 5), (5, 4), (5,)))
    y, final = hm.short_conv(x, w, b, None, None, "silu")
    xe = torch.cat([torch.zeros(3, 5, dtype=torch.float64), x]).t().unsqueeze(0)
    want = torch.nn.functional.silu(torch.nn.functional.conv1d(xe, w.unsqueeze(1), b, groups=5))[0].t()
    assert torch.allclose(y, want, rtol=1e-13, atol=1e-13) and torch.equal(final[0], x[-3:])


def test_scan_restatement_is_the_weighted_sum_of_its_inputs():
    """h[t] = sum_s exp(A (dt[s + 1] + .. + dt[t])) dt[s] u[s] B[s], written out."""
    g = torch.Generator().manual_seed(1)
    n, d, s = 7, 3, 4
    u, delta, z = (torch.randn(n, d, generator=g, dtype=torch.float64) for _ in range(3))
    A = -torch.rand(d, s, generator=g, dtype=torch.float64)
    B, C = (torch.randn(n, 1, s, generator=g, dtype=torch.float64) for _ in range(2))
    y, final = hm.selective_scan(u, delta, A, B, C, None, None, None, None, None, True)
    dt = torch.nn.functional.softplus(delta)
    total = dt.cumsum(0)
    for t in range(n):
        h = sum(torch.exp((total[t] - total[k]).unsqueeze(1) * A) * (dt[k] * u[k]).unsqueeze(1) * B[k] for k in range(t + 1))
        assert torch.allclose(y[t], (h * C[t]).sum(1), rtol=1e-12, atol=1e-12)
    assert torch.allclose(final[0], h, rtol=1e-12, atol=1e-12)
