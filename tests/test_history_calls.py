"""CPU: what the event-history modules and entries do with arguments at the edge of
what they document."""
import ctypes

import torch


def test_last_row_of_an_empty_history_is_zero_whatever_its_neighbours_hold():
    from fast_b200.history import HistoryEncoder
    rows = torch.tensor([[1.0, 2.0], [3.0, 4.0], [float("inf"), float("nan")], [5.0, 6.0]], requires_grad=True)
    starts = torch.tensor([0, 0, 3, 3, 4, 4])
    out = HistoryEncoder.last(rows, starts)
    assert torch.equal(out[[0, 2, 4]], torch.zeros(3, 2)) and torch.equal(out[3], rows[3])
    assert bool(torch.isinf(out[1, 0])) and bool(torch.isnan(out[1, 1]))
    # an empty history hands no gradient to the row in front of it
    grad, = torch.autograd.grad(out[[0, 2, 4]].sum() + out[3].sum(), rows)
    assert torch.equal(grad, torch.tensor([[0.0, 0.0], [0.0, 0.0], [0.0, 0.0], [1.0, 1.0]]))


def test_last_rows_stay_inside_the_rows():
    """starts beyond the rows are clamped to them, as the operators do, and not left to an index out of range."""
    from fast_b200.history import HistoryEncoder
    rows = torch.arange(8.0).view(4, 2)
    assert torch.equal(HistoryEncoder.last(rows, torch.tensor([0, 2, 9, 9, 12])), torch.stack([rows[1], rows[3], *torch.zeros(2, 2)]))
    assert torch.equal(HistoryEncoder.last(rows, torch.tensor([-3, -1, 4])), torch.stack([torch.zeros(2), rows[3]]))


def _refuses(entry, struct, ok, bad, *rest):
    for name, values in bad.items():
        for v in values:
            a = struct()
            for k, w in dict(ok, **{name: v}).items():
                setattr(a, k, w)
            assert entry(ctypes.byref(a), *rest) == 1, (name, v)


def test_entries_refuse_operands_off_their_elements():
    """FB_ERR_ARG from every C entry for every pointer that is not aligned to what it points to, and for negative pitches: what a
    kernel would fault on."""
    from fast_b200.capi import SelectiveScan, SelectiveScanEvent, ShortConv, lib
    buf = ctypes.create_string_buffer(80)
    p = (ctypes.addressof(buf) + 15) & ~15
    for type_, odd in ((0, (p + 1, p + 2)), (1, (p + 1,))):                  # rows of fp32, of bf16
        conv = dict(type=type_, act=0, starts_type=1, D=8, K=4, rows=2, seqs=1, starts=p, x=p, ldx=8, w=p, bias=p, init=p, final=p, y=p,
                    ldy=8, dy=p, lddy=8, dfinal=p, dx=p, lddx=8, dw=p, dbias=p, dinit=p)
        fwd, bwd = lib.fb_short_conv_fwd, lib.fb_short_conv_bwd
        _refuses(fwd, ShortConv, conv, dict.fromkeys(("x", "init", "final", "y"), odd), p, 64, None)
        _refuses(bwd, ShortConv, conv, dict.fromkeys(("x", "init", "dy", "dfinal", "dx", "dinit"), odd), p, 64, None)
        for entry in (fwd, bwd):
            _refuses(entry, ShortConv, conv, dict(w=(p + 2,), bias=(p + 2,), starts=(p + 4,)), p, 64, None)
            _refuses(entry, ShortConv, dict(conv, starts_type=0), dict(starts=(p + 2,)), p, 64, None)
        _refuses(bwd, ShortConv, conv, dict(dw=(p + 2,), dbias=(p + 1,)), p, 64, None)

        scan = dict(type=type_, starts_type=1, D=8, N=4, G=2, rows=2, seqs=1, starts=p, u=p, ldu=8, delta=p, ld_delta=8, B=p, ldb=8,
                    ldb_group=4, C=p, ldc=8, ldc_group=4, z=p, ldz=8, A=p, skip=p, delta_bias=p, init=p, keep=p, final=p, y=p, ldy=8,
                    dy=p, lddy=8, dfinal=p, du=p, ddelta=p, dz=p, dB=p, dC=p, dA=p, dD=p, ddelta_bias=p, dinit=p)
        fwd, bwd, four = lib.fb_selective_scan_fwd, lib.fb_selective_scan_bwd, (p + 2, p + 1)
        _refuses(fwd, SelectiveScan, scan, dict.fromkeys(("u", "delta", "B", "C", "z", "y"), odd), p, 64, None)
        _refuses(bwd, SelectiveScan, scan, dict.fromkeys(("u", "delta", "B", "C", "z", "dy", "du", "ddelta", "dz", "dB", "dC"), odd), p, 64, None)
        for entry in (fwd, bwd):
            _refuses(entry, SelectiveScan, scan, dict.fromkeys(("A", "skip", "delta_bias", "init", "keep"), four), p, 64, None)
            _refuses(entry, SelectiveScan, scan, dict(starts=(p + 4,), ldb=(-8,), ldb_group=(-4,), ldc=(-8,), ldc_group=(-4,)), p, 64, None)
        _refuses(fwd, SelectiveScan, scan, dict(final=four), p, 64, None)
        _refuses(bwd, SelectiveScan, scan, dict.fromkeys(("dfinal", "dA", "dD", "ddelta_bias", "dinit"), four), p, 64, None)

        event = dict(type=type_, D=8, N=4, G=2, n=2, states=4, index=p, u=p, ldu=8, delta=p, ld_delta=8, B=p, ldb=8, ldb_group=4, C=p, ldc=8,
                     ldc_group=4, z=p, ldz=8, A=p, skip=p, delta_bias=p, state=p, y=p, ldy=8)
        bad = dict(dict.fromkeys(("u", "delta", "B", "C", "z", "y"), odd), **dict.fromkeys(("A", "skip", "delta_bias", "state"), four))
        bad.update(index=(p + 4,), ldb=(-8,), ldb_group=(-4,), ldc=(-8,), ldc_group=(-4,))
        _refuses(lib.fb_selective_scan_step, SelectiveScanEvent, event, bad, p, 64, None)

        step = dict(type=type_, act=0, x=p, ldx=8, w=p, bias=p, state=p, states=4, index=p, y=p, ldy=8, n=2, D=8, K=4, ws=p, nb=64, stream=None)
        for name, values in dict(x=odd, y=odd, state=odd, w=four, bias=four, index=(p + 4,)).items():
            for v in values:
                assert lib.fb_short_conv_step(*dict(step, **{name: v}).values()) == 1, (name, v)
        drop = dict(type=type_, x=p, ldx=8, res=p, ldr=8, y=p, ldy=8, rows=2, D=8, p=0.5, seed=1, offset=0, offset_dev=p, stream=None)
        for name, values in dict(x=odd, res=odd, y=odd, offset_dev=(p + 4,)).items():
            for v in values:
                assert lib.fb_dropout(*dict(drop, **{name: v}).values()) == 1, (name, v)


def test_dropout_refuses_widths_its_columns_do_not_count():
    """FB_ERR_UNSUPPORTED above the width the other event-history entries take, too."""
    from fast_b200.capi import lib
    buf = ctypes.create_string_buffer(80)
    p = (ctypes.addressof(buf) + 15) & ~15
    for width in ((1 << 20) + 1, (1 << 31) - 1):
        assert lib.fb_dropout(1, p, width, None, 0, p, width, 2, width, 0.5, 1, 0, None, None) == 3
