"""CPU: refusals of the node-ranking head's operators, before any launch: the
wrappers raise ValueError, the C entries return FB_ERR_ARG (1) or
FB_ERR_UNSUPPORTED (3)."""
import ctypes

import pytest
import torch


def test_wrappers_refuse_bad_operands():
    from fast_b200 import ops
    x, v = torch.zeros(4, 8), torch.zeros(8)
    t = torch.zeros(4, dtype=torch.int64)
    for bad in (x.half(), x.double(), x):                       # type; not on a GPU
        with pytest.raises(ValueError):
            ops.layer_norm_fwd(bad, v)
        with pytest.raises(ValueError):
            ops.gated_ffn_fwd(bad, x, x, x)
        with pytest.raises(ValueError):
            ops.softmax_xent_fwd(bad, x, t)
    with pytest.raises(ValueError):
        ops.gated_ffn_fwd(x, x, x, x, act="tanh")


def _addr():
    buf = ctypes.create_string_buffer(64)
    return buf, ctypes.addressof(buf)


def test_layer_norm_entry_refuses():
    from fast_b200.capi import lib
    buf, p = _addr()
    ok = dict(type=0, x=p, ldx=8, res=None, ldr=0, gamma=p, beta=p, param_type=0, eps=1e-5, sum=None, lds=0, y=p, ldy=8,
              mean=p, rstd=p, n=2, D=8, stream=None)
    for rc, bad in ((1, dict(type=2)), (1, dict(type=0, param_type=1)), (1, dict(D=0)), (1, dict(n=-1)),
                    (1, dict(x=None)), (1, dict(gamma=None)), (1, dict(ldx=7)), (1, dict(ldy=4)), (1, dict(res=p, ldr=8)),
                    (1, dict(eps=-1.0)), (1, dict(eps=float("nan"))),
                    (3, dict(D=16385, ldx=16385, ldy=16385))):
        assert lib.fb_layer_norm_fwd(*dict(ok, **bad).values()) == rc, bad
    assert lib.fb_layer_norm_fwd(*dict(ok, n=0).values()) == 0
    okb = dict(type=1, dy=p, lddy=8, x=p, ldx=8, gamma=p, param_type=0, mean=p, rstd=p, ds=None, ldds=0, dx=p, lddx=8,
               dgamma=p, dbeta=p, accumulate=0, n=2, D=8, ws=p, ws_bytes=64, stream=None)
    for rc, bad in ((1, dict()), (1, dict(ws=None)), (1, dict(dx=None)), (1, dict(mean=None)), (1, dict(lddy=3)),
                    (3, dict(accumulate=1, param_type=1)), (3, dict(D=20000, lddy=20000, ldx=20000, lddx=20000))):
        assert lib.fb_layer_norm_bwd(*dict(okb, **bad).values()) == rc, bad       # {}: the workspace is too small


def test_gated_ffn_entry_refuses():
    from fast_b200.capi import GatedFfn, lib
    buf, p = _addr()

    def args(**kw):
        a = GatedFfn(0, 0, 0, 0, 2, 8, 16, p, 8, p, 8, p, 8, p, 16, p, 8, p, 8, p, 8, p, 8, p, 8, p, 16)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for rc, bad in ((1, dict(type=5)), (1, dict(act=3)), (1, dict(D=0)), (1, dict(F=0)), (1, dict(n=-1)), (1, dict(x=None)),
                    (1, dict(w_up=None)), (1, dict(ldx=7)), (1, dict(ld_down=8)), (1, dict(y=None)), (1, dict(ldy=2)),
                    (3, dict(n=1 << 31)), (3, dict(D=1 << 21, ldx=1 << 21))):
        a = args(**bad)
        assert lib.fb_gated_ffn_fwd(a, p, 1 << 40, None) == rc, bad
        assert lib.fb_gated_ffn_ws_bytes(a, 0) == 256
    assert lib.fb_gated_ffn_fwd(args(), None, 0, None) == 1
    assert lib.fb_gated_ffn_fwd(args(), p, 64, None) == 1                          # workspace too small
    assert lib.fb_gated_ffn_fwd(args(n=0, x=None, y=None), None, 0, None) == 0
    for rc, bad in ((1, dict(dy=None)), (1, dict(lddx=3)), (1, dict(ldd_down=8)), (1, dict(type=0, grad_type=1)),
                    (3, dict(type=1, grad_type=1, accumulate=1))):
        assert lib.fb_gated_ffn_bwd(args(**bad), p, 1 << 40, None) == rc, bad
    assert lib.fb_gated_ffn_fwd(None, p, 64, None) == 1


def test_softmax_xent_entry_refuses():
    from fast_b200.capi import SoftmaxXent, lib
    buf, p = _addr()

    def args(**kw):
        a = SoftmaxXent(1, 1, 0, 8, 2, 30, p, 8, p, 8, p, p, p, p, p, 8, p, 8)
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for rc, bad in ((1, dict(type=2)), (1, dict(V=0)), (1, dict(D=0)), (1, dict(n=-2)), (1, dict(h=None)), (1, dict(w=None)),
                    (1, dict(target=None)), (1, dict(loss=None)), (1, dict(ldw=5)), (3, dict(V=1 << 31)),
                    (3, dict(n=1 << 31))):
        assert lib.fb_softmax_xent_fwd(args(**bad), p, 1 << 40, None) == rc, bad
    assert lib.fb_softmax_xent_fwd(args(), p, 64, None) == 1
    assert lib.fb_softmax_xent_fwd(args(n=0), None, 0, None) == 0
    for rc, bad in ((1, dict(dloss=None)), (1, dict(lddh=4)), (1, dict(grad_type=3)), (3, dict(accumulate=1))):
        assert lib.fb_softmax_xent_bwd(args(**bad), p, 1 << 40, None) == rc, bad


def test_module_refuses_an_unknown_activation():
    from fast_b200.ranking import GatedFeedForward, NodeRankingHead
    with pytest.raises(ValueError):
        GatedFeedForward(8, 16, act="tanh")
    head = NodeRankingHead(8, 20, hidden=12)
    assert {n: tuple(p.shape) for n, p in head.named_parameters()} == {
        "node_table": (20, 8), "norm1.weight": (8,), "norm1.bias": (8,), "norm2.weight": (8,), "norm2.bias": (8,),
        "ffn.w_gate": (12, 8), "ffn.w_up": (12, 8), "ffn.w_down": (8, 12)}


def test_backward_wrappers_refuse_a_gradient_type():
    from fast_b200 import ops
    x, v, t = torch.zeros(4, 8), torch.zeros(4), torch.zeros(4, dtype=torch.int64)
    for bad in (torch.float16, torch.bfloat16, torch.float64):
        with pytest.raises(ValueError, match="grad_dtype"):
            ops.gated_ffn_bwd(x, x, x, x, x, grad_dtype=bad)
        with pytest.raises(ValueError, match="grad_dtype"):
            ops.softmax_xent_bwd(x, x, t, v, v, grad_dtype=bad)


def test_entries_refuse_a_workspace_that_is_not_aligned():
    """The workspace's pieces are accessed 16 bytes at a time and mapped for bulk copies: refused before any launch."""
    from fast_b200.capi import GatedFfn, SoftmaxXent, lib
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    f = GatedFfn(0, 0, 0, 0, 2, 8, 16, p, 8, p, 8, p, 8, p, 16, p, 8, p, 8, p, 8, p, 8, p, 8, p, 16)
    x = SoftmaxXent(1, 1, 0, 8, 2, 30, p, 8, p, 8, p, p, p, p, p, 8, p, 8)
    for off in (1, 4, 8):
        assert lib.fb_gated_ffn_fwd(f, p + off, 1 << 40, None) == 1
        assert lib.fb_gated_ffn_bwd(f, p + off, 1 << 40, None) == 1
        assert lib.fb_softmax_xent_fwd(x, p + off, 1 << 40, None) == 1
        assert lib.fb_softmax_xent_bwd(x, p + off, 1 << 40, None) == 1
        assert lib.fb_layer_norm_bwd(0, p, 8, p, 8, p, 0, p, p, None, 0, p, 8, p, p, 0, 2, 8, p + off, 1 << 20, None) == 1
