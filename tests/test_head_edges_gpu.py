"""GPU: the node-ranking head's operators where the caller, single values or rows are out of the ordinary, against fp64
restatements.  Bounds are test_head_gpu.py's: c = (K + 64) 2^-22 of the terms' sum for a product of K terms, 2^-8 for a
rounding to bf16."""
import math
import threading

import pytest
import torch

from test_head_gpu import _c, _check, _gen, _mat

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
