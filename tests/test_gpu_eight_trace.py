"""Operators in 8 bits under a trace: their launches are not of the trace, which would replay the memory that
they wrote into, so every one refuses it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_traces_are_refused(m3, dev):
    T = m3.eightbit
    x, gain = torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    w, g = T.pack8(torch.randn(64, 48, device=dev)), T.pack8(torch.randn(64, 64, device=dev), gated=True)
    q = T.quantize8(x)
    for call in (lambda t: T.quantize8(t).values.float(), lambda t: T.rms_norm8(t, gain, 1e-5)[0], lambda t: T.matmul8(t, w),
                 lambda t: T.swiglu8(t, g).values.float(), lambda t: q.dequantize() + t.to(torch.bfloat16),
                 lambda t: q.dequantize(torch.float32) + t):
        with pytest.raises(ValueError, match="no trace"):
            torch.jit.trace(call, (x,), check_trace=False)
        call(x)


def test_tangents_are_refused(m3, dev):
    import torch.autograd.forward_ad as fwd_ad

    T = m3.eightbit
    x = torch.randn(4, 64, device=dev)
    w = T.pack8(torch.randn(64, 48, device=dev))
    with fwd_ad.dual_level():
        dual = fwd_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: T.quantize8(dual), lambda: T.matmul8(dual, w)):
            with pytest.raises(ValueError, match="tangent"):
                call()
