"""torch.ops.picotron_b200.logit_loss_backward called directly, as a graph or a user's own autograd
Function calls it: what is not a forward's statistics is refused before any launch."""

from __future__ import annotations

import pytest
import torch

import gpu_utils as gu
from picotron_b200 import _capi, kernels
from picotron_b200.errors import TritonLogitLossUnavailable

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def test_statistics_and_grad_are_checked():
    x, t = gu.randn((2, 5, 40), 1), torch.zeros(2, 5, dtype=torch.long, device=gu.DEV)
    coef = gu.randn((2, 5), 2)
    _, stats = torch.ops.picotron_b200.token_logps(x, t, -100)
    back = torch.ops.picotron_b200.logit_loss_backward
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(kernels.token_log_probs(leaf, t), leaf, coef)
    one = torch.ones((), device=gu.DEV)
    for grad in (None, one, one[None], one.double()):
        assert torch.equal(back(x, t, stats, coef, grad, -100), want)
    off = torch.zeros(stats.numel() + 1, device=gu.DEV)[1:].view(stats.shape)  # 4 modulo 8
    off.copy_(stats)
    assert off.is_contiguous() and off.data_ptr() % 8 == 4
    for bad in (off, stats.bfloat16(), stats.double(), stats.cpu(), stats[:1], stats[..., :1],
                stats.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(TritonLogitLossUnavailable, match="stats"):
            back(x, t, bad, coef, None, -100)
    for bad in (one.cpu(), torch.ones(2, device=gu.DEV), torch.ones(0, device=gu.DEV)):
        with pytest.raises(TritonLogitLossUnavailable, match="grad"):
            back(x, t, stats, coef, bad, -100)


def test_statistics_of_c_callers_are_checked():
    x, t = gu.randn((5, 40), 1), torch.zeros(5, dtype=torch.long, device=gu.DEV)
    held = torch.zeros(11, device=gu.DEV)
    lp = torch.zeros(5, device=gu.DEV)
    work = torch.zeros(1 << 16, dtype=torch.uint8, device=gu.DEV)
    for at, refused in ((held[:10], False), (held[1:], True)):
        call = lambda: _capi.token_logps_fwd(  # noqa: E731
            (x.data_ptr(), 200, 40), 40, 1, 5, (t.data_ptr(), 5, 1), -100, lp.data_ptr(),
            at.data_ptr(), work.data_ptr(), work.numel(), 0, gu.stream())
        if refused:
            with pytest.raises(_capi.PtError, match="stats"):
                call()
        else:
            call()
    # (m, 1 / sum e^(x - m)) with m from the maximum to 9 above it
    m, inv = held[:10].view(5, 2).double().unbind(-1)
    gap = m - x.double().amax(-1)
    assert (gap >= 0).all() and (gap <= 9).all()
    want = 1 / (x.double() - m[:, None]).exp().sum(-1)
    torch.testing.assert_close(inv, want, rtol=1e-5, atol=0)
