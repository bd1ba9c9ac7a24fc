"""Forward-mode differentiation is refused by the post-training operators, never dropped."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import gpu_utils as gu
from picotron_b200 import kernels

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def test_tangents_are_refused():
    x, t = gu.randn((2, 3, 40), 1), torch.zeros(2, 3, dtype=torch.long, device=gu.DEV)
    f = torch.zeros(2, 3, device=gu.DEV)
    q, freq = gu.randn((1, 2, 3, 8), 2), kernels.rotary_frequencies(8, device=gu.DEV)[0]
    at = torch.arange(3, device=gu.DEV)
    calls = [
        lambda: kernels.token_log_probs(dual, t),
        lambda: kernels.preference_loss(dual, t, f),
        lambda: kernels.policy_loss(dual, t, f, f),
        lambda: kernels.apply_rotary_positions(dual_q, q, at, freq),
        lambda: kernels.apply_rotary_positions(q, dual_q, at, freq),
        lambda: torch.ops.picotron_b200.token_logps(dual, t, -100),
    ]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        dual_q = forward_ad.make_dual(q, torch.ones_like(q))
        for call in calls:
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                call()
        # Tensors without a tangent are taken as ever.
        assert torch.isfinite(kernels.token_log_probs(x, t)).all()
        with torch.no_grad():
            assert torch.isfinite(kernels.token_log_probs(x, t)).all()
    assert torch.isfinite(kernels.token_log_probs(x, t)).all()
