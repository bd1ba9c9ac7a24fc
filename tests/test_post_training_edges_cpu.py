"""Refusals of the post-training operators before any launch, next to those of
test_post_training_cpu.py."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from picotron_b200 import _capi
from picotron_b200.kernels import AdamW8bit


def test_wait_limits_of_the_self_test_are_checked():
    for limit in (-2, 2_000_000_001):
        with pytest.raises(_capi.PtError, match="limit_cycles"):
            _capi.selftest_policy_wait(limit)
    _capi.selftest_policy_wait(2_000_000_000)  # as without it


def test_an_eps_below_what_the_states_can_drop_is_refused():
    """Blocks whose largest exp_avg_sq is below 255^4 times the smallest normal number keep none of
    it, so that eps alone is left in the denominator of the next step."""

    p = torch.nn.Parameter(torch.zeros(4))
    for eps in (0.0, 1e-45, 1e-30, 1e-13):
        with pytest.raises(ValueError, match="eps"):
            AdamW8bit([p], eps=eps)
    AdamW8bit([p], eps=1e-12)
    lib = _capi.library()
    one = (ctypes.c_void_p * 1)(None)
    n, step = (ctypes.c_int64 * 1)(0), (ctypes.c_int64 * 1)(1)
    lr = (ctypes.c_double * 1)(0.1)
    for eps, want in ((0.0, _capi.PT_ERR_INVALID_ARGUMENT), (1e-13, _capi.PT_ERR_INVALID_ARGUMENT),
                      (math.nan, _capi.PT_ERR_INVALID_ARGUMENT)):
        assert lib.pt_adamw8_step(one, one, one, one, one, one, n, step, lr, lr, 1, 0.9, 0.99, eps, 0,
                                  0, None) == want
        assert "eps" in _capi.last_error()


def test_factors_that_fp32_does_not_hold_are_refused():
    """A gradient formed with 1e-50 or 1e39 is 0 or infinite, and no rescaling brings it back."""

    lib, arg = _capi.library(), _capi.PT_ERR_INVALID_ARGUMENT
    for expected in (1e-50, -1e-40, 1e39, math.inf, math.nan, 0.0):
        assert lib.pt_rescale_logits_grad(None, 8, 0, 1, 8, 8, None, expected, 2, None) == arg
    for expected in (2.0 ** -126, -3e38):
        assert lib.pt_rescale_logits_grad(None, 8, 0, 1, 8, 8, None, expected, 2, None) == _capi.PT_OK
    rows = (None, 0, 0)
    for grad in (1e39, math.inf, math.nan):
        assert lib.pt_policy_loss_grad(None, 8, 2, 3, 24, 8, *rows, -100, *rows, *rows, *rows, 0.2, 0.2,
                                       0.0, 0, grad, None, None, None, None, *rows, None, 0, 2,
                                       None) == arg
        assert "grad" in _capi.last_error()
