"""Refusals of the post-training operators before any launch, next to those of
test_post_training_cpu.py."""

from __future__ import annotations

import pytest

from picotron_b200 import _capi


def test_wait_limits_of_the_self_test_are_checked():
    for limit in (-2, 2_000_000_001):
        with pytest.raises(_capi.PtError, match="limit_cycles"):
            _capi.selftest_policy_wait(limit)
    _capi.selftest_policy_wait(2_000_000_000)  # as without it
