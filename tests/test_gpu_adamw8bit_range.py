"""The 8-bit AdamW step at the ends of what its states can hold, and what a refused one leaves."""

from __future__ import annotations

import pytest
import torch

import gpu_utils as gu
from picotron_b200.errors import TritonAdamWUnavailable
from picotron_b200.kernels import AdamW8bit, adamw8bit_moments, adamw8bit_step

pytestmark = pytest.mark.gpu

LR = 1e-2


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def _fresh(n, seed):
    p, g = gu.randn((n,), seed, torch.float32, 0.05), gu.randn((n,), seed + 1, torch.float32, 1e-3)
    blocks = (n + 255) // 256
    return p, g, [torch.zeros(n, dtype=torch.int8, device=gu.DEV),
                  torch.zeros(blocks, device=gu.DEV),
                  torch.zeros(n, dtype=torch.uint8, device=gu.DEV),
                  torch.zeros(blocks, device=gu.DEV)]


def _call(p, g, state, step, b1=0.9, b2=0.95, eps=1e-8):
    adamw8bit_step([p], [g], *([t] for t in state), step=step, lr=LR, beta1=b1, beta2=b2, eps=eps,
                   weight_decay=0.0)


def test_denominators_of_forgotten_squares_keep_steps_small():
    """A block of tiny gradients, whose exp_avg_sq falls below what its scale can hold, and then a
    gradient of zero: the step has eps alone for a denominator, which is refused where it would
    carry parameters away and bounds the step to the learning rate where it is not."""

    for eps in (0.0, 1e-30, 1e-13):
        p, g, state = _fresh(600, 21)
        keep = [t.clone() for t in (p, *state)]
        with pytest.raises(TritonAdamWUnavailable, match="eps"):
            _call(p, g, state, 1, eps=eps)
        assert all(torch.equal(a, b) for a, b in zip(keep, (p, *state)))
    for b1, b2 in ((0.9, 0.999), (0.9, 0.95), (0.5, 0.99999)):
        p, g, state = _fresh(600, 21)
        # exp_avg_sq just below the smallest that is kept, 255^4 * 2^-126.
        g = torch.sign(g) * (0.99 * 255.0 ** 4 * 2.0 ** -126 / (1 - b2)) ** 0.5
        _call(p, g, state, 1, b1=b1, b2=b2, eps=1e-12)
        assert (state[3] == 0).all() and (state[1] > 0).all()
        before = p.clone()
        _call(p, torch.zeros_like(g), state, 2, b1=b1, b2=b2, eps=1e-12)
        # lr / (1 - b1^2) * b1 (1 - b1) |g| / eps, and the parameter's own rounding
        bound = LR / (1 - b1 ** 2) * b1 * (1 - b1) * g.abs().max().item() / 1e-12
        assert bound <= LR
        assert (p - before).abs().max().item() <= 1.02 * bound + 2.0 ** -24 * p.abs().max().item()


def test_squares_beyond_the_range_count_as_not_finite():
    """A finite gradient whose square passes fp32's range loses its block's exp_avg_sq, as a
    gradient that is not finite does; the other blocks keep theirs."""

    p, g, state = _fresh(1000, 22)
    q, _, other = _fresh(1000, 22)
    clean = g.clone()
    g[300] = 1e20
    _call(p, g, state, 1)
    _call(q, clean, other, 1)
    assert torch.isfinite(p).all()
    m, v = adamw8bit_moments(*([t] for t in state))
    assert torch.isnan(v[0][256:512]).all() and torch.isfinite(m[0]).all()
    for s in (slice(0, 256), slice(512, 1000)):
        assert torch.equal(p[s], q[s]) and torch.isfinite(v[0][s]).all()


def test_a_step_that_is_refused_for_one_group_takes_none():
    """Groups of other betas or types are launches of their own; all are checked before the first."""

    good = [torch.nn.Parameter(gu.randn((40, 3), 1)), torch.nn.Parameter(gu.randn((9,), 2))]
    bad = torch.nn.Parameter(gu.randn((6, 4), 3).t())
    opt = AdamW8bit([{"params": good}, {"params": [bad], "betas": (0.8, 0.9)}])
    for p in (*good, bad):
        p.grad = torch.ones_like(p)
    before = [p.detach().clone() for p in (*good, bad)]
    with pytest.raises(TritonAdamWUnavailable):
        opt.step()
    assert len(opt.state) == 0
    assert all(torch.equal(p, b) for p, b in zip((*good, bad), before))
    bad.grad = None
    opt.step()
    assert [opt.state[p]["step"] for p in good] == [1, 1] and len(opt.state) == 2
    bad.grad = torch.ones_like(bad)
    before = [p.detach().clone() for p in good]
    with pytest.raises(TritonAdamWUnavailable):
        opt.step()
    assert [opt.state[p]["step"] for p in good] == [1, 1]
    assert all(torch.equal(p, b) for p, b in zip(good, before))
    bad.grad = None
    opt.param_groups[0]["eps"] = 0.0  # may be set, or loaded, after construction
    with pytest.raises(TritonAdamWUnavailable, match="eps"):
        opt.step()
    assert all(torch.equal(p, b) for p, b in zip(good, before))


def test_states_that_share_memory_across_lists_are_refused():
    p, g, state = _fresh(600, 31)
    mc, ms, vc, vs = state
    flat = torch.zeros(5000, dtype=torch.uint8, device=gu.DEV)
    inside = flat[:2400].view(torch.float32)  # a parameter of 600 elements over its own codes
    for params, held in ((p, [mc, ms, mc.view(torch.uint8), vs]), (p, [mc, ms, vc, ms]),
                         (inside, [flat[2399:2999].view(torch.int8), ms, vc, vs]),
                         (p, [mc, flat[1000:1012].view(torch.float32), flat[411:1011], vs])):
        before = [t.clone() for t in (params, *held)]
        with pytest.raises(TritonAdamWUnavailable, match="share memory"):
            _call(params, g, held, 1)
        assert all(torch.equal(a, b) for a, b in zip((params, *held), before))
    _call(inside, g, [flat[2400:3000].view(torch.int8), ms, vc, vs], 1)  # next to one another
