"""policy_loss on inputs that are not numbers, and on what else its callers may hand it: NaN and
infinities in every input, targets outside the vocabulary, ratios beyond the range of 32 bits,
gradients that are not finite, and a backward pass that is captured by itself.

Rows are compared bit for bit with those of a call on clean inputs: a row's gradient depends on
that row and on the number of positions with a target alone.
"""

from __future__ import annotations

import math

import pytest
import torch

import gpu_utils as gu
from picotron_b200 import _capi, kernels
from picotron_b200.errors import TritonLogitLossUnavailable

pytestmark = pytest.mark.gpu

IGNORE = -100
AT = (0, 2)  # the row that is broken; it has a target
# A path of the implementation: shape, dtype, whether the logits need a gradient, and what
# expected_grad is given. float16 without a hint forms its gradient in backward.
PATHS = {
    "one pass": ((2, 5, 1003), torch.bfloat16, True, None),
    "one pass, a cluster per row": ((1, 3, 100_003), torch.float32, True, None),
    "two passes": ((2, 5, 1003), torch.float16, True, None),
    "no gradient": ((2, 5, 1003), torch.float32, False, None),
    "many short rows": ((3, 2000, 37), torch.bfloat16, True, None),
    "many short rows, two passes": ((3, 2000, 37), torch.float16, True, None),
}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()
    _capi.take_device_error()


def _inputs(shape, dtype):
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(shape, generator=g) * 2.0).to(dtype).to(gu.DEV)
    t = torch.randint(0, shape[-1], shape[:2], generator=g)
    t.view(-1)[1::4] = IGNORE
    t = t.to(gu.DEV)
    old = kernels.token_log_probs(x, t) + 0.01  # ratios next to 1, inside the clipping range
    return x, t, old, old - 0.02, gu.randn(shape[:2], 6) + 3.0


def _call(x, t, old, ref, adv, kl, path):
    _, _, grad, expected = PATHS[path]
    leaf = x.detach().requires_grad_(grad)
    loss, lp = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref if kl else None,
                                   kl_coef=kl, expected_grad=expected)
    dx = torch.autograd.grad(loss, leaf)[0] if grad else None
    return loss.detach(), lp, dx


def _set(tensor, value):
    out = tensor.clone()
    out[AT] = value
    return out


BREAK = {
    "NaN among the logits": lambda x, t, old, ref, adv: (_at(x, 7, math.nan), t, old, ref, adv),
    "infinite logit": lambda x, t, old, ref, adv: (_at(x, 7, math.inf), t, old, ref, adv),
    "no finite logit": lambda x, t, old, ref, adv: (_set(x, -math.inf), t, old, ref, adv),
    "NaN old": lambda x, t, old, ref, adv: (x, t, _set(old, math.nan), ref, adv),
    "NaN advantage": lambda x, t, old, ref, adv: (x, t, old, ref, _set(adv, math.nan)),
    "NaN reference": lambda x, t, old, ref, adv: (x, t, old, _set(ref, math.nan), adv),
    "both -inf": lambda x, t, old, ref, adv: (
        _at(x, int(t[AT]), -math.inf), t, _set(old, -math.inf), ref, adv),
}


def _at(x, column, value):
    out = x.clone()
    out[(*AT, column)] = value
    return out


@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("broken", BREAK)
@pytest.mark.parametrize("path", PATHS)
def test_what_is_not_a_number_stays_so(path, broken, kl):
    clean = _inputs(*PATHS[path][:2])
    for sign in (1.0, -1.0):
        args = [*clean[:4], clean[4] * sign]
        want_loss, _, want = _call(*args, kl, path)
        loss, _, dx = _call(*BREAK[broken](*args), kl, path)
        if broken == "NaN reference" and not kl:  # not read
            assert torch.equal(loss, want_loss) and (dx is None or torch.equal(dx, want))
            continue
        assert torch.isfinite(want_loss) and torch.isnan(loss)
        if dx is not None:
            assert torch.isnan(dx[AT]).all()
            rest = torch.ones(dx.shape[:2], dtype=torch.bool, device=gu.DEV)
            rest[AT] = False
            assert torch.equal(dx[rest], want[rest])
    assert _capi.take_device_error() == 0


@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("target", [-1, "vocab"])
@pytest.mark.parametrize("path", PATHS)
def test_a_target_outside_the_vocabulary(path, target, kl):
    x, t, old, ref, adv = _inputs(*PATHS[path][:2])
    _, _, want = _call(x, t, old, ref, adv, kl, path)
    bad = _set(t, x.size(-1) if target == "vocab" else target)
    loss, lp, dx = _call(x, bad, old, ref, adv, kl, path)
    assert torch.isnan(loss) and torch.isnan(lp[AT])
    if dx is not None:
        assert (dx[AT] == 0).all()
        want = want.clone()
        want[AT] = 0
        assert torch.equal(dx, want)
    assert _capi.take_device_error() == 2 and _capi.take_device_error() == 0


@pytest.mark.parametrize("path", PATHS)
def test_ratios_beyond_the_range_of_32_bits(path):
    """exp(logp - old) above 3.4e38: a zero advantage still costs nothing, a positive one is
    clipped, and a negative one weighs a finite product."""

    x, t, old, ref, adv = _inputs(*PATHS[path][:2])
    n = int((t != IGNORE).sum())
    lp = kernels.token_log_probs(x, t)
    old = lp.clone()  # every other ratio is 1 up to the rounding of its log-probability
    old[AT] = -100.0 + lp[AT].double().item()
    exact = math.exp(lp[AT].double().item() - float(old[AT]))
    for a, loss64, coef64 in ((0.0, 0.0, 0.0), (2.0, -2.4, 0.0),
                              (-1e-30, 1e-30 * exact, 1e-30 * exact)):
        advantages = _set(torch.zeros_like(adv), a)
        loss, _, dx = _call(x, t, old, ref, advantages, 0.0, path)
        # The log-probability is known to 2^-24 of itself, the loss is rounded once (2^-24), and a
        # softmax value is off by 2 eps: its exponential by 2^-22 + 146 * 2^-24, its sum by
        # V / 256 + 56 roundings more.
        lp_error = 2.0 ** -22 + 2.0 ** -24 * abs(lp[AT].item())
        eps = 2.0 ** -22 + 2.0 ** -24 * (x.size(-1) / 256 + 202)
        assert abs(loss.item() - loss64 / n) <= 2 * lp_error * abs(loss64) / n
        if dx is None:
            continue
        hot = torch.zeros(x.size(-1), dtype=torch.float64, device=gu.DEV)
        hot[t[AT]] = 1.0
        want = coef64 / n * (hot - torch.softmax(x[AT].double(), -1))
        info = torch.finfo(x.dtype)
        tol = ((2 * lp_error + 2 * eps) * abs(coef64) / n + want.abs() * info.eps
               + info.smallest_normal)
        fits = want.abs() < info.max  # float16 has no such gradients
        assert ((dx[AT].double() - want).abs()[fits] <= tol[fits]).all()
        assert (dx[t == IGNORE] == 0).all()


def test_a_backward_that_is_captured_by_itself_can_be_replayed():
    """The forward ran outside of the graph: its gradient, formed for another factor than it gets,
    must not be rescaled once more by every replay."""

    x, t, old, ref, adv = _inputs(*PATHS["one pass"][:2])
    leaf = x.detach().requires_grad_()
    up = torch.tensor(2.0, device=gu.DEV)

    def loss():
        return kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1)[0]

    (want,) = torch.autograd.grad(loss(), leaf, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(loss(), leaf, up)
        kept = loss()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (dx,) = torch.autograd.grad(kept, leaf, up)
    results = []
    for _ in range(3):
        graph.replay()
        results.append(dx.clone())
    up.fill_(4.0)
    graph.replay()
    torch.cuda.synchronize()
    for got in results:
        assert torch.equal(got, want)  # twice a bf16 value: no rounding on either way
    assert torch.equal(dx, 2.0 * want)


def test_a_forward_and_backward_that_are_captured_together_can_be_replayed():
    x, t, old, ref, adv = _inputs(*PATHS["one pass"][:2])
    leaf = x.detach().requires_grad_()
    up = torch.tensor(2.0, device=gu.DEV)

    def step():
        loss, _ = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1)
        return torch.autograd.grad(loss, leaf, up)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dx = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want)


@pytest.mark.parametrize("up", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("vocab", [37, 1003, 1024])
def test_ignored_rows_stay_zero_under_a_gradient_that_is_not_finite(vocab, up):
    x, t, old, ref, adv = _inputs((2, 5, vocab), torch.bfloat16)
    leaf = x.detach().requires_grad_()
    loss, _ = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1)
    grads = [torch.autograd.grad(loss, leaf, torch.tensor(up, device=gu.DEV),
                                 retain_graph=True)[0] for _ in range(2)]
    for dx in grads:  # formed in the forward's pass, and in backward
        assert (dx[t == IGNORE] == 0).all()
        assert not torch.isfinite(dx[t != IGNORE]).any()


@pytest.mark.parametrize("limit", [-1, 0])
@pytest.mark.parametrize("path", PATHS)
def test_waits_that_run_out_leave_nan_and_the_error_word(path, limit):
    """Waits that are given up at once (-1), or after one look (0, which may see the data): what was
    not waited for is NaN and said so; nothing of it reaches the next call."""

    args = (*_inputs(*PATHS[path][:2]), 0.1, path)
    want_loss, want_lp, want = _call(*args)
    t = args[1]
    _capi.selftest_policy_wait(limit)
    loss, lp, dx = _call(*args)
    code = _capi.take_device_error()
    if path.startswith("one pass") and limit < 0:
        assert code == 1 and torch.isnan(loss)
        assert torch.isnan(dx[t != IGNORE]).all() and torch.isnan(lp[t != IGNORE]).all()
    elif path.startswith("one pass") and code:
        assert code == 1 and (torch.isnan(dx) | (dx == want)).all()
    else:
        assert code == 0 and torch.equal(loss, want_loss) and torch.equal(lp, want_lp)
        assert dx is None or torch.equal(dx, want)
    assert dx is None or (dx[t == IGNORE] == 0).all()
    _capi.selftest_policy_wait(2_000_000_000)
    loss, lp, dx = _call(*args)
    assert torch.equal(loss, want_loss) and (dx is None or torch.equal(dx, want))
    assert _capi.take_device_error() == 0


def test_expected_gradients_that_fp32_does_not_hold_are_refused():
    x, t, old, _, adv = _inputs(*PATHS["one pass"][:2])
    for expected in (1e-50, -1e-40, 1e39):
        with pytest.raises(TritonLogitLossUnavailable, match="expected_grad"):
            kernels.policy_loss(x, t, old, adv, expected_grad=expected)


@pytest.mark.parametrize("path", PATHS)
def test_clipped_terms_are_rounded_once(path):
    """Where every position is clipped the loss hangs on no log-probability, so that the one rounding
    to fp32 (2^-24 relative) is all that may be off; the gradient is zero."""

    x, t, _, _, _ = _inputs(*PATHS[path][:2])
    lp, keep = kernels.token_log_probs(x, t), t != IGNORE
    for seed in range(12):
        adv = gu.randn(t.shape, seed)
        old = lp - torch.sign(adv) * 0.6  # ratios of 1.8 and 0.55
        loss, _, dx = _call(x, t, old, None, adv, 0.0, path)
        border = torch.where(adv > 0, 1.0 + 0.2 * torch.ones_like(adv, dtype=torch.float64), 1.0 - 0.2)
        want = -(adv.double() * border)[keep].mean().item()
        assert abs(loss.item() - want) <= 1.001 * 2.0 ** -24 * abs(want)
        assert dx is None or not dx.any()
