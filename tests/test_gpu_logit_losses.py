"""Log-probabilities, preference loss and policy loss against their definitions in 64 bits.

Tolerances, for a row of V logits (u = 2^-24, the half step of fp32):
* each term e^(x - m) is off by at most 2^-22 (the exponential) plus 2.3 u |x - m| log2 e (the
  difference, the constant and the product rounded); terms with |x - m| above 44 are below u of
  the sum, so 146 u covers the second part; a thread's two partial sums take at most V / 256 + 16
  additions each (u apiece), the merges 40 roundings more. So s is off by at most
  EPS = 2^-22 + u (V / 256 + 202) relative, which is the log-probability's error, plus half a step
  of its own rounding;
* a softmax value is one more such term over s: at most 2 EPS; dx = c (onehot - p) then has an
  absolute error of |c| p 2 EPS + |dc| + |dx| (4 u + half a step of the logits' type), and, where
  the type's smallest step is coarser than that, half of it;
* the exponential's results below 2^-126 are 0. They are taken relative to a reference that is at
  most 9 above the row's maximum, so s >= e^-9 (1 - EPS) and a softmax value below
  2^-126 e^9 < 2^-113 may be 0 instead: another |c| 2^-113.
dc is the error that the coefficient takes from the log-probabilities, derived per loss below.
"""

from __future__ import annotations

import math

import pytest
import torch

import gpu_utils as gu
from picotron_b200 import _capi, kernels
from picotron_b200.errors import TritonLogitLossUnavailable
from picotron_b200.ops import DTYPE_CODES

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (1, 1, 2), (2, 3, 7), (1, 5, 8), (2, 4, 129), (4, 5, 1000), (2, 129, 321),
          (1, 300, 33), (2, 3, 50257), (2, 2, 128256)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def _eps(vocab: int) -> float:
    return 2.0 ** -22 + U * (vocab / 256 + 202)


def _data(shape, dtype, seed=0, ignore=True):
    b, s, v = shape
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * 3.0).to(dtype)
    t = torch.randint(0, v, (b, s), generator=g)
    if ignore and b * s > 3:
        t.view(-1)[1::4] = IGNORE
    return x.to(gu.DEV), t.to(gu.DEV)


def _logps64(x, t):
    """Log-probabilities in 64 bits on the CPU, 0 where ignored."""

    lp = torch.log_softmax(x.double().cpu(), -1)
    lp = lp.gather(-1, t.cpu().clamp_min(0).unsqueeze(-1)).squeeze(-1)
    return torch.where(t.cpu() == IGNORE, torch.zeros_like(lp), lp)


def _grad64(x, t, coef):
    """coef (onehot - softmax) in 64 bits, and softmax; zeros where ignored."""

    p = torch.softmax(x.double().cpu(), -1)
    hot = torch.zeros_like(p).scatter_(-1, t.cpu().clamp_min(0).unsqueeze(-1), 1.0)
    d = coef.double().cpu().unsqueeze(-1) * (hot - p)
    return torch.where((t.cpu() == IGNORE).unsqueeze(-1), torch.zeros_like(d), d), p


def _check_logps(got, x, t):
    want = _logps64(x, t)
    err = (got.double().cpu() - want).abs()
    assert (err <= _eps(x.size(-1)) + U * want.abs()).all(), err.max()
    assert (got.cpu()[t.cpu() == IGNORE] == 0).all()
    return want


def _check_grad(got, x, t, coef, dcoef=0.0):
    assert got.shape == x.shape and got.dtype == x.dtype
    want, p = _grad64(x, t, coef)
    c = coef.double().cpu().abs().unsqueeze(-1)
    dc = torch.as_tensor(dcoef, dtype=torch.float64)
    dc = dc.unsqueeze(-1) if dc.dim() else dc
    info = torch.finfo(x.dtype)
    tol = c * (p * 2 * _eps(x.size(-1)) + 2.0 ** -113) + dc + want.abs() * (4 * U + info.eps / 2)
    tol = tol + info.smallest_normal * info.eps / 2
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), f"{(err - tol).max()} over at {want.abs().max()}"
    assert (got.cpu()[t.cpu() == IGNORE] == 0).all()


# ------------------------------------------------------------------ log-probabilities --


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_token_log_probs_forward_and_backward(shape, dtype):
    x, t = _data(shape, dtype, seed=1)
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    assert lp.dtype == torch.float32 and lp.shape == t.shape
    _check_logps(lp.detach(), x.detach(), t)
    dlp = gu.randn(t.shape, 2)
    (dx,) = torch.autograd.grad(lp, x, dlp)
    _check_grad(dx, x.detach(), t, dlp)
    assert _capi.take_device_error() == 0


VIEWS = {
    "2-D": lambda x, t: (x[0], t[0]),
    "without the last position": lambda x, t: (x[:, :-1], t[:, 1:]),
    "without the first position": lambda x, t: (x[:, 1:], t[:, 1:]),
    "last positions": lambda x, t: (x[:, -2:], t[:, -2:]),
    "every other sequence": lambda x, t: (x[::2], t[::2]),
    "classes outside": lambda x, t: (x.transpose(1, 2).contiguous().transpose(1, 2), t),
    "sequence outside": lambda x, t: (x.transpose(0, 1).contiguous().transpose(0, 1), t.t()
                                      .contiguous().t()),
    "one sequence expanded": lambda x, t: (x[:1].expand_as(x), t),
    "part of the classes": lambda x, t: (x[..., 3:], t.clamp(max=x.size(-1) - 4)),
    "no positions": lambda x, t: (x[:, :0], t[:, :0]),
    "no sequences": lambda x, t: (x[:0], t[:0]),
}


@pytest.mark.parametrize("vocab", [65, 512])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("view", VIEWS)
def test_token_log_probs_of_views(view, dtype, vocab):
    x, t = _data((4, 6, vocab), dtype, seed=3)
    x, t = VIEWS[view](x, t)
    leaf = x.detach().requires_grad_()
    lp = kernels.token_log_probs(leaf, t)
    _check_logps(lp.detach(), x, t)
    dlp = gu.randn((*t.shape, 2), 4)[..., 0]  # a strided gradient
    (dx,) = torch.autograd.grad(lp, leaf, dlp)
    _check_grad(dx, x, t, dlp)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_masked_logits(dtype):
    x, t = _data((2, 6, 1003), dtype, seed=5, ignore=False)
    low = torch.finfo(dtype).min
    x[0, 0, 100:] = -math.inf          # a vocabulary mask, target inside
    t[0, 0] = 5
    x[0, 1, 100:] = low                # the type's lowest value as a mask
    t[0, 1] = 5
    x[0, 2, :] = low                   # a mask that leaves nothing: uniform
    x[0, 3, :900] = -math.inf          # whole vectors of -inf before the first finite logit
    t[0, 3] = 950
    x[0, 4, 7] = -math.inf             # the target masked: log-probability -inf
    t[0, 4] = 7
    x[1, 0, :] = math.nan              # ignored rows may hold anything
    x[1, 1, 4] = math.inf
    x[1, 2, :] = -math.inf
    t[1, :3] = IGNORE
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    want = _logps64(x.detach(), t)
    assert lp[0, 4].item() == -math.inf
    fine = torch.isfinite(want)
    err = (lp.detach().double().cpu() - want).abs()[fine]
    assert (err <= _eps(1003) + U * want.abs()[fine]).all()
    assert lp[0, 2].item() == pytest.approx(-math.log(1003), rel=1e-6)
    dlp = gu.randn(t.shape, 6)
    (dx,) = torch.autograd.grad(lp, x, dlp)
    clean = x.detach().clone()
    clean[1, :3] = 0.0
    _check_grad(dx, clean, t, dlp)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_near_certain_targets_and_large_logits(dtype):
    """Targets far above the rest (log-probabilities next to 0, never above), and logits of any
    size that the type holds."""

    x, t = _data((4, 8, 515), dtype, seed=10, ignore=False)
    top = torch.finfo(dtype).max
    x[0].scatter_(-1, t[0, :, None], 40.0)
    x[1] = (x[1].double() * 1000).to(dtype)
    x[2] = torch.where(x[2] > 0, x[2].abs() + top / 4, x[2]).to(dtype)
    x[3] += -top / 2
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    assert (lp <= 0).all() and (lp[0] > -1e-6).all()
    _check_logps(lp.detach(), x.detach(), t)
    (dx,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    _check_grad(dx, x.detach(), t, torch.ones(t.shape))


def test_rows_without_a_finite_logit_are_nan():
    x, t = _data((1, 4, 300), torch.float32, seed=7, ignore=False)
    x[0, 0] = -math.inf
    x[0, 1, 10] = math.nan
    x[0, 2, 299] = math.inf
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    assert torch.isnan(lp[0, :3]).all() and torch.isfinite(lp[0, 3])
    (dx,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert torch.isnan(dx[0, 0]).all() and torch.isfinite(dx[0, 3]).all()


def test_bad_target_gives_nan_and_the_error_word():
    x, t = _data((1, 3, 100), torch.bfloat16, seed=8, ignore=False)
    t[0, 1] = 100
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    (dx,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert torch.isnan(lp[0, 1]) and torch.isfinite(lp[0, ::2]).all()
    assert (dx[0, 1] == 0).all()
    assert _capi.take_device_error() == 2 and _capi.take_device_error() == 0


def test_other_ignore_index():
    x, t = _data((2, 3, 50), torch.float32, seed=9, ignore=False)
    t[0, 0] = 7
    lp = kernels.token_log_probs(x, t, ignore_index=7)
    assert lp[0, 0].item() == 0.0 and (lp.view(-1)[1:][t.view(-1)[1:] != 7] < 0).all()


# --------------------------------------------------------------------- preference loss --


def _preference64(lp, ref, t, beta, smoothing):
    keep = (t != IGNORE).cpu()
    rewards = beta * torch.where(keep, lp - ref.double().cpu(), torch.zeros_like(lp)).sum(-1)
    pairs = t.size(0) // 2
    z = rewards[:pairs] - rewards[pairs:]
    loss = ((1 - smoothing) * torch.nn.functional.softplus(-z)
            + smoothing * torch.nn.functional.softplus(z)).mean()
    dz = (smoothing - torch.sigmoid(-z)) / pairs
    return loss, rewards, beta * torch.cat((dz, -dz))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape,beta,smoothing", [
    ((2, 1, 5), 0.1, 0.0), ((4, 9, 301), 0.1, 0.1), ((6, 40, 1000), 0.5, 0.0),
    ((2, 700, 64), 0.05, 0.3), ((4, 3, 50257), 0.1, 0.0), ((2, 3, 128256), -0.2, 0.0),
], ids=str)
def test_preference_loss(shape, beta, smoothing, dtype):
    x, t = _data(shape, dtype, seed=11)
    ref = (_logps64(x, t) + 0.5 * torch.randn(t.shape, generator=torch.Generator().manual_seed(1),
                                              dtype=torch.float64)).float().to(gu.DEV)
    x.requires_grad_()
    loss, rewards = kernels.preference_loss(x, t, ref, beta=beta, label_smoothing=smoothing)
    assert loss.dtype == torch.float32 and loss.shape == () and not rewards.requires_grad
    want, rewards64, coef = _preference64(_logps64(x.detach(), t), ref, t, beta, smoothing)
    # Each of the sequence's positions adds its log-probability's error (unrounded), times beta.
    dr = abs(beta) * shape[1] * _eps(shape[2])
    assert ((rewards.double().cpu() - rewards64).abs() <= dr + U * rewards64.abs()).all()
    assert abs(loss.item() - want.item()) <= 2 * dr + U * abs(want.item())
    for scale in (None, 3.0):
        up = None if scale is None else torch.tensor(scale, device=gu.DEV)
        (dx,) = torch.autograd.grad(loss, x, up, retain_graph=True)
        s = scale or 1.0
        c = (s * coef)[:, None].expand(t.shape)
        # sigmoid' <= 1/4, z off by 2 dr; the coefficient rounded twice.
        _check_grad(dx, x.detach(), t, c, s * abs(beta) * 0.5 * dr / (shape[0] // 2)
                    + 2 * U * c.abs())


def test_preference_pair_without_positions():
    x, t = _data((4, 7, 90), torch.bfloat16, seed=12)
    t[1] = IGNORE
    t[3] = IGNORE
    ref = torch.full(t.shape, math.nan, device=gu.DEV)  # ignored positions may hold anything
    ref[t != IGNORE] = -4.0
    x.requires_grad_()
    loss, rewards = kernels.preference_loss(x, t, ref)
    want, rewards64, coef = _preference64(_logps64(x.detach(), t), ref.nan_to_num(), t, 0.1, 0.0)
    assert rewards[1].item() == 0.0 and rewards[3].item() == 0.0
    assert abs(loss.item() - want.item()) <= 2 * 0.7 * _eps(90) + U * abs(want.item())
    (dx,) = torch.autograd.grad(loss, x)
    _check_grad(dx, x.detach(), t, coef[:, None].expand(t.shape), 0.1 * _eps(90))
    assert (dx[1] == 0).all() and (dx[3] == 0).all()


def test_preference_extreme_margins():
    x, t = _data((4, 3, 40), torch.float32, seed=13, ignore=False)
    ref = torch.zeros(t.shape, device=gu.DEV)
    ref[0], ref[1] = -1e4, 1e4  # z far to both sides
    x.requires_grad_()
    loss, _ = kernels.preference_loss(x, t, ref, beta=1.0)
    want, _, coef = _preference64(_logps64(x.detach(), t), ref, t, 1.0, 0.0)
    assert abs(loss.item() - want.item()) <= 6 * _eps(40) + U * abs(want.item())
    (dx,) = torch.autograd.grad(loss, x)
    _check_grad(dx, x.detach(), t, coef[:, None].expand(t.shape), 2 * U)


def test_no_pairs_and_no_positions():
    x, t = _data((2, 3, 40), torch.float32, seed=14)
    loss, rewards = kernels.preference_loss(x[:0], t[:0], torch.zeros(0, 3, device=gu.DEV))
    assert math.isnan(loss.item()) and rewards.shape == (0,)
    leaf = x[:, :0].detach().requires_grad_()
    loss, rewards = kernels.preference_loss(leaf, t[:, :0], torch.zeros(2, 0, device=gu.DEV))
    assert loss.item() == pytest.approx(math.log(2.0), rel=1e-6) and (rewards == 0).all()
    (dx,) = torch.autograd.grad(loss, leaf)
    assert dx.shape == (2, 0, 40)


# ------------------------------------------------------------------------- policy loss --


def _policy64(lp, old, adv, ref, t, low, high, kl, by_sequence):
    """(loss, d loss / d lp, bound of |d2 loss / d lp2| in units of the log-probability's error)."""

    keep = (t != IGNORE).cpu()
    old, adv = old.double().cpu(), adv.double().cpu()
    adv = adv.unsqueeze(-1) if adv.dim() < t.dim() else adv
    adv = adv.expand(t.shape)
    r = (lp - old).exp()
    term = torch.maximum(-adv * r, -adv * r.clamp(1 - low, 1 + high))
    inside = torch.where(adv > 0, r <= 1 + high, r >= 1 - low)
    coef = torch.where(inside, -adv * r, torch.zeros_like(r))
    bend = coef.abs()
    if kl:
        g = ref.double().cpu() - lp
        term = term + kl * (g.exp() - g - 1)
        coef = coef + kl * (1 - g.exp())
        bend = bend + abs(kl) * g.exp()
    n = keep.sum(-1, keepdim=True) if keep.dim() > 1 else keep.sum()
    if by_sequence and keep.dim() > 1:
        w = keep.double() / (n.clamp_min(1) * (n > 0).sum())
    else:
        w = keep.double() / keep.sum()
    zero = torch.zeros_like(term)
    slope = torch.where(keep, coef.abs(), zero)
    return (torch.where(keep, term * w, zero).sum(), torch.where(keep, coef * w, zero),
            torch.where(keep, bend * w, zero), (slope * w).sum())


def _policy_inputs(x, t, seed, low=0.2, high=0.2):
    """Old log-probabilities whose ratios keep 1e-3 away from the clipping borders (a ratio within
    rounding of a border may fall on either side), reference ones, and advantages."""

    g = torch.Generator().manual_seed(seed)
    lp = _logps64(x, t)
    drift = 0.3 * torch.randn(t.shape, generator=g, dtype=torch.float64)
    for border in (math.log(1 - low), math.log(1 + high)):
        drift = torch.where((drift - border).abs() < 1e-3, drift + 4e-3, drift)
    old = (lp - drift).float().to(gu.DEV)
    ref = (lp + 0.3 * torch.randn(t.shape, generator=g, dtype=torch.float64)).float().to(gu.DEV)
    adv = torch.randn(t.shape, generator=g).to(gu.DEV)
    adv.view(-1)[::7] = 0.0
    return old, ref, adv


def _check_policy(x, t, old, adv, ref, kl, aggregate, low=0.2, high=0.2, scales=(None, 0.25)):
    x = x.detach().requires_grad_()
    loss, lp = kernels.policy_loss(x, t, old, adv, reference_log_probs=ref if kl else None,
                                   kl_coef=kl, clip_low=low, clip_high=high, aggregate=aggregate)
    lp64 = _check_logps(lp, x.detach(), t)
    assert not lp.requires_grad
    want, coef, bend, slope = _policy64(lp64, old, adv, ref, t, low, high, kl,
                                        aggregate == "sequence")
    eps = _eps(x.size(-1))
    assert abs(loss.item() - want.item()) <= 1.01 * eps * slope.item() + U * abs(want.item()), (
        loss.item(), want.item())
    for scale in scales:
        up = None if scale is None else torch.tensor(scale, device=gu.DEV)
        (dx,) = torch.autograd.grad(loss, x, up, retain_graph=True)
        s = scale or 1.0
        # The coefficient moves by bend * eps and is rounded twice.
        _check_grad(dx, x.detach(), t, s * coef, s * (1.01 * eps * bend + 2 * U * coef.abs()))
    return loss.detach(), dx


@pytest.mark.parametrize("aggregate", ["token", "sequence"])
@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES[2:], ids=str)
def test_policy_loss(shape, dtype, kl, aggregate):
    x, t = _data(shape, dtype, seed=21)
    old, ref, adv = _policy_inputs(x, t, 22)
    _check_policy(x, t, old, adv, ref, kl, aggregate)


@pytest.mark.parametrize("aggregate", ["token", "sequence"])
def test_policy_sequences_without_tokens_and_junk_where_ignored(aggregate):
    x, t = _data((5, 11, 200), torch.bfloat16, seed=23)
    t[2] = IGNORE
    t[4, 1:] = IGNORE
    old, ref, adv = _policy_inputs(x, t, 24)
    x[2, 3] = math.nan
    x[4, 5] = math.inf
    for value in (old, ref, adv):
        value[t == IGNORE] = math.nan
    clean, junk = x.clone(), t == IGNORE
    clean[junk] = 0.0
    leaf = x.detach().requires_grad_()
    loss, lp = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1,
                                   aggregate=aggregate)
    (dx,) = torch.autograd.grad(loss, leaf)
    want, dwant = _check_policy(clean, t, old.nan_to_num(), adv.nan_to_num(), ref.nan_to_num(), 0.1,
                                aggregate, scales=(None,))
    assert torch.equal(loss.detach(), want) and torch.equal(dx, dwant)


def test_policy_advantage_per_sequence_equals_broadcast():
    x, t = _data((3, 8, 128), torch.bfloat16, seed=25)
    old, ref, adv = _policy_inputs(x, t, 26)
    one = adv[:, 0].contiguous()
    a, da = _check_policy(x, t, old, one, ref, 0.1, "sequence")
    b, db = _check_policy(x, t, old, one[:, None].expand(t.shape).contiguous(), ref, 0.1,
                          "sequence")
    assert torch.equal(a, b) and torch.equal(da, db)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("expected", [None, 1.0, 0.25, 3.0, -2.0])
def test_policy_expected_gradient(dtype, expected):
    """The gradient is right whatever the loss's gradient turns out to be; formed for another
    factor it is rounded twice."""

    x, t = _data((3, 7, 1003), dtype, seed=33)
    old, ref, adv = _policy_inputs(x, t, 34)
    _, coef, bend, _ = _policy64(_logps64(x, t), old, adv, ref, t, 0.2, 0.2, 0.1, False)
    eps, info = _eps(1003), torch.finfo(dtype)
    for up in (1.0, 0.25, 3.0):
        leaf = x.detach().requires_grad_()
        loss, _ = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1,
                                      expected_grad=expected)
        grads = [torch.autograd.grad(loss, leaf, torch.tensor(up, device=gu.DEV),
                                     retain_graph=True)[0] for _ in range(3)]
        assert torch.equal(grads[1], grads[2])  # the second and third are formed in backward
        # Formed once at full precision.
        _check_grad(grads[1], x, t, up * coef, up * (1.01 * eps * bend + 2 * U * coef.abs()))
        want, p = _grad64(x, t, up * coef)
        formed = expected or 1.0
        extra = 0.0 if up == expected else (
            info.eps / 2 * want.abs() + abs(up / formed) * info.smallest_normal * info.eps)
        tol = (up * coef.abs().unsqueeze(-1) * p * 2 * eps
               + up * (1.01 * eps * bend + 2 * U * coef.abs()).unsqueeze(-1)
               + want.abs() * (8 * U + info.eps / 2) + info.smallest_normal * info.eps + extra)
        assert ((grads[0].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("vocab,dtype", [(400_001, torch.float32), (786_440, torch.bfloat16)],
                         ids=str)
def test_policy_rows_that_do_not_fit_on_chip(vocab, dtype):
    x, t = _data((1, 3, vocab), dtype, seed=35, ignore=False)
    old, ref, adv = _policy_inputs(x, t, 36)
    assert not _capi.policy_loss_grad_supported(vocab, 1, 3, DTYPE_CODES[dtype])
    _check_policy(x, t, old, adv, ref, 0.1, "token", scales=(None,))


@pytest.mark.parametrize("vocab,dtype", [(393_216, torch.float32), (262_145, torch.float32),
                                         (262_144, torch.bfloat16), (262_151, torch.bfloat16)],
                         ids=str)
def test_policy_rows_that_just_fit_on_chip(vocab, dtype):
    x, t = _data((1, 3, vocab), dtype, seed=37, ignore=False)
    old, ref, adv = _policy_inputs(x, t, 38)
    _check_policy(x, t, old, adv, ref, 0.1, "token", scales=(None,))


@pytest.mark.parametrize("view", VIEWS)
def test_policy_of_views(view):
    for dtype, vocab in ((torch.bfloat16, 1001), (torch.float32, 64)):
        x, t = _data((4, 6, vocab), dtype, seed=39)
        x, t = VIEWS[view](x, t)
        if t.numel() == 0:
            continue
        old, ref, adv = _policy_inputs(x, t, 40)
        _check_policy(x, t, old, adv, ref, 0.1, "token", scales=(None,))


@pytest.mark.parametrize("vocab", [65, 512])
def test_gradients_through_a_slice_and_saved_on_the_host(vocab):
    """The whole logits' gradient where the losses read a slice of them, and the same bits with
    saved tensors kept in host memory (where strided views come back contiguous)."""

    x, t = _data((4, 7, vocab), torch.bfloat16, seed=49)
    old, ref, adv = (v[:, 1:] for v in _policy_inputs(x, t, 50))
    leaf = x.detach().requires_grad_()
    results = []
    for hooks in (None, torch.autograd.graph.save_on_cpu()):
        if hooks:
            hooks.__enter__()
        cut, want = leaf[:, :-1], t[:, 1:]
        lp = kernels.token_log_probs(cut, want)
        pref, _ = kernels.preference_loss(cut, want, ref)
        pol, _ = kernels.policy_loss(cut, want, old, adv, reference_log_probs=ref, kl_coef=0.1)
        if hooks:
            hooks.__exit__(None, None, None)
        results.append([torch.autograd.grad(v, leaf, u, retain_graph=True)[0]
                        for v, u in ((lp, adv), (pref, None), (pol, None), (pol, None))])
    for got in results:
        for a, b in zip(got, results[0]):
            assert torch.equal(a, b) and (a[:, -1] == 0).all()
    _check_grad(results[0][0][:, :-1], x[:, :-1], t[:, 1:], adv)


def test_empty_batches_have_empty_gradients():
    x, t = _data((2, 3, 64), torch.bfloat16, seed=52)
    f = torch.zeros(t.shape, device=gu.DEV)
    for cut in ((slice(0, 0), slice(None)), (slice(None), slice(0, 0))):
        leaf = x[cut].detach().requires_grad_()
        loss, _ = kernels.policy_loss(leaf, t[cut], f[cut], f[cut])
        (dx,) = torch.autograd.grad(loss, leaf)
        assert math.isnan(loss.item()) and dx.shape == leaf.shape
        loss, _ = kernels.preference_loss(leaf, t[cut], f[cut])
        (dx,) = torch.autograd.grad(loss, leaf)
        assert dx.shape == leaf.shape
        lp = kernels.token_log_probs(leaf, t[cut])
        (dx,) = torch.autograd.grad(lp.sum(), leaf)
        assert dx.shape == leaf.shape


def test_second_derivatives_are_refused():
    x, t = _data((2, 3, 64), torch.float32, seed=53, ignore=False)
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    (dx,) = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad((dx * dx).sum(), x)


def test_compiled_graphs_agree():
    x, t = _data((2, 6, 501), torch.bfloat16, seed=47)
    old, ref, adv = _policy_inputs(x, t, 48)

    def run(leaf):
        lp = kernels.token_log_probs(leaf, t)
        pref, _ = kernels.preference_loss(leaf, t, ref)
        pol, _ = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1)
        return lp.sum() + pref + pol

    grads = []
    for f in (run, torch.compile(run, backend="aot_eager", fullgraph=True)):
        leaf = x.detach().requires_grad_()
        loss = f(leaf)
        loss.backward()
        grads.append((loss.detach(), leaf.grad))
    assert torch.equal(grads[0][0], grads[1][0])
    # Three gradients added in bf16, each rounded: half a step of the largest partial sums.
    assert (grads[0][1] - grads[1][1]).abs().max() <= 2 ** -7 * grads[0][1].abs().max()


def test_policy_2d_and_unclipped():
    x, t = _data((1, 50, 777), torch.float32, seed=27)
    old, ref, adv = _policy_inputs(x, t, 28, 0.9, 2.0)
    _check_policy(x[0], t[0], old[0], adv[0], ref[0], 0.05, "token", low=0.9, high=2.0)
    loss, _ = kernels.policy_loss(x[0], t[0], old[0], adv[0], clip_low=1.0, clip_high=math.inf)
    keep = t[0].cpu() != IGNORE
    r = (_logps64(x[0], t[0]) - old[0].double().cpu()).exp()
    want = (-adv[0].double().cpu() * r)[keep].mean().item()
    assert loss.item() == pytest.approx(want, abs=1e-5)


def test_policy_without_tokens_is_nan_with_zero_gradient():
    x, t = _data((2, 3, 64), torch.bfloat16, seed=29)
    t[:] = IGNORE
    old, ref, adv = (torch.zeros(t.shape, device=gu.DEV) for _ in range(3))
    for aggregate in ("token", "sequence"):
        leaf = x.detach().requires_grad_()
        loss, lp = kernels.policy_loss(leaf, t, old, adv, aggregate=aggregate)
        (dx,) = torch.autograd.grad(loss, leaf)
        assert math.isnan(loss.item()) and (dx == 0).all() and (lp == 0).all()
    loss, _ = kernels.policy_loss(x[:0], t[:0], old[:0], adv[:0])
    assert math.isnan(loss.item())


def test_policy_gradient_against_differences():
    """Central differences in 64 bits of the loss that the kernel evaluates, along a direction."""

    x, t = _data((2, 5, 24), torch.float32, seed=30)
    old, ref, adv = _policy_inputs(x, t, 31)
    leaf = x.detach().requires_grad_()
    loss, _ = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.2)
    (dx,) = torch.autograd.grad(loss, leaf)
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(32), dtype=torch.float64)
    h = 1e-5
    f = [_policy64(_logps64(x.double().cpu() + s * h * d, t), old, adv, ref, t, 0.2, 0.2, 0.2,
                   False)[0] for s in (1, -1)]
    want = ((f[0] - f[1]) / (2 * h)).item()
    assert (dx.double().cpu() * d).sum().item() == pytest.approx(want, rel=1e-4, abs=1e-6)


# ------------------------------------------------------- streams, graphs, repeats, sizes --


def _all_losses(x, t, old, adv, ref):
    leaf = x.detach().requires_grad_()
    lp = kernels.token_log_probs(leaf, t)
    (d0,) = torch.autograd.grad(lp, leaf, adv)
    pref, rewards = kernels.preference_loss(leaf, t, ref)
    (d1,) = torch.autograd.grad(pref, leaf)
    pol, lp2 = kernels.policy_loss(leaf, t, old, adv, reference_log_probs=ref, kl_coef=0.1)
    (d2,) = torch.autograd.grad(pol, leaf)
    return [lp.detach(), d0, pref.detach(), rewards, d1, pol.detach(), lp2, d2]


@pytest.mark.parametrize("vocab", [1000, 50257])
def test_repeats_streams_and_graphs_give_the_same_bits(vocab):
    x, t = _data((4, 16, vocab), torch.bfloat16, seed=41)
    old, ref, adv = _policy_inputs(x, t, 42)
    want = _all_losses(x, t, old, adv, ref)
    again = _all_losses(x, t, old, adv, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _all_losses(x, t, old, adv, ref)
    torch.cuda.current_stream().wait_stream(side)
    # Two captured graphs, replayed on new inputs in turn.
    sx, sold = torch.zeros_like(x), torch.zeros_like(old)
    graphs, outs = [], []
    with torch.cuda.stream(side):
        _all_losses(sx, t, sold, adv, ref)
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all_losses(sx, t, sold, adv, ref))
        graphs.append(g)
    sx.copy_(x)
    sold.copy_(old)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for got in (again, other, *outs):
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_many_rows():
    x, t = _data((2, 20000, 16), torch.bfloat16, seed=43)
    lp = kernels.token_log_probs(x, t)
    _check_logps(lp, x, t)
    old, ref, adv = _policy_inputs(x, t, 44)
    _check_policy(x, t, old, adv, ref, 0.1, "sequence", scales=(None,))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [2, 9, 333, 1003, 2048, 4103, 8192])
def test_many_short_rows(vocab, dtype):
    """Enough rows that a warp takes a row each (4736 on B200), aligned and not, whole batches and
    a slice of them, with rows that have no target and rows of every mask."""

    shape = (5, 1201, vocab)
    x, t = _data(shape, dtype, seed=54)
    x[0, 0, 1:] = -math.inf
    x[0, 2, :] = torch.finfo(dtype).min
    t[0, :3] = 0
    x[1, 1, :] = math.nan
    t[1, 1] = IGNORE
    clean = x.clone()
    clean[1, 1] = 0.0
    cut = (slice(None), slice(1, None))
    for view in (slice(None), cut):
        leaf = x[view].detach().requires_grad_()
        lp = kernels.token_log_probs(leaf, t[view])
        _check_logps(lp.detach(), clean[view], t[view])
        dlp = gu.randn(t[view].shape, 55)
        (dx,) = torch.autograd.grad(lp, leaf, dlp)
        _check_grad(dx, clean[view], t[view], dlp)
    old, ref, adv = _policy_inputs(clean, t, 56)
    old[torch.isinf(old)] = -60.0
    ref[torch.isinf(ref)] = -60.0
    _check_policy(clean, t, old, adv, ref, 0.1, "sequence", scales=(None, 0.25))


@pytest.mark.parametrize("aggregate", ["token", "sequence"])
@pytest.mark.parametrize("shape", [(3, 30000, 12), (9000, 9, 12)], ids=str)
def test_policy_weights_of_many_tokens(shape, aggregate):
    """More tokens than one CTA counts, in few sequences and in many, some without a target."""

    x, t = _data(shape, torch.float32, seed=57)
    t[::3] = IGNORE
    old, ref, adv = _policy_inputs(x, t, 58)
    _check_policy(x, t, old, adv, ref, 0.1, aggregate, scales=(None,))


def test_offsets_beyond_32_bits():
    """Rows whose byte and element offsets pass 2^31 and 2^32."""

    rows, vocab = 33000, 131072
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=gu.DEV)
    t = torch.full((rows,), IGNORE, device=gu.DEV)
    at = torch.tensor([0, 16383, 16385, 32767, 32769, rows - 1], device=gu.DEV)
    x[at] = gu.randn((len(at), vocab), 45, torch.bfloat16)
    t[at] = torch.arange(len(at), device=gu.DEV) * 1111
    x.requires_grad_()
    lp = kernels.token_log_probs(x, t)
    _check_logps(lp.detach()[at], x.detach()[at], t[at])
    dlp = gu.randn((rows,), 46)
    (dx,) = torch.autograd.grad(lp, x, dlp)
    _check_grad(dx[at], x.detach()[at], t[at], dlp[at])
    assert torch.count_nonzero(dx[1:16383]).item() == 0


# ------------------------------------------------------------------------------ refusals --


def test_refusals():
    x, t = _data((2, 3, 32), torch.float32, seed=51)
    f = torch.zeros(t.shape, device=gu.DEV)
    bad = [
        lambda: kernels.token_log_probs(x.cpu(), t),
        lambda: kernels.token_log_probs(x, t.cpu()),
        lambda: kernels.token_log_probs(x.double(), t),
        lambda: kernels.token_log_probs(x, t.int()),
        lambda: kernels.token_log_probs(x, t[:, :2]),
        lambda: kernels.token_log_probs(x[..., :0], t),
        lambda: kernels.token_log_probs(x[None], t[None]),
        lambda: kernels.preference_loss(x[:1], t[:1], f[:1]),
        lambda: kernels.preference_loss(x[0], t[0], f[0]),
        lambda: kernels.preference_loss(x, t, f[:, 0]),
        lambda: kernels.preference_loss(x, t, f, label_smoothing=1.5),
        lambda: kernels.preference_loss(x, t, f, beta=math.nan),
        lambda: kernels.policy_loss(x, t, f, f, kl_coef=0.1),
        lambda: kernels.policy_loss(x, t, f, f[:, :1]),
        lambda: kernels.policy_loss(x, t, f, f, clip_low=-0.1),
        lambda: kernels.policy_loss(x, t, f, f, clip_high=math.nan),
        lambda: kernels.policy_loss(x, t, f, f, aggregate="sum"),
        lambda: kernels.policy_loss(x, t, f, f, expected_grad=0.0),
        lambda: kernels.policy_loss(x, t, f, f, expected_grad=math.nan),
        lambda: kernels.policy_loss(x, t, f.cpu(), f),
    ]
    for call in bad:
        with pytest.raises(TritonLogitLossUnavailable):
            call()
