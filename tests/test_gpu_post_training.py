"""A post-training run of the operators together, as a trainer uses them: a frozen reference model
scores packed sequences (RoPE by positions that restart in every document), the preference and
the policy loss train the policy through the same kernels, and the 8-bit AdamW takes the steps.

Losses and parameter gradients are compared with the same model in float64 built from plain
operations. The float32 model's products sum up to 512 terms (VOCAB) six times in a row, so a
gradient is off by at most about 6 * 512 * 2^-24 < 2e-4 of the largest terms that meet in it;
2e-3 of the parameter's largest gradient leaves room for terms that cancel.
"""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

import gpu_utils as gu
from picotron_b200 import _capi
from picotron_b200.kernels import (
    AdamW8bit,
    AdamWStepWithFallback,
    policy_loss,
    preference_loss,
    token_log_probs,
)
from picotron_b200.modules import RMSNorm, RotaryEmbedding, SwiGLU

pytestmark = pytest.mark.gpu

B, S, HEADS, D, VOCAB, INTER = 4, 48, 4, 32, 509, 96
HIDDEN = HEADS * D
IGNORE = -100
SCALING = {"scaling": "yarn", "factor": 4.0, "original_length": 64}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


class Model(nn.Module):
    def __init__(self, fast: bool) -> None:
        super().__init__()
        self.embedding = nn.Embedding(VOCAB, HIDDEN)
        self.norm = RMSNorm(HIDDEN, 1e-5, use_triton_rmsnorm=fast)
        self.q_proj = nn.Linear(HIDDEN, HIDDEN, bias=False)
        self.k_proj = nn.Linear(HIDDEN, HIDDEN // 2, bias=False)
        self.rope = RotaryEmbedding(D, 10_000.0, use_triton_rope=fast)
        self.rope.rotary_dim, self.rope.scaling = 24, SCALING
        self.mlp = SwiGLU(HIDDEN, INTER, use_triton_swiglu=fast)
        self.output = nn.Linear(HIDDEN, VOCAB, bias=False)

    def forward(self, ids, positions):
        x = self.embedding(ids)
        n = self.norm(x)
        q = self.q_proj(n).view(B, S, HEADS, D).transpose(1, 2)
        k = self.k_proj(n).view(B, S, HEADS // 2, D).transpose(1, 2)
        q, k = self.rope(q, k, positions)
        k = k.repeat_interleave(2, dim=1)
        mixed = q * torch.sigmoid((q * k).sum(-1, keepdim=True) / D ** 0.5) + k
        h = x + mixed.transpose(1, 2).reshape(B, S, HIDDEN)
        return self.output(h + self.mlp(h))


def _batch(seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, (B, S), generator=g)
    targets = torch.full_like(ids, IGNORE)
    targets[:, 9:-7] = ids[:, 10:-6]  # shifted by one; prompt and padding ignored
    at = torch.arange(S).expand(B, S)
    positions = torch.where(at < 20, at, at - 20) + 1000 * torch.arange(B)[:, None]
    return ids, targets, positions


def _logps64(logits, targets):
    lp = torch.log_softmax(logits.double(), -1)
    lp = lp.gather(-1, targets.clamp_min(0)[..., None])[..., 0]
    return torch.where(targets == IGNORE, torch.zeros_like(lp), lp)


def _plain_preference(lp, ref, beta):
    rewards = beta * (lp - ref).sum(-1)
    z = rewards[: B // 2] - rewards[B // 2:]
    return -torch.nn.functional.logsigmoid(z).mean()


def _plain_policy(lp, old, ref, adv, keep, kl):
    r = (lp - old).exp()
    a = adv[:, None]
    term = torch.maximum(-a * r, -a * r.clamp(0.8, 1.2))
    term = term + kl * ((ref - lp).exp() - (ref - lp) - 1)
    return (term * keep).sum() / keep.sum()


def _models():
    torch.manual_seed(5)
    policy = Model(True).to(gu.DEV)
    reference = copy.deepcopy(policy)
    with torch.no_grad():
        for p in policy.parameters():  # a policy that has moved away from its reference
            p.add_(0.02 * gu.randn(p.shape, p.numel()))
    plain = Model(False).double()
    plain.load_state_dict({k: v.double().cpu() for k, v in policy.state_dict().items()})
    plain_reference = Model(False).double()
    plain_reference.load_state_dict({k: v.double().cpu()
                                     for k, v in reference.state_dict().items()})
    return policy, reference, plain, plain_reference


def _compare(policy, plain, loss, want):
    assert abs(loss.item() - want.item()) <= 1e-4 * max(1.0, abs(want.item()))
    for (name, p), q in zip(policy.named_parameters(), plain.parameters()):
        err = (p.grad.double().cpu() - q.grad).abs().max().item()
        assert err <= 2e-3 * q.grad.abs().max().item(), f"{name}: {err}"


def _check_first_step(policy, before, lr, decay):
    """AdamW's first step is lr * g / (|g| + eps) whatever the moments' precision."""

    for p, old in zip(policy.parameters(), before):
        g = p.grad.double()
        want = old.double() * (1 - lr * decay) - lr * g / (g.abs() + 1e-8)
        assert (p.detach().double() - want).abs().max().item() <= lr * 2.0 ** -18 + 2.0 ** -22


def test_preference_step():
    policy, reference, plain, plain_reference = _models()
    ids, targets, positions = _batch(1)
    on = [t.to(gu.DEV) for t in (ids, targets, positions)]
    with torch.no_grad():
        ref = token_log_probs(reference(on[0], on[2]), on[1])
    loss, rewards = preference_loss(policy(on[0], on[2]), on[1], ref, beta=0.3)
    optimizer = AdamW8bit(policy.parameters(), lr=1e-3, weight_decay=0.1)
    loss.backward()
    with torch.no_grad():
        ref64 = _logps64(plain_reference(ids, positions), targets)
    want = _plain_preference(_logps64(plain(ids, positions), targets), ref64, 0.3)
    want.backward()
    _compare(policy, plain, loss, want)
    assert rewards.shape == (B,) and not policy.rope._triton_fallback_warned
    before = [p.detach().clone() for p in policy.parameters()]
    AdamWStepWithFallback(use_triton=True).step(optimizer)
    _check_first_step(policy, before, 1e-3, 0.1)
    assert _capi.take_device_error() == 0


@pytest.mark.parametrize("micro", [1, 2])
def test_policy_step_with_accumulation(micro):
    policy, reference, plain, plain_reference = _models()
    optimizer = AdamW8bit(policy.parameters(), lr=1e-3, weight_decay=0.0)
    adv = torch.tensor([1.0, -0.5, 0.25, -2.0])
    total = want_total = 0.0
    for k in range(micro):
        ids, targets, positions = _batch(10 + k)
        on = [t.to(gu.DEV) for t in (ids, targets, positions)]
        with torch.no_grad():
            ref = token_log_probs(reference(on[0], on[2]), on[1])
            old = token_log_probs(policy(on[0], on[2]), on[1]) + 0.05  # ratios below 1, unclipped
        loss, lp = policy_loss(policy(on[0], on[2]), on[1], old, adv.to(gu.DEV),
                               reference_log_probs=ref, kl_coef=0.1, expected_grad=1.0 / micro)
        (loss / micro).backward()
        with torch.no_grad():
            ref64 = _logps64(plain_reference(ids, positions), targets)
            old64 = _logps64(plain(ids, positions), targets) + 0.05
        want = _plain_policy(_logps64(plain(ids, positions), targets), old64, ref64, adv.double(),
                             (targets != IGNORE).double(), 0.1)
        (want / micro).backward()
        total, want_total = total + loss.detach() / micro, want_total + want.detach() / micro
        assert (lp[on[1] != IGNORE] < 0).all() and (lp[on[1] == IGNORE] == 0).all()
    _compare(policy, plain, total, want_total)
    before = [p.detach().clone() for p in policy.parameters()]
    AdamWStepWithFallback(use_triton=True).step(optimizer)
    _check_first_step(policy, before, 1e-3, 0.0)
    assert all(optimizer.state[p]["step"] == 1 for p in policy.parameters())
    assert _capi.take_device_error() == 0
