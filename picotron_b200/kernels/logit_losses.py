"""Post-training losses that read logits: log-probabilities, preference and policy losses.

The reference's post-training package (src/picotron_sft, src/picotron_dpo) evaluates such losses
in PyTorch; these run the sm_100a kernels of ``csrc/logit_loss.cu`` through
``torch.ops.picotron_b200.*``, next to ``cross_entropy``. All of them take

* ``logits`` [B, S, V] (or [N, V], one sequence) in float32, float16 or bfloat16, strided views
  included (the class dimension is copied if it is not contiguous), and
* ``targets`` [B, S] (or [N]), int64, where ``targets[b, s]`` is the token that
  ``logits[b, s]`` predicts (shift the ids before the call) and ``ignore_index`` marks positions
  without one: prompts and padding. Their logits are not read and get a gradient of zeros,
  whatever they hold.

The logits gradient is the only one: per-token inputs and returned log-probabilities or rewards
of the losses carry none. Targets outside [0, V) give NaN and set the library's device error
word (a kernel cannot raise); their logits get a gradient of zeros. NaN, and what has no value in
64 bits either, in the logits or per-token inputs of a position with a target makes the loss and
that position's gradient NaN (in the preference loss, its pair's). Calls that cannot run raise
:class:`TritonLogitLossUnavailable`.
"""

from __future__ import annotations

import torch
from torch import Tensor

from picotron_b200 import ops
from picotron_b200.errors import TritonLogitLossUnavailable


_FP32 = torch.finfo(torch.float32)


def _check_tensors(**tensors) -> None:
    for name, t in tensors.items():
        if not isinstance(t, Tensor):
            raise TritonLogitLossUnavailable(f"{name} must be a tensor.")
        if not t.is_cuda:
            raise TritonLogitLossUnavailable(f"sm_100a losses require CUDA tensors ({name}).")


def _per_token(t: Tensor, targets: Tensor, name: str) -> Tensor:
    if t.shape != targets.shape:
        raise TritonLogitLossUnavailable(
            f"{name} must have the targets' shape {tuple(targets.shape)}, not {tuple(t.shape)}")
    if t.dtype is torch.float32 and not t.requires_grad:
        return t
    return t.detach().to(torch.float32)


def token_log_probs(logits: Tensor, targets: Tensor, *, ignore_index: int = -100) -> Tensor:
    """``log_softmax(logits)[..., targets]`` in float32, shaped like ``targets``; 0 where the
    target is ``ignore_index``.

    One pass over the logits of rows with a target; with autograd (any gradient of the result
    costs one more read and one write of the logits' size). Under ``torch.no_grad`` this scores
    a batch with a frozen reference model for the losses below.
    """

    _check_tensors(logits=logits, targets=targets)
    return ops.token_logps(logits, targets, int(ignore_index))[0]


def preference_loss(logits: Tensor, targets: Tensor, reference_log_probs: Tensor, *,
                    beta: float = 0.1, label_smoothing: float = 0.0,
                    ignore_index: int = -100) -> tuple[Tensor, Tensor]:
    """Preference loss of paired log ratios; returns ``(loss, rewards)``.

    ``logits`` [2P, S, V] holds P chosen sequences, then their P rejected ones;
    ``reference_log_probs`` [2P, S] is :func:`token_log_probs` of the frozen reference model.
    With ``rewards[q] = beta * sum(log_probs - reference_log_probs)`` over the positions of q
    that have a target and ``z = rewards[:P] - rewards[P:]``::

        loss = mean((1 - label_smoothing) * softplus(-z) + label_smoothing * softplus(z))

    ``rewards`` [2P] is returned for logging and carries no gradient.
    """

    _check_tensors(logits=logits, targets=targets, reference_log_probs=reference_log_probs)
    reference = _per_token(reference_log_probs, targets, "reference_log_probs")
    loss, rewards, _, _ = ops.preference_loss(
        logits, targets, reference, float(beta), float(label_smoothing), int(ignore_index))
    return loss, rewards


def policy_loss(logits: Tensor, targets: Tensor, old_log_probs: Tensor, advantages: Tensor, *,
                reference_log_probs: Tensor | None = None, kl_coef: float = 0.0,
                clip_low: float = 0.2, clip_high: float = 0.2, aggregate: str = "token",
                ignore_index: int = -100,
                expected_grad: float | None = None) -> tuple[Tensor, Tensor]:
    """Clipped policy-gradient loss with a KL term; returns ``(loss, log_probs)``.

    With ``r = exp(log_probs - old_log_probs)``, ``A = advantages`` ([B], one per sequence, or
    the targets' shape) and ``g = reference_log_probs - log_probs``, a position with a target
    costs::

        max(-A * r, -A * clip(r, 1 - clip_low, 1 + clip_high)) + kl_coef * (exp(g) - g - 1)

    (no second term for ``kl_coef`` 0). ``aggregate="token"`` averages over all positions with a
    target, ``"sequence"`` over the means of the sequences that have any; the loss is NaN when
    there are none. ``log_probs`` is shaped like ``targets`` (0 where ignored) and carries no
    gradient.

    Where the logits need a gradient it is formed with the loss, in one pass over them, for the
    gradient that the loss is expected to receive; ``backward`` then only compares. That is 1 by
    default (``loss.backward()``); give ``expected_grad`` where the loss is scaled before it, e.g.
    ``1 / steps`` for ``(loss / steps).backward()`` or a loss scaler's scale. Any other gradient
    is still right but costs a pass to rescale, and rounds the result once more: to the logits'
    type's smallest steps at the expected factor, so a guess that is far too small loses what is
    below them. float16 logits form their gradient in ``backward`` unless ``expected_grad`` is
    given, since it would underflow without the loss scale.
    """

    _check_tensors(logits=logits, targets=targets, old_log_probs=old_log_probs,
                   advantages=advantages)
    if aggregate not in ("token", "sequence"):
        raise TritonLogitLossUnavailable(
            f'aggregate must be "token" or "sequence", not {aggregate!r}')
    if expected_grad is not None and not _FP32.tiny <= abs(expected_grad) <= _FP32.max:
        raise TritonLogitLossUnavailable("expected_grad must be finite and not 0 in float32.")
    reference = None
    if kl_coef != 0.0:
        if reference_log_probs is None:
            raise TritonLogitLossUnavailable("a KL term needs reference_log_probs.")
        _check_tensors(reference_log_probs=reference_log_probs)
        reference = _per_token(reference_log_probs, targets, "reference_log_probs")
    if targets.dim() == 2 and advantages.shape == targets.shape[:1]:
        advantages = advantages[:, None].expand(targets.shape)
    loss, log_probs, _, _ = ops.policy_loss(
        logits, targets, _per_token(old_log_probs, targets, "old_log_probs"),
        _per_token(advantages, targets, "advantages"), reference, float(clip_low),
        float(clip_high), float(kl_coef), aggregate == "sequence", int(ignore_index),
        None if expected_grad is None else float(expected_grad))
    return loss, log_probs
