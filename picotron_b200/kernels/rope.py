"""RoPE entry point with the reference's name and contract.

``triton_apply_rotary_embedding`` keeps the signature and error type of the reference
(src/picotron/nn/triton_kernels/rope.py:52-91) but, unlike the reference's
inference-only kernel, supports autograd (the backward is the inverse rotation on the
same kernel) and reads strided [B, H, S, D] views in place without ``.contiguous()``.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from picotron_b200 import ops
from picotron_b200.errors import TritonRoPEUnavailable


def _validate(states: Tensor, cosine: Tensor, sine: Tensor) -> None:
    """Reject inputs the kernel cannot take (reference triton_kernels/rope.py:56-74)."""

    for t in (states, cosine, sine):
        if not isinstance(t, Tensor):
            raise TritonRoPEUnavailable("RoPE expects tensors.")
    if not states.is_cuda or not cosine.is_cuda or not sine.is_cuda:
        raise TritonRoPEUnavailable("sm_100a RoPE requires CUDA tensors.")
    ops.check_device(states.device, TritonRoPEUnavailable)
    if (
        states.ndim != 4
        or states.size(-1) != cosine.size(-1) * 2
        or cosine.shape != sine.shape
        or cosine.size(0) != states.size(-2)
    ):
        raise TritonRoPEUnavailable("sm_100a RoPE requires compatible [B,H,S,D] / [S,D/2] tensors.")


def triton_apply_rotary_embedding(
    states: Tensor, cosine: Tensor, sine: Tensor, *, layout: str = "interleaved"
) -> Tensor:
    """Rotate ``(batch, heads, sequence, head_dim)`` states by the RoPE tables.

    ``layout="interleaved"`` (default) rotates pairs (x[2i], x[2i+1]) exactly like the
    reference; ``layout="rotate_half"`` rotates (x[i], x[i + D/2]).
    """

    _validate(states, cosine, sine)
    if layout not in ops.LAYOUTS:
        raise TritonRoPEUnavailable(f"unknown RoPE layout {layout!r}")
    return torch.ops.picotron_b200.rope(states, cosine, sine, ops.LAYOUTS[layout])


def rotary_frequencies(rotary_dim: int, theta: float = 10_000.0, *, scaling: str | None = None,
                       factor: float = 1.0, original_length: int | None = None,
                       beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[Tensor, float]:
    """Frequencies of :func:`apply_rotary_positions` (float64 [rotary_dim / 2]) and its ``scale``.

    Without ``scaling``: ``theta ** (-2 i / rotary_dim)`` and 1, the reference's
    (src/picotron/nn/rope.py:13-32) in 64 bits. For contexts ``factor`` times as long as the
    model was trained on:

    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"ntk"``: theta raised to ``theta * factor ** (R / (R - 2))``, which keeps the highest
      frequency and divides the lowest by ``factor``;
    * ``"yarn"``: by wavelength. A pair that turns more than ``beta_fast`` times within
      ``original_length`` tokens keeps its frequency, one that turns less than ``beta_slow``
      times has it divided by ``factor``, with a linear ramp over the pair index between; the
      scale is ``0.1 ln(factor) + 1`` (Peng et al., "YaRN: Efficient Context Window Extension of
      Large Language Models", 2023).
    """

    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError("rotary_dim must be even and at least 2.")
    if theta <= 0:
        raise ValueError("rope_theta must be positive.")
    if factor < 1.0:
        raise ValueError("the scaling factor must be at least 1.")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown RoPE scaling {scaling!r}")
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    scale = 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair.")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv_freq = torch.pow(torch.tensor(float(theta), dtype=torch.float64), -exponent)
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("yarn scaling needs original_length.")
        if theta == 1.0:
            raise ValueError("yarn scaling needs theta other than 1.")
        # The pair index whose wavelength fits `turns` times into original_length tokens.
        pair = lambda turns: (rotary_dim * math.log(original_length / (turns * 2 * math.pi))  # noqa: E731
                              / (2 * math.log(theta)))
        low = max(math.floor(pair(beta_fast)), 0)
        high = min(math.ceil(pair(beta_slow)), rotary_dim - 1)
        index = torch.arange(rotary_dim // 2, dtype=torch.float64)
        ramp = ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        inv_freq = inv_freq / factor * ramp + inv_freq * (1.0 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return inv_freq.to(device), scale


def apply_rotary_positions(query: Tensor, key: Tensor, positions: Tensor, inv_freq: Tensor, *,
                           layout: str = "interleaved",
                           scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """Rotate query and key ``(batch, heads, sequence, head_dim)`` by explicit positions.

    ``positions`` ([S] or [B, S], int64) may be in any order and far: packed documents that
    restart at 0, left-padded batches, the next token of a decoding batch. Angles are
    ``positions * inv_freq`` in 64 bits, so no table is built or kept; ``inv_freq`` (float64
    [R / 2]) and ``scale`` come from :func:`rotary_frequencies`, on the states' device. With
    R smaller than head_dim only the first R elements of a head are rotated. Strided views are
    read in place; with autograd for query and key.
    """

    for t in (query, key, positions, inv_freq):
        if not isinstance(t, Tensor):
            raise TritonRoPEUnavailable("RoPE expects tensors.")
        if not t.is_cuda:
            raise TritonRoPEUnavailable("sm_100a RoPE requires CUDA tensors.")
    if layout not in ops.LAYOUTS:
        raise TritonRoPEUnavailable(f"unknown RoPE layout {layout!r}")
    return ops.rope_positions(query, key, positions, inv_freq, ops.LAYOUTS[layout], float(scale))
