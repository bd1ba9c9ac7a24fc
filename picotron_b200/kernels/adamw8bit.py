"""AdamW with its moments in 8 bits.

``AdamW8bit`` is a ``torch.optim.Optimizer`` whose two moments take 2.03 bytes per parameter
(8-bit codes in blocks of 256 with an fp32 scale each) instead of 8, with one sm_100a launch per
step for a whole list of tensors. ``adamw8bit_step`` is the step on plain tensor lists and
``adamw8bit_moments`` the fp32 moments that the states stand for. The update is
torch.optim.AdamW's (decoupled weight decay, no amsgrad), which the reference's training loop
builds (src/picotron/training/train_loop.py:302-325); the codes are described at
``pt_adamw8_step`` in ``include/picotron_b200.h``.
"""

from __future__ import annotations

from collections import defaultdict
from collections.abc import Sequence

import torch
from torch import Tensor
from torch.optim import Optimizer

from picotron_b200 import _capi, ops
from picotron_b200.errors import TritonAdamWUnavailable

BLOCK = 256  # elements that share a scale
LEAST_EPS = 1e-12  # what a block's exp_avg_sq may be dropped next to (see pt_adamw8_step)
_STATE = {"exp_avg_codes": torch.int8, "exp_avg_scales": torch.float32,
          "exp_avg_sq_codes": torch.uint8, "exp_avg_sq_scales": torch.float32}


def _scales(numel: int) -> int:
    return (numel + BLOCK - 1) // BLOCK


def _addresses(name: str, tensors: Sequence[Tensor], sizes: Sequence[int], dtype: torch.dtype,
               device: int) -> list[int]:
    """Data addresses of contiguous tensors with these sizes, dtype and CUDA device."""

    if len(tensors) != len(sizes):
        raise TritonAdamWUnavailable("all tensor lists must have the same length.")
    for t, n in zip(tensors, sizes):
        if (t.dtype is not dtype or t.numel() != n or t.get_device() != device
                or not t.is_contiguous()):
            raise TritonAdamWUnavailable(
                f"{name} must be contiguous {dtype} tensors of {n} elements on one CUDA device; "
                f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    return [t.data_ptr() for t in tensors]


def _state_addresses(lists: Sequence[Sequence[Tensor]], sizes: Sequence[int], device: int):
    scales = [(n + BLOCK - 1) // BLOCK for n in sizes]
    return [_addresses(name, values, scales if name.endswith("scales") else sizes, dtype, device)
            for values, (name, dtype) in zip(lists, _STATE.items())], scales


def _per_tensor(value, count: int, name: str) -> list:
    if isinstance(value, Sequence):
        if len(value) != count:
            raise TritonAdamWUnavailable(f"{name} must be one value or one per tensor.")
        return list(value)
    return [value] * count


def _refuse_shared(spans: list[tuple[int, int]]) -> None:
    """(address, bytes) of all that a step writes. Memory that two entries share, of one list or of
    two, would be updated twice at once."""

    end = 0
    for at, size in sorted(spans):
        if at < end and size:
            raise TritonAdamWUnavailable("two of the parameters and states share memory.")
        if size:
            end = at + size


@torch.no_grad()
def adamw8bit_step(params: Sequence[Tensor], grads: Sequence[Tensor],
                   exp_avg_codes: Sequence[Tensor], exp_avg_scales: Sequence[Tensor],
                   exp_avg_sq_codes: Sequence[Tensor], exp_avg_sq_scales: Sequence[Tensor], *,
                   step: int | Sequence[int], lr: float | Sequence[float], beta1: float = 0.9,
                   beta2: float = 0.999, eps: float = 1e-8,
                   weight_decay: float | Sequence[float] = 0.01, maximize: bool = False) -> None:
    """One AdamW step, in place, on lists of contiguous CUDA tensors of one device and dtype
    (float32, float16 or bfloat16; gradients like their parameters).

    Per tensor of n elements the state is ``exp_avg_codes`` int8 [n], ``exp_avg_scales`` float32
    [ceil(n / 256)], ``exp_avg_sq_codes`` uint8 [n] and ``exp_avg_sq_scales`` float32 [ceil(n /
    256)] (any shape with that many elements; zeros before the first step). ``step`` counts this
    step (1 for the first); ``step``, ``lr`` and ``weight_decay`` are one value or one per tensor.
    ``eps`` is at least 1e-12: squares below 5e-29 are not kept, which leaves ``eps`` alone in the
    denominator. A gradient that is not finite, or whose square is not (beyond 1.8e19), spoils the
    moments of its block of 256.
    Nothing is changed when the call is refused. The step's scalars are host values, so a captured
    CUDA graph would replay the same step count.
    """

    _checked_step(params, grads, exp_avg_codes, exp_avg_scales, exp_avg_sq_codes,
                  exp_avg_sq_scales, step, lr, beta1, beta2, eps, weight_decay, maximize)()


def _checked_step(params, grads, exp_avg_codes, exp_avg_scales, exp_avg_sq_codes,
                  exp_avg_sq_scales, step, lr, beta1, beta2, eps, weight_decay, maximize):
    """adamw8bit_step's checks; returns the step itself, to be called under no_grad."""

    count = len(params)
    if count == 0 and not any(map(len, (grads, exp_avg_codes, exp_avg_scales, exp_avg_sq_codes,
                                        exp_avg_sq_scales))):
        return lambda: None
    if count == 0:
        raise TritonAdamWUnavailable("all tensor lists must have the same length.")
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and eps >= LEAST_EPS):
        raise TritonAdamWUnavailable(f"betas must be in [0, 1) and eps at least {LEAST_EPS}.")
    steps = _per_tensor(step, count, "step")
    if min(steps) < 1:
        raise TritonAdamWUnavailable("step counts the step that is taken: at least 1.")
    lrs, decays = _per_tensor(lr, count, "lr"), _per_tensor(weight_decay, count, "weight_decay")
    first = params[0]
    ops.check_device(first.device, TritonAdamWUnavailable)
    code = ops._dtype_code(first, TritonAdamWUnavailable)
    dtype, device = first.dtype, first.get_device()
    sizes = [p.numel() for p in params]
    at_params = _addresses("parameters", params, sizes, dtype, device)
    at_grads = _addresses("gradients", grads, sizes, dtype, device)
    for p, g in zip(params, grads):
        if p.shape != g.shape:
            raise TritonAdamWUnavailable("parameters and gradients must have the same shapes.")
    at_states, scales = _state_addresses(
        (exp_avg_codes, exp_avg_scales, exp_avg_sq_codes, exp_avg_sq_scales), sizes, device)
    width = first.element_size()
    extents = ([n * width for n in sizes], sizes, [4 * n for n in scales])
    _refuse_shared([span for at, which in zip((at_params, *at_states), (0, 1, 2, 1, 2))
                    for span in zip(at, extents[which])])

    def run() -> None:
        with ops._OnDevice(first.device):
            _capi.adamw8_step(at_params, at_grads, *at_states, sizes, steps, lrs, decays, beta1,
                              beta2, eps, maximize, code, ops._raw_stream(first.device),
                              TritonAdamWUnavailable)
        # As an in-place torch operation does: a backward that saved a parameter notices.
        torch.autograd.graph.increment_version(params)

    return run


@torch.no_grad()
def adamw8bit_moments(exp_avg_codes: Sequence[Tensor], exp_avg_scales: Sequence[Tensor],
                      exp_avg_sq_codes: Sequence[Tensor],
                      exp_avg_sq_scales: Sequence[Tensor]) -> tuple[list[Tensor], list[Tensor]]:
    """The fp32 ``(exp_avg, exp_avg_sq)`` lists that 8-bit states stand for, shaped like their
    codes: for inspection, or to carry on with an optimizer that keeps 32-bit states."""

    held = (exp_avg_codes, exp_avg_scales, exp_avg_sq_codes, exp_avg_sq_scales)
    if not any(map(len, held)):
        return [], []
    if len(exp_avg_codes) == 0:
        raise TritonAdamWUnavailable("all tensor lists must have the same length.")
    device = exp_avg_codes[0].device
    ops.check_device(device, TritonAdamWUnavailable)
    sizes = [c.numel() for c in exp_avg_codes]
    at_states, _ = _state_addresses(held, sizes, exp_avg_codes[0].get_device())
    exp_avg, exp_avg_sq = ([torch.empty(c.shape, dtype=torch.float32, device=device)
                            for c in exp_avg_codes] for _ in range(2))
    with ops._OnDevice(device):
        _capi.adamw8_moments(*at_states, sizes, [t.data_ptr() for t in exp_avg],
                             [t.data_ptr() for t in exp_avg_sq], ops._raw_stream(device),
                             TritonAdamWUnavailable)
    return exp_avg, exp_avg_sq


class AdamW8bit(Optimizer):
    """AdamW whose moments are held in 8 bits (see the module's description).

    Parameters: dense contiguous CUDA tensors in float32, float16 or bfloat16, updated in their
    own dtype (no separate master copy). Arguments as torch.optim.AdamW's, with ``eps`` at least
    1e-12; amsgrad is not offered. ``state_dict`` holds the codes and scales; ``load_state_dict``
    keeps their dtypes.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *,
                 maximize: bool = False) -> None:
        if lr < 0 or weight_decay < 0:
            raise ValueError("lr and weight_decay must be >= 0")
        if not eps >= LEAST_EPS:
            raise ValueError(f"eps must be at least {LEAST_EPS}: {eps}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas must be in [0, 1): {betas}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      maximize=maximize))

    def _new_state(self, p: Tensor) -> dict:
        sizes = {name: _scales(p.numel()) if name.endswith("scales") else p.shape
                 for name in _STATE}
        return {"step": 0, **{name: torch.zeros(sizes[name], dtype=dtype, device=p.device)
                              for name, dtype in _STATE.items()}}

    @torch.no_grad()
    def step(self, closure=None):
        """One step over all parameters that have a gradient: one launch per device, dtype and
        (betas, eps, maximize)."""

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = defaultdict(list)
        for group in self.param_groups:
            key = (float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]),
                   bool(group["maximize"]))
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse or not p.is_cuda:
                    raise TritonAdamWUnavailable("AdamW8bit takes dense CUDA parameters.")
                calls[(p.device, p.dtype, *key)].append((p, group))
        steps = []  # all checked before the first is taken: a refused step changes nothing
        for (_, _, beta1, beta2, eps, maximize), items in calls.items():
            params = [p for p, _ in items]
            # Not self.state[p], which would leave an empty entry behind a refused step.
            states = [self.state.get(p) or self._new_state(p) for p in params]
            steps.append((params, states, _checked_step(
                params, [p.grad for p in params], *([s[name] for s in states] for name in _STATE),
                [s["step"] + 1 for s in states], [float(g["lr"]) for _, g in items], beta1, beta2,
                eps, [float(g["weight_decay"]) for _, g in items], maximize)))
        for params, states, run in steps:
            run()
            for p, s in zip(params, states):
                s["step"] += 1
                self.state[p] = s
        return loss

    def moments(self) -> dict[Tensor, tuple[Tensor, Tensor]]:
        """The fp32 ``(exp_avg, exp_avg_sq)`` of every parameter that has taken a step."""

        result = {}
        devices = defaultdict(list)
        for p, s in self.state.items():
            devices[p.device].append((p, s))
        for items in devices.values():
            exp_avg, exp_avg_sq = adamw8bit_moments(*([s[name] for _, s in items]
                                                      for name in _STATE))
            result.update({p: pair for (p, _), *pair in zip(items, exp_avg, exp_avg_sq)})
        return {p: tuple(pair) for p, pair in result.items()}

    def load_state_dict(self, state_dict) -> None:
        """torch's, with codes and scales kept in their own dtypes (the base class would cast
        them to the parameters')."""

        for held in state_dict["state"].values():
            if not {"step", *_STATE} <= held.keys():
                raise ValueError("the state is not an AdamW8bit's: it lacks codes or scales")
        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for index, p in zip(saved["params"], group["params"]):
                if index in state_dict["state"]:
                    held = state_dict["state"][index]
                    self.state[p] = {"step": int(held["step"]),
                                     **{name: held[name].detach().to(p.device, dtype, copy=True)
                                        for name, dtype in _STATE.items()}}
