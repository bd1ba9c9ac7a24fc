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
_STATE = {"exp_avg_codes": torch.int8, "exp_avg_scales": torch.float32,
          "exp_avg_sq_codes": torch.uint8, "exp_avg_sq_scales": torch.float32}


def _scales(numel: int) -> int:
    return (numel + BLOCK - 1) // BLOCK


def _check_states(lists: Sequence[Sequence[Tensor]], numels: Sequence[int] | None):
    """Validate the four state lists; returns (device, numels)."""

    if len(lists[0]) == 0:
        return None, []
    device = lists[0][0].device
    sizes = [t.numel() for t in lists[0]]
    if numels is not None and sizes != list(numels):
        raise TritonAdamWUnavailable("exp_avg codes must have one element per parameter element.")
    for values, (name, dtype) in zip(lists, _STATE.items()):
        if len(values) != len(sizes):
            raise TritonAdamWUnavailable("all tensor lists must have the same length.")
        for t, n in zip(values, sizes):
            if t.dtype != dtype or t.device != device or not t.is_contiguous():
                raise TritonAdamWUnavailable(
                    f"{name} must be contiguous {dtype} tensors on one device.")
            if t.numel() != (_scales(n) if name.endswith("scales") else n):
                raise TritonAdamWUnavailable(f"{name} has the wrong number of elements.")
    return device, sizes


def _per_tensor(value, count: int, name: str) -> list:
    if isinstance(value, Sequence):
        if len(value) != count:
            raise TritonAdamWUnavailable(f"{name} must be one value or one per tensor.")
        return list(value)
    return [value] * count


def _refuse_shared(name: str, tensors: Sequence[Tensor]) -> None:
    """Two entries over the same memory would be updated by two blocks at once."""

    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                   for t in tensors if t.numel())
    if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
        raise TritonAdamWUnavailable(f"two of the {name} share memory.")


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
    Nothing is changed when the call is refused. The step's scalars are host values, so a captured
    CUDA graph would replay the same step count.
    """

    count = len(params)
    device, numels = _check_states(
        (exp_avg_codes, exp_avg_scales, exp_avg_sq_codes, exp_avg_sq_scales),
        [p.numel() for p in params])
    if count != len(grads) or count != len(numels):
        raise TritonAdamWUnavailable("all tensor lists must have the same length.")
    if count == 0:
        return
    ops.check_device(device, TritonAdamWUnavailable)
    dtype = params[0].dtype
    code = ops._dtype_code(params[0], TritonAdamWUnavailable)
    for p, g in zip(params, grads):
        if p.dtype != dtype or g.dtype != dtype or p.device != device or g.device != device:
            raise TritonAdamWUnavailable("parameters and gradients must share dtype and device.")
        if p.shape != g.shape or not p.is_contiguous() or not g.is_contiguous():
            raise TritonAdamWUnavailable(
                "parameters and gradients must be contiguous and of the same shape.")
    for name, values in (("parameters", params), ("exp_avg codes", exp_avg_codes),
                         ("exp_avg scales", exp_avg_scales),
                         ("exp_avg_sq codes", exp_avg_sq_codes),
                         ("exp_avg_sq scales", exp_avg_sq_scales)):
        _refuse_shared(name, values)
    address = lambda values: [t.data_ptr() for t in values]  # noqa: E731
    with ops._OnDevice(device):
        _capi.adamw8_step(address(params), address(grads), address(exp_avg_codes),
                          address(exp_avg_scales), address(exp_avg_sq_codes),
                          address(exp_avg_sq_scales), numels, _per_tensor(step, count, "step"),
                          _per_tensor(lr, count, "lr"),
                          _per_tensor(weight_decay, count, "weight_decay"), beta1, beta2, eps,
                          maximize, code, ops._stream(device), TritonAdamWUnavailable)


@torch.no_grad()
def adamw8bit_moments(exp_avg_codes: Sequence[Tensor], exp_avg_scales: Sequence[Tensor],
                      exp_avg_sq_codes: Sequence[Tensor],
                      exp_avg_sq_scales: Sequence[Tensor]) -> tuple[list[Tensor], list[Tensor]]:
    """The fp32 ``(exp_avg, exp_avg_sq)`` lists that 8-bit states stand for, shaped like their
    codes: for inspection, or to carry on with an optimizer that keeps 32-bit states. The tensors
    of one call share one allocation."""

    held = (exp_avg_codes, exp_avg_scales, exp_avg_sq_codes, exp_avg_sq_scales)
    device, numels = _check_states(held, None)
    if not numels:
        return [], []
    ops.check_device(device, TritonAdamWUnavailable)
    # 32-byte aligned pieces of one buffer.
    room = [(n + 7) // 8 * 8 for n in numels]
    buffer = torch.empty(2 * sum(room), dtype=torch.float32, device=device)
    pieces = buffer.split(room + room)
    moments = [t[:n].view(c.shape) for t, n, c in
               zip(pieces, numels + numels, [*exp_avg_codes, *exp_avg_codes])]
    exp_avg, exp_avg_sq = moments[:len(numels)], moments[len(numels):]
    address = lambda values: [t.data_ptr() for t in values]  # noqa: E731
    with ops._OnDevice(device):
        _capi.adamw8_moments(*(address(v) for v in held), numels, address(exp_avg),
                             address(exp_avg_sq), ops._stream(device), TritonAdamWUnavailable)
    return exp_avg, exp_avg_sq


class AdamW8bit(Optimizer):
    """AdamW whose moments are held in 8 bits (see the module's description).

    Parameters: dense contiguous CUDA tensors in float32, float16 or bfloat16, updated in their
    own dtype (no separate master copy). Arguments as torch.optim.AdamW's; amsgrad is not
    offered. ``state_dict`` holds the codes and scales; ``load_state_dict`` keeps their dtypes.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *,
                 maximize: bool = False) -> None:
        if lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError("lr, eps and weight_decay must be >= 0")
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
        for (_, _, beta1, beta2, eps, maximize), items in calls.items():
            params = [p for p, _ in items]
            states = [self.state[p] if self.state[p] else self._new_state(p) for p in params]
            adamw8bit_step(params, [p.grad for p in params],
                           *([s[name] for s in states] for name in _STATE),
                           step=[s["step"] + 1 for s in states],
                           lr=[float(g["lr"]) for _, g in items], beta1=beta1, beta2=beta2,
                           eps=eps, weight_decay=[float(g["weight_decay"]) for _, g in items],
                           maximize=maximize)
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

        super().load_state_dict(state_dict)
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for index, p in zip(saved["params"], group["params"]):
                if index in state_dict["state"]:
                    held = state_dict["state"][index]
                    self.state[p] = {"step": int(held["step"]),
                                     **{name: held[name].detach().to(p.device, dtype, copy=True)
                                        for name, dtype in _STATE.items()}}
