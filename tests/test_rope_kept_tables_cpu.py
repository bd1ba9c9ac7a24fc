"""RotaryEmbedding keeps its tables and frequencies between calls: what it keeps has to serve a
call in any other mode."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import picotron_b200 as pb

SETTINGS = {
    "tables": lambda rope: None,
    "positions": lambda rope: torch.arange(6) + 3,
    "part of the head": lambda rope: setattr(rope, "rotary_dim", 8),
    "scaling": lambda rope: setattr(rope, "scaling", {"scaling": "linear", "factor": 2.0}),
}


def _states():
    g = torch.Generator().manual_seed(1)
    return torch.randn(2, 3, 6, 16, generator=g), torch.randn(2, 1, 6, 16, generator=g)


@pytest.mark.parametrize("setting", SETTINGS)
def test_inference_first_then_training(setting):
    rope = pb.RotaryEmbedding(16)
    positions = SETTINGS[setting](rope)
    q, k = _states()
    with torch.inference_mode():
        first = rope(q, k, positions)
    q.requires_grad_()
    out = rope(q, k, positions)
    (dq,) = torch.autograd.grad(out[0].square().sum(), q)
    assert torch.equal(out[0].detach(), first[0]) and torch.equal(out[1], first[1])
    torch.testing.assert_close(dq, 2 * q.detach(), rtol=1e-5, atol=1e-5)  # a rotation
    with torch.inference_mode():
        again = rope(q, k, positions)
    assert torch.equal(again[0], first[0])


@pytest.mark.parametrize("setting", SETTINGS)
def test_fake_tensors_are_not_kept(setting):
    rope, other = pb.RotaryEmbedding(16), pb.RotaryEmbedding(16)
    positions = SETTINGS[setting](rope)
    SETTINGS[setting](other)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        q, k = (mode.from_tensor(x) for x in _states())
        out = rope(q, k, None if positions is None else mode.from_tensor(positions))
        assert out[0].shape == q.shape
    q, k = _states()
    for a, b in zip(rope(q, k, positions), other(q, k, positions)):
        assert type(a) is torch.Tensor and torch.equal(a, b)


def test_modules_from_before_positions_still_run():
    """A module that was pickled whole by a version without the attributes for explicit
    positions, and one that has them."""

    rope = pb.RotaryEmbedding(16)
    old = pb.RotaryEmbedding.__new__(pb.RotaryEmbedding)
    old.__setstate__({name: value for name, value in rope.__dict__.items()
                      if name not in ("rotary_dim", "scaling", "_frequencies")})
    q, k = _states()
    for positions in (None, torch.arange(6)):
        for a, b in zip(old(q, k, positions), rope(q, k, positions)):
            assert torch.equal(a, b)
    rope.rotary_dim = 8
    for twin in (copy.deepcopy(rope), pickle.loads(pickle.dumps(rope))):
        assert twin.rotary_dim == 8
        assert torch.equal(twin(q, k)[0], rope(q, k)[0])
