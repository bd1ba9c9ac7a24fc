"""RotaryEmbedding on the GPU: the tables and frequencies it keeps between calls serve a call in any
other mode."""

from __future__ import annotations

import pytest
import torch

import gpu_utils as gu
from picotron_b200 import RotaryEmbedding

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def test_module_used_in_inference_mode_first_then_trained():
    """The frequencies that a module keeps serve autograd whatever mode the first call ran in."""

    for positions in (None, torch.arange(6, device=gu.DEV) + 3):
        rope = RotaryEmbedding(16, use_triton_rope=True)
        if positions is None:
            rope.rotary_dim = 8
        q, k = gu.randn((2, 3, 6, 16), 1), gu.randn((2, 1, 6, 16), 2)
        with torch.inference_mode():
            first = rope(q, k, positions)
        q.requires_grad_()
        out = rope(q, k, positions)
        (dq,) = torch.autograd.grad(out[0].square().sum(), q)
        assert torch.equal(out[0].detach(), first[0]) and torch.equal(out[1], first[1])
        torch.testing.assert_close(dq, 2 * q.detach(), rtol=1e-5, atol=1e-5)  # a rotation


def test_tables_of_a_captured_first_call_are_not_kept():
    """A table built while capturing holds nothing until the graph is replayed."""

    rope = RotaryEmbedding(16, use_triton_rope=True)
    q, k = gu.randn((2, 3, 6, 16), 1), gu.randn((2, 1, 6, 16), 2)
    want = RotaryEmbedding(16, use_triton_rope=True)(q, k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rope(q, k)
    for got, w in zip(rope(q, k), want):  # before any replay
        assert torch.equal(got, w)
    graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(captured, want):
        assert torch.equal(got, w)
