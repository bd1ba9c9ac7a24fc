"""RoPE by explicit positions against complex rotation in 64 bits.

The angle is formed in 64 bits and its fraction of a turn rounded once to fp32 (2^-24 of at most
half a turn: 2^-24 pi radian), cosine and sine are within 2 ulp (2^-22) and scaled once (2^-24),
each output is two products and a sum (3 * 2^-24 of the terms) rounded once to its type. So an
output is off by at most half a step of its type plus
(2^-24 pi + 2^-22 + 4 * 2^-24) * scale * (|x_1| + |x_2|) < 2^-21 * scale * (|x_1| + |x_2|).
"""

from __future__ import annotations

import itertools

import pytest
import torch

import gpu_utils as gu
import picotron_b200 as pb
from picotron_b200 import kernels
from picotron_b200.errors import TritonRoPEUnavailable
from picotron_b200.kernels import apply_rotary_positions, rotary_frequencies

pytestmark = pytest.mark.gpu

LAYOUTS = ["interleaved", "rotate_half"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def _parts(x, rotary, layout):
    body = x[..., :rotary]
    if layout == "interleaved":
        return body[..., 0::2], body[..., 1::2]
    return body[..., :rotary // 2], body[..., rotary // 2:]


def _check(got, x, positions, inv_freq, layout, scale, sign):
    """sign +1: the rotation; -1: its transpose."""

    assert got.shape == x.shape and got.dtype == x.dtype
    rotary = 2 * inv_freq.numel()
    x64 = x.double().cpu()
    a = positions.cpu().double().unsqueeze(-1) * inv_freq.cpu()
    turn = torch.polar(torch.full_like(a, scale), sign * a)
    turn = turn if positions.dim() == 1 else turn.unsqueeze(1)
    z = torch.complex(*(t.contiguous() for t in _parts(x64, rotary, layout))) * turn
    size = sum(t.abs() for t in _parts(x64, rotary, layout))
    g64 = got.double().cpu()
    eps = torch.finfo(x.dtype).eps / 2
    for g, w in zip(_parts(g64, rotary, layout), (z.real, z.imag)):
        tol = 2.0 ** -21 * scale * size + eps * w.abs() + torch.finfo(x.dtype).smallest_normal * eps
        err = (g - w).abs()
        assert (err <= tol).all(), (err - tol).max()
    assert torch.equal(got[..., rotary:], x[..., rotary:])


def _run(q, k, positions, inv_freq, layout, scale=1.0):
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    oq, ok = apply_rotary_positions(q, k, positions, inv_freq, layout=layout, scale=scale)
    _check(oq.detach(), q.detach(), positions, inv_freq, layout, scale, 1)
    _check(ok.detach(), k.detach(), positions, inv_freq, layout, scale, 1)
    dq, dk = gu.randn(oq.shape, 8, oq.dtype), gu.randn(ok.shape, 9, ok.dtype)
    gq, gk = torch.autograd.grad((oq, ok), (q, k), (dq, dk))
    _check(gq, dq, positions, inv_freq, layout, scale, -1)
    _check(gk, dk, positions, inv_freq, layout, scale, -1)
    return oq.detach(), ok.detach(), gq, gk


def _positions(shape, seed=0, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-far // 4, far, shape, generator=g).to(gu.DEV)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("b,s,hq,hk,d,r", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 128, 128), (1, 5, 3, 1, 96, 40), (2, 7, 2, 2, 64, 32),
    (3, 2, 5, 1, 78, 66), (1, 33, 1, 1, 8, 6), (2, 9, 7, 1, 80, 16), (1, 2, 32, 8, 256, 256),
    (4, 1, 40, 8, 128, 64), (1, 3, 2, 1, 8192, 8192), (2, 129, 1, 1, 16, 2),
], ids=str)
def test_layouts_sizes_and_types(b, s, hq, hk, d, r, layout, dtype):
    q = gu.randn((b, s, hq, d), 1, dtype).transpose(1, 2)  # the attention layer's view
    k = gu.randn((b, s, hk, d), 2, dtype).transpose(1, 2)
    inv_freq, _ = rotary_frequencies(r, 500_000.0, device=gu.DEV)
    _run(q, k, _positions((b, s)), inv_freq, layout, 1.25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("s,hq,hk,d,r", [
    (1, 1, 1, 2, 2), (5, 1, 1, 6, 4), (700, 3, 1, 10, 10), (33, 20, 5, 78, 66), (300, 1, 2, 30, 2),
    (9, 7, 3, 226, 226), (3, 129, 1, 22, 14), (1, 2, 1, 4094, 4094), (2, 60, 0, 78, 40),
    (3, 250, 1, 82, 82),
], ids=str)
def test_rows_of_odd_heads(s, hq, hk, d, r, layout, dtype):
    """Heads that are no whole 16-byte vectors, in rows that start anywhere: the attention layer's
    view, a slice of a fused projection (whose rows the gradient's do not match) and one token."""

    fused = gu.randn((2, s, (hq + hk) * d), 1, dtype)
    q = fused[..., : hq * d].unflatten(-1, (hq, d)).transpose(1, 2)
    k = fused[..., hq * d:].unflatten(-1, (hk, d)).transpose(1, 2)
    inv_freq, _ = rotary_frequencies(r, device=gu.DEV)
    pos = _positions((2, s))
    a = _run(q, k, pos, inv_freq, layout, 0.75)
    b = _run(q.transpose(1, 2).contiguous().transpose(1, 2),
             k.transpose(1, 2).contiguous().transpose(1, 2), pos, inv_freq, layout, 0.75)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def _shifted(shape, seed, dtype, shift):
    """A dense tensor that starts `shift` elements into its storage."""

    n = torch.Size(shape).numel()
    return gu.randn((n + shift,), seed, dtype)[shift:].view(shape)


VIEWS = {
    "heads outside": lambda t: t.contiguous(),
    "sequence outside": lambda t: t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3),
    "every other token": lambda t: t[:, :, ::2],
    "part of a fused projection": lambda t: torch.cat((t, t), -1)[..., : t.size(-1)],
    "odd row stride": lambda t: torch.nn.functional.pad(t, (0, 3))[..., : t.size(-1)],
    "head_dim not innermost": lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
    "one sequence expanded": lambda t: t[:1].expand(2, -1, -1, -1),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("view", VIEWS)
def test_views(view, layout, dtype):
    q, k = (VIEWS[view](gu.randn((2, h, 6, 64), h, dtype)) for h in (4, 2))
    inv_freq, _ = rotary_frequencies(48, device=gu.DEV)
    _run(q, k, _positions((2, 6))[:, : q.size(2)], inv_freq, layout)


@pytest.mark.parametrize("shift", [1, 2, 4])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_unaligned_storage_gives_the_same_bits(dtype, layout, shift):
    q, k = _shifted((2, 3, 5, 64), 1, dtype, shift), _shifted((2, 1, 5, 64), 2, dtype, shift)
    inv_freq, _ = rotary_frequencies(32, device=gu.DEV)
    pos = _positions((2, 5))
    a = _run(q, k, pos, inv_freq, layout)
    b = _run(q.clone(), k.clone(), pos, inv_freq, layout)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_matches_the_table_path_for_consecutive_positions():
    q = gu.randn((2, 32, 8, 128), 1).transpose(1, 2)
    k = gu.randn((2, 32, 2, 128), 2).transpose(1, 2)
    inv_freq, scale = rotary_frequencies(128, 500_000.0, device=gu.DEV)
    assert scale == 1.0
    oq, ok = apply_rotary_positions(q, k, torch.arange(32, device=gu.DEV), inv_freq)
    rope = pb.RotaryEmbedding(128, theta=500_000.0, use_triton_rope=True)
    tq, tk = rope(q, k)
    # The table's angles are fp32 products of fp32 frequencies: up to 31 * 2^-22 radian off.
    assert (oq - tq).abs().max() <= 31 * 2.0 ** -21 * 2 * q.abs().max()
    assert (ok - tk).abs().max() <= 31 * 2.0 ** -21 * 2 * k.abs().max()


def test_shared_positions_far_positions_and_strides():
    q, k = gu.randn((2, 4, 6, 32), 1), gu.randn((2, 2, 6, 32), 2)
    inv_freq, _ = rotary_frequencies(32, device=gu.DEV)
    pos = _positions((6,))
    a = _run(q, k, pos, inv_freq, "interleaved")
    b = _run(q, k, pos.expand(2, 6), inv_freq, "interleaved")
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    wide = torch.stack((_positions((6, 2), 3), _positions((6, 2), 4)), -1)[..., 0].t()
    _run(q, k, wide, inv_freq, "rotate_half")
    _run(q, k, torch.tensor([0, -1, 2**31 + 7, 2**33, 2**36, -(2**35)], device=gu.DEV),
         inv_freq, "rotate_half")


def test_rotation_inverts_and_keeps_relative_positions():
    q, k = gu.randn((1, 2, 40, 64), 1), gu.randn((1, 2, 40, 64), 2)
    inv_freq, _ = rotary_frequencies(64, device=gu.DEV)
    pos = torch.arange(40, device=gu.DEV)
    dots = []
    for offset in (0, 1_000_003):
        oq, ok = apply_rotary_positions(q, k, pos + offset, inv_freq, layout="rotate_half")
        dots.append(oq @ ok.transpose(2, 3))
    # 64 products of rotated values, each off by 2^-21 of its terms on either side.
    bound = 2.0 ** -19 * 2 * (q.abs().sum(-1).max() * k.abs().max()).item() * 2
    assert (dots[0] - dots[1]).abs().max().item() <= bound


def test_gradient_of_one_output_and_differences():
    q, k = gu.randn((1, 2, 3, 16), 1), gu.randn((1, 1, 3, 16), 2)
    inv_freq, _ = rotary_frequencies(10, device=gu.DEV)
    pos = torch.tensor([[5, 1, 99]], device=gu.DEV)
    q.requires_grad_()
    oq, _ = apply_rotary_positions(q, k, pos, inv_freq, scale=0.7)
    w = gu.randn(oq.shape, 3)
    (gq,) = torch.autograd.grad(oq, q, w)
    d, h = gu.randn(q.shape, 4), 0.5  # linear: a large step loses nothing
    with torch.no_grad():
        up, _ = apply_rotary_positions(q + h * d, k, pos, inv_freq, scale=0.7)
        down, _ = apply_rotary_positions(q - h * d, k, pos, inv_freq, scale=0.7)
    want = ((up - down).double() * w.double()).sum() / (2 * h)
    assert (gq.double() * d.double()).sum().item() == pytest.approx(want.item(), rel=1e-4)


def test_empty_and_one_side_empty():
    inv_freq, _ = rotary_frequencies(16, device=gu.DEV)
    q, k = gu.randn((2, 3, 0, 16), 1), gu.randn((2, 1, 0, 16), 2)
    oq, ok = apply_rotary_positions(q, k, _positions((2, 0)), inv_freq)
    assert oq.shape == q.shape and ok.shape == k.shape
    q, k = gu.randn((2, 3, 4, 16), 1), gu.randn((2, 0, 4, 16), 2)
    pos = _positions((2, 4))
    oq, ok = apply_rotary_positions(q, k, pos, inv_freq)
    _check(oq, q, pos, inv_freq, "interleaved", 1.0, 1)
    assert ok.shape == k.shape


def test_offsets_beyond_32_bits():
    d, s = 64, 1 << 20
    q = torch.zeros(1, 66, s, d, dtype=torch.bfloat16, device=gu.DEV)  # 4.4e9 elements
    k = gu.randn((1, 1, 1, d), 1, torch.bfloat16).expand(1, 1, s, d)
    at = torch.tensor([0, 1 << 19, s - 1], device=gu.DEV)
    q[0, 65, at] = gu.randn((3, d), 2, torch.bfloat16)
    inv_freq, _ = rotary_frequencies(d, device=gu.DEV)
    pos = torch.arange(s, device=gu.DEV)
    oq, ok = apply_rotary_positions(q, k, pos, inv_freq)
    _check(oq[:, 65:, at], q[:, 65:, at], pos[at], inv_freq, "interleaved", 1.0, 1)
    _check(ok[:, :, at], k[:, :, at], pos[at], inv_freq, "interleaved", 1.0, 1)


def test_streams_and_graph_replays():
    q, k = gu.randn((2, 4, 8, 128), 1, torch.bfloat16), gu.randn((2, 2, 8, 128), 2, torch.bfloat16)
    inv_freq, _ = rotary_frequencies(128, device=gu.DEV)
    pos = _positions((2, 8))
    want = _run(q, k, pos, inv_freq, "rotate_half")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sq, sk, sp = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(pos)
    with torch.cuda.stream(side):
        got = _run(q, k, pos, inv_freq, "rotate_half")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary_positions(sq, sk, sp, inv_freq, layout="rotate_half")
    for p in (pos, pos + 77):
        sq.copy_(q), sk.copy_(k), sp.copy_(p)
        graph.replay()
        eager = apply_rotary_positions(q, k, p, inv_freq, layout="rotate_half")
        assert all(torch.equal(x, y) for x, y in zip(out, eager))


def test_module_takes_positions_partial_heads_and_scaling():
    q, k = gu.randn((2, 8, 4, 64), 1).transpose(1, 2), gu.randn((2, 8, 2, 64), 2).transpose(1, 2)
    pos = _positions((2, 8))
    for rotary, scaling in itertools.product((None, 32), (None, {
            "scaling": "yarn", "factor": 8.0, "original_length": 4096})):
        fast = pb.RotaryEmbedding(64, 500_000.0, use_triton_rope=True)
        eager = pb.RotaryEmbedding(64, 500_000.0)
        for module in (fast, eager):
            module.rotary_dim, module.scaling = rotary, scaling
        inv_freq, scale = rotary_frequencies(rotary or 64, 500_000.0, device=gu.DEV,
                                             **(scaling or {}))
        for p in (pos, pos[0], None):
            if p is None and rotary is None and scaling is None:
                continue
            at = torch.arange(8, device=gu.DEV) if p is None else p
            for module in (fast, eager):
                oq, ok = module(q, k, p)
                _check(oq, q, at, inv_freq, "interleaved", scale, 1)
                _check(ok, k, at, inv_freq, "interleaved", scale, 1)
        assert not fast._triton_fallback_warned


def test_refusals():
    q, k = gu.randn((2, 4, 6, 32), 1), gu.randn((2, 2, 6, 32), 2)
    inv_freq, _ = rotary_frequencies(32, device=gu.DEV)
    pos = torch.arange(6, device=gu.DEV)

    def call(q=q, k=k, pos=pos, inv_freq=inv_freq, **kw):
        return lambda: kernels.apply_rotary_positions(q, k, pos, inv_freq, **kw)

    for bad in (call(q=q.cpu()), call(q=q.double(), k=k.double()), call(k=k.half()),
                call(k=k[:1]), call(k=k[:, :, :5]), call(k=k[..., :16]), call(q=q[0]),
                call(pos=pos[:5]), call(pos=pos.int()), call(pos=pos.expand(3, 6)),
                call(pos=pos.cpu()), call(inv_freq=inv_freq.float()), call(inv_freq=inv_freq[:0]),
                call(inv_freq=torch.cat((inv_freq, inv_freq))), call(inv_freq=inv_freq[None]),
                call(layout="half")):
        with pytest.raises(TritonRoPEUnavailable):
            bad()
