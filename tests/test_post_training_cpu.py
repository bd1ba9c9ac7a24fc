"""Post-training operators without a GPU: refusals before any launch (Python and C ABI), the
frequencies of long-context RoPE, the eager module path, fake implementations, 8-bit state dicts."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import picotron_b200 as pb
from picotron_b200 import _capi, kernels, ops
from picotron_b200.errors import (
    TritonAdamWUnavailable,
    TritonLogitLossUnavailable,
    TritonRoPEUnavailable,
)
from picotron_b200.kernels import AdamW8bit, rotary_frequencies


def test_cpu_tensors_are_refused():
    x, t, f = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for call in (lambda: kernels.token_log_probs(x, t), lambda: kernels.preference_loss(x, t, f),
                 lambda: kernels.policy_loss(x, t, f, f),
                 lambda: kernels.token_log_probs(x.tolist(), t)):
        with pytest.raises(TritonLogitLossUnavailable):
            call()
    q = torch.randn(1, 2, 3, 8)
    inv_freq, _ = rotary_frequencies(8)
    with pytest.raises(TritonRoPEUnavailable):
        kernels.apply_rotary_positions(q, q, torch.arange(3), inv_freq)
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    opt = AdamW8bit([p])
    with pytest.raises(TritonAdamWUnavailable):
        opt.step()
    assert not opt.state[p] and (p == 0).all()


def _rows(p=None, a=0, b=0):
    return p, a, b


def test_loss_entry_points_reject_bad_arguments_before_cuda():
    lib = _capi.library()
    i64 = ctypes.c_int64(0)
    shape, dtype, arg = (_capi.PT_ERR_SHAPE, _capi.PT_ERR_UNSUPPORTED_DTYPE,
                         _capi.PT_ERR_INVALID_ARGUMENT)
    assert lib.pt_logit_loss_workspace(8, 2, 3, 2, None) == arg
    assert lib.pt_logit_loss_workspace(8, -1, 3, 2, ctypes.byref(i64)) == shape
    assert lib.pt_logit_loss_workspace(0, 2, 3, 2, ctypes.byref(i64)) == shape
    assert lib.pt_logit_loss_workspace(8, 2**40, 2**40, 2, ctypes.byref(i64)) == shape
    assert lib.pt_logit_loss_workspace(8, 2, 3, 9, ctypes.byref(i64)) == dtype
    logits = lambda outer, vocab=8: (None, vocab, outer, 3, 24, 8, *_rows(), -100)  # noqa: E731
    assert lib.pt_token_logps_fwd(*logits(-1), None, None, None, 0, 2, None) == shape
    assert lib.pt_token_logps_fwd(*logits(1, 0), None, None, None, 0, 2, None) == shape
    assert lib.pt_token_logps_fwd(*logits(1), None, None, None, 0, 5, None) == dtype
    tail = (None, None, None, None, None, 0, 2, None)
    assert lib.pt_preference_loss_fwd(*logits(3), *_rows(), 0.1, 0.0, *tail) == shape
    assert lib.pt_preference_loss_fwd(*logits(2), *_rows(), math.inf, 0.0, *tail) == arg
    assert lib.pt_preference_loss_fwd(*logits(2), *_rows(), 0.1, -0.1, *tail) == arg
    policy = lambda low, high, kl: lib.pt_policy_loss_fwd(  # noqa: E731
        *logits(2), *_rows(), *_rows(), *_rows(), low, high, kl, 0, *tail)
    assert policy(-0.1, 0.2, 0.0) == arg
    assert policy(0.2, math.nan, 0.0) == arg
    assert policy(0.2, 0.2, math.inf) == arg
    assert "kl_coef" in _capi.last_error()


def test_policy_gradient_support_and_rescaling_are_checked_before_cuda():
    lib, flag = _capi.library(), ctypes.c_int(-1)
    ask = lambda vocab, outer=1, dtype=2: (  # noqa: E731
        lib.pt_policy_loss_grad_supported(vocab, outer, 1, dtype, ctypes.byref(flag)), flag.value)
    assert ask(128256) == (_capi.PT_OK, 1) and ask(786432) == (_capi.PT_OK, 1)
    assert ask(786433) == (_capi.PT_OK, 0) and ask(400_000, dtype=0) == (_capi.PT_OK, 0)
    assert ask(8, 2**29) == (_capi.PT_OK, 0) and ask(8, 2**31)[0] == _capi.PT_ERR_SHAPE
    assert ask(0)[0] == _capi.PT_ERR_SHAPE and ask(8, dtype=4)[0] == _capi.PT_ERR_UNSUPPORTED_DTYPE
    rescale = lambda expected, dtype=2, outer=1: lib.pt_rescale_logits_grad(  # noqa: E731
        None, 8, outer, 1, 8, 8, None, expected, dtype, None)
    assert rescale(0.0) == rescale(math.nan) == _capi.PT_ERR_INVALID_ARGUMENT
    assert rescale(1.0, dtype=3) == _capi.PT_ERR_UNSUPPORTED_DTYPE
    assert rescale(1.0, outer=-1) == _capi.PT_ERR_SHAPE
    assert rescale(1.0, outer=0) == _capi.PT_OK


def test_adamw8_entry_points_reject_bad_arguments_before_cuda():
    lib = _capi.library()
    one = (ctypes.c_void_p * 1)(None)
    n, bad, step, zero = ((ctypes.c_int64 * 1)(v) for v in (0, -1, 1, 0))
    lr = (ctypes.c_double * 1)(0.1)

    def call(numel=n, steps=step, count=1, b1=0.9, b2=0.99, eps=1e-8, dtype=0, first=one):
        return lib.pt_adamw8_step(first, one, one, one, one, one, numel, steps, lr, lr, count, b1,
                                  b2, eps, 0, dtype, None)

    assert call(count=-1) == _capi.PT_ERR_INVALID_ARGUMENT
    assert call(count=0) == _capi.PT_OK
    assert call(dtype=7) == _capi.PT_ERR_UNSUPPORTED_DTYPE
    assert call(first=None) == _capi.PT_ERR_INVALID_ARGUMENT
    assert call(b1=1.0) == call(b2=-1.0) == call(eps=-1.0) == _capi.PT_ERR_INVALID_ARGUMENT
    assert call(numel=bad) == _capi.PT_ERR_SHAPE
    assert call(steps=zero) == _capi.PT_ERR_INVALID_ARGUMENT
    assert lib.pt_adamw8_moments(one, one, one, one, bad, one, one, 1, None) == _capi.PT_ERR_SHAPE
    assert lib.pt_adamw8_moments(one, one, one, None, n, one, one, 1,
                                 None) == _capi.PT_ERR_INVALID_ARGUMENT


def test_rope_positions_rejects_bad_arguments_before_cuda():
    lib, st = _capi.library(), _capi._i64x4
    strides = st([64, 32, 8, 1])

    def call(sizes=(1, 2, 4, 8), k_sizes=(1, 1, 4, 8), xs=strides, rotary=8, layout=0, dtype=2,
             ps=1):
        return lib.pt_rope_positions(None, xs, None, strides, st(sizes), None, strides, None,
                                     strides, st(k_sizes), None, 0, ps, None, rotary, 1.0, 0,
                                     layout, dtype, None)

    shape = _capi.PT_ERR_SHAPE
    assert call(layout=2) == _capi.PT_ERR_INVALID_ARGUMENT
    assert call(dtype=3) == _capi.PT_ERR_UNSUPPORTED_DTYPE
    assert call(xs=st([64, 32, 8, 2])) == call(xs=st([-64, 32, 8, 1])) == shape
    assert call(k_sizes=(1, 1, 5, 8)) == call(k_sizes=(2, 1, 4, 8)) == shape
    assert call(rotary=0) == call(rotary=3) == call(rotary=10) == call(ps=-1) == shape
    assert call(sizes=(1, 2, 4, 7), k_sizes=(1, 1, 4, 7), rotary=6) == shape
    assert call(sizes=(0, 2, 4, 8), k_sizes=(0, 1, 4, 8)) == _capi.PT_OK


def test_rotary_frequencies():
    base, one = rotary_frequencies(64, 10_000.0)
    want = torch.tensor([10_000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    torch.testing.assert_close(base, want, rtol=1e-14, atol=0.0)
    assert one == 1.0 and base.dtype == torch.float64
    linear, one = rotary_frequencies(64, 10_000.0, scaling="linear", factor=4.0)
    assert torch.equal(linear, base / 4.0) and one == 1.0
    ntk, one = rotary_frequencies(64, 10_000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and one == 1.0
    assert ntk[-1].item() == pytest.approx(base[-1].item() / 4.0, rel=1e-12)
    assert (ntk <= base).all() and (ntk >= base / 4.0 * (1 - 1e-12)).all()
    yarn, scale = rotary_frequencies(64, 10_000.0, scaling="yarn", factor=4.0,
                                     original_length=4096)
    turns = 4096 * base / (2 * math.pi)
    assert scale == pytest.approx(0.1 * math.log(4.0) + 1.0)
    # One pair beyond the ramp's ends (they are rounded outwards to whole pairs).
    step = 10_000.0 ** (2 / 64)
    torch.testing.assert_close(yarn[turns > 32 * step], base[turns > 32 * step])
    torch.testing.assert_close(yarn[turns < 1 / step], base[turns < 1 / step] / 4.0)
    assert (yarn.diff() < 0).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, theta=0.0),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="yarn", factor=2.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0),
                dict(rotary_dim=8, theta=1.0, scaling="yarn", factor=2.0, original_length=64)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_eager_module_with_positions_partial_heads_and_scaling():
    q, k = torch.randn(2, 4, 6, 16, dtype=torch.float64), torch.randn(2, 2, 6, 16)
    rope = pb.RotaryEmbedding(16)
    plain = rope(q, k.double())
    moved = rope(q, k.double(), torch.arange(6))
    for a, b in zip(plain, moved):  # the table path rounds angles to fp32
        torch.testing.assert_close(a, b, rtol=0, atol=1e-5)
    pos = torch.randint(-5, 1000, (2, 6))
    rope.rotary_dim, rope.scaling = 8, {"scaling": "linear", "factor": 2.0}
    oq, ok = rope(q, k.double(), pos)
    a = pos.double()[:, None, :, None] * rotary_frequencies(8)[0] / 2.0
    z = torch.view_as_complex(q[..., :8].unflatten(-1, (4, 2)).contiguous())
    z = z * torch.polar(torch.ones_like(a), a)
    torch.testing.assert_close(oq[..., :8], torch.view_as_real(z).flatten(-2))
    assert torch.equal(oq[..., 8:], q[..., 8:]) and ok.shape == k.shape
    rope.use_triton_rope = True
    with pytest.warns(RuntimeWarning, match="Triton RoPE unavailable"):
        again, _ = rope(q, k.double(), pos)
    assert torch.equal(again, oq)
    rope.rotary_dim = 18
    with pytest.raises(ValueError):
        rope(q, k.double(), pos)
    assert list(rope.state_dict()) == []


def test_fake_implementations_match_shapes_and_strides():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 3, 65, dtype=torch.bfloat16, device="cuda")
        t = torch.empty(2, 3, dtype=torch.long, device="cuda")
        f = torch.empty(2, 3, device="cuda")
        lp, stats = torch.ops.picotron_b200.token_logps(x, t, -100)
        assert lp.shape == (2, 3) and lp.dtype == torch.float32 and stats.shape == (2, 3, 2)
        out = torch.ops.picotron_b200.preference_loss(x, t, f, 0.1, 0.0, -100)
        assert [tuple(o.shape) for o in out] == [(), (2,), (2, 3, 2), (2,)]
        out = torch.ops.picotron_b200.policy_loss(x, t, f, f, None, 0.2, 0.2, 0.0, False, -100,
                                                  None)
        assert [tuple(o.shape) for o in out] == [(), (2, 3), (2, 3, 2), (2, 3)]
        back = torch.ops.picotron_b200.logit_loss_backward
        assert back(x, t, stats, f, None, -100).stride() == x.stride()
        # Odd rows of a strided view keep its strides (equal addresses modulo 16 bytes).
        assert back(x[:, 1:], t[:, 1:], stats[:, 1:], f[:, 1:], None, -100).stride() == x.stride()
        q = torch.empty(2, 8, 4, 32, device="cuda").transpose(1, 2)
        k = torch.empty(2, 8, 2, 32, device="cuda").transpose(1, 2)
        freq = torch.empty(16, dtype=torch.float64, device="cuda")
        oq, ok = torch.ops.picotron_b200.rope_positions(q, k, t[0], freq, 0, 1.0)
        assert oq.stride() == q.stride() and ok.shape == k.shape


def test_overlapping_and_strided_logits_are_copied_only_when_needed():
    x = torch.randn(4, 6, 8)
    same = [x, x[:, :-1], x[::2], x[..., 2:], x.transpose(0, 1), x[:0], x[:, :0], x[:1]]
    for view in same:
        assert ops._ll_logits(view) is view
    for view in (x[:1].expand(4, 6, 8), x.transpose(1, 2), x[:, :1].expand(4, 6, 8),
                 x.view(-1).as_strided((4, 6, 8), (8, 8, 1))):
        copied = ops._ll_logits(view)
        assert copied.is_contiguous() and torch.equal(copied, view)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_adamw8bit_state_dict_keeps_codes_and_scales(dtype):
    p = torch.nn.Parameter(torch.zeros(300, dtype=dtype))
    opt = AdamW8bit([p], lr=1e-2)
    state = opt._new_state(p)
    assert [tuple(state[n].shape) for n in ("exp_avg_codes", "exp_avg_scales")] == [(300,), (2,)]
    state["step"] = 4
    state["exp_avg_codes"] += 3
    state["exp_avg_scales"] += 1.2345678
    opt.state[p] = state
    q = torch.nn.Parameter(torch.zeros(300, dtype=dtype))
    other = AdamW8bit([q])
    other.load_state_dict(opt.state_dict())
    assert other.state[q]["step"] == 4 and other.param_groups[0]["lr"] == 1e-2
    for name, t in state.items():
        if name != "step":
            got = other.state[q][name]
            assert got.dtype == t.dtype and torch.equal(got, t) and got is not t
    foreign = torch.optim.AdamW([q])
    foreign.state[q] = {"step": torch.tensor(1.0), "exp_avg": torch.zeros(300),
                        "exp_avg_sq": torch.zeros(300)}
    with pytest.raises(ValueError, match="not an AdamW8bit"):
        AdamW8bit([q]).load_state_dict(foreign.state_dict())
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(1.0, 0.9)),
                dict(betas=(0.9, -0.1))):
        with pytest.raises(ValueError):
            AdamW8bit([q], **bad)
