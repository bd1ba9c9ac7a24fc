"""AdamW with 8-bit states against its definition.

The oracle evaluates the moments with numpy's fp32 arithmetic (every product and sum rounded, as
the definition says), so scales and codes have to be equal; codes are chosen there in 64 bits.
Parameters: the update is one quotient of fp32 values; the square root (2^-23), its scaling and
sum (2^-24 each), the quotient (2^-22) and the step size (2^-24) put it within 2^-21 relative, the
decayed parameter and the sum within 2 * 2^-24, and the result is rounded once to its type.
"""

from __future__ import annotations

import copy
import warnings

import numpy as np
import pytest
import torch

import gpu_utils as gu
from picotron_b200 import kernels
from picotron_b200.errors import TritonAdamWUnavailable
from picotron_b200.kernels import AdamW8bit, adamw8bit_moments, adamw8bit_step

pytestmark = pytest.mark.gpu

F = np.float32
SIZES = [1, 2, 255, 256, 257, 511, 4096, 8192, 8193, 100_003]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    gu.require_gpu()


def _blocks(a):
    return np.pad(a, (0, -a.size % 256)).reshape(-1, 256)


def _spread(s, n):
    return np.repeat(s, 256)[:n]


def _values(mc, ms, vc, vs):
    c, d = mc.astype(np.int32), vc.astype(np.int32)
    d2 = (d * d).astype(F)
    return (c * np.abs(c)).astype(F) * _spread(ms, c.size), d2 * d2 * _spread(vs, d.size)


def _codes(a, power, top):
    """(codes, scales) of |a| in blocks of 256, codes nearest in the root's domain."""

    with np.errstate(divide="ignore", invalid="ignore", under="ignore"):
        s = _blocks(a).max(1) * F(1.0 / top ** power)
        s = np.where(s < np.finfo(F).tiny, F(0), s)
        q = np.where(_spread(s, a.size) > 0,
                     a.astype(np.float64) / _spread(s, a.size).astype(np.float64), 0.0)
    return np.minimum(np.rint(q ** (1.0 / power) if power == 2 else np.sqrt(np.sqrt(q))), top), s


def _step64(p, g, mc, ms, vc, vs, step, lr, b1, b2, eps, wd, maximize=False):
    m, v = _values(mc, ms, vc, vs)
    g = -g if maximize else g
    m = m * F(b1) + g * F(1.0 - b1)
    v = v * F(b2) + (g * g) * F(1.0 - b2)
    m64, v64 = m.astype(np.float64), v.astype(np.float64)
    update = lr / (1 - b1 ** step) * m64 / (np.sqrt(v64 / (1 - b2 ** step)) + eps)
    new = p.astype(np.float64) * (1 - lr * wd) - update
    mcode, ms = _codes(np.abs(m), 2, 127)
    vcode, vs = _codes(v, 4, 255)
    vcode = np.where((v > 0) & (_spread(vs, v.size) > 0), np.maximum(vcode, 1), vcode)
    return new, update, (mcode * np.sign(m)).astype(np.int8), ms, vcode.astype(np.uint8), vs


def _check_param(got, new, update, old):
    eps = torch.finfo(got.dtype).eps
    tol = (2.0 ** -21 * np.abs(update) + 2.0 ** -23 * (np.abs(old) + np.abs(new))
           + eps / 2 * np.abs(new) + torch.finfo(got.dtype).smallest_normal * eps)
    err = np.abs(got.double().cpu().numpy().ravel() - new)
    assert (err <= tol).all(), (err - tol).max()


def _fresh(n, dtype, seed, scale=1e-3):
    p = gu.randn((n,), seed, dtype, 0.05)
    g = gu.randn((n,), seed + 1, dtype, scale)
    blocks = (n + 255) // 256
    state = [torch.zeros(n, dtype=torch.int8, device=gu.DEV),
             torch.zeros(blocks, device=gu.DEV),
             torch.zeros(n, dtype=torch.uint8, device=gu.DEV), torch.zeros(blocks, device=gu.DEV)]
    return p, g, state


def _np(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


KW = dict(lr=1e-2, b1=0.9, b2=0.95, eps=1e-8, wd=0.1)


def _call(ps, gs, states, step, maximize=False, **kw):
    a = {**KW, **kw}
    adamw8bit_step(ps, gs, *zip(*states), step=step, lr=a["lr"], beta1=a["b1"], beta2=a["b2"],
                   eps=a["eps"], weight_decay=a["wd"], maximize=maximize)


@pytest.mark.parametrize("maximize", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_three_steps_of_a_list(dtype, maximize):
    ps, gs, states = map(list, zip(*(_fresh(n, dtype, 10 * i) for i, n in enumerate(SIZES))))
    for step in (1, 2, 3):
        before = [([_np(t) for t in s], _np(p), _np(g)) for p, g, s in zip(ps, gs, states)]
        _call(ps, gs, states, step, maximize)
        for (s, p0, g0), p, state in zip(before, ps, states):
            new, update, *want = _step64(p0, g0, *s, step, *KW.values(), maximize)
            for got, w in zip(state, want):
                assert np.array_equal(_np(got), w)
            _check_param(p, new, update, p0)
        gs = [gu.randn(g.shape, 100 * step + i, dtype, 1e-3) for i, g in enumerate(gs)]
    m, v = adamw8bit_moments(*map(list, zip(*states)))
    for a, b, state in zip(m, v, states):
        wm, wv = _values(*map(_np, state))
        assert np.array_equal(_np(a), wm) and np.array_equal(_np(b), wv)


def test_many_values_next_to_code_borders():
    """Moments on and around every border between two codes: beta 0 makes the moments the
    gradient (and its square), so the borders can be hit exactly."""

    c = np.arange(127)
    border = ((2 * c + 1) / 2.0) ** 2
    g = border.astype(F)
    g = np.concatenate([g, np.nextafter(g, F(0)), np.nextafter(g, F(1e9)), -g])
    for scale in (F(1.0), F(0.37), F(1.7e-5)):
        a = (g * scale).astype(F)
        a = _blocks(a)
        a[:, -1] = F(16129.0) * scale  # every block's scale is `scale` up to rounding
        a = a.ravel()
        n = a.size
        p, _, state = _fresh(n, torch.float32, 5)
        p0 = _np(p)
        grad = torch.from_numpy(a).to(gu.DEV)
        before = [_np(t) for t in state]
        _call([p], [grad], [state], 1, b1=0.0, b2=0.0)
        kw = {**KW, "b1": 0.0, "b2": 0.0}
        new, update, *want = _step64(p0, a, *before, 1, *kw.values())
        for got, w in zip(state, want):
            assert np.array_equal(_np(got), w)


def test_zero_tiny_and_huge_gradients():
    for scale in (0.0, 1e-30, 1e-20, 1e-12, 1e4, 1e15):
        p, g, state = _fresh(700, torch.float32, 6, scale=1.0)
        g = (g.double() * scale).float()
        g[256:512] = 0.0
        p0, g0, before = _np(p), _np(g), [_np(t) for t in state]
        _call([p], [g], [state], 1)
        new, update, *want = _step64(p0, g0, *before, 1, *KW.values())
        for got, w in zip(state, want):
            assert np.array_equal(_np(got), w)
        if scale <= 1e15:
            _check_param(p, new, update, p0)
        assert torch.isfinite(p).all()


def test_non_finite_gradient_stays_in_its_block():
    p, g, state = _fresh(1000, torch.float32, 7)
    q, _, other = _fresh(1000, torch.float32, 7)
    clean = g.clone()
    g[300], g[700] = float("nan"), float("inf")
    _call([p], [g], [state], 1)
    _call([q], [clean], [other], 1)
    m, v = adamw8bit_moments(*([t] for t in state))
    for b in (0, 3):
        s = slice(256 * b, min(1000, 256 * (b + 1)))
        assert torch.equal(p[s], q[s])
        for x, y in zip(state[::2], other[::2]):
            assert torch.equal(x[s], y[s])
    assert torch.isnan(m[0][256:768]).all() and torch.isnan(v[0][256:512]).all()
    assert torch.isfinite(m[0][:256]).all() and torch.isfinite(m[0][768:]).all()


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_unaligned_slices_and_untouched_neighbours(dtype, shift):
    n = 1500
    p, g, state = _fresh(n, dtype, 8)
    big = [torch.full((n + 8,), 7, dtype=t.dtype, device=gu.DEV)
           for t in (p, g, state[0], state[2])]
    views = [b[shift:shift + n] for b in big]
    for view, t in zip(views, (p, g, state[0], state[2])):
        view.copy_(t)
    shifted = [views[2], state[1].clone(), views[3], state[3].clone()]
    _call([p], [g], [state], 1)
    _call([views[0]], [views[1]], [shifted], 1)
    assert torch.equal(views[0], p)
    for a, b in zip(shifted, state):
        assert torch.equal(a, b)
    for b in big:
        assert (b[:shift] == 7).all() and (b[shift + n:] == 7).all()
    m, v = adamw8bit_moments(*([t] for t in state))
    m2, v2 = adamw8bit_moments(*([t] for t in shifted))
    assert torch.equal(m[0], m2[0]) and torch.equal(v[0], v2[0])


def test_more_tensors_than_one_launch_and_per_tensor_scalars():
    ps, gs, states = map(list, zip(*(_fresh(1 + 37 * i, torch.float32, i) for i in range(250))))
    single = [(p.clone(), [t.clone() for t in s]) for p, s in zip(ps, states)]
    steps, lrs = [1 + i % 5 for i in range(250)], [1e-3 * (1 + i % 3) for i in range(250)]
    adamw8bit_step(ps, gs, *zip(*states), step=steps, lr=lrs, weight_decay=[0.0] * 250)
    for (p, s), g, got, state, step, lr in zip(single, gs, ps, states, steps, lrs):
        adamw8bit_step([p], [g], *([t] for t in s), step=step, lr=lr, weight_decay=0.0)
        assert torch.equal(p, got) and all(torch.equal(a, b) for a, b in zip(s, state))


def test_first_step_is_32_bit_adamws():
    """The first update of AdamW is lr * sign(g) whatever precision the states are kept in."""

    p8 = torch.nn.Parameter(gu.randn((64, 40), 3))
    p32 = torch.nn.Parameter(p8.detach().clone())
    a, b = AdamW8bit([p8], lr=1e-2), torch.optim.AdamW([p32], lr=1e-2)
    g = gu.randn((64, 40), 4)
    p8.grad, p32.grad = g.clone(), g.clone()
    a.step()
    b.step()
    assert (p8 - p32).abs().max().item() <= 1e-2 * 2.0 ** -20 + 5 * 2.0 ** -23


def _params(seed, dtype=torch.float32):
    ps = [torch.nn.Parameter(gu.randn(s, seed + i, dtype, 0.1))
          for i, s in enumerate([(300, 7), (5,), (64, 64)])]
    return ps


def _set_grads(ps, seed):
    for i, p in enumerate(ps):
        p.grad = gu.randn(p.shape, seed + i, p.dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_optimizer_groups_state_dict_and_moments(dtype):
    ps = _params(1, dtype)
    frozen = torch.nn.Parameter(gu.randn((9,), 50, dtype))
    opt = AdamW8bit([{"params": ps[:2], "lr": 1e-2}, {"params": [ps[2], frozen],
                                                      "betas": (0.8, 0.9)}], weight_decay=0.1)
    assert len(opt.moments()) == 0
    for k in range(3):
        _set_grads(ps, 10 * k)
        opt.step()
    assert frozen not in opt.state and opt.state[ps[0]]["step"] == 3
    saved = copy.deepcopy(opt.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in (*ps, frozen)]
    other = AdamW8bit([{"params": twins[:2]}, {"params": twins[2:]}])
    other.load_state_dict(saved)
    for p, q in zip(ps, twins):
        for name, t in opt.state[p].items():
            u = other.state[q][name]
            assert t == u if name == "step" else (t.dtype == u.dtype and torch.equal(t, u)
                                                  and t.data_ptr() != u.data_ptr())
    for o, group in ((opt, ps), (other, twins[:3])):
        _set_grads(group, 77)
        o.step()
    for p, q in zip(ps, twins):
        assert torch.equal(p, q)
    moments = opt.moments()
    assert len(moments) == 3
    for p in ps:
        m, v = moments[p]
        assert m.shape == p.shape and m.dtype == torch.float32 and (v >= 0).all()


def test_training_loop_step_object_runs_it():
    ps = _params(2)
    _set_grads(ps, 3)
    opt = AdamW8bit(ps)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        kernels.AdamWStepWithFallback(use_triton=True).step(opt)
    assert all(opt.state[p]["step"] == 1 for p in ps)


def test_parameters_notice_the_step():
    """A graph that saved a parameter before the step refuses to go back through it after."""

    p = torch.nn.Parameter(gu.randn((8, 8), 5))
    p.grad = gu.randn((8, 8), 6)
    x = gu.randn((8, 8), 7).requires_grad_()
    out = (x @ p).sum()
    AdamW8bit([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_captured_step_and_refused_step():
    p, g, state = _fresh(5000, torch.bfloat16, 12)
    q, s2 = p.clone(), [t.clone() for t in state]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _call([q], [g], [s2], 1)
    for _ in range(2):  # a graph repeats the step that it captured, with its step count
        graph.replay()
        _call([p], [g], [state], 1)
    assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(state, s2))
    bad = torch.nn.Parameter(gu.randn((6, 4), 1).t())
    bad.grad = torch.zeros_like(bad)
    opt = AdamW8bit([bad])
    with pytest.raises(TritonAdamWUnavailable):
        opt.step()
    assert opt.moments() == {} and len(opt.state) == 0


def test_streams_give_the_same_bits():
    p, g, state = _fresh(100_000, torch.float32, 9)
    q, s2 = p.clone(), [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _call([q], [g], [s2], 1)
    _call([p], [g], [state], 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(state, s2))


def test_refusals_change_nothing():
    p, g, state = _fresh(600, torch.float32, 11)
    keep = [t.clone() for t in (p, *state)]
    short = [t[:1] for t in state]

    def step(ps=(p,), gs=(g,), st=(state,), **kw):
        adamw8bit_step(list(ps), list(gs), *zip(*st), **{"step": 1, "lr": 1e-3, **kw})

    bad = [
        lambda: step(gs=[g.bfloat16()]), lambda: step(gs=[g[:599]]), lambda: step(gs=[]),
        lambda: step(ps=[p.cpu()]), lambda: step(ps=[p.double()], gs=[g.double()]),
        lambda: step(ps=[p.view(20, 30).t()], gs=[g.view(20, 30).t()]),
        lambda: step(st=[short]), lambda: step(st=[[state[0].float(), *state[1:]]]),
        lambda: step(st=[[state[2], state[1], state[0], state[3]]]),
        lambda: step(ps=[p, p], gs=[g, g], st=[state, [t.clone() for t in state]]),
        lambda: step(ps=[p, p.clone()], gs=[g, g], st=[state, state]),
        lambda: step(step=0), lambda: step(beta1=1.0), lambda: step(beta2=-0.1),
        lambda: step(eps=-1.0), lambda: step(lr=[1e-3, 1e-3]),
    ]
    for call in bad:
        with pytest.raises(TritonAdamWUnavailable):
            call()
    for a, b in zip(keep, (p, *state)):
        assert torch.equal(a, b)
    with pytest.raises(TritonAdamWUnavailable):
        adamw8bit_moments([state[0].cpu()], [state[1].cpu()], [state[2].cpu()], [state[3].cpu()])
    adamw8bit_step([], [], [], [], [], [], step=1, lr=1e-3)
    assert adamw8bit_moments([], [], [], []) == ([], [])
    q = torch.nn.Parameter(torch.zeros(4))
    q.grad = torch.zeros(4)
    with pytest.raises(TritonAdamWUnavailable):
        AdamW8bit([q]).step()
