"""Workloads of the post-training operators: the losses that read logits, the 8-bit AdamW step,
and rotary embedding by explicit positions.

``listed()`` names fixed workloads and ``draw()`` more of the same ranges; ``prepare`` makes a
workload's inputs on the GPU from a seed, ``run`` makes one pass over them, ``work`` counts the
bytes and operations a pass cannot do without, and ``exact`` evaluates the definition in 64 bits.
With ``own`` false a pass is written in elementary torch operations; with ``own`` true it makes
the calls a user of ``picotron_b200`` makes.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100
LARGEST = 8 * 1024 * 128256  # logits of the largest loss workloads
BLOCK = 256  # elements that share one scale in an 8-bit optimizer state


def listed():
    return [
        # Token log-probabilities with their gradient, one short sample (a weighted SFT term).
        {"name": "logps sample", "op": "logps", "batch": 1, "seq": 48, "vocab": 32000,
         "dtype": "fp32", "grad": True},
        # A frozen reference model scores a whole batch: forward only, vocabulary of an 8B decoder.
        {"name": "logps reference", "op": "logps", "batch": 8, "seq": 1024, "vocab": 128256,
         "dtype": "bf16", "grad": False},
        # Two short preference pairs, odd vocabulary (rows start at every alignment).
        {"name": "preference short", "op": "preference", "batch": 4, "seq": 96, "vocab": 50257,
         "dtype": "bf16", "smoothing": 0.1},
        # A full preference batch of four pairs.
        {"name": "preference batch", "op": "preference", "batch": 8, "seq": 1024,
         "vocab": 128256, "dtype": "bf16", "smoothing": 0.0},
        # A small group of rollouts, no KL term.
        {"name": "policy group", "op": "policy", "batch": 4, "seq": 64, "vocab": 32000,
         "dtype": "bf16", "kl": 0.0, "aggregate": "token", "per_token": False, "empty": 0},
        # fp16 training under a loss scale, per-token advantages, one rollout without tokens.
        {"name": "policy fp16 odd", "op": "policy", "batch": 6, "seq": 333, "vocab": 50257,
         "dtype": "fp16", "kl": 0.05, "aggregate": "sequence", "per_token": True, "empty": 1},
        # A full policy step with the KL term.
        {"name": "policy batch", "op": "policy", "batch": 16, "seq": 512, "vocab": 128256,
         "dtype": "bf16", "kl": 0.04, "aggregate": "token", "per_token": False, "empty": 0},
        # The quickstart-sized block (hidden 128, intermediate 256), bf16 parameters.
        {"name": "adamw8 small", "op": "adamw8", "hidden": 128, "inter": 256, "layers": 2,
         "odd": 77, "dtype": "bf16"},
        # Two decoder layers of hidden 4096, intermediate 14336, fp32 parameters.
        {"name": "adamw8 layers", "op": "adamw8", "hidden": 4096, "inter": 14336, "layers": 2,
         "odd": 0, "dtype": "fp32"},
        # One decoded token for each of 32 sequences, far into a long context.
        {"name": "rotary decode", "op": "rotary", "batch": 32, "seq": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "rotate_half", "dtype": "bf16",
         "far": 1000000, "factor": 8.0, "grad": False},
        # A packed training batch, forward and backward.
        {"name": "rotary packed", "op": "rotary", "batch": 8, "seq": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "interleaved", "dtype": "bf16",
         "far": 0, "factor": 1.0, "grad": True},
        # Part of the head rotated, odd sizes, fp32.
        {"name": "rotary partial", "op": "rotary", "batch": 3, "seq": 777, "heads": 14,
         "kv_heads": 2, "dim": 96, "rotary": 40, "layout": "rotate_half", "dtype": "fp32",
         "far": 4096, "factor": 4.0, "grad": True},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logps", "preference", "policy", "adamw8", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("logps", "preference", "policy"):
        vocab = _log_int(rng, 300, 128256)
        batch = _log_int(rng, 1, 16)
        if op == "preference":
            batch += batch % 2
        seq = _log_int(rng, 1 if op == "logps" else 8, max(8, min(4096, LARGEST // (batch * vocab))))
        if dtype == "fp32":
            seq = max(1, seq // 2)
        case = {"op": op, "batch": batch, "seq": seq, "vocab": vocab, "dtype": dtype}
        if op == "logps":
            case["grad"] = rng.random() < 0.5
        elif op == "preference":
            case["smoothing"] = rng.choice([0.0, 0.05, 0.2])
        else:
            case.update(kl=rng.choice([0.0, 0.02, 0.1]), aggregate=rng.choice(["token", "sequence"]),
                        per_token=rng.random() < 0.5, empty=int(batch > 3 and rng.random() < 0.5))
        return case
    if op == "adamw8":
        hidden = _log_int(rng, 64, 4096)
        return {"op": op, "hidden": hidden, "inter": _log_int(rng, hidden, hidden * 7 // 2),
                "layers": rng.randint(1, 2), "odd": rng.choice([0, 1, rng.randint(2, 5000)]),
                "dtype": dtype}
    dim = 2 * rng.randint(16, 128)
    kv = _log_int(rng, 1, 8)
    heads = kv * rng.randint(1, 4)
    batch = _log_int(rng, 1, 64)
    room = 8 * 2048 * 40 * 128 // (batch * (heads + kv) * dim * (2 if dtype == "fp32" else 1))
    return {"op": op, "batch": batch, "seq": _log_int(rng, 1, max(1, min(8192, room))),
            "heads": heads, "kv_heads": kv, "dim": dim,
            "rotary": rng.choice([dim, 2 * rng.randint(1, dim // 2)]),
            "layout": rng.choice(["interleaved", "rotate_half"]), "dtype": dtype,
            "far": rng.choice([0, 4096, 1000000]), "factor": rng.choice([1.0, 4.0, 32.0]),
            "grad": rng.random() < 0.6}


# ---------------------------------------------------------------------------- inputs --


def _shapes(case):
    """The parameter shapes of `layers` decoder blocks, and one odd-sized tensor."""

    h, i = case["hidden"], case["inter"]
    kv = max(1, h // 4)
    block = [(h,), (h, h), (kv, h), (kv, h), (h, h), (h,), (i, h), (i, h), (h, i)]
    return block * case["layers"] + ([(case["odd"],)] if case["odd"] else [])


def _targets(case, gen):
    """Targets with the prompt and the padding ignored; the last `empty` rows ignored whole."""

    b, s = case["batch"], case["seq"]
    t = torch.randint(0, case["vocab"], (b, s), generator=gen, device=DEV)
    if s >= 8:
        at = torch.arange(s, device=DEV)
        prompt = (torch.rand(b, 1, generator=gen, device=DEV) * s * 0.4).long()
        end = s - (torch.rand(b, 1, generator=gen, device=DEV) * s * 0.3).long()
        keep = (at >= prompt) & (at < end)
        if case.get("empty"):
            keep[b - case["empty"]:] = False
        t = torch.where(keep, t, torch.full_like(t, IGNORE))
    return t


def _logits(case, targets, gen):
    """Logits with the spread of a trained head: the target a few units above the rest."""

    b, s, v = case["batch"], case["seq"], case["vocab"]
    x = torch.empty(b, s, v, dtype=DTYPES[case["dtype"]], device=DEV)
    for i in range(b):
        row = torch.randn(s, v, generator=gen, device=DEV) * 2.0
        lift = torch.rand(s, 1, generator=gen, device=DEV) * 9.0
        row.scatter_add_(1, targets[i].clamp_min(0)[:, None], lift)
        x[i] = row.to(x.dtype)
    return x


def _exact_logps(logits, targets):
    """Log-probabilities in 64 bits, one sequence at a time."""

    out = []
    for x, t in zip(logits, targets):
        lp = torch.log_softmax(x.double(), -1).gather(-1, t.clamp_min(0)[:, None])[:, 0]
        out.append(torch.where(t == IGNORE, torch.zeros_like(lp), lp))
    return torch.stack(out)


def _quantise(m, v, pad):
    """Codes and scales of 8-bit moments in blocks of 256: exp_avg is sign(c) c^2 scale with c in
    [-127, 127], exp_avg_sq is c^4 scale with c in [0, 255]; each code is the one nearest in the
    root's domain, found in 64 bits, and a positive exp_avg_sq keeps a code of at least 1."""

    n = m.numel()
    m, v = (torch.nn.functional.pad(x, (0, pad)).view(-1, BLOCK) for x in (m, v))
    tiny = torch.finfo(torch.float32).tiny
    ms = m.abs().amax(1) * torch.tensor(1.0 / 16129.0, dtype=torch.float32, device=DEV)
    vs = v.amax(1) * torch.tensor(1.0 / 4228250625.0, dtype=torch.float32, device=DEV)
    ms = torch.where(ms < tiny, torch.zeros_like(ms), ms)
    vs = torch.where(vs < tiny, torch.zeros_like(vs), vs)
    mr = torch.where(ms > 0, 1.0 / ms.double(), 0.0)[:, None]
    vr = torch.where(vs > 0, 1.0 / vs.double(), 0.0)[:, None]
    mc = (m.abs().double() * mr).sqrt().round().clamp_max(127) * torch.sign(m).double()
    vc = (v.double() * vr).sqrt().sqrt().round().clamp_max(255)
    vc = torch.where((v > 0) & (vr > 0), vc.clamp_min(1), vc)
    return (mc.to(torch.int8).view(-1)[:n].clone(), ms, vc.to(torch.uint8).view(-1)[:n].clone(), vs)


def _moments(mc, ms, vc, vs, pad):
    """The fp32 moments that codes and scales stand for."""

    n = mc.numel()
    c, d = (torch.nn.functional.pad(x, (0, pad)).view(-1, BLOCK).float() for x in (mc, vc))
    d = d * d
    return (c * c.abs() * ms[:, None]).view(-1)[:n], (d * d * vs[:, None]).view(-1)[:n]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = {"case": case}
    op = case["op"]
    if op in ("logps", "preference", "policy"):
        t = state["targets"] = _targets(case, gen)
        x = state["logits"] = _logits(case, t, gen)
        noise = torch.randn(t.shape, generator=gen, device=DEV)
        if op == "logps":
            state["grad"] = noise / max(1, t.numel())
        elif op == "preference":
            # The reference's log-probabilities, and a policy that has moved away from them.
            state["reference"] = (_exact_logps(x, t) + 0.3 * noise).float()
        else:
            # The sampling policy's log-probabilities. Ratios within 1e-4 of a clipping border are
            # moved off it: which side such a token falls on is the last bit's choice.
            lp, drift = _exact_logps(x, t), 0.15 * noise.double()
            for border in (math.log(0.8), math.log(1.25)):
                drift = torch.where((drift - border).abs() < 1e-4, drift + 3e-4, drift)
            state["old"] = (lp - drift).float()
            state["reference"] = (lp + 0.2 * torch.randn(t.shape, generator=gen, device=DEV)).float()
            shape = t.shape if case["per_token"] else t.shape[:1]
            state["advantages"] = 0.4 + torch.randn(shape, generator=gen, device=DEV)
            state["loss_grad"] = torch.tensor(4096.0 if case["dtype"] == "fp16" else 1.0, device=DEV)
        return state
    dtype = DTYPES[case["dtype"]]
    if op == "adamw8":
        for name in ("params", "grads", "mc", "ms", "vc", "vs"):
            state[name] = []
        for shape in _shapes(case):
            n = math.prod(shape)
            p, g, m, r = (torch.randn(n, generator=gen, device=DEV) for _ in range(4))
            v = (1e-3 * (1.0 + 0.5 * r)) ** 2
            codes = _quantise(3e-4 * m, v, -n % BLOCK)
            state["params"].append((0.02 * p).to(dtype).view(shape))
            state["grads"].append((1e-3 * g).to(dtype).view(shape))
            for name, value in zip(("mc", "ms", "vc", "vs"), codes):
                state[name].append(value)
        return state
    b, s, d = case["batch"], case["seq"], case["dim"]

    def states(heads):  # [B, H, S, D] views of [B, S, H, D] projections
        x = torch.randn(b, s, heads, d, generator=gen, device=DEV).to(dtype)
        return x.transpose(1, 2)

    state["q"], state["k"] = states(case["heads"]), states(case["kv_heads"])
    if case["grad"]:
        state["dq"], state["dk"] = states(case["heads"]), states(case["kv_heads"])
    # Packed documents restart their positions; a far context adds an offset.
    cut = torch.rand(b, s, generator=gen, device=DEV) < 4.0 / (s + 4)
    at = torch.arange(s, device=DEV).expand(b, s)
    start = torch.where(cut, at, torch.zeros_like(at)).cummax(1).values
    offset = torch.randint(0, case["far"] + 1, (b, 1), generator=gen, device=DEV)
    state["positions"] = at - start + offset
    pair = torch.arange(0, case["rotary"], 2, device=DEV, dtype=torch.float64) / case["rotary"]
    state["inv_freq"] = (500000.0 ** -pair) / case["factor"]
    state["scale"] = 1.0 + 0.1 * math.log(case["factor"])
    return state


# ------------------------------------------------------------------------ plain forms --


def _softmax_parts(logits, targets):
    """exp(x - max), its sum (64-bit accumulation) and the targets' log-probabilities."""

    x = logits.float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, dtype=torch.float64)
    at = targets.clamp_min(0)[..., None]
    lp = x.gather(-1, at)[..., 0].double() - m[..., 0].double() - torch.log(total)
    return e, total, torch.where(targets == IGNORE, torch.zeros_like(lp), lp)


def _logits_grad(e, total, targets, coef, dtype):
    """coef (onehot - softmax), zero where the target is ignored."""

    coef = torch.where(targets == IGNORE, torch.zeros_like(coef), coef)
    g = e.mul_((-coef / total).float()[..., None])
    g.scatter_add_(-1, targets.clamp_min(0)[..., None], coef.float()[..., None])
    return g.to(dtype)


def _plain_logps(state):
    x, t = state["logits"], state["targets"]
    e, total, lp = _softmax_parts(x, t)
    out = {"log_probs": lp.float()}
    if state["case"]["grad"]:
        out["grad"] = _logits_grad(e, total, t, state["grad"].double(), x.dtype)
    return out


def _plain_preference(state, beta=0.1):
    x, t, smoothing = state["logits"], state["targets"], state["case"]["smoothing"]
    e, total, lp = _softmax_parts(x, t)
    keep = t != IGNORE
    ratio = torch.where(keep, lp - state["reference"].double(), torch.zeros_like(lp)).sum(-1)
    pairs = t.size(0) // 2
    z = beta * (ratio[:pairs] - ratio[pairs:])
    soft = torch.clamp_min(-z, 0) + torch.log1p(torch.exp(-z.abs()))  # -log sigmoid(z)
    loss = (soft + smoothing * z).mean()
    dz = (smoothing - 1.0 / (1.0 + torch.exp(z))) / pairs
    coef = beta * torch.cat((dz, -dz))[:, None].expand(t.shape)
    return {"loss": loss.float(), "rewards": (beta * ratio).float(),
            "grad": _logits_grad(e, total, t, coef, x.dtype)}


def _plain_policy(state, low=0.2, high=0.25):
    x, t, case = state["logits"], state["targets"], state["case"]
    e, total, lp = _softmax_parts(x, t)
    keep = t != IGNORE
    adv = state["advantages"].double()
    adv = adv if case["per_token"] else adv[:, None]
    ratio = torch.exp(lp - state["old"].double())
    term = torch.maximum(-adv * ratio, -adv * ratio.clamp(1.0 - low, 1.0 + high))
    inside = torch.where(adv > 0, ratio <= 1.0 + high, ratio >= 1.0 - low)
    coef = torch.where(inside, -adv * ratio, torch.zeros_like(ratio))
    if case["kl"]:
        gap = state["reference"].double() - lp
        term = term + case["kl"] * (torch.exp(gap) - gap - 1.0)
        coef = coef + case["kl"] * (1.0 - torch.exp(gap))
    if case["aggregate"] == "token":
        weight = keep.double() / keep.sum()
    else:
        count = keep.sum(-1, keepdim=True)
        weight = keep.double() / (count.clamp_min(1) * (count > 0).sum())
    loss = torch.where(keep, term * weight, torch.zeros_like(term)).sum()
    coef = coef * weight * state["loss_grad"].double()
    return {"loss": loss.float(), "log_probs": lp.float(),
            "grad": _logits_grad(e, total, t, coef, x.dtype)}


ADAMW = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1, "step": 1000}


def _plain_adamw8_tensor(p, g, mc, ms, vc, vs):
    """One tensor's step. The new moments are fp32 with each product and sum rounded; their codes
    are the nearest ones."""

    a, pad = ADAMW, -p.numel() % BLOCK
    m, v = _moments(mc, ms, vc, vs, pad)
    gf = g.reshape(-1).float()
    m = m * a["beta1"] + gf * (1.0 - a["beta1"])
    v = v * a["beta2"] + (gf * gf) * (1.0 - a["beta2"])
    size = a["lr"] / (1.0 - a["beta1"] ** a["step"])
    root = 1.0 / math.sqrt(1.0 - a["beta2"] ** a["step"])
    new = p.reshape(-1).float() * (1.0 - a["lr"] * a["weight_decay"])
    new = new - size * (m / (v.sqrt() * root + a["eps"]))
    p.copy_(new.to(p.dtype).view(p.shape))
    for old, now in zip((mc, ms, vc, vs), _quantise(m, v, pad)):
        old.copy_(now)
    return _moments(mc, ms, vc, vs, pad)


def _plain_adamw8(state):
    lists = [state[k] for k in ("params", "grads", "mc", "ms", "vc", "vs")]
    moments = [_plain_adamw8_tensor(*tensors) for tensors in zip(*lists)]
    return {"params": state["params"], "exp_avg": [m for m, _ in moments],
            "exp_avg_sq": [v for _, v in moments]}


def _rotate(x, cosine, sine, layout):
    half = cosine.size(-1)
    body, rest = x[..., : 2 * half].float(), x[..., 2 * half:]
    if layout == "interleaved":
        a, b = body[..., 0::2], body[..., 1::2]
        out = torch.stack((a * cosine - b * sine, a * sine + b * cosine), -1).flatten(-2)
    else:
        a, b = body[..., :half], body[..., half:]
        out = torch.cat((a * cosine - b * sine, a * sine + b * cosine), -1)
    return torch.cat((out.to(x.dtype), rest), -1)


def _plain_rotary(state):
    angle = state["positions"].double()[:, None, :, None] * state["inv_freq"]
    cosine = (angle.cos() * state["scale"]).float()
    sine = (angle.sin() * state["scale"]).float()
    layout = state["case"]["layout"]
    out = {n: _rotate(state[n], cosine, sine, layout) for n in ("q", "k")}
    if state["case"]["grad"]:
        out.update({n: _rotate(state[n], cosine, -sine, layout) for n in ("dq", "dk")})
    return out


# ------------------------------------------------------------------- the framework's --


def _own_logps(state):
    from picotron_b200.kernels import token_log_probs

    if not state["case"]["grad"]:
        return {"log_probs": token_log_probs(state["logits"], state["targets"])}
    x = state["logits"].detach().requires_grad_()
    lp = token_log_probs(x, state["targets"])
    (grad,) = torch.autograd.grad(lp, x, state["grad"])
    return {"log_probs": lp.detach(), "grad": grad}


def _own_preference(state):
    from picotron_b200.kernels import preference_loss

    x = state["logits"].detach().requires_grad_()
    loss, rewards = preference_loss(x, state["targets"], state["reference"], beta=0.1,
                                    label_smoothing=state["case"]["smoothing"])
    (grad,) = torch.autograd.grad(loss, x)
    return {"loss": loss.detach(), "rewards": rewards, "grad": grad}


def _own_policy(state):
    from picotron_b200.kernels import policy_loss

    case = state["case"]
    x = state["logits"].detach().requires_grad_()
    loss, lp = policy_loss(x, state["targets"], state["old"], state["advantages"],
                           reference_log_probs=state["reference"] if case["kl"] else None,
                           kl_coef=case["kl"], clip_low=0.2, clip_high=0.25,
                           aggregate=case["aggregate"])
    (grad,) = torch.autograd.grad(loss, x, state["loss_grad"])
    return {"loss": loss.detach(), "log_probs": lp, "grad": grad}


def _own_adamw8(state):
    from picotron_b200.kernels import adamw8bit_moments, adamw8bit_step

    a, held = ADAMW, [state[k] for k in ("mc", "ms", "vc", "vs")]
    adamw8bit_step(state["params"], state["grads"], *held, step=a["step"], lr=a["lr"],
                   beta1=a["beta1"], beta2=a["beta2"], eps=a["eps"],
                   weight_decay=a["weight_decay"])
    exp_avg, exp_avg_sq = adamw8bit_moments(*held)
    return {"params": state["params"], "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}


def _own_rotary(state):
    from picotron_b200.kernels import apply_rotary_positions

    args = (state["positions"], state["inv_freq"])
    kind = {"layout": state["case"]["layout"], "scale": state["scale"]}
    if not state["case"]["grad"]:
        q, k = apply_rotary_positions(state["q"], state["k"], *args, **kind)
        return {"q": q, "k": k}
    q, k = state["q"].detach().requires_grad_(), state["k"].detach().requires_grad_()
    oq, ok = apply_rotary_positions(q, k, *args, **kind)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (state["dq"], state["dk"]))
    return {"q": oq.detach(), "k": ok.detach(), "dq": dq, "dk": dk}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"logps": _own_logps, "preference": _own_preference, "policy": _own_policy,
                "adamw8": _own_adamw8, "rotary": _own_rotary}[op](state)
    return {"logps": _plain_logps, "preference": _plain_preference, "policy": _plain_policy,
            "adamw8": _plain_adamw8, "rotary": _plain_rotary}[op](state)


# --------------------------------------------------------------------- work and truth --


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("logps", "preference", "policy"):
        rows = case["batch"] * case["seq"]
        # About two thirds of a batch's rows carry a target (prompts and padding do not); only
        # those rows' logits have to be read, while the gradient is written whole.
        share = 0.65 if case["seq"] >= 8 else 1.0
        share *= 1.0 - case.get("empty", 0) / case["batch"]
        grad = case.get("grad", True)
        vocab = case["vocab"]
        return {"bytes": int(rows * vocab * size * (share + (1.0 if grad else 0.0)) + rows * 32),
                "flops": int(rows * vocab * share * (8 if grad else 4))}
    if case["op"] == "adamw8":
        n = sum(math.prod(s) for s in _shapes(case))
        # Parameter read and written, gradient read, two codes read and written; the moments
        # that the codes stand for, as returned, written in fp32.
        return {"bytes": n * (3 * size + 4 + 8), "flops": n * 30}
    rows = case["batch"] * case["seq"]
    n = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
    passes = 2 if case["grad"] else 1
    return {"bytes": passes * 2 * n * size + rows * 8, "flops": passes * 3 * n}


def _exact_loss(case, state):
    """Losses and their gradients from log_softmax and autograd in 64 bits."""

    x = state["logits"].double().requires_grad_(case.get("grad", True))
    t = state["targets"]
    keep = t != IGNORE
    lp = torch.log_softmax(x, -1).gather(-1, t.clamp_min(0).unsqueeze(-1)).squeeze(-1)
    lp = lp.masked_fill(~keep, 0.0)
    if case["op"] == "logps":
        if not case["grad"]:
            return {"log_probs": lp}
        (grad,) = torch.autograd.grad(lp, x, state["grad"].double())
        return {"log_probs": lp.detach(), "grad": grad}
    ref = state["reference"].double()
    if case["op"] == "preference":
        rewards = 0.1 * (lp - ref).masked_fill(~keep, 0.0).sum(1)
        chosen, rejected = rewards.chunk(2)
        good = torch.nn.functional.logsigmoid(chosen - rejected)
        bad = torch.nn.functional.logsigmoid(rejected - chosen)
        loss = -((1 - case["smoothing"]) * good + case["smoothing"] * bad).mean()
        (grad,) = torch.autograd.grad(loss, x)
        return {"loss": loss.detach(), "rewards": rewards.detach(), "grad": grad}
    adv = state["advantages"].double().view(t.size(0), -1)
    ratio = (lp - state["old"].double()).exp()
    gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.25) * adv)
    each = (case["kl"] * ((ref - lp).expm1() - (ref - lp)) - gain).masked_fill(~keep, 0.0)
    if case["aggregate"] == "token":
        loss = each.sum() / keep.sum()
    else:
        some = keep.any(1)
        loss = (each.sum(1)[some] / keep.sum(1)[some]).mean()
    (grad,) = torch.autograd.grad(loss, x, state["loss_grad"].double())
    return {"loss": loss.detach(), "log_probs": lp.detach(), "grad": grad}


def _exact_adamw8(state):
    """The step in 64 bits. The moments are fp32 by definition (every product and sum rounded), so
    the codes are chosen from those: the number of code borders that a moment has reached."""

    a = ADAMW
    out = {"params": [], "exp_avg": [], "exp_avg_sq": []}
    f32 = lambda y: y.float().double()  # noqa: E731  (one rounding to fp32)
    steps = torch.arange(0, 255, device=DEV, dtype=torch.float64) + 0.5
    for p, g, mc, ms, vc, vs in zip(*(state[k] for k in ("params", "grads", "mc", "ms", "vc", "vs"))):
        n = p.numel()
        spread = lambda s: s.double().repeat_interleave(BLOCK)[:n]  # noqa: E731
        p, g = p.double().flatten(), g.double().flatten()
        m0 = f32(mc.double() ** 2 * mc.double().sign() * spread(ms))
        v0 = f32(f32(vc.double() ** 4) * spread(vs))
        b1, w1, b2, w2 = (f32(torch.tensor(w, dtype=torch.float64, device=DEV)) for w in
                          (a["beta1"], 1 - a["beta1"], a["beta2"], 1 - a["beta2"]))
        m = f32(f32(b1 * m0) + f32(w1 * g))
        v = f32(f32(b2 * v0) + f32(w2 * f32(g * g)))
        m64, v64 = a["beta1"] * m0 + (1 - a["beta1"]) * g, a["beta2"] * v0 + (1 - a["beta2"]) * g * g
        hat = m64 / (1 - a["beta1"] ** a["step"])
        root = (v64 / (1 - a["beta2"] ** a["step"])).sqrt()
        p = p * (1 - a["lr"] * a["weight_decay"]) - a["lr"] * hat / (root + a["eps"])
        out["params"].append(p)
        tops = [torch.nn.functional.pad(y, (0, -n % BLOCK)).view(-1, BLOCK).amax(1)
                for y in (m.abs(), v)]
        third, fourth = (f32(torch.tensor(1.0 / k, dtype=torch.float64, device=DEV))
                         for k in (127 ** 2, 255 ** 4))
        ms, vs = spread(f32(tops[0] * third)), spread(f32(tops[1] * fourth))
        c = torch.bucketize(m.abs() / ms, steps[:127] ** 2)
        d = torch.bucketize(v / vs, steps ** 4)
        d = torch.where(v > 0, d.clamp_min(1), d)
        out["exp_avg"].append(c.double() ** 2 * m.sign() * ms)
        out["exp_avg_sq"].append(d.double() ** 4 * vs)
    return out


def _exact_rotary(case, state):
    turn = torch.polar(torch.full((), state["scale"], dtype=torch.float64, device=DEV),
                       state["positions"].double().unsqueeze(-1) * state["inv_freq"]).unsqueeze(1)
    r = case["rotary"]

    def by(x, turn):
        x = x.double()
        y = x[..., :r].unflatten(-1, (-1, 2) if case["layout"] == "interleaved" else (2, -1))
        axis = -1 if case["layout"] == "interleaved" else -2
        z = torch.complex(*y.unbind(axis)) * turn
        return torch.cat((torch.stack((z.real, z.imag), axis).flatten(-2), x[..., r:]), -1)

    out = {"q": by(state["q"], turn), "k": by(state["k"], turn)}
    if case["grad"]:
        out.update(dq=by(state["dq"], turn.conj()), dk=by(state["dk"], turn.conj()))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "adamw8":
        return _exact_adamw8(state)
    return _exact_rotary(case, state) if case["op"] == "rotary" else _exact_loss(case, state)
