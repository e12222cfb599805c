"""Timed cases of the sequence operators: what a token model built from recurrences has the framework do, in training and serving.

Operators (`op`):
  recurrence  gated linear recurrence over T steps, [T, N, D] with the steps outermost, or a batch-first tensor seen that way ("batch_first")
  norm        norm of a block's output, its gate and scale, residual addition, norm in front of the next block, [rows, D]
  scores      log probability of one given token a row, entropy of the row, the largest alternatives, [rows, V]

"grad" cases are training steps: forward, then the gradients of all floating inputs for given gradients of all outputs.
The plain forms compute in float32 and round once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
DEVICE = "cuda:0"
EPS = 1e-6


def listed():
    return [
        # one token for each of 16 requests: the recurrence of one layer, where the latency of a call counts
        {"name": "recurrence_step_16x1024_bf16", "op": "recurrence", "t": 1, "n": 16, "d": 1024, "dtype": "bf16", "form": "leaky", "grad": False,
         "starts": False, "lengths": False, "batch_first": False},
        # the prompt of one request: a long sequence over few channels, which fills the chip only if time is split
        {"name": "recurrence_prompt_8192x1x1024_bf16", "op": "recurrence", "t": 8192, "n": 1, "d": 1024, "dtype": "bf16", "form": "leaky", "grad": False,
         "starts": False, "lengths": False, "batch_first": True},
        # a training step on packed documents: states start anew inside the sequences
        {"name": "recurrence_train_4096x8x2048_bf16", "op": "recurrence", "t": 4096, "n": 8, "d": 2048, "dtype": "bf16", "form": "leaky", "grad": True,
         "starts": True, "lengths": False, "batch_first": True},
        # a training step on a padded batch with an odd number of channels and decays that the program computed itself
        {"name": "recurrence_padded_1531x5x777_f16", "op": "recurrence", "t": 1531, "n": 5, "d": 777, "dtype": "f16", "form": "linear", "grad": True,
         "starts": False, "lengths": True, "batch_first": False},
        # between two blocks of a layer, one token for each of 16 requests
        {"name": "norm_step_16x1024_bf16", "op": "norm", "rows": 16, "d": 1024, "dtype": "bf16", "kind": "rms", "gate": "silu", "scale": True, "grad": False},
        # the same for the tokens of a batch of prompts
        {"name": "norm_prompt_8192x2048_bf16", "op": "norm", "rows": 8192, "d": 2048, "dtype": "bf16", "kind": "rms", "gate": "silu", "scale": True, "grad": False},
        # a training step
        {"name": "norm_train_32768x2048_bf16", "op": "norm", "rows": 32768, "d": 2048, "dtype": "bf16", "kind": "rms", "gate": "silu", "scale": True, "grad": True},
        # a training step in float32 with an odd width, the mean taken out, no gate
        {"name": "norm_odd_1531x777_f32", "op": "norm", "rows": 1531, "d": 777, "dtype": "f32", "kind": "layer", "gate": "none", "scale": False, "grad": True},
        # the next token of 16 requests, with 8 alternatives each: few rows, which fill the chip only if they are split
        {"name": "scores_step_16x32000_bf16", "op": "scores", "rows": 16, "v": 32000, "dtype": "bf16", "k": 8, "masked": False, "grad": False},
        # the answer of a classifier network on a batch: the five best of 1000 classes
        {"name": "scores_classes_64x1000_f32", "op": "scores", "rows": 64, "v": 1000, "dtype": "f32", "k": 5, "masked": False, "grad": False},
        # a training step: log probability and entropy of every token of a batch
        {"name": "scores_train_8192x32000_bf16", "op": "scores", "rows": 8192, "v": 32000, "dtype": "bf16", "k": 0, "masked": False, "grad": True},
        # scoring prompts under a vocabulary mask, an odd number of tokens (every second row starts off the alignment)
        {"name": "scores_masked_500x50021_bf16", "op": "scores", "rows": 500, "v": 50021, "dtype": "bf16", "k": 20, "masked": True, "grad": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["recurrence", "norm", "scores"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    size = SIZES[dtype]
    if op == "recurrence":
        d = _spread(rng, 64, 4096)
        d = d if rng.random() < 0.4 else max(64, d // 64 * 64)
        grad = rng.random() < 0.5
        most = 4096 * 8 * 2048 * 2 * (1 if grad else 2) // size
        n = _spread(rng, 1, 64)
        t = min(_spread(rng, 1, 16384), max(1, most // (n * d)))
        return {"op": op, "t": t, "n": n, "d": d, "dtype": dtype, "form": rng.choice(["leaky", "linear"]), "grad": grad,
                "starts": rng.random() < 0.4, "lengths": rng.random() < 0.4, "batch_first": rng.random() < 0.5}
    if op == "norm":
        d = _spread(rng, 64, 8192)
        d = d if rng.random() < 0.4 else max(64, d // 64 * 64)
        grad = rng.random() < 0.5
        most = 32768 * 2048 * 2 * (1 if grad else 2) // size
        rows = min(_spread(rng, 1, 32768), most // d)
        return {"op": op, "rows": rows, "d": d, "dtype": dtype, "kind": rng.choice(["rms", "rms", "layer"]),
                "gate": rng.choice(["silu", "sigmoid", "none"]), "scale": rng.random() < 0.7, "grad": grad}
    v = _spread(rng, 1000, 131072)
    v = v if rng.random() < 0.4 else max(1000, v // 8 * 8)
    grad = rng.random() < 0.5
    most = 8192 * 32000 * 2 * (1 if grad else 2) // (3 * size)
    rows = min(_spread(rng, 1, 8192), max(1, most // v))
    return {"op": op, "rows": rows, "v": v, "dtype": dtype, "k": 0 if grad else rng.choice([0, 1, 5, 8, 20]), "masked": rng.random() < 0.3, "grad": grad}


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, to=dtype):
        return (torch.randn(shape, generator=g, device=DEVICE) * std + mean).to(to)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEVICE)

    state = {"case": dict(case)}
    if case["op"] == "recurrence":
        t, n, d = case["t"], case["n"], case["d"]
        order = (n, t) if case["batch_first"] else (t, n)

        def steps(make):                                   # [T, N, D] as the program holds it
            a = make(*order, d)
            return a.transpose(0, 1) if case["batch_first"] else a

        # Channels remember over a few to a few thousand steps.
        memory = torch.exp(uniform(d) * 7.0 + 0.7)
        if case["form"] == "leaky":
            gate = steps(lambda *s: (torch.randn(s, generator=g, device=DEVICE) + torch.log(memory)).to(dtype))
        else:
            gate = steps(lambda *s: torch.exp(-torch.exp(0.5 * torch.randn(s, generator=g, device=DEVICE)) / memory).to(dtype))
        state.update(x=steps(normal), gate=gate, state=normal(n, d, std=0.5, to=torch.float32), starts=None, lengths=None)
        if case["starts"]:
            state["starts"] = uniform(t, n) < 1.0 / 512
        if case["lengths"]:
            state["lengths"] = torch.randint(max(1, t // 3), t + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32)
        if case["grad"]:
            state.update(dh=steps(normal), dstate=normal(n, d, to=torch.float32))
        leaves = ("x", "gate", "state")
    elif case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        state.update(residual=normal(rows, d, std=2.0), branch=normal(rows, d, mean=0.2, std=0.7), branch_weight=normal(d, mean=1.0, std=0.1),
                     next_weight=normal(d, mean=1.0, std=0.1), gate=None if case["gate"] == "none" else normal(rows, d), scale=None)
        if case["scale"]:
            state["scale"] = normal(d, mean=0.5, std=0.2)
        if case["grad"]:
            state.update(dresidual=normal(rows, d), dnormed=normal(rows, d))
        leaves = ("residual", "branch", "gate", "branch_weight", "next_weight", "scale")
    else:
        rows, v = case["rows"], case["v"]
        logits = torch.randn((rows, v), generator=g, device=DEVICE) * 2.5
        tokens = torch.randint(0, v, (rows,), generator=g, device=DEVICE)
        logits.scatter_add_(1, tokens[:, None], 8.0 * uniform(rows, 1))
        if case["masked"]:
            logits.masked_fill_((uniform(v) < 0.3)[None, :], -math.inf)
            logits.scatter_(1, tokens[:, None], 4.0)
            tokens = torch.where(uniform(rows) < 0.1, torch.full_like(tokens, -100), tokens)      # rows that no token is given for
        state.update(logits=logits.to(dtype), tokens=tokens)
        if case["grad"]:
            state.update(dlogprob=normal(rows, mean=-1.0 / rows, std=0.3 / rows, to=torch.float32), dentropy=normal(rows, mean=-0.01 / rows, std=0.003 / rows, to=torch.float32))
        leaves = ("logits",)
    if case["grad"]:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------------------------
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first dimension, by doubling the span that each element covers."""
    span = 1
    while span < a.shape[0]:
        b = torch.cat([b[:span], b[span:] + a[span:] * b[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return b


def _plain_recurrence(s):
    case = s["case"]
    dtype = s["x"].dtype
    x, gate = s["x"].detach().float(), s["gate"].detach().float()
    h0 = s["state"].detach()
    a, keep = (torch.sigmoid(gate), torch.sigmoid(-gate)) if case["form"] == "leaky" else (gate, None)
    b = x if keep is None else keep * x
    carried = a if s["starts"] is None else torch.where(s["starts"][:, :, None], 0.0, a)
    inside = None
    if s["lengths"] is not None:
        inside = (torch.arange(case["t"], device=DEVICE)[:, None] < s["lengths"][None, :])[:, :, None]
        carried, b = torch.where(inside, carried, 1.0), torch.where(inside, b, 0.0)
    h = _scan(carried, torch.cat([b[:1] + carried[:1] * h0, b[1:]]))
    last = h[-1].clone()
    shown = h if inside is None else torch.where(inside, h, 0.0)
    out = [shown.to(dtype), last]
    if case["grad"]:
        dh = s["dh"].float()
        if inside is not None:
            dh = torch.where(inside, dh, 0.0)
        dh = torch.cat([dh[:-1], dh[-1:] + s["dstate"]])
        behind = torch.cat([carried[1:], torch.zeros_like(carried[:1])])
        total = _scan(behind.flip(0), dh.flip(0)).flip(0)
        before = torch.cat([h0[None], h[:-1]])
        if s["starts"] is not None:
            before = torch.where(s["starts"][:, :, None], 0.0, before)
        dx, dgate = (total, total * before) if keep is None else (total * keep, total * (before - x) * (a * keep))
        if inside is not None:
            dx, dgate = torch.where(inside, dx, 0.0), torch.where(inside, dgate, 0.0)
        out += [dx.to(dtype), dgate.to(dtype), carried[0] * total[0]]
    return out


def _plain_norm(s):
    case = s["case"]
    dtype = s["branch"].dtype
    d = case["d"]
    residual, branch = s["residual"].detach().float(), s["branch"].detach().float()
    wb, wn = s["branch_weight"].detach().float(), s["next_weight"].detach().float()
    scale = 1.0 if s["scale"] is None else s["scale"].detach().float()
    layer = case["kind"] == "layer"

    def whiten(v):
        v = v - v.mean(1, keepdim=True) if layer else v
        r = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
        return v * r, r

    def whiten_gradient(dy, y, r):
        dv = dy - y * (dy * y).mean(1, keepdim=True)
        return r * (dv - dy.mean(1, keepdim=True) if layer else dv)

    unit, r1 = whiten(branch)
    if s["gate"] is None:
        gate, act = None, 1.0
    else:
        gate = s["gate"].detach().float()
        sig = torch.sigmoid(gate)
        act = gate * sig if case["gate"] == "silu" else sig
    u = unit * wb
    total = residual + scale * act * u
    normed, r2 = whiten(total)
    out = [total.to(dtype), (normed * wn).to(dtype)]
    if case["grad"]:
        dn, dt = s["dnormed"].float(), s["dresidual"].float()
        dt = dt + whiten_gradient(dn * wn, normed, r2)
        du = dt * scale * act
        out += [dt.to(dtype), whiten_gradient(du * wb, unit, r1).to(dtype)]
        if gate is not None:
            slope = sig * (1.0 + gate * (1.0 - sig)) if case["gate"] == "silu" else sig * (1.0 - sig)
            out.append((dt * scale * u * slope).to(dtype))
        out += [(du * unit).sum(0).to(dtype), (dn * normed).sum(0).to(dtype)]
        if s["scale"] is not None:
            out.append((dt * act * u).sum(0).to(dtype))
    return out


def _plain_scores(s):
    case = s["case"]
    logits, tokens = s["logits"].detach(), s["tokens"]
    x = logits.float()
    peak = x.max(1, keepdim=True).values
    e = torch.exp(x - peak)
    total = e.sum(1, keepdim=True)
    lse = peak + torch.log(total)
    p = e / total
    logp = x - lse
    surprise = torch.where(p > 0, p * logp, 0.0)
    entropy = -surprise.sum(1)
    given = tokens >= 0
    index = tokens.clamp(min=0)[:, None]
    out = [torch.where(given, logp.gather(1, index)[:, 0], 0.0), entropy]
    if case["k"]:
        best = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["k"]]      # ties: the lowest index first
        out += [logp.gather(1, best), best]
    if case["grad"]:
        pull = torch.where(given, s["dlogprob"], 0.0)[:, None]
        d = -pull * p - s["dentropy"][:, None] * torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
        out.append(d.scatter_add(1, index, pull).to(logits.dtype))
    return out


# ------------------------------------------------------------------------------------------------------------------
# The framework's operators
# ------------------------------------------------------------------------------------------------------------------
def _own_recurrence(s):
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    h, last = run_hip_gated_recurrence(s["x"], s["gate"], s["state"], form=s["case"]["form"], starts=s["starts"], lengths=s["lengths"])
    if not s["case"]["grad"]:
        return [h, last]
    return [h, last, *torch.autograd.grad([h, last], [s["x"], s["gate"], s["state"]], [s["dh"], s["dstate"]])]


def _own_norm(s):
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    residual, normed = run_hip_block_norm(s["residual"], s["branch"], gate=s["gate"], branch_weight=s["branch_weight"], next_weight=s["next_weight"],
                                          scale=s["scale"], kind=s["case"]["kind"], gate_form="silu" if s["gate"] is None else s["case"]["gate"], eps=EPS)
    if not s["case"]["grad"]:
        return [residual, normed]
    leaves = [s[name] for name in ("residual", "branch", "gate", "branch_weight", "next_weight", "scale") if s[name] is not None]
    return [residual, normed, *torch.autograd.grad([residual, normed], leaves, [s["dresidual"], s["dnormed"]])]


def _own_scores(s):
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    scores = run_hip_token_scores(s["logits"], s["tokens"], top_k=s["case"]["k"])
    out = [scores.logprob, scores.entropy]
    if s["case"]["k"]:
        out += [scores.top_logprob, scores.top_token]
    if s["case"]["grad"]:
        out += torch.autograd.grad(out, [s["logits"]], [s["dlogprob"], s["dentropy"]])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"recurrence": _own_recurrence, "norm": _own_norm, "scores": _own_scores}[op](state)
    return {"recurrence": _plain_recurrence, "norm": _plain_norm, "scores": _plain_scores}[op](state)


# ------------------------------------------------------------------------------------------------------------------
# Work and exact values
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "recurrence":
        t, n, d = case["t"], case["n"], case["d"]
        elements = t * n * d
        small = (t * n if case["starts"] else 0) + (4 * n if case["lengths"] else 0)
        if case["grad"]:                                   # x, gate, dh in; h, dx, dgate out; the state and its gradient in and out
            return {"bytes": 6 * elements * size + 16 * n * d + small, "flops": 24 * elements}
        return {"bytes": 3 * elements * size + 8 * n * d + small, "flops": 8 * elements}
    if case["op"] == "norm":
        elements, d = case["rows"] * case["d"], case["d"]
        gated, vectors = case["gate"] != "none", 2 + case["scale"]
        if case["grad"]:
            return {"bytes": (8 + 2 * gated) * elements * size + 2 * vectors * d * size, "flops": 44 * elements}
        return {"bytes": (4 + gated) * elements * size + vectors * d * size, "flops": 14 * elements}
    rows, v = case["rows"], case["v"]
    answers = rows * (8 + 4 + 4 + 12 * case["k"])
    if case["grad"]:
        return {"bytes": 2 * rows * v * size + answers + 8 * rows, "flops": 14 * rows * v}
    return {"bytes": rows * v * size + answers, "flops": 6 * rows * v}


def _exact_recurrence(case, s):
    t, n = case["t"], case["n"]
    x, gate, h = s["x"].detach().double(), s["gate"].detach().double(), s["state"].detach().double()
    leaky = case["form"] == "leaky"
    a = 1.0 / (1.0 + torch.exp(-gate)) if leaky else gate
    into = 1.0 / (1.0 + torch.exp(gate)) if leaky else torch.ones_like(gate)
    starts = torch.zeros(t, n, 1, dtype=torch.bool, device=DEVICE) if s["starts"] is None else s["starts"][:, :, None]
    lengths = torch.full((n,), t, device=DEVICE) if s["lengths"] is None else s["lengths"]
    inside = (torch.arange(t, device=DEVICE)[:, None] < lengths[None, :])[:, :, None]
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    before, after = torch.empty_like(x), torch.empty_like(x)
    drive = into * x
    for i in range(t):
        before[i] = torch.where(starts[i], zero, h)
        h = torch.where(inside[i], torch.addcmul(drive[i], a[i], before[i]), h)
        after[i] = h
    out = [torch.where(inside, after, zero), h]
    if case["grad"]:
        del after, drive
        later, dx, dgate, dh = s["dstate"].double(), torch.empty_like(x), torch.empty_like(x), s["dh"].double()
        slope = a * into if leaky else into
        for i in range(t - 1, -1, -1):
            total = later + dh[i]
            dx[i] = torch.where(inside[i], total * into[i], zero)
            dgate[i] = torch.where(inside[i], total * (before[i] - x[i] if leaky else before[i]) * slope[i], zero)
            later = torch.where(inside[i], torch.where(starts[i], zero, total * a[i]), later)
        out += [dx, dgate, later]
    return out


def _exact_norm(case, s):
    names = [name for name in ("residual", "branch", "gate", "branch_weight", "next_weight", "scale") if s[name] is not None]
    v = {name: s[name].detach().double().requires_grad_(case["grad"]) for name in names}

    def norm(a):
        if case["kind"] == "layer":
            return (a - a.mean(-1, keepdim=True)) / torch.sqrt(a.var(-1, unbiased=False, keepdim=True) + EPS)
        return a / torch.sqrt(a.pow(2).mean(-1, keepdim=True) + EPS)

    block = norm(v["branch"]) * v["branch_weight"]
    if "gate" in v:
        block = block / (1.0 + torch.exp(-v["gate"])) * (v["gate"] if case["gate"] == "silu" else 1.0)
    if "scale" in v:
        block = block * v["scale"]
    residual = v["residual"] + block
    normed = norm(residual) * v["next_weight"]
    out = [residual.detach(), normed.detach()]
    if case["grad"]:
        out += torch.autograd.grad([residual, normed], [v[name] for name in names], [s["dresidual"].double(), s["dnormed"].double()])
    return out


def _exact_scores(case, s):
    x, tokens = s["logits"].detach().double(), s["tokens"]
    rows = torch.arange(case["rows"], device=DEVICE)
    lse = torch.logsumexp(x, 1)
    logp = x - lse[:, None]
    p = torch.exp(logp)
    finite = torch.where(p > 0, logp, 0.0)
    entropy = -(p * finite).sum(1)
    given = tokens >= 0
    at = tokens.clamp(min=0)
    out = [torch.where(given, logp[rows, at], 0.0), entropy]
    if case["k"]:
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["k"]]
        out += [logp.gather(1, best), best]
    if case["grad"]:
        pull = torch.where(given, s["dlogprob"].double(), 0.0)
        d = p * (-pull[:, None] - s["dentropy"].double()[:, None] * (finite + entropy[:, None]))
        d[rows, at] += pull
        out.append(d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "norm": _exact_norm, "scores": _exact_scores}[case["op"]](case, s)
