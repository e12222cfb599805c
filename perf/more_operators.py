"""Timed cases of two more sequence operators: the gated delta rule, in training and serving, and the verification of drafted tokens.

Operators (`op`):
  delta   gated delta rule over T steps, heads of [Dk] queries and keys and [Dv] values, [T, N, heads, D] with the steps outermost, or a batch-first
          tensor seen that way ("batch_first"); a state of [Dk, Dv] in float32 for each sequence and value head
  verify  drafted tokens against the target's distribution, [N, K + 1, V] logits, from given random numbers

"grad" cases are training steps: forward, then the gradients of all floating inputs for given gradients of all outputs.
The plain forms compute in float32 and round once at the end; in float64 the sums of logarithms of decays, of which differences are taken, and what
decides between tokens.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
DEVICE = "cuda:0"
CHUNK = 64


def listed():
    return [
        # one token for each of 16 requests: one layer's step, which reads and writes the states
        {"name": "delta_step_16x16x128_bf16", "op": "delta", "t": 1, "n": 16, "h": 8, "hv": 16, "dk": 128, "dv": 128, "dtype": "bf16", "gates": "f32",
         "grad": False, "starts": False, "lengths": False, "batch_first": False},
        # the same for drafted tokens, of which each request keeps as many as were accepted
        {"name": "delta_drafts_5x16x16x128_bf16", "op": "delta", "t": 5, "n": 16, "h": 8, "hv": 16, "dk": 128, "dv": 128, "dtype": "bf16", "gates": "f32",
         "grad": False, "starts": False, "lengths": True, "batch_first": True},
        # the prompt of one request: a long sequence over few heads
        {"name": "delta_prompt_8192x1x16x128_bf16", "op": "delta", "t": 8192, "n": 1, "h": 8, "hv": 16, "dk": 128, "dv": 128, "dtype": "bf16", "gates": "f32",
         "grad": False, "starts": False, "lengths": False, "batch_first": True},
        # prompts of a batch, padded to the longest
        {"name": "delta_prompts_2048x16x16x128_bf16", "op": "delta", "t": 2048, "n": 16, "h": 16, "hv": 16, "dk": 128, "dv": 128, "dtype": "bf16", "gates": "f32",
         "grad": False, "starts": False, "lengths": True, "batch_first": True},
        # a training step on packed documents: states start anew inside the sequences
        {"name": "delta_train_4096x4x16x128_bf16", "op": "delta", "t": 4096, "n": 4, "h": 16, "hv": 16, "dk": 128, "dv": 128, "dtype": "bf16", "gates": "bf16",
         "grad": True, "starts": True, "lengths": False, "batch_first": True},
        # a training step on a padded batch with heads of odd sizes, two value heads to a key head
        {"name": "delta_padded_1531x3x6x80_f16", "op": "delta", "t": 1531, "n": 3, "h": 3, "hv": 6, "dk": 96, "dv": 80, "dtype": "f16", "gates": "f16",
         "grad": True, "starts": False, "lengths": True, "batch_first": False},
        # a training step in float32
        {"name": "delta_train_1000x2x5x65_f32", "op": "delta", "t": 1000, "n": 2, "h": 5, "hv": 5, "dk": 64, "dv": 65, "dtype": "f32", "gates": "f32",
         "grad": True, "starts": False, "lengths": False, "batch_first": True},
        # four drafts of one request
        {"name": "verify_step_1x4x32000_bf16", "op": "verify", "n": 1, "k": 4, "v": 32000, "dtype": "bf16", "draft": True, "temperature": "one", "lengths": False},
        # drafts that were looked up and have no distribution, numbers of them that differ
        {"name": "verify_lookup_32x8x32000_f32", "op": "verify", "n": 32, "k": 8, "v": 32000, "dtype": "f32", "draft": False, "temperature": "each", "lengths": True},
        # a batch with an odd vocabulary, temperatures and numbers of drafts of its requests
        {"name": "verify_batch_64x5x50021_bf16", "op": "verify", "n": 64, "k": 5, "v": 50021, "dtype": "bf16", "draft": True, "temperature": "each", "lengths": True},
        # a large batch and vocabulary
        {"name": "verify_batch_256x4x128000_bf16", "op": "verify", "n": 256, "k": 4, "v": 128000, "dtype": "bf16", "draft": True, "temperature": "one", "lengths": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    size = SIZES[dtype]
    if rng.random() < 0.6:
        grad = rng.random() < 0.5
        group = rng.choice([1, 1, 2, 4])
        h = _spread(rng, 1, 16)
        dk, dv = (_spread(rng, 16, 128), _spread(rng, 16, 256)) if rng.random() < 0.4 else (rng.choice([64, 128]), rng.choice([64, 128]))
        n = min(_spread(rng, 1, 64), 256 // (h * group))
        most = 4096 * 4 * 16 * 128 * 2 // (2 * size)
        t = rng.choice([1, 2, 4, 7]) if rng.random() < 0.25 else _spread(rng, 16, 8192)
        t = max(1, min(t, most // (max(1, n) * h * group * max(dk, dv))))
        return {"op": "delta", "t": t, "n": max(1, n), "h": h, "hv": h * group, "dk": dk, "dv": dv, "dtype": dtype, "gates": dtype if grad else rng.choice([dtype, "f32"]),
                "grad": grad, "starts": rng.random() < 0.3, "lengths": rng.random() < 0.4, "batch_first": rng.random() < 0.5}
    v = _spread(rng, 1000, 131072)
    v = v if rng.random() < 0.4 else max(1000, v // 8 * 8)
    k = rng.randint(1, 8)
    draft = rng.random() < 0.7
    most = 256 * 4 * 128000 * 2 // size
    n = max(1, min(_spread(rng, 1, 256), most // (v * (2 * k + 1 if draft else k + 1))))
    return {"op": "verify", "n": n, "k": k, "v": v, "dtype": dtype, "draft": draft, "temperature": rng.choice(["one", "each"]), "lengths": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEVICE)
    state = {"case": dict(case)}
    if case["op"] == "delta":
        t, n, h, hv, dk, dv = (case[name] for name in ("t", "n", "h", "hv", "dk", "dv"))
        gates = DTYPES[case["gates"]]

        def steps(make, *rest):                            # [T, N, ...] as the program holds it
            a = make(*((n, t) if case["batch_first"] else (t, n)), *rest)
            return a.transpose(0, 1) if case["batch_first"] else a

        def rows(*rest):                                   # what a projection and an activation leave, brought to length 1
            a = torch.nn.functional.silu(normal(*rest))
            return (a / a.norm(dim=-1, keepdim=True)).to(dtype)

        # Heads remember over a few to a few thousand steps.
        memory = torch.exp(uniform(hv) * 6.0 + 1.0)
        state.update(query=steps(rows, h, dk), key=steps(rows, h, dk), value=steps(lambda *s: normal(*s).to(dtype), hv, dv),
                     gate=steps(lambda *s: (-torch.exp(0.5 * normal(*s)) / memory).to(gates), hv), beta=steps(lambda *s: torch.sigmoid(normal(*s)).to(gates), hv),
                     state=normal(n, hv, dk, dv) * 0.3, starts=None, lengths=None)
        if case["starts"]:
            state["starts"] = uniform(t, n) < 1.0 / 512
        if case["lengths"]:
            state["lengths"] = torch.randint(max(1, t // 3), t + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32)
        if case["grad"]:
            state.update(dout=steps(lambda *s: normal(*s).to(dtype), hv, dv), dstate=normal(n, hv, dk, dv) * 0.3)
            for name in ("query", "key", "value", "gate", "beta", "state"):
                state[name].requires_grad_(True)
        return state
    n, k, v = case["n"], case["k"], case["v"]
    logits = normal(n, k + 1, v) * 2.5
    peaks = torch.randint(0, v, (n, k + 1, 4), generator=g, device=DEVICE)           # a few tokens are likely
    logits.scatter_add_(2, peaks, 11.0 * uniform(n, k + 1, 4))
    draft = logits[:, :k] + 0.8 * normal(n, k, v)                                    # a smaller model's idea of them
    state.update(logits=logits.to(dtype), draft_logits=draft.to(dtype) if case["draft"] else None, temperature=1.0, lengths=None,
                 uniforms=uniform(n, k), noise=-torch.log(1.0 - uniform(n, v)).clamp(min=1e-12))
    if case["temperature"] == "each":                                                # a quarter of the requests are answered greedily
        state["temperature"] = torch.where(uniform(n) < 0.25, 0.0, 0.5 + uniform(n))
    if case["lengths"]:
        state["lengths"] = torch.randint(0, k + 1, (n,), generator=g, device=DEVICE, dtype=torch.int32)
    state["drafts"] = (draft - torch.log(-torch.log(uniform(n, k, v).clamp(min=1e-12)).clamp(min=1e-12))).argmax(2)       # drawn from it
    if not case["draft"]:
        state["drafts"] = torch.where(uniform(n, k) < 0.7, logits[:, :k].argmax(2), state["drafts"])
    return state


# ------------------------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------------------------
def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular matrices of 2^j rows, from the inverses of their diagonal blocks."""
    size = a.shape[-1]
    inverse, block = torch.ones_like(a[..., :1]).unsqueeze(-1), 1                     # [..., blocks, block, block]
    while block < size:
        count = size // (2 * block)
        tiles = a.unflatten(-1, (count, 2, block)).unflatten(-4, (count, 2, block))   # [..., count, 2, block, count, 2, block]
        below = torch.diagonal(tiles[..., 1, :, :, 0, :], dim1=-4, dim2=-2).movedim(-1, -3)
        inverse = inverse.unflatten(-3, (count, 2))
        first, second = inverse[..., 0, :, :], inverse[..., 1, :, :]
        corner = -(second @ below @ first)
        inverse = torch.cat([torch.cat([first, torch.zeros_like(first)], -1), torch.cat([corner, second], -1)], -2)
        block *= 2
    return inverse[..., 0, :, :]


def _plain_delta_forward(s, query, key, value, gate, beta, state):
    case = s["case"]
    t, n, dk = case["t"], case["n"], case["dk"]
    inside = torch.ones(t, n, dtype=torch.bool, device=DEVICE) if s["lengths"] is None else torch.arange(t, device=DEVICE)[:, None] < s["lengths"][None, :]
    starts = torch.zeros(t, n, dtype=torch.bool, device=DEVICE) if s["starts"] is None else s["starts"] & inside
    chunk = min(CHUNK, 1 << (t - 1).bit_length())
    count = -(-t // chunk)

    def chunks(a, heads):                                  # [T, N, H, ...] to [count, N, Hv, chunk, ...]
        a = torch.where(inside.reshape(t, n, *[1] * (a.dim() - 2)), a.float(), 0.0)
        a = torch.cat([a, a.new_zeros(count * chunk - t, *a.shape[1:])]).unflatten(0, (count, chunk))
        a = a.movedim(1, 3)
        return a if heads == case["hv"] else a.repeat_interleave(case["hv"] // heads, 2)

    q, k, v = chunks(query, case["h"]), chunks(key, case["h"]), chunks(value, case["hv"])
    g, b = chunks(gate, case["hv"]), chunks(beta, case["hv"])
    fresh = torch.cat([starts, starts.new_zeros(count * chunk - t, n)]).unflatten(0, (count, chunk)).movedim(1, 2)[:, :, None]
    g = torch.where(fresh, 0.0, g)
    part = fresh.cumsum(3)                                 # 0 as long as the state before the chunk lasts
    total = g.double().cumsum(3)
    between = total[..., :, None] - total[..., None, :]
    lower = torch.ones(chunk, chunk, dtype=torch.bool, device=DEVICE).tril()
    decay = torch.where(lower & (part[..., :, None] == part[..., None, :]), between, -math.inf).float().exp()
    since = torch.where(part == 0, total, -math.inf).float().exp()[..., None]
    until = torch.where(part == part[..., -1:], total[..., -1:] - total, -math.inf).float().exp()[..., None]
    kt = k.transpose(-1, -2)
    inverse = _unit_lower_inverse((k @ kt * decay * b[..., None]).tril(-1))
    scores = q @ kt * decay * dk ** -0.5
    outs = []
    for c in range(count):
        u = inverse[c] @ (b[c][..., None] * (v[c] - since[c] * (k[c] @ state)))
        outs.append(dk ** -0.5 * since[c] * (q[c] @ state) + scores[c] @ u)
        state = since[c][..., -1:, :] * state + kt[c] @ (until[c] * u)
    out = torch.stack(outs).movedim(3, 1).flatten(0, 1)[:t]
    return torch.where(inside[:, :, None, None], out, 0.0).to(value.dtype), state


def _plain_delta(s):
    leaves = [s[name] for name in ("query", "key", "value", "gate", "beta", "state")]
    if not s["case"]["grad"]:
        return list(_plain_delta_forward(s, *leaves))
    leaves = [a.detach().float().requires_grad_(True) for a in leaves]                # their gradients are rounded once, at the end
    out, last = _plain_delta_forward(s, *leaves)
    grads = torch.autograd.grad([out, last], leaves, [s["dout"].float(), s["dstate"]])
    dtype, gates = DTYPES[s["case"]["dtype"]], DTYPES[s["case"]["gates"]]
    return [out.detach().to(dtype), last.detach(), *(d.to(kind) for d, kind in zip(grads, (dtype, dtype, dtype, gates, gates, torch.float32)))]


def _temperatures(s):
    t = s["temperature"]
    return t.double() if isinstance(t, torch.Tensor) else torch.full((s["case"]["n"],), float(t), dtype=torch.float64, device=DEVICE)


def _plain_verify(s):
    n, k = s["case"]["n"], s["case"]["k"]
    t = _temperatures(s)[:, None, None]
    greedy = t == 0
    row = torch.arange(n, device=DEVICE)

    def probabilities(x):
        first = torch.zeros_like(x, dtype=torch.float64).scatter_(2, x.argmax(2, keepdim=True), 1.0)
        x = x.double() / torch.where(greedy, 1.0, t)
        e = torch.exp(x - x.max(2, keepdim=True).values)
        return torch.where(greedy, first, e / e.sum(2, keepdim=True))

    drafts = s["drafts"]
    p = probabilities(s["logits"])
    q = torch.zeros_like(p[:, :k]).scatter_(2, drafts[..., None], 1.0)
    if s["draft_logits"] is not None:
        q = torch.where(greedy, q, probabilities(s["draft_logits"]))
    length = torch.full((n,), k, device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    pd, qd = p[:, :k].gather(2, drafts[..., None])[..., 0], q.gather(2, drafts[..., None])[..., 0]
    places = torch.arange(k + 1, device=DEVICE)[None]
    taken = (s["uniforms"].double() * qd < pd) & (places[:, :k] < length[:, None])
    accepted = taken.long().cumprod(1).sum(1)
    at = p[row, accepted]
    less = torch.where((accepted < length)[:, None], q[row, accepted.clamp(max=k - 1)], 0.0)
    rest = (at - less).clamp(min=0)
    rest = torch.where(rest.amax(1, keepdim=True) > 0, rest, at)
    token = (rest / s["noise"].double()).argmax(1)
    tokens = torch.where(places < accepted[:, None], torch.cat([drafts, drafts[:, :1]], 1), torch.where(places == accepted[:, None], token[:, None], -100))
    return [tokens, accepted.int()]


# ------------------------------------------------------------------------------------------------------------------
# The framework's operators
# ------------------------------------------------------------------------------------------------------------------
def _own_delta(s):
    from triton_snn_fusion_amd.runtime.hip_delta_rule_backend import run_hip_delta_rule
    leaves = [s[name] for name in ("query", "key", "value", "gate", "beta", "state")]
    out, last = run_hip_delta_rule(*leaves, starts=s["starts"], lengths=s["lengths"])
    if not s["case"]["grad"]:
        return [out, last]
    return [out, last, *torch.autograd.grad([out, last], leaves, [s["dout"], s["dstate"]])]


def _own_verify(s):
    from triton_snn_fusion_amd.runtime.hip_draft_verification_backend import run_hip_draft_verification
    answer = run_hip_draft_verification(s["logits"], s["drafts"], s["uniforms"], s["noise"], draft_logits=s["draft_logits"], temperature=s["temperature"],
                                        lengths=s["lengths"])
    return [answer.tokens, answer.accepted]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"delta": _own_delta, "verify": _own_verify}[op](state)
    return {"delta": _plain_delta, "verify": _plain_verify}[op](state)


# ------------------------------------------------------------------------------------------------------------------
# Work and exact values
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "verify":
        n, k, v = case["n"], case["k"], case["v"]
        rows = n * (k + 1 + (k if case["draft"] else 0))
        return {"bytes": rows * v * size + 4 * n * v + 24 * n * k, "flops": 6 * rows * v + 8 * n * v}
    t, n, h, hv, dk, dv = (case[name] for name in ("t", "n", "h", "hv", "dk", "dv"))
    moved = t * n * (size * (2 * h * dk + 2 * hv * dv) + 2 * SIZES[case["gates"]] * hv) + 8 * n * hv * dk * dv
    if case["starts"]:
        moved += t * n
    if case["grad"]:      # the inputs are read and gradients of all of them written; the gradient of the output comes in
        moved += t * n * (size * (2 * h * dk + 2 * hv * dv) + 2 * SIZES[case["gates"]] * hv) + 8 * n * hv * dk * dv
    # each step's key with the state, its correction, its query with the state: three products of Dk x Dv, and twice that many backwards
    return {"bytes": moved, "flops": (18 if case["grad"] else 6) * t * n * hv * dk * dv}


def _exact_delta(case, s):
    t, n, h, hv, dk, dv = (case[name] for name in ("t", "n", "h", "hv", "dk", "dv"))
    wide = lambda a: a.detach().double().repeat_interleave(hv // a.shape[2], 2)
    q, k, v, g, b = (wide(s[name]) for name in ("query", "key", "value", "gate", "beta"))
    scale = 1.0 / math.sqrt(dk)
    a = torch.exp(g)
    if s["starts"] is not None:
        a = a * (~s["starts"])[:, :, None]
    last_step = torch.full((n,), t, device=DEVICE) if s["lengths"] is None else s["lengths"]
    live = (torch.arange(t, device=DEVICE)[:, None] < last_step[None, :]).double()[:, :, None]
    # a step that is not live neither decays nor learns
    a, b = torch.where(live > 0, a, 1.0), b * live
    column = lambda x: x[..., None]
    across = lambda x: x[..., None, :]

    def step(state, i):
        held = state * column(column(a[i]))
        delta = v[i] - (across(k[i]) @ held)[..., 0, :]
        return held, delta, held + column(k[i]) @ across(b[i][..., None] * delta)

    state, out, marks = s["state"].detach().double(), torch.zeros(t, n, hv, dv, dtype=torch.float64, device=DEVICE), []
    for i in range(t):
        if i % 64 == 0:
            marks.append(state)
        _, _, state = step(state, i)
        out[i] = scale * live[i][..., None] * (across(q[i]) @ state)[..., 0, :]
    if not case["grad"]:
        return [out, state]
    last = state
    do, later = s["dout"].double() * live[..., None], s["dstate"].double()
    dq, dk_, dv_, dg, db = (torch.zeros_like(x) for x in (q, k, v, g, b))
    for first in range((t - 1) // 64 * 64, -1, -64):
        states = [marks.pop()]
        for i in range(first, min(first + 64, t)):
            states.append(step(states[-1], i)[2])
        for i in range(min(first + 64, t) - 1, first - 1, -1):
            held, delta, now = step(states[i - first], i)
            dq[i] = scale * (now @ column(do[i]))[..., 0]
            later = later + scale * column(q[i]) @ across(do[i])
            du = (across(k[i]) @ later)[..., 0, :]
            dk_[i] = (later @ column(b[i][..., None] * delta))[..., 0]
            db[i] = (du * delta).sum(-1) * live[i]
            dv_[i] = b[i][..., None] * du
            later = later - column(k[i]) @ across(dv_[i])
            dk_[i] -= (held @ column(dv_[i]))[..., 0]
            dg[i] = (later * held).sum((-1, -2)) * live[i]
            later = later * column(column(a[i]))
    fold = lambda x: x.unflatten(2, (h, hv // h)).sum(3)
    return [out, last, fold(dq), fold(dk_), dv_, dg, db, later]


def _exact_verify(case, s):
    n, k = case["n"], case["k"]
    t = _temperatures(s)
    tokens = torch.full((n, k + 1), -100, dtype=torch.int64, device=DEVICE)
    accepted = torch.zeros(n, dtype=torch.int32, device=DEVICE)
    for i in range(n):
        def distribution(x):
            if float(t[i]) == 0.0:
                return (torch.arange(x.shape[0], device=DEVICE) == x.argmax()).double()
            return torch.softmax(x.double() / t[i], 0)

        count = k if s["lengths"] is None else int(s["lengths"][i])
        j = 0
        while True:
            p = distribution(s["logits"][i, j])
            if j == count:
                break
            x = int(s["drafts"][i, j])
            if s["draft_logits"] is None or float(t[i]) == 0.0:
                q = torch.zeros_like(p)
                q[x] = 1.0
            else:
                q = distribution(s["draft_logits"][i, j])
            if not bool(s["uniforms"][i, j].double() * q[x] < p[x]):
                less = torch.clamp(p - q, min=0.0)
                p = less if bool(less.any()) else p
                break
            tokens[i, j] = x
            j += 1
        tokens[i, j] = torch.argmax(p / s["noise"][i].double())
        accepted[i] = j
    return [tokens, accepted]


def exact(case, seed):
    s = prepare(case, seed)
    return {"delta": _exact_delta, "verify": _exact_verify}[case["op"]](case, s)
