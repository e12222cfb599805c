"""The delta rule and the verification of drafts as they are used with the other sequence operators: a layer in training with its gradients, serving with drafts whose
rejected steps the state never takes, captured and replayed, on streams of their own, traced and observed.

Tolerances of the layer: as in test_gpu_sequence_operators.py, every stage moved by what its own test allows it (256 u of its largest output, and half a step where it rounds to
16 bits; with the terms that 16-bit calls of the delta rule leave out, 2^-14), in float64 on the CPU, four times the largest deviation seen."""
import pytest
import torch

import test_gpu_sequence_operators as sequence
from helpers import DEV, gen
from test_gpu_sequence_operators import Moved, far_apart, near

H, HV, DK, DV = 2, 4, 24, 16
D, VOCABULARY = HV * DV, 211
SIZES = [H * DK, H * DK, HV * DV, HV, HV, D]


def run_delta(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_delta_rule_backend import run_hip_delta_rule
    return run_hip_delta_rule(*args, **kwargs)


def run_verification(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_draft_verification_backend import run_hip_draft_verification
    return run_hip_draft_verification(*args, **kwargs)


def weights(dtype, seed):
    g = gen(seed)
    draw = lambda *shape: (torch.randn(*shape, generator=g) * shape[0] ** -0.5).to(dtype)
    vector = lambda n, mean: (mean + 0.1 * torch.randn(n, generator=g)).to(dtype)
    return {"w_in": draw(D, sum(SIZES)), "w_out": draw(D, VOCABULARY), "n1": vector(D, 1.0), "n2": vector(D, 1.0), "n3": vector(D, 1.0), "scale": vector(D, 0.5)}


def plain(p, residual, state, tokens, starts=None, lengths=None, moved=lambda y: y):
    """float64, [T, N, D]."""
    norm = lambda v: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    T, N = residual.shape[:2]
    both = moved(moved(norm(residual) * p["n1"]) @ p["w_in"])
    q, k, v, gate, beta, out_gate = both.split(SIZES, -1)
    heads = lambda x, n: x.unflatten(-1, (n, -1))
    q, k = (moved(norm(heads(x, H)) * DK ** -0.5).repeat_interleave(HV // H, 2) for x in (q, k))
    v, gate, beta = heads(v, HV), moved(-torch.nn.functional.softplus(gate) * 0.25), moved(torch.sigmoid(beta))
    S, outs = state, []
    for t in range(T):
        held = torch.exp(gate[t])[..., None, None] * S
        if starts is not None:
            held = torch.where(starts[t][:, None, None, None], torch.zeros_like(held), held)
        delta = v[t] - (k[t][..., None] * held).sum(-2)
        new = held + k[t][..., None] * (beta[t][..., None] * delta)[..., None, :]
        live = (torch.ones(N, dtype=torch.bool) if lengths is None else t < lengths)[:, None, None, None]
        S = torch.where(live, new, S)
        out = DK ** -0.5 * (q[t][..., None] * new).sum(-2)
        outs.append(torch.where(live[..., 0], out, torch.zeros_like(out)))
    branch = moved(torch.stack(outs).flatten(2))
    after = residual + p["scale"] * out_gate * torch.sigmoid(out_gate) * norm(branch) * p["n2"]
    logp = torch.log_softmax(moved(moved(norm(after) * p["n3"]) @ p["w_out"]), -1)
    given = tokens >= 0
    logprob = torch.where(given, logp.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], torch.zeros_like(logp[..., 0]))
    return moved(logprob), moved(-(logp.exp() * logp).sum(-1)), moved(after), moved(S)


def layer(p, residual, state, starts=None, lengths=None, state_out=None):
    """(logits, residual, state, what the delta rule was given)"""
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    unit = torch.full((DK,), DK ** -0.5, dtype=residual.dtype, device=residual.device)
    _, normed = run_hip_block_norm(residual, next_weight=p["n1"])
    q, k, v, gate, beta, out_gate = (normed @ p["w_in"]).split(SIZES, -1)
    q, k = (run_hip_block_norm(x.unflatten(-1, (H, DK)), next_weight=unit)[1] for x in (q, k))
    given = (q, k, v.unflatten(-1, (HV, DV)), -torch.nn.functional.softplus(gate) * 0.25, torch.sigmoid(beta))
    out, state = run_delta(*given, state, starts=starts, lengths=lengths, state_out=state_out)
    after, normed = run_hip_block_norm(residual, out.flatten(2), out_gate, p["n2"], p["n3"], p["scale"])
    return normed @ p["w_out"], after, state, given


def fused(p, residual, state, tokens, starts=None, lengths=None):
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    logits, after, state, _ = layer(p, residual, state, starts, lengths)
    return run_hip_token_scores(logits, tokens), after, state


def operands(T, N, dtype, seed):
    g = gen(seed)
    residual, state = torch.randn(T, N, D, generator=g).to(dtype), torch.randn(N, HV, DK, DV, generator=g)
    tokens = torch.randint(0, VOCABULARY, (T, N), generator=g)
    tokens[torch.rand(T, N, generator=g) < 0.1] = -100
    return residual, state, tokens


def stage_error(dtype):
    return 256 * 2.0 ** -24 + (torch.finfo(dtype).eps / 2 + 2.0 ** -14 if dtype != torch.float32 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,N,masks", [(1, 3, ""), (24, 5, ""), (24, 5, "starts"), (90, 2, "starts lengths")])
def test_a_layer_in_training(hip_ops, T, N, masks, dtype):
    p, (residual, state, tokens) = weights(dtype, 1), operands(T, N, dtype, 2)
    starts, lengths = sequence.cases(T, N, masks)
    if lengths is not None:
        tokens = torch.where(torch.arange(T)[:, None] < lengths, tokens, torch.full_like(tokens, -100))
    d = torch.randn(tokens.shape, generator=gen(5))

    def once(moved):
        leaves = {k: v.double().requires_grad_(True) for k, v in {**p, "residual": residual, "state": state}.items()}
        outs = plain({k: leaves[k] for k in p}, leaves["residual"], leaves["state"], tokens, starts, lengths, moved)
        loss = (outs[0] * d).sum() + 0.1 * outs[1].sum() + (outs[3] ** 2).sum()
        return list(outs), torch.autograd.grad(loss, list(leaves.values()))

    outs, grads = once(lambda y: y)
    off = [0.0] * (len(outs) + len(grads))
    for k in range(8):
        g = gen(100 + k)
        o, r = once(lambda y: Moved.apply(y, stage_error(dtype), g))
        off = [max(m, float((a - b).detach().abs().max())) for m, a, b in zip(off, [*o, *r], [*outs, *grads])]
    off = [4 * m for m in off]
    leaves = {k: v.to(DEV).requires_grad_(True) for k, v in {**p, "residual": residual, "state": state}.items()}
    on = lambda t: None if t is None else t.to(DEV)
    scores, after, last = fused(leaves, leaves["residual"], leaves["state"], tokens.to(DEV), on(starts), on(lengths))
    loss = (scores.logprob * d.to(DEV)).sum() + 0.1 * scores.entropy.sum() + (last ** 2).sum()
    got = torch.autograd.grad(loss, list(leaves.values()))
    for what, a, b, m in zip(("logprob", "entropy", "residual", "state"), (scores.logprob, scores.entropy, after, last), outs, off):
        near(a, b, m, what)
    for what, a, b, m in zip(leaves, got, grads, off[4:]):
        assert a.dtype == leaves[what].dtype and a.shape == leaves[what].shape
        near(a, b, m, "gradient of " + what)


# ------------------------------------------------------------------------------------------------------------------
# Serving with drafts
# ------------------------------------------------------------------------------------------------------------------
def decode(p, embedding, first, state, count, drafted, temperature):
    """`count` tokens of each request, drafts of each round from `drafted`, which gets (the number of tokens so far [N], the last token [N]). The state takes a step only once its token stands."""
    N, V = first.shape[0], VOCABULARY
    state, last = state.clone(), first.clone()
    done, tokens = torch.zeros(N, dtype=torch.long, device=DEV), torch.full((N, count + 16), -1, dtype=torch.long, device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    rounds = 0
    while int(done.min()) < count:
        drafts = drafted(done, last)
        K = drafts.shape[1]
        steps = torch.cat([last[:, None], drafts], 1).t()                              # [K + 1, N]
        logits, _, _, given = layer(p, embedding[steps], state)
        answer = run_verification(logits.transpose(0, 1), drafts, torch.rand(N, K, generator=g, device=DEV),
                                  torch.empty(N, V, device=DEV).exponential_(generator=g).clamp(min=1e-9), temperature=temperature)
        run_delta(*given, state, lengths=answer.accepted + 1, state_out=state)
        rows, places = torch.arange(N, device=DEV), torch.arange(K + 1, device=DEV)
        kept = places[None] <= answer.accepted[:, None]
        at = (done[:, None] + places[None])
        inside = kept & (at < tokens.shape[1])
        tokens[rows[:, None].expand_as(at)[inside], at[inside]] = answer.tokens[inside]
        last = answer.tokens[rows, answer.accepted.long()]
        done += answer.accepted + 1
        rounds += 1
    return tokens[:, :count], state, done, rounds


@pytest.mark.gpu
def test_greedy_decoding_with_drafts_and_without(hip_ops):
    """The same tokens whatever the drafts are, right ones, wrong ones or none; right ones take fewer rounds; the state after them is that of the tokens one by one."""
    N, count = 5, 24
    p = {k: v.to(DEV) for k, v in weights(torch.float32, 1).items()}
    embedding = torch.randn(VOCABULARY, D, generator=gen(2)).to(DEV)
    first = torch.randint(0, VOCABULARY, (N,), generator=gen(3)).to(DEV)
    state = torch.randn(N, HV, DK, DV, generator=gen(4)).to(DEV)
    none = lambda done, last: torch.zeros(N, 0, dtype=torch.long, device=DEV)
    long = 5 * count + 8                                        # as far as a request may get while the slowest one gets to `count`
    want, _, _, rounds = decode(p, embedding, first, state, long, none, 0.0)
    assert rounds == long
    g = torch.Generator(device=DEV)
    g.manual_seed(9)
    right = lambda done, last: torch.stack([want[n, int(done[n]):][:4] if int(done[n]) + 4 <= want.shape[1] else torch.zeros(4, dtype=torch.long, device=DEV) for n in range(N)])
    half = lambda done, last: torch.where(torch.rand(N, 4, generator=g, device=DEV) < 0.6, right(done, last), 7)
    for drafted, most in ((right, count // 4), (half, count), (lambda done, last: torch.full((N, 3), 5, device=DEV), count)):
        got, last_state, done, rounds = decode(p, embedding, first, state, count, drafted, 0.0)
        assert torch.equal(got, want[:, :count]) and rounds <= most
        # the last token stands and has not been taken yet
        for n in range(N):
            taken = torch.cat([first[n:n + 1], want[n]])[:int(done[n])]
            alone = state[n:n + 1]
            for token in taken:
                alone = layer(p, embedding[token][None, None], alone)[2]
            # projections of several rows at once are summed in another order, 64 u of the largest, remembered over 30 steps
            assert float((alone[0] - last_state[n]).abs().max()) <= 64 * 30 * 2.0 ** -24 * float(alone.abs().max())


@pytest.mark.gpu
def test_a_round_of_drafts_captured(hip_ops):
    """The round as one graph, replayed on new drafts with eager work between, the state kept in place: the same bits as without a graph."""
    N, K = 6, 3
    p = {k: v.to(DEV) for k, v in weights(torch.bfloat16, 1).items()}
    embedding = torch.randn(VOCABULARY, D, generator=gen(2)).to(DEV, torch.bfloat16)
    state = torch.randn(N, HV, DK, DV, generator=gen(4)).to(DEV)
    steps, uniforms, noise = torch.zeros(K + 1, N, dtype=torch.long, device=DEV), torch.zeros(N, K, device=DEV), torch.ones(N, VOCABULARY, device=DEV)

    def turn(state):
        logits, _, _, given = layer(p, embedding[steps], state)
        answer = run_verification(logits.transpose(0, 1), steps[1:].t().contiguous(), uniforms, noise, temperature=0.8)
        run_delta(*given, state, lengths=answer.accepted + 1, state_out=state)
        return answer
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            turn(state.clone())
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        cell, graph = state.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            answer = turn(cell)
        eager = state.clone()
        cell.copy_(state)
        for seed in range(6):
            g = gen(seed)
            steps.copy_(torch.randint(0, VOCABULARY, (K + 1, N), generator=g))
            uniforms.copy_(torch.rand(N, K, generator=g) * 0.01)
            noise.copy_(torch.empty(N, VOCABULARY).exponential_(generator=g))
            graph.replay()
            want = turn(eager)
            torch.cuda.synchronize()
            assert torch.equal(answer.tokens, want.tokens) and torch.equal(answer.accepted, want.accepted) and torch.equal(cell, eager)


# ------------------------------------------------------------------------------------------------------------------
# Graphs and streams
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_two_captured_training_steps(hip_ops):
    graphs = []
    for seed, (T, N) in enumerate([(300, 2), (40, 9)]):
        p, (residual, state, tokens) = weights(torch.bfloat16, seed), operands(T, N, torch.bfloat16, 20 + seed)
        leaves = {k: v.to(DEV).requires_grad_(True) for k, v in {**p, "residual": residual, "state": state}.items()}
        tokens = tokens.to(DEV)

        def step(leaves=leaves, tokens=tokens):
            scores, _, last = fused(leaves, leaves["residual"], leaves["state"], tokens)
            ones = torch.ones_like(scores.logprob)
            return torch.autograd.grad([scores.logprob, scores.entropy, last], list(leaves.values()), [ones, ones, torch.ones_like(last)])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step, side))
    for _ in range(4):
        for graph, out, _, side in graphs:
            for t in out:
                t.zero_()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for graph, out, step, _ in graphs:
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_calls_at_once_on_three_streams(hip_ops):
    runs = []
    for seed, (T, N) in enumerate([(1000, 3), (500, 9), (2000, 1)]):
        p, (residual, state, tokens) = weights(torch.bfloat16, seed), operands(T, N, torch.bfloat16, 30 + seed)
        leaves = {k: v.to(DEV).requires_grad_(True) for k, v in {**p, "residual": residual, "state": state}.items()}
        tokens = tokens.to(DEV)

        def step(leaves=leaves, tokens=tokens):
            scores, after, last = fused(leaves, leaves["residual"], leaves["state"], tokens)
            grads = torch.autograd.grad([scores.logprob, last], list(leaves.values()), [torch.ones_like(scores.logprob), torch.ones_like(last)])
            return [scores.logprob.detach(), after.detach(), last.detach(), *grads]
        want = step()
        torch.cuda.synchronize()
        runs.append((step, want, torch.cuda.Stream()))
    for _ in range(3):
        got = []
        for step, _, side in runs:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append([step() for _ in range(3)][-1])
        torch.cuda.synchronize()
        for (_, want, _), out in zip(runs, got):
            assert all(torch.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------------------------------------------------------
# Memory
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("strides", ["steps", "sequences", "heads"])
@pytest.mark.parametrize("T", [5, 70])
def test_offsets_past_32_bits(hip_ops, T, strides):
    g, far = gen(11), 1 << 30
    N, heads = (1, 2) if strides == "steps" else ((4, 1) if strides == "sequences" else (1, 4))
    small = [torch.randn(T, N, heads, 16, generator=g).to(torch.bfloat16).to(DEV) * 0.2 for _ in range(3)] + [-torch.rand(T, N, heads, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]

    def place(t):
        inner = (heads * t[0, 0, 0].numel(), t[0, 0, 0].numel(), 1)[-(t.dim() - 1):] if t.dim() == 4 else (heads, 1)
        step, row, head = {"steps": (far // T * 4, inner[0], inner[1]), "sequences": (inner[0], far, inner[1]), "heads": (inner[1], inner[1], far)}[strides]
        return far_apart(t, step, row, head, *([1] if t.dim() == 4 else []))
    answers = []
    for given in (small, [place(t) for t in small]):
        leaves = [t.requires_grad_(True) for t in given]
        out, last = run_delta(*leaves)
        answers.append([out, last, *torch.autograd.grad([out, last], leaves, [torch.ones_like(out), torch.ones_like(last)])])
        del leaves, given
    assert all(torch.equal(a, b) for a, b in zip(*answers))


@pytest.mark.gpu
def test_many_heads_and_steps(hip_ops):
    """More chunks than a launch has threads for along x, the last of them as by themselves; marks and workspaces past 2^32 bytes."""
    N, heads, T = 40000, 8, 500
    x = torch.zeros(T, N, heads, 4, dtype=torch.bfloat16, device=DEV)
    x[:, -2:] = torch.randn(T, 2, heads, 4, generator=gen(5)).to(DEV) * 0.3
    gate = torch.full((T, N, heads), -0.1, dtype=torch.bfloat16, device=DEV)
    with torch.no_grad():
        out, last = run_delta(x, x, x, gate)
        want, want_last = run_delta(x[:, -2:], x[:, -2:], x[:, -2:], gate[:, -2:])
    assert torch.equal(out[:, -2:], want) and torch.equal(last[-2:], want_last) and not bool(out[:, :-2].any())
    del out, last
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_verification_past_32_bits(hip_ops):
    V, far = 300, 1 << 31
    g = gen(7)
    logits, theirs = torch.randn(3, 2, V, generator=g).to(torch.bfloat16).to(DEV), torch.randn(3, 1, V, generator=g).to(torch.bfloat16).to(DEV)
    drafts, uniforms, noise = torch.randint(0, V, (3, 1), generator=g).to(DEV), torch.rand(3, 1, generator=g).to(DEV), torch.empty(3, V).exponential_(generator=g).to(DEV)
    want = run_verification(logits, drafts, uniforms, noise, draft_logits=theirs)
    got = run_verification(far_apart(logits, far, 400, 1), drafts, uniforms, far_apart(noise, far, 1), draft_logits=far_apart(theirs, far, 400, 1))
    assert torch.equal(want.tokens, got.tokens) and torch.equal(want.accepted, got.accepted)
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------------------------
# Both implementations of a call, and what follows it from outside
# ------------------------------------------------------------------------------------------------------------------
def without_module(monkeypatch):
    from triton_snn_fusion_amd.runtime import _sequence_common, hip_delta_rule_backend, hip_draft_verification_backend
    for backend in (_sequence_common, hip_delta_rule_backend, hip_draft_verification_backend):
        monkeypatch.setattr(backend, "native", lambda t: None)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 70])
def test_the_dispatch_module_and_python_give_the_same_bits(hip_ops, monkeypatch, T):
    """With operands left out, in-place states and some gradients; and the module takes these calls."""
    from triton_snn_fusion_amd import _dispatch
    g = gen(9)
    N = 3
    q, k = (torch.randn(T, N, H, DK, generator=g).to(DEV) * 0.2 for _ in range(2))
    v = torch.randn(T, N, HV, DV, generator=g).to(DEV)
    gate, beta = (-torch.rand(T, N, HV, generator=g).to(DEV) for _ in range(2))
    state, lengths = torch.randn(N, HV, DK, DV, generator=g).to(DEV), torch.tensor([T, 0, 2], dtype=torch.int32, device=DEV)
    starts = (torch.rand(T, N, generator=g) < 0.2).to(DEV)

    def answers():
        found = []
        for options in ({}, {"gate": gate}, {"beta": beta, "state": state}, {"gate": gate, "beta": beta, "state": state, "starts": starts, "lengths": lengths, "scale": 2}):
            found += run_delta(q, k, v, **options)
            leaves = [t.clone().requires_grad_(i != 1) for i, t in enumerate((q, k, v))]
            more = {name: t.clone().requires_grad_(True) if name in ("gate", "beta", "state") else t for name, t in options.items()}
            wanted = [*leaves[::2], *(t for name, t in more.items() if name in ("gate", "beta", "state"))]
            out, last = run_delta(*leaves, **more)
            found += [out, last, *torch.autograd.grad([out.sum() + (last * last).sum()], wanted)]
        cell = state.clone()
        out, last = run_delta(q, k, v, gate, beta, cell, state_out=cell)
        assert last is cell
        return found + [out, cell]
    module = _dispatch.module()
    assert module.delta_rule(q, k, v, gate, beta, state, None, starts, lengths, None) is not None
    fast = answers()
    without_module(monkeypatch)
    assert all(torch.equal(a, b) for a, b in zip(fast, answers()))


@pytest.mark.gpu
def test_verification_from_the_dispatch_module_and_python(hip_ops, monkeypatch):
    from test_gpu_draft_verification import operands as drafted
    from triton_snn_fusion_amd import _dispatch
    args, theirs = drafted(7, 3, 999, torch.float16, 5)
    each, lengths = torch.rand(7, device=DEV), torch.randint(0, 4, (7,), dtype=torch.int32, device=DEV)
    assert _dispatch.module().verify_drafts(*args, theirs, each, lengths) is not None
    calls = [lambda: run_verification(*args), lambda: run_verification(*args, draft_logits=theirs, temperature=each, lengths=lengths), lambda: run_verification(*args, temperature=0)]
    fast = [t for call in calls for t in call()]
    without_module(monkeypatch)
    assert all(torch.equal(a, b) for a, b in zip(fast, [t for call in calls for t in call()]))


def _operators():
    return {"delta": (lambda x, other: run_delta(x, other, other)[0], (5, 2, 1, 8))}


def test_what_follows_a_call_from_outside_is_refused_without_a_gpu(monkeypatch):
    monkeypatch.setattr(sequence, "_operators", _operators)
    sequence._observed("delta", "cpu")


@pytest.mark.gpu
def test_what_follows_a_call_from_outside_is_refused(hip_ops, monkeypatch):
    monkeypatch.setattr(sequence, "_operators", _operators)
    sequence._observed("delta", DEV)
    without_module(monkeypatch)
    sequence._observed("delta", DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_operands_whose_elements_lie_elsewhere_are_refused(hip_ops, monkeypatch, python):
    from torch.testing._internal.two_tensor import TwoTensor
    if python:
        without_module(monkeypatch)
    wrap = lambda t: TwoTensor(t, t.clone())
    x, gate, state = torch.randn(4, 2, 1, 8, device=DEV), -torch.rand(4, 2, 1, device=DEV), torch.zeros(2, 1, 8, 8, device=DEV)
    logits, drafts, noise = torch.randn(2, 2, 9, device=DEV), torch.zeros(2, 1, dtype=torch.long, device=DEV), torch.ones(2, 9, device=DEV)
    for call in (lambda: run_delta(wrap(x), x, x), lambda: run_delta(x, x, x, gate=wrap(gate)), lambda: run_delta(x, x, x, state=wrap(state)),
                 lambda: run_delta(x, x, x, state_out=wrap(state)), lambda: run_delta(x, x, x, lengths=wrap(torch.ones(2, dtype=torch.int32, device=DEV))),
                 lambda: run_verification(wrap(logits), drafts, noise[:, :1], noise), lambda: run_verification(logits, drafts, noise[:, :1], noise, temperature=wrap(torch.ones(2, device=DEV))),
                 lambda: run_verification(logits, drafts, noise[:, :1], noise, draft_logits=wrap(logits[:, :1].contiguous()))):
        with pytest.raises(RuntimeError, match="unsupported_subclass"):
            call()
    with pytest.raises(RuntimeError, match="unsupported_transform"):
        torch.vmap(lambda t: run_verification(t, drafts, noise[:, :1], noise).tokens)(torch.stack([logits, logits]))


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_outputs_may_be_written_over(hip_ops, monkeypatch, python):
    if python:
        without_module(monkeypatch)
    g = gen(5)
    x, y = (torch.randn(3, 20, 2, 16, generator=g).to(DEV).requires_grad_(True) for _ in range(2))
    for order in (lambda t: t, lambda t: t.transpose(0, 1)):
        for k in range(2):
            answers = []
            for in_place in (False, True):
                out = run_delta(order(x) * 0.2, order(y) * 0.2, order(x))[k]
                cover = torch.ones_like(out, dtype=torch.bool).tril()
                out = (out.add_(1.0).masked_fill_(cover, 0.0) if in_place else (out + 1.0).masked_fill(cover, 0.0))
                answers.append([out.detach(), *torch.autograd.grad((out * out).sum(), [x, y])])
            assert all(torch.equal(a, b) for a, b in zip(*answers))


@pytest.mark.gpu
def test_differentiated_twice_is_refused(hip_ops):
    x = (torch.randn(20, 1, 1, 8, generator=gen(6)).to(DEV) * 0.3).requires_grad_(True)
    out, _ = run_delta(x, x, x)
    first = torch.autograd.grad(out.sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice|once_differentiable|differentiable once"):
        (first * x).sum().backward()


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        for name, value in weights(torch.float32, 7).items():
            setattr(self, name, torch.nn.Parameter(value))

    def forward(self, q, k, v, gate, drafts, uniforms, noise):
        out, state = run_delta(q, k, v, gate, scale=0.5)
        logits = out.flatten(2).transpose(0, 1) @ self.w_out
        return out, state, run_verification(logits, drafts, uniforms, noise, temperature=0.5).tokens


def test_a_symbolic_trace_holds_the_operators():
    names = [node.target.__name__ for node in torch.fx.symbolic_trace(Layer()).graph.nodes if node.op == "call_function" and node.target.__name__.startswith("run_hip")]
    assert names == ["run_hip_delta_rule", "run_hip_draft_verification"]


@pytest.mark.gpu
def test_a_traced_module_runs_as_it_is_written(hip_ops):
    g, module = gen(3), Layer().to(DEV)
    given = [torch.randn(4, 2, H, DK, generator=g), torch.randn(4, 2, H, DK, generator=g) * 0.2, torch.randn(4, 2, HV, DV, generator=g), -torch.rand(4, 2, HV, generator=g),
             torch.randint(0, VOCABULARY, (2, 3), generator=g), torch.rand(2, 3, generator=g), torch.empty(2, VOCABULARY).exponential_(generator=g)]
    given = [t.to(DEV) for t in given]
    assert all(torch.equal(a, b) for a, b in zip(module(*given), torch.fx.symbolic_trace(module)(*given)))
