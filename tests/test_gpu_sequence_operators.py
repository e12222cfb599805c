"""The sequence operators as they are used together: norm, projections, recurrence, gate and norm and residual, logits, scores. Training with its
gradients, a prompt followed by single tokens, and both captured in graphs and replayed.

Tolerances. Every stage by itself is off by at most 128 u (u = 2^-24) of its largest output, as the operators' own tests bound it, with a product
over 64 channels at 64 u among them, and by half a step of its type where it rounds to 16 bits. What that comes to at the end is worked out in
float64 on the CPU: the same run with each stage's output, and in the backward pass each stage's gradient, moved by that much with random signs,
eight times. Those are worst cases of all stages at once, so four times the largest deviation seen bounds what a right run may be off by."""
import pytest
import torch

from helpers import DEV, gen

D, VOCABULARY = 64, 211
DTYPES = [torch.float32, torch.bfloat16]


class Moved(torch.autograd.Function):
    """y with each element, and its gradient, moved by `by` of the largest, in random directions."""

    @staticmethod
    def forward(ctx, y, by, g):
        ctx.by, ctx.g = by, g
        return Moved.move(y, by, g)

    @staticmethod
    def backward(ctx, d):
        return Moved.move(d, ctx.by, ctx.g), None, None

    @staticmethod
    def move(y, by, g):
        signs = torch.randint(0, 2, y.shape, generator=g).to(y.dtype) * 2 - 1
        return y + signs * by * y.abs().max() if y.numel() else y


def weights(dtype, seed):
    g = gen(seed)
    draw = lambda *shape: (torch.randn(*shape, generator=g) * shape[0] ** -0.5).to(dtype)
    return {"w_in": draw(D, 3 * D), "w_out": draw(D, VOCABULARY), "n1": (1 + 0.1 * torch.randn(D, generator=g)).to(dtype),
            "n2": (1 + 0.1 * torch.randn(D, generator=g)).to(dtype), "n3": (1 + 0.1 * torch.randn(D, generator=g)).to(dtype),
            "scale": (0.5 + 0.1 * torch.randn(D, generator=g)).to(dtype)}


def plain(p, residual, state, tokens, starts=None, lengths=None, moved=lambda y: y):
    """float64, [T, N, D]."""
    norm = lambda v: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    T = residual.shape[0]
    both = moved(norm(residual) * p["n1"]) @ p["w_in"]
    x, gate, out_gate = moved(both).split(D, -1)
    h, hs = state, []
    for t in range(T):
        a = torch.sigmoid(gate[t])
        before = h if starts is None else torch.where(starts[t][:, None], torch.zeros_like(h), h)
        new = a * before + (1 - a) * x[t]
        live = torch.ones(residual.shape[1], dtype=torch.bool) if lengths is None else t < lengths
        h = torch.where(live[:, None], new, h)
        hs.append(torch.where(live[:, None], new, torch.zeros_like(new)))
    branch = moved(torch.stack(hs))
    after = residual + p["scale"] * out_gate * torch.sigmoid(out_gate) * norm(branch) * p["n2"]
    logits = moved(moved(norm(after) * p["n3"]) @ p["w_out"])
    logp = torch.log_softmax(logits, -1)
    given = tokens >= 0
    logprob = torch.where(given, logp.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], torch.zeros_like(logp[..., 0]))
    return moved(logprob), moved(-(logp.exp() * logp).sum(-1)), moved(after), moved(h)


def fused(p, residual, state, tokens, starts=None, lengths=None, top_k=0):
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    _, normed = run_hip_block_norm(residual, next_weight=p["n1"])
    x, gate, out_gate = (normed @ p["w_in"]).split(D, -1)
    h, state = run_hip_gated_recurrence(x, gate, state, starts=starts, lengths=lengths)
    after, normed = run_hip_block_norm(residual, h, out_gate, p["n2"], p["n3"], p["scale"])
    return run_hip_token_scores(normed @ p["w_out"], tokens, top_k=top_k), after, state


def operands(T, N, dtype, seed):
    g = gen(seed)
    residual = torch.randn(T, N, D, generator=g).to(dtype)
    state = torch.randn(N, D, generator=g)
    tokens = torch.randint(0, VOCABULARY, (T, N), generator=g)
    tokens[torch.rand(T, N, generator=g) < 0.1] = -100
    return residual, state, tokens


def stage_error(dtype):
    return 128 * 2.0 ** -24 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0)


def expected(p, residual, state, tokens, dtype, **masks):
    """Float64 outputs and gradients, and what each may be off by."""
    d = torch.randn(tokens.shape, generator=gen(5))

    def once(moved):
        leaves = {k: v.double().requires_grad_(True) for k, v in {**p, "residual": residual, "state": state}.items()}
        w = {k: v for k, v in leaves.items() if k not in ("residual", "state")}
        outs = plain(w, leaves["residual"], leaves["state"], tokens, moved=moved, **masks)
        loss = (outs[0] * d).sum() + 0.1 * outs[1].sum() + (outs[3] ** 2).sum()
        return list(outs), torch.autograd.grad(loss, list(leaves.values()))

    outs, grads = once(lambda y: y)
    off = [0.0] * (len(outs) + len(grads))
    for k in range(8):
        g = gen(100 + k)
        o, q = once(lambda y: Moved.apply(y, stage_error(dtype), g))
        off = [max(m, float((a - b).detach().abs().max())) for m, a, b in zip(off, [*o, *q], [*outs, *grads])]
    return d, outs, grads, [4 * m for m in off]


def near(got, want, off, what):
    diff = (got.detach().double().cpu() - want.detach()).abs().max()
    assert float(diff) <= off, f"{what}: off by {float(diff):.3e}, may be {off:.3e} (largest {float(want.abs().max()):.3e})"


def cases(T, N, masks):
    starts = (torch.rand(T, N, generator=gen(3)) < 0.1) if "starts" in masks else None
    lengths = torch.randint(0, T + 1, (N,), generator=gen(4)) if "lengths" in masks else None
    return starts, lengths


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,masks", [(1, 3, ""), (24, 5, ""), (24, 5, "starts"), (30, 4, "starts lengths"), (300, 2, "lengths")])
def test_training(hip_ops, T, N, masks, dtype):
    p, (residual, state, tokens) = weights(dtype, 1), operands(T, N, dtype, 2)
    starts, lengths = cases(T, N, masks)
    if lengths is not None:  # padding carries no token
        tokens = torch.where(torch.arange(T)[:, None] < lengths, tokens, torch.full_like(tokens, -100))
    d, outs, grads, off = expected(p, residual, state, tokens, dtype, starts=starts, lengths=lengths)
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_and_then_single_tokens(hip_ops, dtype):
    """One captured step replayed for every token, its state kept in place, against the whole sequence at once."""
    T, N, prompt = 40, 6, 29
    p, (residual, state, tokens) = weights(dtype, 1), operands(T, N, dtype, 7)
    _, outs, _, off = expected(p, residual, state, tokens, dtype)
    p, residual, state, tokens = {k: v.to(DEV) for k, v in p.items()}, residual.to(DEV), state.to(DEV), tokens.to(DEV)
    with torch.no_grad():
        whole, after, last = fused(p, residual, state, tokens)
        near(whole.logprob, outs[0], off[0], "logprob")
        head, _, kept = fused(p, residual[:prompt], state, tokens[:prompt])
        near(head.logprob, outs[0][:prompt], off[0], "logprob of the prompt")
        step_residual, step_token = residual[prompt:prompt + 1].clone(), tokens[prompt:prompt + 1].clone()
        cell = kept.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fused(p, step_residual, cell, step_token, top_k=4)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scores, step_after, new = fused(p, step_residual, cell, step_token, top_k=4)
            cell.copy_(new)
        eager = kept.clone()
        for t in range(prompt, T):
            step_residual.copy_(residual[t:t + 1])
            step_token.copy_(tokens[t:t + 1])
            graph.replay()
            want, want_after, eager = fused(p, residual[t:t + 1], eager, tokens[t:t + 1], top_k=4)
            torch.cuda.synchronize()
            for a, b in zip((*scores, step_after, cell), (*want, want_after, eager)):
                assert torch.equal(a, b)
            near(scores.logprob[0], outs[0][t], off[0], f"logprob of token {t}")
            near(scores.entropy[0], outs[1][t], off[1], f"entropy of token {t}")
            near(step_after[0], outs[2][t], off[2], f"residual of token {t}")
        near(cell, outs[3], off[3], "state")


@pytest.mark.gpu
def test_two_captured_training_steps(hip_ops):
    """Two graphs of forward and backward, replayed in turn on their own streams with eager work between: each has scratch memory of its own."""
    graphs = []
    for seed, (T, N) in enumerate([(300, 2), (40, 64)]):
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
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_at_once_on_three_streams(hip_ops):
    """Long sequences whose tiles wait for each other, training passes among them, with the chip shared: results as alone."""
    runs = []
    for seed, (T, N) in enumerate([(3000, 3), (2500, 9), (9000, 1)]):
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


@pytest.mark.gpu
def test_no_rows_are_still_differentiable(hip_ops):
    """A shard of a batch that got nothing: gradients of no elements, zeros for the parameters."""
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    rows, vectors = [torch.empty(0, 8, device=DEV, requires_grad=True) for _ in range(3)], [torch.ones(8, device=DEV, requires_grad=True) for _ in range(3)]
    out, normed = run_hip_block_norm(*rows, *vectors)
    assert out.shape == normed.shape == (0, 8)
    for k in (out, normed):
        for t, g in zip((*rows, *vectors), torch.autograd.grad(k.sum(), (*rows, *vectors), retain_graph=True)):
            assert g.shape == t.shape and bool((g == 0).all())
    scores = run_hip_token_scores(rows[0], torch.empty(0, dtype=torch.int64, device=DEV), top_k=2)
    assert torch.autograd.grad((scores.logprob + scores.entropy).sum(), rows[0])[0].shape == (0, 8)
    for shape in ((0, 2, 8), (3, 0, 8)):
        x, gate = torch.empty(shape, device=DEV, requires_grad=True), torch.empty(shape, device=DEV, requires_grad=True)
        state = torch.ones(shape[1:], device=DEV, requires_grad=True)
        h, last = run_hip_gated_recurrence(x, gate, state)
        grads = torch.autograd.grad(h.sum() + last.sum(), (x, gate, state))
        assert [g.shape for g in grads] == [x.shape, gate.shape, state.shape] and bool((grads[2] == 1).all())


def far_apart(t, *strides):
    """t's elements with these strides, in memory of its own."""
    span = 1 + sum((n - 1) * s for n, s in zip(t.shape, strides))
    out = torch.empty(span, dtype=t.dtype, device=DEV).as_strided(t.shape, strides)
    out.copy_(t)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("operator", ["steps", "sequences", "norm", "scores"])
def test_offsets_past_32_bits(hip_ops, operator):
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    g = gen(11)
    far = 1 << 30
    if operator in ("steps", "sequences"):
        T, N, D = (70, 1, 96) if operator == "steps" else (20, 4, 96)
        near_by = [torch.randn(T, N, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
        strides = (far >> 4, D, 1) if operator == "steps" else (D, far, 1)
        call = run_hip_gated_recurrence
    else:
        near_by = [torch.randn(4, 200, generator=g).to(torch.bfloat16).to(DEV) for _ in range(1 if operator == "scores" else 2)]
        strides = (far, 1)
        tokens = torch.tensor([3, 199, 0, 7], device=DEV)
        call = run_hip_block_norm if operator == "norm" else (lambda x: run_hip_token_scores(x, tokens, top_k=3))
    answers = []
    for operands_ in (near_by, [far_apart(t, *strides) for t in near_by]):
        leaves = [t.requires_grad_(True) for t in operands_]
        out = [t for t in call(*leaves) if t.is_floating_point()]
        used = [t for t in out if t.requires_grad]
        answers.append([*out, *torch.autograd.grad(used, leaves, [torch.ones_like(t) for t in used])])
        del leaves, operands_
    for a, b in zip(*answers):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_steps_too_far_apart_are_refused(hip_ops, monkeypatch):
    """Sixteen steps more than 2 GiB apart, from the dispatch module and from Python, with and without gradients."""
    from triton_snn_fusion_amd.runtime import hip_gated_recurrence_backend as backend
    x = torch.empty(19 * (1 << 27) + 8, dtype=torch.bfloat16, device=DEV).as_strided((20, 1, 8), (1 << 27, 8, 1))
    for _ in range(2):
        for gradient in (False, True):
            with pytest.raises(RuntimeError, match="unsupported_stride"):
                backend.run_hip_gated_recurrence(x.detach().requires_grad_(gradient), x)
        monkeypatch.setattr(backend, "native", lambda t: None)
    x = x[::10]
    assert backend.run_hip_gated_recurrence(x[:1].zero_(), x[:1])[0].shape == (1, 1, 8)


@pytest.mark.gpu
def test_orders_that_differ_between_operands(hip_ops):
    """x with steps outermost, the gate with sequences outermost, gradients with either, channels apart: the same bits."""
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    g = gen(14)
    T, N, D = 270, 3, 130
    x, gate, dh = (torch.randn(T, N, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3))
    orders = [lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: t.permute(2, 0, 1).contiguous().permute(1, 2, 0),
              lambda t: torch.stack([t, t], -1)[..., 0]]
    answers = []
    for a, b, c in ((0, 0, 0), (0, 1, 1), (1, 0, 0), (2, 3, 2), (3, 1, 3), (1, 2, 0)):
        leaves = [orders[a](x).detach().requires_grad_(True), orders[b](gate).detach().requires_grad_(True)]
        h, last = run_hip_gated_recurrence(*leaves)
        answers.append([h, last, *torch.autograd.grad([h, last], leaves, [orders[c](dh), torch.ones_like(last)])])
    for other in answers[1:]:
        for p, q in zip(answers[0], other):
            assert torch.equal(p, q)


@pytest.mark.gpu
def test_one_tensor_in_several_places(hip_ops):
    """The same leaf as x and gate, as residual, branch and gate, as all three vectors: its gradient is the sum."""
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    g = gen(15)
    t = torch.randn(33, 2, 70, generator=g).to(DEV)
    w = torch.rand(70, generator=g).to(DEV)
    for call, roles in ((lambda *a: run_hip_gated_recurrence(*a), (t, t)),
                        (lambda *a: run_hip_block_norm(*a), (t, t, t, w, w, w))):
        one = {id(r): r.clone().requires_grad_(True) for r in roles}
        apart = [r.clone().requires_grad_(True) for r in roles]
        out, want = call(*(one[id(r)] for r in roles)), call(*apart)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        got = torch.autograd.grad(out, list(one.values()), [torch.ones_like(a) for a in out])
        separate = torch.autograd.grad(want, apart, [torch.ones_like(a) for a in want])
        for k, grad in zip(one, got):
            parts = [s for s, r in zip(separate, roles) if id(r) == k]
            # sums of at most six terms in either order
            assert bool(((grad - sum(parts)).abs() <= 6 * 2.0 ** -24 * sum(p.abs() for p in parts)).all())


@pytest.mark.gpu
def test_more_elements_than_32_bits_count(hip_ops):
    """Rows of one tensor with more than 2^31 elements, against the last of them by themselves."""
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    rows, width = (1 << 20) + 5, 2056
    x = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    x[:-9].fill_(0.25)
    x[-9:] = torch.randn(9, width, generator=gen(12)).to(torch.bfloat16).to(DEV)
    x.requires_grad_(True)
    tail = x.detach()[-9:].clone().requires_grad_(True)
    tokens = torch.arange(rows, device=DEV) % width
    for call in (lambda t: run_hip_block_norm(t, t), lambda t: run_hip_token_scores(t, tokens[rows - t.shape[0]:])[:2],
                 lambda t: run_hip_gated_recurrence(t[None], t[None])):
        big, small = call(x), call(tail)
        grad = torch.autograd.grad(big, x, [torch.ones_like(t) for t in big])[0][-9:]
        want = torch.autograd.grad(small, tail, [torch.ones_like(t) for t in small])[0]
        for a, b in zip(big, small):
            assert torch.equal(a.reshape(-1, *a.shape[1:] if a.shape[0] == rows else a.shape[2:])[-9:], b.reshape(-1, *b.shape[1:] if b.shape[0] == 9 else b.shape[2:]))
        assert torch.equal(grad, want)
        del big, grad


@pytest.mark.gpu
def test_more_rows_than_a_launch_has_threads_for(hip_ops):
    """17 million short rows, a workgroup each: the last of them as by themselves."""
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    rows, width = (1 << 24) + 3, 10
    x = torch.zeros(rows, width, device=DEV)
    x[-9:] = torch.randn(9, width, generator=gen(13)).to(DEV)
    x.requires_grad_(True)
    tail = x.detach()[-9:].clone().requires_grad_(True)
    tokens = torch.arange(rows, device=DEV) % width
    big, small = run_hip_token_scores(x, tokens, top_k=2), run_hip_token_scores(tail, tokens[-9:], top_k=2)
    for a, b in zip(big, small):
        assert torch.equal(a[-9:], b)
    ones = torch.ones(rows, device=DEV)
    grad = torch.autograd.grad([big.logprob, big.entropy], x, [ones, ones])[0]
    assert torch.equal(grad[-9:], torch.autograd.grad([small.logprob, small.entropy], tail, [ones[:9], ones[:9]])[0])


# ------------------------------------------------------------------------------------------------------------------
# What the kernels do not see of a call
# ------------------------------------------------------------------------------------------------------------------
def _operators():
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    return {"recurrence": (lambda x, other: run_hip_gated_recurrence(x, other)[0], (5, 2, 8)),
            "norm": (lambda x, other: run_hip_block_norm(x, other)[1], (5, 8)),
            "norm without a branch": (lambda x, other: run_hip_block_norm(x, next_weight=other[0].contiguous())[1], (5, 8)),
            "scores": (lambda x, other: run_hip_token_scores(x * other).entropy, (5, 8))}


def _observed(operator, device):
    """Every way in which torch follows a call from outside, each refused by name."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    call, shape = _operators()[operator]
    x, other = torch.randn(shape, generator=gen(1)).to(device), torch.randn(shape, generator=gen(2)).to(device)
    for which in range(2):
        for differentiated in (False, True):
            leaves = [x.clone().requires_grad_(differentiated), other.clone().requires_grad_(differentiated)]
            with forward_ad.dual_level():
                leaves[which] = forward_ad.make_dual(leaves[which], torch.ones_like(x))
                with pytest.raises(RuntimeError, match="unsupported_forward_ad"):
                    call(*leaves)
                with torch.no_grad(), pytest.raises(RuntimeError, match="unsupported_forward_ad"):
                    call(*leaves)
    with pytest.raises(RuntimeError, match="unsupported_tracing"):
        torch.jit.trace(call, (x, other), check_trace=False)
    with pytest.raises(RuntimeError, match="unsupported_tracing"):
        make_fx(call)(x, other)
    stacked = torch.stack([x, x])
    transformed = [lambda: torch.vmap(call, in_dims=(0, None))(stacked, other), lambda: torch.func.grad(lambda t: call(t, other).sum())(x),
                   lambda: torch.vmap(call, in_dims=(None, 0))(x, stacked)]
    for call_of in transformed:
        with pytest.raises(RuntimeError, match="unsupported_transform"):
            call_of()
    if device == "cpu":
        return
    leaf = x.clone().requires_grad_(True)
    out = call(leaf, other)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="unsupported_forward_ad"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
    with pytest.raises(RuntimeError, match="unsupported_transform"):
        torch.autograd.grad(out, leaf, torch.ones(2, *out.shape, dtype=out.dtype, device=device), retain_graph=True, is_grads_batched=True)
    with pytest.raises(RuntimeError, match="unsupported_tracing"):
        make_fx(lambda d: torch.autograd.grad(out, leaf, d, retain_graph=True)[0])(torch.ones_like(out))
    assert torch.autograd.grad(out, leaf, torch.ones_like(out))[0].shape == leaf.shape


@pytest.mark.parametrize("operator", ["recurrence", "norm", "norm without a branch", "scores"])
def test_what_follows_a_call_from_outside_is_refused_without_a_gpu(operator):
    _observed(operator, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("operator", ["recurrence", "norm", "norm without a branch", "scores"])
def test_what_follows_a_call_from_outside_is_refused(hip_ops, monkeypatch, operator):
    """A tangent would be lost and a trace would hold memory that nothing fills; through the dispatch module and without it. Where forward-mode
    differentiation is off a tangent is none, and the call runs."""
    from torch.autograd import forward_ad
    from triton_snn_fusion_amd.runtime import _sequence_common, hip_block_norm_backend, hip_gated_recurrence_backend, hip_token_scores_backend
    call, shape = _operators()[operator]
    x, other = torch.randn(shape, generator=gen(1)).to(DEV), torch.randn(shape, generator=gen(2)).to(DEV)
    want = call(x, other)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(call(dual, other), want)
    _observed(operator, DEV)
    for backend in (_sequence_common, hip_block_norm_backend, hip_gated_recurrence_backend, hip_token_scores_backend):
        monkeypatch.setattr(backend, "native", lambda t: None)
    _observed(operator, DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_outputs_may_be_written_over(hip_ops, monkeypatch, python):
    """An addition or a mask in place on an output is the one out of place, whichever implementation ran the call."""
    from triton_snn_fusion_amd.runtime import hip_block_norm_backend, hip_gated_recurrence_backend, hip_token_scores_backend
    if python:
        for backend in (hip_block_norm_backend, hip_gated_recurrence_backend, hip_token_scores_backend):
            monkeypatch.setattr(backend, "native", lambda t: None)
    g = gen(5)
    x, gate, logits = (torch.randn(2, 40, 64, generator=g).to(DEV).requires_grad_(True) for _ in range(3))
    tokens = torch.randint(0, 64, (2, 40), generator=g).to(DEV)
    mask = (torch.rand(2, 40, generator=g) < 0.5).to(DEV)

    def recurrence(batch_first):
        order = (lambda t: t.transpose(0, 1)) if batch_first else (lambda t: t)
        return hip_gated_recurrence_backend.run_hip_gated_recurrence(order(x), order(gate))
    calls = [(lambda: recurrence(True), [x, gate], 2), (lambda: recurrence(False), [x, gate], 2),
             (lambda: hip_block_norm_backend.run_hip_block_norm(x, gate), [x, gate], 2),
             (lambda: hip_token_scores_backend.run_hip_token_scores(logits, tokens, 3), [logits], 1)]      # entropy is saved for the gradient
    for call, leaves, n_written in calls:
        for k in range(n_written):
            answers = []
            for in_place in (False, True):
                out = call()[k]
                cover = mask if out.shape == mask.shape else torch.ones_like(out, dtype=torch.bool).tril()
                out = (out.add_(1.0).masked_fill_(cover, 0.0) if in_place else (out + 1.0).masked_fill(cover, 0.0))
                answers.append([out.detach(), *torch.autograd.grad((out * out).sum(), leaves)])
            assert all(torch.equal(a, b) for a, b in zip(*answers))


# ------------------------------------------------------------------------------------------------------------------
# torch.fx
# ------------------------------------------------------------------------------------------------------------------
class Block(torch.nn.Module):
    """One layer of a token model with its scores."""

    def __init__(self, seed=7):
        super().__init__()
        for name, value in weights(torch.float32, seed).items():
            setattr(self, name, torch.nn.Parameter(value))

    def forward(self, residual, tokens, state=None):
        from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
        from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
        from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
        _, normed = run_hip_block_norm(residual, next_weight=self.n1)
        x, gate, out_gate = (normed @ self.w_in).split(D, -1)
        h, state = run_hip_gated_recurrence(x, gate, state, form="leaky")
        residual, normed = run_hip_block_norm(residual, h, out_gate, self.n2, self.n3, self.scale, gate_form="silu")
        scores = run_hip_token_scores(normed @ self.w_out, tokens, top_k=3)
        return scores.logprob, scores.entropy, scores.top_token, state


def test_a_symbolic_trace_holds_the_operators():
    """torch.fx records each call as one node, as it does torch's own functions; a module that uses them can be traced without a GPU."""
    traced = torch.fx.symbolic_trace(Block())
    names = [node.target.__name__ for node in traced.graph.nodes if node.op == "call_function" and node.target.__name__.startswith("run_hip")]
    assert names == ["run_hip_block_norm", "run_hip_gated_recurrence", "run_hip_block_norm", "run_hip_token_scores"]
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    with pytest.raises(RuntimeError, match="must be a tensor"):
        run_hip_token_scores("no tensor")


@pytest.mark.gpu
def test_a_traced_module_runs_as_it_is_written(hip_ops):
    block = Block().to(DEV)
    traced = torch.fx.symbolic_trace(block)
    g = gen(3)
    residual, tokens = torch.randn(6, 2, D, generator=g).to(DEV).requires_grad_(True), torch.randint(0, VOCABULARY, (6, 2), generator=g).to(DEV)
    state = torch.randn(2, D, generator=g).to(DEV)
    answers = []
    for module in (block, traced):
        out = module(residual, tokens, state)
        answers.append([*out, *torch.autograd.grad(out[0].sum() + out[1].sum() + out[3].sum(), [residual, *block.parameters()])])
    assert all(torch.equal(a, b) for a, b in zip(*answers))


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_operands_whose_elements_lie_elsewhere_are_refused(hip_ops, monkeypatch, python):
    """A subclass that wraps other tensors has no address, and an operand without one must not pass for one that a call lacks."""
    from torch.testing._internal.two_tensor import TwoTensor
    from triton_snn_fusion_amd.runtime import _sequence_common, hip_block_norm_backend, hip_gated_recurrence_backend, hip_token_scores_backend
    if python:
        for backend in (_sequence_common, hip_block_norm_backend, hip_gated_recurrence_backend, hip_token_scores_backend):
            monkeypatch.setattr(backend, "native", lambda t: None)
    x, vector, rows = torch.randn(4, 2, 8, device=DEV), torch.randn(8, device=DEV), torch.randn(2, 8, device=DEV)
    wrap = lambda t: TwoTensor(t, t.clone())
    recurrence, norm = hip_gated_recurrence_backend.run_hip_gated_recurrence, hip_block_norm_backend.run_hip_block_norm
    for call in (lambda: recurrence(x, x, wrap(rows)), lambda: recurrence(x, x, starts=wrap(torch.ones(4, 2, dtype=torch.bool, device=DEV))),
                 lambda: recurrence(x, x, lengths=wrap(torch.ones(2, dtype=torch.int32, device=DEV))), lambda: recurrence(wrap(x), x),
                 lambda: norm(x, x, gate=wrap(x)), lambda: norm(x, x, next_weight=wrap(vector)), lambda: norm(x, x, scale=wrap(vector)),
                 lambda: hip_token_scores_backend.run_hip_token_scores(rows, wrap(torch.zeros(2, dtype=torch.int64, device=DEV)))):
        with pytest.raises(RuntimeError, match="unsupported_subclass"):
            call()
