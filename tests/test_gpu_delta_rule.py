"""Gated delta rule and its gradient against the formulas in float64 on the CPU, step by step.

Tolerances. An output is rounded once, half a step of its type (`eps / 2` relative). Before that: keys have length 1 and beta lies in 0..1, so that a step's
map of the state does not expand it and errors add up. A chunk adds some 64 roundings of u = 2^-24 of the largest column of the state: products over the
head in float32 and in terms that leave 2^-24 (16), the inverse by substitution over 16 steps and three joins of blocks (40), the decays and sums (8). Gates
remember over at most 56 steps, so that two chunks count: 128 u in units of what the formula's factors can make at most (the lengths of the vectors and the
Frobenius norm of the states that an output is a product of). Gradients are products of two such: 256 u. Outputs and gradients of 16-bit tensors, other than the states', leave out terms
below 2^-16 of the factors, in up to four products: 2^-14."""
import itertools

import pytest
import torch

from helpers import DEV, gen

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def reference(query, key, value, gate, beta, state, scale, starts=None, lengths=None, dout=None, dlast=None):
    """float64: out, last and, with dout, (dquery, dkey, dvalue, dgate, dbeta, dstate); and what each may be at most by the lengths of its factors."""
    T, N, H, DK = query.shape
    HV, DV = value.shape[2:]
    G = HV // H
    q, k = (t.double().cpu().repeat_interleave(G, 2) for t in (query, key))
    v = value.double().cpu()
    g = torch.zeros(T, N, HV, dtype=torch.float64) if gate is None else gate.double().cpu()
    b = torch.ones(T, N, HV, dtype=torch.float64) if beta is None else beta.double().cpu()
    S = torch.zeros(N, HV, DK, DV, dtype=torch.float64) if state is None else state.double().cpu()
    limit = torch.full((N,), T) if lengths is None else lengths.cpu().clamp(0, T)
    live = torch.arange(T)[:, None] < limit[None, :]
    a = torch.exp(g) * (g >= -104)
    if starts is not None:
        a = torch.where(starts.cpu()[..., None], torch.zeros_like(a), a)
    out = torch.zeros(T, N, HV, DV, dtype=torch.float64)
    kept, deltas, after = [], [], []
    for t in range(T):
        on = live[t][:, None, None, None]
        held = torch.where((a[t] == 0)[..., None, None], torch.zeros_like(S), a[t][..., None, None] * S)
        delta = v[t] - (k[t][..., None] * held).sum(-2)
        new = held + k[t][..., None] * (b[t][..., None] * delta)[..., None, :]
        kept.append(held), deltas.append(delta)
        S = torch.where(on, new, S)
        after.append(S)
        out[t] = torch.where(on[..., 0], scale * (q[t][..., None] * new).sum(-2), out[t])
    size = max(float(torch.linalg.matrix_norm(s).max()) for s in [*after, *kept])
    length = lambda x: float(torch.where(live[:, :, None, None], x, 0.0).norm(dim=-1).max())
    most = [scale * length(q) * size, size]
    if dout is None:
        return [out, S], most
    d = dout.double().cpu()
    R = torch.zeros_like(S) if dlast is None else dlast.double().cpu()
    grads = [torch.zeros_like(x) for x in (q, k, v, g, b)]
    back = float(torch.linalg.matrix_norm(R).max())
    for t in range(T - 1, -1, -1):
        on = live[t][:, None, None]
        do = torch.where(on, d[t], 0.0)
        R1 = R + scale * q[t][..., None] * do[..., None, :]
        u = b[t][..., None] * deltas[t]
        du = (k[t][..., None] * R1).sum(-2)
        dv = b[t][..., None] * du
        R0 = R1 - k[t][..., None] * dv[..., None, :]
        new = (scale * (after[t] * do[..., None, :]).sum(-1), (R1 * u[..., None, :]).sum(-1) - (kept[t] * dv[..., None, :]).sum(-1), dv,
               (R0 * kept[t]).sum((-1, -2)), (du * deltas[t]).sum(-1))
        for x, y in zip(grads, new):
            x[t] = torch.where(on if y.dim() == 3 else on[..., 0], y, x[t])
        back = max(back, float(torch.where(on[..., None], torch.linalg.matrix_norm(R1)[..., None, None], 0.0).max()))
        R = torch.where(on[..., None], a[t][..., None, None] * R0, R)
    grads[0], grads[1] = (x.unflatten(2, (H, G)).sum(3) for x in grads[:2])
    deep = length(torch.stack(deltas))
    most += [G * scale * size * length(d), G * back * (deep + size), back, back * size * 4, back * deep, back]
    return [out, S, *grads, R], most


def operands(T, N, H, HV, DK, DV, dtype, seed, gates=None, batch_first=False):
    g = gen(seed)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp(min=1e-30)
    to = lambda t, kind=dtype: (t.transpose(0, 1).contiguous().to(DEV, kind).transpose(0, 1) if batch_first else t.to(DEV, kind))
    q, k = (to(unit(torch.randn(T, N, H, DK, generator=g) + 0.3)) for _ in range(2))
    v, dout = (to(torch.randn(T, N, HV, DV, generator=g)) for _ in range(2))
    gate = to(-torch.exp(torch.rand(T, N, HV, generator=g) * 3.0 - 4.0), gates or dtype)                # 1/56 to 1/2.7
    beta = to(torch.rand(T, N, HV, generator=g), gates or dtype)
    state, dlast = (torch.randn(N, HV, DK, DV, generator=g) * 0.3 for _ in range(2))
    return [q, k, v, gate, beta, state.to(DEV)], dout, dlast.to(DEV)


def near(got, want, dtype, extra, what):
    got, want = got.detach().double().cpu(), want.double()
    room = (torch.finfo(dtype).eps / 2) * want.abs() + extra + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (got - want).abs()
    assert bool((off <= room).all()), f"{what}: off by {float((off - room).max()):.3g} over the tolerance, at most {float(off.max()):.3g} of {float(want.abs().max()):.3g}"


def run(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_delta_rule_backend import run_hip_delta_rule
    return run_hip_delta_rule(*args, **kwargs)


NAMES = ("out", "last state", "dquery", "dkey", "dvalue", "dgate", "dbeta", "dstate")


def check(shape, dtype, seed, grad=True, gates=None, batch_first=False, starts=None, lengths=None, without=(), scale=None):
    leaves, dout, dlast = operands(*shape, dtype, seed, gates, batch_first)
    for i in without:
        leaves[i] = None
    factor = shape[4] ** -0.5 if scale is None else scale
    want, most = reference(*leaves, factor, starts, lengths, *((dout, dlast) if grad else ()))
    if grad:
        leaves = [None if t is None else t.requires_grad_(True) for t in leaves]
    out, last = run(*leaves, scale=scale, starts=starts, lengths=lengths)
    got = [out, last]
    if grad:
        grads = iter(torch.autograd.grad([out, last], [t for t in leaves if t is not None], [dout, dlast]))
        got += [None if t is None else next(grads) for t in leaves]
    torch.cuda.synchronize()
    kinds = [dtype, torch.float32] + [torch.float32 if t is None else t.dtype for t in leaves]
    for i, (a, b, m, kind) in enumerate(zip(got, want, most, kinds)):
        if a is None:
            continue
        assert a.dtype == kind and a.shape == b.shape
        coarse = 2.0 ** -14 if dtype != torch.float32 and i not in (1, 4, 7) else 0.0
        near(a, b, kind, ((128 if i < 2 else 256) * U + coarse) * m, NAMES[i])
    order = lambda t: t.shape[0] == 1 or t.shape[1] == 1 or (t.stride(1) > t.stride(0)) == batch_first
    assert order(out) and out.stride(-1) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1), (2, 3, 2, 4, 16, 17), (16, 2, 1, 1, 128, 64), (17, 1, 2, 2, 33, 129), (63, 2, 1, 3, 64, 64), (64, 1, 1, 1, 65, 20),
                                   (65, 2, 2, 2, 128, 128), (128, 1, 3, 3, 8, 200), (200, 3, 1, 2, 96, 80), (333, 1, 1, 1, 127, 63)])
def test_sizes(hip_ops, shape, dtype):
    check(shape, dtype, 100 + shape[0])
    check(shape, dtype, 200 + shape[0], grad=False)


def check_padded(shape, lengths, starts, dtype):
    for grad, wide in ((False, torch.int32), (True, torch.int64)):
        leaves, dout, dlast = operands(*shape, dtype, 300 + shape[0])
        want, most = reference(*leaves, 0.2, starts, lengths, dout, dlast)
        dead = (torch.arange(shape[0])[:, None] >= lengths.clamp(0, shape[0])[None, :]).to(DEV)
        for t in (*leaves[:5], dout):
            t[dead] = float("nan")
        leaves = [t.requires_grad_(grad) for t in leaves]
        out, last = run(*leaves, scale=0.2, starts=(starts.to(DEV) | dead), lengths=lengths.to(DEV, wide))
        got = [out, last, *(torch.autograd.grad([out, last], leaves, [dout, dlast]) if grad else ())]
        torch.cuda.synchronize()
        kinds = [dtype, torch.float32] + [t.dtype for t in leaves]
        for i, a in enumerate(got):
            coarse = 2.0 ** -14 if dtype != torch.float32 and i not in (1, 4, 7) else 0.0
            near(a, want[i], kinds[i], ((128 if i < 2 else 256) * U + coarse) * most[i], NAMES[i])
            if i not in (1, 7):
                assert bool((a[dead] == 0).all()), NAMES[i]
        empty = lengths <= 0
        assert torch.equal(last[empty], leaves[5][empty])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 3, 16, 17, 70, 150])
def test_starts_and_lengths(hip_ops, T, dtype):
    """Padding holds NaN in every operand, and starts of its own."""
    N, shape = 5, (T, 5, 1, 2, 40, 24)
    lengths = torch.tensor([0, T, (T + 1) // 2, -3, T + 9], dtype=torch.int32)
    starts = torch.rand(T, N, generator=gen(T)) < 0.1
    starts[0, 1] = True
    check_padded(shape, lengths, starts, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1100, 5, 1, 2, 40, 24), (1234, 4, 2, 2, 17, 33), (1111, 2, 1, 1, 128, 70)])
def test_long_sequences_of_few_heads(hip_ops, shape, dtype):
    """Chunks in segments of some, of which sequences have all, some, one or none; starts in few of them. A segment's matrix times a state adds 128 u of what is left of that after 3 chunks
    at least, 3 % with these gates."""
    T, N = shape[:2]
    lengths = torch.tensor([T, 449, 0, T - 1, 5][:N], dtype=torch.int32)
    starts = torch.rand(T, N, generator=gen(T)) < 0.003
    check_padded(shape, lengths, starts, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(70, 260, 1, 1, 17, 73), (65, 130, 1, 1, 24, 48), (65, 130, 1, 1, 70, 40), (66, 256, 1, 1, 72, 72)])
def test_many_heads(hip_ops, shape, dtype):
    check(shape, dtype, 400 + shape[4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(40, 1, 1, 64, 16, 16), (70, 1, 1, 1, 1, 1024), (1200, 1, 1, 1, 1, 700), (1200, 1, 1, 1, 128, 96), (20, 700, 1, 1, 8, 8), (65, 1, 64, 64, 4, 4)])
def test_extremes(hip_ops, shape, dtype):
    check(shape, dtype, 500 + shape[5])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences_on_two_streams(hip_ops, dtype):
    one, _, _ = operands(1400, 1, 2, 4, 64, 64, dtype, 44)
    two, _, _ = operands(1500, 2, 1, 1, 128, 128, dtype, 45)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        want = [*run(*one), *run(*two)]
        for _ in range(3):
            torch.cuda.synchronize()
            got = []
            for leaves, stream in zip((one, two), streams):
                with torch.cuda.stream(stream):
                    got += run(*leaves)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_long_sequence_in_pieces(hip_ops):
    """60000 steps at once, in segments, and in pieces of 8 chunks that are walked in one go: either way a state is off by 128 u of its size at most."""
    leaves, _, _ = operands(60000, 1, 1, 1, 32, 32, torch.float32, 46)
    with torch.no_grad():
        out, last = run(*leaves)
        state, outs = leaves[5], []
        for i in range(0, 60000, 500):
            piece, state = run(*(t[i:i + 500] for t in leaves[:5]), state)
            outs.append(piece)
    size = float(torch.linalg.matrix_norm(last).max().clamp(min=8.0))
    near(torch.cat(outs), out.cpu(), torch.float32, 256 * U * size, "out")
    near(state, last.cpu(), torch.float32, 256 * U * size, "last state")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences_forget(hip_ops, dtype):
    """An infinite state is gone behind a start, whichever segment that is in, and a vanishing gate."""
    T = 1150
    leaves, _, _ = operands(T, 2, 1, 1, 32, 32, dtype, 41)
    starts = torch.zeros(T, 2, dtype=torch.bool, device=DEV)
    starts[500, 0] = True
    leaves[3][300, 1] = -200.0
    state = leaves[5].clone()
    state[0, 0, 3], state[1, 0, 5] = float("inf"), float("nan")
    with torch.no_grad():
        a, b = run(*leaves[:5], state, starts=starts), run(*leaves[:5], None, starts=starts)
    assert torch.equal(a[0][500:, 0], b[0][500:, 0]) and torch.equal(a[0][300:, 1], b[0][300:, 1]) and torch.equal(a[1], b[1])
    assert not bool(torch.isfinite(a[0][499, 0]).all()) and bool(torch.isfinite(a[1]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [12, 100, 260])
def test_infinities_end_at_starts(hip_ops, T, dtype):
    """What a state and values hold of infinities and NaN reaches the steps of its own part, from the first of them on, and no others, in their own columns."""
    leaves, _, _ = operands(T, 2, 1, 2, 16, 40, dtype, 43)
    starts = torch.rand(T, 2, generator=gen(T)) < 0.15
    starts[4], starts[7, 0], starts[8, 1] = True, True, True
    parts = starts.cumsum(0)
    value, state = leaves[2].clone(), leaves[5].clone()
    state[1, :, :, 2] = float("inf")
    value[5, 0, 0, 3], value[5, 0, 1, 30], value[T - 2, 1, 0, 7] = float("nan"), float("inf"), -float("inf")
    with torch.no_grad():
        want, last = run(*leaves, starts=starts.to(DEV))
        out, state_out = run(leaves[0], leaves[1], value, *leaves[3:5], state, starts=starts.to(DEV))
    reached = torch.zeros(T, 2, 2, 40, dtype=torch.bool)
    reached[:, 1, :, 2] = (parts[:, 1] == 0)[:, None]
    for t, n, h, c in ((5, 0, 0, 3), (5, 0, 1, 30), (T - 2, 1, 0, 7)):
        reached[t:, n, h, c] |= parts[t:, n] == parts[t, n]
    assert torch.equal(out.isfinite().cpu(), ~reached)
    assert torch.equal(out[~reached.to(DEV)], want[~reached.to(DEV)])
    assert torch.equal(state_out.isfinite().all(2).cpu(), ~reached[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("without", [(3,), (4,), (3, 4), (5,), (3, 4, 5)])
@pytest.mark.parametrize("T", [7, 90])
def test_operands_left_out(hip_ops, T, without):
    check((T, 2, 2, 2, 32, 48), torch.float32, 11, without=without, scale=1.5)
    check((T, 2, 2, 2, 32, 48), torch.bfloat16, 12, without=without, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [5, 100])
def test_gates_in_float32(hip_ops, T, dtype):
    check((T, 2, 1, 2, 64, 64), dtype, 13, gates=torch.float32, batch_first=True)
    check((T, 2, 1, 2, 64, 64), dtype, 14, gates=torch.float32, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 100])
def test_gates_that_forget(hip_ops, T):
    """Minus infinity, below the threshold and just above it, and 0: what the state held, infinities among it, ends where nothing of it is left."""
    leaves, dout, dlast = operands(T, 2, 1, 2, 16, 16, torch.float32, 21)
    leaves[3][:, :, 0] = 0.0
    leaves[3][1, 0] = -float("inf")
    leaves[3][2, 1] = -105.0
    if T > 60:
        leaves[3][40, 0], leaves[3][55, 1, 1], leaves[3][70, 1, 0] = -103.0, -float("inf"), -1000.0
    want, most = reference(*leaves, 0.25, None, None, dout, dlast)
    leaves = [t.requires_grad_(True) for t in leaves]
    out, last = run(*leaves)
    grads = torch.autograd.grad([out, last], leaves, [dout, dlast])
    for i, a in enumerate([out, last, *grads]):
        near(a, want[i], torch.float32, (128 if i < 2 else 256) * U * (2 + T / 64) * most[i], NAMES[i])       # without decay every chunk counts
    state = leaves[5].detach().clone()
    state[0, :, 3] = float("inf")
    state[1, 1] = float("nan")
    starts = torch.zeros(T, 2, dtype=torch.bool, device=DEV)
    starts[0] = True
    with torch.no_grad():
        a, b = run(*leaves[:5], state, starts=starts), run(*leaves[:5], None)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def layouts(t):
    """The same elements: steps first, sequences first, slices of a wider tensor, elements apart."""
    yield t.contiguous()
    yield t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(*t.shape[:2], t.shape[2] + 1, *(n + 3 for n in t.shape[3:]), dtype=t.dtype, device=t.device)
    part = wide[:, :, 1:, 3:] if t.dim() == 4 else wide[:, :, 1:]
    yield part.copy_(t)
    yield t.transpose(2, -1).contiguous().transpose(2, -1)
    yield torch.stack([t, t], -1)[..., 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [6, 70])
def test_layouts_give_the_same_bits(hip_ops, T, dtype):
    leaves, dout, dlast = operands(T, 3, 2, 4, 37, 21, dtype, 31)
    state = leaves.pop()
    answers = []
    for *moved, d, last in itertools.islice(zip(*(layouts(t) for t in (*leaves, dout)), [dlast, dlast.transpose(2, 3).contiguous().transpose(2, 3)] * 3), 5):
        moved = [t.detach().requires_grad_(True) for t in (*moved, state)]
        with torch.no_grad():
            free = run(*moved)
        out, now = run(*moved)
        answers.append([*free, out, now, *torch.autograd.grad([out, now], moved, [d, last])])
    assert len(answers) == 5
    for other in answers[1:]:
        for a, b in zip(answers[0], other):
            assert torch.equal(a, b)
    expanded = run(leaves[0][:, :1].expand(-1, 3, -1, -1), leaves[1], leaves[2], leaves[3], leaves[4][:1].expand(T, -1, -1), state)
    again = run(leaves[0][:, :1].expand(-1, 3, -1, -1).contiguous(), leaves[1], leaves[2], leaves[3], leaves[4][:1].expand(T, -1, -1).contiguous(), state)
    assert torch.equal(expanded[0], again[0]) and torch.equal(expanded[1], again[1])


@pytest.mark.gpu
def test_long_sequence_without_decay(hip_ops):
    """2000 steps that all count: the state after them, and gradients of the first step. Errors add up over 32 chunks: 32 x 64 u, twice that for gradients."""
    leaves, dout, dlast = operands(2000, 1, 1, 1, 32, 16, torch.float32, 41)
    leaves[3] = torch.full_like(leaves[3], -1e-4)
    want, most = reference(*leaves, 32 ** -0.5, None, None, dout, dlast)
    leaves = [t.requires_grad_(True) for t in leaves]
    out, last = run(*leaves)
    for i, a in enumerate([out, last, *torch.autograd.grad([out, last], leaves, [dout, dlast])]):
        near(a, want[i], torch.float32, (2048 if i < 2 else 4096) * U * most[i], NAMES[i])


@pytest.mark.gpu
def test_large_decays_next_to_small_ones(hip_ops):
    """A strong decay at the head of a chunk takes nothing from the precision of those behind it: differences of sums are taken in float64."""
    leaves, _, _ = operands(64, 1, 1, 1, 16, 16, torch.float32, 43)
    leaves[3][:8], leaves[3][8:] = -100.0, -1e-3
    want, most = reference(*leaves, 0.25)
    out, last = run(*leaves)
    near(out, want[0], torch.float32, 128 * U * most[0], "out")
    near(last, want[1], torch.float32, 128 * U * most[1], "last state")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 80])
def test_gradient_against_differences(hip_ops, T):
    """Along a random direction, of a scalar of both outputs, in float32: (f(x + e d) - f(x - e d)) / 2e with e = 2^-6 is off by e^2 / 6 of the third derivative, here at most of the
    size of the derivative's bound times |d|^2, and by the outputs' roundings over e, 128 u / e of theirs."""
    leaves, dout, dlast = operands(T, 2, 1, 2, 16, 8, torch.float32, 51)
    leaves = [t.requires_grad_(True) for t in leaves]
    f = lambda xs: sum((a.double() * w.double()).sum() for a, w in zip(run(*xs), (dout, dlast)))
    grads = torch.autograd.grad(list(run(*leaves)), leaves, [dout, dlast])
    e = 2.0 ** -6
    for i, (x, g) in enumerate(zip(leaves, grads)):
        d = torch.randn(x.shape, generator=gen(60 + i)).to(DEV)
        d = d / d.norm()
        with torch.no_grad():
            up, down = ([*leaves[:i], x + s * e * d, *leaves[i + 1:]] for s in (1, -1))
            slope = float(f(up) - f(down)) / (2 * e)
            weight = sum(float((a.abs().double() * w.abs().double()).sum()) for a, w in zip(run(*leaves), (dout, dlast)))
        want = float((g.double() * d.double()).sum())
        assert abs(slope - want) <= e * e * float(g.norm()) + 128 * U / e * weight, (NAMES[2 + i], slope, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6, 40])
def test_state_in_place(hip_ops, T):
    leaves, _, _ = operands(T, 3, 1, 2, 50, 70, torch.bfloat16, 61)
    want = run(*leaves)
    state = leaves[5].clone()
    out, last = run(*leaves[:5], state, state_out=state)
    assert last is state and torch.equal(out, want[0]) and torch.equal(state, want[1])
    other = torch.empty_like(state)
    out, last = run(*leaves, state_out=other)
    assert last is other and torch.equal(out, want[0]) and torch.equal(other, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_state_in_place_of_long_sequences(hip_ops, dtype):
    leaves, _, _ = operands(1200, 2, 1, 2, 50, 70, dtype, 62)
    lengths = torch.tensor([1200, 130], dtype=torch.int32, device=DEV)
    want = run(*leaves, lengths=lengths)
    for _ in range(3):
        state = leaves[5].clone()
        out, last = run(*leaves[:5], state, lengths=lengths, state_out=state)
        assert last is state and torch.equal(out, want[0]) and torch.equal(state, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences_in_a_graph(hip_ops, dtype):
    """Replays with other work and another call of the same kind between them."""
    leaves, _, _ = operands(1200, 1, 1, 2, 30, 40, dtype, 63)
    other, _, _ = operands(1300, 2, 1, 1, 30, 40, dtype, 64)
    with torch.no_grad():
        expected = run(*other)
        run(*leaves)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, last = run(*leaves)
        for i in range(4):
            for t in leaves[2:3] + leaves[5:]:
                t.mul_(0.5)
            graph.replay()
            again = run(*other)
            want = run(*leaves)
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(last, want[1]) and torch.equal(again[0], expected[0]) and torch.equal(again[1], expected[1])


@pytest.mark.gpu
def test_steps_one_by_one_and_together(hip_ops):
    """A sequence in pieces, the state handed on: each piece is right for itself, so the whole is."""
    leaves, _, _ = operands(100, 2, 1, 2, 64, 32, torch.float32, 71)
    want, most = reference(*leaves, 0.125)
    state, outs, at = leaves[5], [], 0
    for size in (1, 1, 5, 16, 17, 30, 30):
        out, state = run(*(t[at:at + size] for t in leaves[:5]), state)
        outs.append(out)
        at += size
    near(torch.cat(outs), want[0], torch.float32, 256 * U * most[0], "out")
    near(state, want[1], torch.float32, 256 * U * most[1], "last state")


@pytest.mark.gpu
def test_no_steps_and_no_sequences(hip_ops):
    for T, N in ((0, 3), (4, 0)):
        leaves, _, _ = operands(T, N, 1, 2, 8, 4, torch.float32, 81)
        leaves = [t.requires_grad_(True) for t in leaves]
        out, last = run(*leaves)
        assert out.shape == (T, N, 2, 4) and torch.equal(last, leaves[5])
        grads = torch.autograd.grad(out.sum() + last.sum(), leaves)
        assert [g.shape for g in grads] == [t.shape for t in leaves] and bool((grads[5] == 1).all())
        assert bool((run(*leaves[:5])[1] == 0).all())


@pytest.mark.gpu
def test_only_some_gradients(hip_ops):
    leaves, dout, dlast = operands(70, 2, 1, 2, 16, 16, torch.bfloat16, 91)
    every = [t.detach().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(list(run(*every)), every, [dout, dlast])
    for i in range(6):
        some = [t.detach() for t in leaves]
        some[i].requires_grad_(True)
        out, last = run(*some)
        assert torch.equal(torch.autograd.grad([out, last], some[i], [dout, dlast])[0], want[i])
    zero = torch.zeros_like(dlast)
    out, last = run(*every)
    a = torch.autograd.grad(out, every, dout, retain_graph=True)
    for x, y in zip(a, torch.autograd.grad([out, last], every, [dout, zero], retain_graph=True)):
        assert torch.equal(x, y)
    for x, y in zip(torch.autograd.grad(last, every, dlast, allow_unused=True, retain_graph=True), torch.autograd.grad([out, last], every, [torch.zeros_like(dout), dlast])):
        assert torch.equal(x, y)


def test_refusals():
    """On the CPU: what is no GPU tensor is refused before anything else is looked at."""
    from triton_snn_fusion_amd.runtime.hip_delta_rule_backend import check_delta_rule_support, run_hip_delta_rule
    t = torch.zeros(2, 3, 1, 8)
    with pytest.raises(RuntimeError, match="unsupported_device"):
        run_hip_delta_rule(t, t, t)
    assert check_delta_rule_support(t.to(torch.float64), t, t)
    assert check_delta_rule_support(None, t, t)


def test_refusals_of_the_c_entries():
    """Before anything is launched: no address here is one of memory."""
    import ctypes

    from triton_snn_fusion_amd import _lib
    lib = _lib.lib()
    heads = lambda at: _lib.Heads(at, 64, 64, 32)
    call = _lib.DeltaRuleCall(2000, 1, 2, 2, 32, 32, _lib.dtype_code(torch.bfloat16), _lib.dtype_code(torch.float32), 1.0, heads(4096), heads(4096), heads(4096), heads(None), heads(None),
                              None, 0, 0, None, None)
    need, back = lib.snnf_delta_rule_workspace_bytes(ctypes.byref(call), 1), lib.snnf_delta_rule_backward_workspace_bytes(ctypes.byref(call))
    assert need % 4 == 0 and back % 4 == 0 and need > 0 and back > need
    out = [heads(8192) for _ in range(6)]
    forward = lambda marks, space, size, o=out[0], last=8192: lib.snnf_delta_rule(ctypes.byref(call), ctypes.byref(o), last, marks, space, size, None)
    backward = lambda marks, space, size, o=out[0]: lib.snnf_delta_rule_backward(ctypes.byref(call), marks, ctypes.byref(o), None, *(ctypes.byref(x) for x in out[1:]), 8192, space, size, None)
    for rc in (forward(8200, 4096, need), forward(8192, 4096, need - 1), forward(8192, 4100, need), forward(8192, None, need), forward(None, 4096, need, heads(None)), forward(8192, 4096, need, last=None),
               backward(8200, 4096, back), backward(8192, 4096, back - 1), backward(8192, 4104, back), backward(None, 4096, back), backward(8192, 4096, back, heads(None))):
        assert rc != 0
    call.value_heads = 3
    assert forward(8192, 4096, need) != 0 and lib.snnf_delta_rule_workspace_bytes(ctypes.byref(call), 1) == 0
    call.value_heads, call.key_size = 2, 129
    assert forward(8192, 4096, need) != 0 and backward(8192, 4096, back) != 0


@pytest.mark.gpu
@pytest.mark.parametrize("what,match", [
    ("key shape", "key must be"), ("rank", "unsupported_rank"), ("heads", "multiple of heads"), ("wide keys", "keys of 1 to 128"), ("wide values", "values of 1 to 1024"),
    ("mixed dtypes", "unsupported_dtype"), ("gate dtype", "gate must be"), ("gates that differ", "beta must be"), ("state dtype", "state must be"), ("state shape", "state must be"),
    ("starts", "starts must be"), ("lengths", "lengths must be"), ("other device", "unsupported_device"), ("double", "unsupported_dtype"), ("out gradient", "unsupported_gradient"),
    ("out overlap", "unsupported_overlap"), ("out strides", "unsupported_stride"), ("no values", "values of 1 to"), ("scale", "scale must be")])
def test_refusals_on_the_gpu(hip_ops, what, match):
    leaves, _, _ = operands(4, 2, 2, 2, 8, 8, torch.bfloat16, 95)
    options = {}
    if what == "key shape": leaves[1] = leaves[1][:3]
    elif what == "rank": leaves[0] = leaves[0][0]
    elif what == "heads": leaves[2] = torch.cat([leaves[2], leaves[2][:, :, :1]], 2)
    elif what == "wide keys": leaves[0] = leaves[1] = torch.zeros(4, 2, 2, 129, dtype=torch.bfloat16, device=DEV)
    elif what == "wide values": leaves[2] = torch.zeros(4, 2, 2, 1025, dtype=torch.bfloat16, device=DEV)
    elif what == "no values": leaves[2] = leaves[2][..., :0]
    elif what == "mixed dtypes": leaves[1] = leaves[1].float()
    elif what == "gate dtype": leaves[3] = leaves[3].half()
    elif what == "gates that differ": leaves[4] = leaves[4].float()
    elif what == "state dtype": leaves[5] = leaves[5].bfloat16()
    elif what == "state shape": leaves[5] = leaves[5][:1]
    elif what == "starts": options["starts"] = torch.zeros(4, 2, device=DEV)
    elif what == "lengths": options["lengths"] = torch.zeros(3, dtype=torch.int32, device=DEV)
    elif what == "other device": options["lengths"] = torch.zeros(2, dtype=torch.int32)
    elif what == "double": leaves = [t.double() for t in leaves]
    elif what == "scale": options["scale"] = torch.ones(())
    elif what == "out gradient":
        leaves[2].requires_grad_(True)
        options["state_out"] = torch.zeros_like(leaves[5])
    elif what == "out overlap":
        space = torch.zeros(2 * leaves[5].numel(), device=DEV)
        leaves[5], options["state_out"] = (space[i:i + leaves[5].numel()].view(leaves[5].shape) for i in (0, 8))
    elif what == "out strides": options["state_out"] = leaves[5].transpose(2, 3)
    with pytest.raises(RuntimeError, match=match):
        run(*leaves, **options)
