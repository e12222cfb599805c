"""Gated linear recurrence and its gradient against the formulas in float64 on the CPU.

Tolerances: an output is rounded once, half a step of its type (`eps / 2` relative). Before that the kernels add float32 roundings: every step
adds at most a few of 2^-24 relative to the largest state (decay, product, sum), a decay below 1 lets `memory` = 1 / (1 - largest decay)
of them accumulate, and a decay that is itself off by a rounding acts like one more per step; runs of steps that are joined add one per
joint. C = 8 covers decay (2), input gate (2), product and sum (1), joints (3)."""
import pytest
import torch

from helpers import DEV, gen

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
C = 8.0


def reference(x, gate, state, form, starts=None, lengths=None, dh=None, dlast=None):
    """float64, step by step: h, last and, with dh, (dx, dgate, dstate), and the largest |h| and |s|."""
    x, gate = x.double().cpu(), gate.double().cpu()
    T, N, D = x.shape
    a, rest = (torch.sigmoid(gate), torch.sigmoid(-gate)) if form == "leaky" else (gate, torch.ones_like(gate))
    h = torch.zeros(N, D, dtype=torch.float64) if state is None else state.double().cpu()
    limit = torch.full((N,), T) if lengths is None else lengths.cpu().clamp(0, T)
    inside = torch.arange(T)[:, None] < limit[None, :]
    drop = torch.zeros(T, N, dtype=torch.bool) if starts is None else starts.cpu()
    out, before = torch.zeros_like(x), torch.zeros_like(x)
    peak = float(h.nan_to_num().abs().max()) if h.numel() else 0.0
    for t in range(T):
        before[t] = torch.where(drop[t][:, None], torch.zeros_like(h), h)
        new = torch.where(drop[t][:, None], rest[t] * x[t], a[t] * h + rest[t] * x[t])
        h = torch.where(inside[t][:, None], new, h)
        out[t] = torch.where(inside[t][:, None], new, torch.zeros_like(new))
        peak = max(peak, float(out[t].nan_to_num().abs().max()))
    if dh is None:
        return out, h, peak
    dh = dh.double().cpu()
    r = torch.zeros(N, D, dtype=torch.float64) if dlast is None else dlast.double().cpu()
    dx, dgate = torch.zeros_like(x), torch.zeros_like(x)
    most = float(r.abs().max())
    for t in range(T - 1, -1, -1):
        on = inside[t][:, None]
        s = dh[t] + r
        most = max(most, float(torch.where(on, s, torch.zeros_like(s)).nan_to_num().abs().max()))
        dx[t] = torch.where(on, s * rest[t], torch.zeros_like(s))
        dgate[t] = torch.where(on, s * (before[t] - x[t]) * a[t] * rest[t] if form == "leaky" else s * before[t], torch.zeros_like(s))
        r = torch.where(on, torch.where(drop[t][:, None], torch.zeros_like(s), a[t] * s), r)
    return out, h, peak, dx, dgate, r, most


def operands(T, N, D, dtype, form, seed, batch_first=False):
    g = gen(seed)
    x, dh = torch.randn(T, N, D, generator=g), torch.randn(T, N, D, generator=g)
    gate = (torch.randn(T, N, D, generator=g) * 1.5 + 1.0).clamp(-6.0, 4.0)                      # memory of at most 56 steps
    if form == "linear":
        gate = torch.sigmoid(gate) * torch.where(torch.rand(T, N, D, generator=g) < 0.1, -1.0, 1.0)
    state, dlast = torch.randn(N, D, generator=g), torch.randn(N, D, generator=g)

    def to(t):
        if batch_first:
            return t.transpose(0, 1).contiguous().to(DEV, dtype).transpose(0, 1)
        return t.to(DEV, dtype)
    return to(x), to(gate), state.to(DEV), to(dh), dlast.to(DEV)


MEMORY = 60.0


def near(got, want, dtype, extra, what):
    got, want = got.double().cpu(), want.double()
    room = torch.finfo(dtype).eps / 2 * (1 if dtype != torch.float32 else 0) * want.abs() + extra
    if dtype == torch.float16:
        room = room + 2.0 ** -25                                                                # half a step of the subnormals
    off = (got - want).abs()
    assert bool((off <= room).all()), f"{what}: off by {float((off - room).max()):.3g} over the tolerance, at most {float(off.max()):.3g}"


def run(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import run_hip_gated_recurrence
    return run_hip_gated_recurrence(*args, **kwargs)


def check(T, N, D, dtype, form, seed, starts=None, lengths=None, batch_first=False, with_state=True, grad=True):
    x, gate, state, dh, dlast = operands(T, N, D, dtype, form, seed, batch_first)
    state = state if with_state else None
    if not grad:
        h, last = run(x, gate, state, form=form, starts=starts, lengths=lengths)
        want = reference(x, gate, state, form, starts, lengths)
    else:
        leaves = [t.requires_grad_(True) for t in (x, gate, state) if t is not None]
        h, last = run(x, gate, state, form=form, starts=starts, lengths=lengths)
        got = torch.autograd.grad([h, last], leaves, [dh, dlast])
        want = reference(x.detach(), gate.detach(), None if state is None else state.detach(), form, starts, lengths, dh, dlast)
    torch.cuda.synchronize()
    peak = want[2]
    err = C * U * MEMORY * peak
    near(h.detach(), want[0], dtype, err, "h")
    near(last.detach(), want[1], torch.float32, err, "last state")
    assert h.stride(2) == 1 and (N == 1 or T == 1 or (h.stride(1) > h.stride(0)) == batch_first)
    if grad:
        dx, dgate, dstate, most = want[3:]
        top = float(x.detach().float().abs().max())
        near(got[0], dx, dtype, C * U * MEMORY * most, "dx")
        near(got[1], dgate, dtype, 2 * C * U * MEMORY * most * (peak + top), "dgate")
        if state is not None:
            near(got[2], dstate, torch.float32, C * U * MEMORY * most, "dstate")


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["leaky", "linear"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,D", [(1, 1, 1), (1, 16, 1024), (2, 3, 65), (15, 2, 130), (16, 2, 128), (17, 1, 64), (33, 2, 192), (65, 1, 63),
                                   (127, 2, 66), (257, 1, 320), (513, 2, 129), (1200, 1, 128), (256, 20, 1280), (2500, 1, 64)])
def test_sizes(hip_ops, T, N, D, dtype, form):
    check(T, N, D, dtype, form, 100 + T)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,N", [(torch.float32, 1500, 96), (torch.bfloat16, 1500, 192), (torch.float32, 4096, 2), (torch.bfloat16, 4096, 2)])
def test_long_memories(hip_ops, dtype, T, N):
    """Channels that remember over m = 300 to 2000 steps, each with one decay for all steps, so that what a step's decay loses to rounding is the same
    every time: the state and the gradient come from runs of S = 8 steps (16 forward where tiles are relayed, N = 2) whose decay is worked out as 1 - c.

    A run adds half a step of 1 - c, 2^-25, and one of its sum, 2^-24; m / S of them are remembered. Inside a run a step adds 2^-24 of the sum and up to 2.5 of the
    decay (1 + e, its reciprocal). 64 for the exponential (16 in 16 bits, twice: decay and input) and the join of a tile (14 runs, each
    half a step of 1 - c, and their sums): 1.5 m / S + 3.5 S + 64 in units of 2^-24 of the largest state. A decay worked out as a product of rounded
    decays instead loses up to 2.5 a step: in float32 arithmetic on the CPU these cases are off by 50 to 100 units so and by 1400 to 2200 as a product."""
    D = 128
    g = gen(29)
    memory = torch.exp(torch.empty(D).uniform_(5.704, 7.6, generator=g))            # 300 to 2000
    gate = torch.log(memory - 1).to(dtype)[None, None].expand(T, N, D).contiguous()
    x, dh = (1 + 0.1 * torch.randn(T, N, D, generator=g)).to(dtype), (1 + 0.1 * torch.randn(T, N, D, generator=g)).to(dtype)
    state, dlast = torch.ones(N, D), 300 * torch.ones(N, D)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gate, state)]
    h, last = run(*leaves)
    dx, dgate, dstate = torch.autograd.grad([h, last], leaves, [dh.to(DEV), dlast.to(DEV)])
    want_h, want_last, peak, want_dx, want_dgate, want_dstate, most = reference(x, gate, state, "leaky", dh=dh, dlast=dlast)
    units = lambda S: U * (1.5 * 2048 / S + 3.5 * S + 64)                           # 2048: a gate in bfloat16 may be half a step of 2^-6 more
    h_off, s_off = units(16 if N == 2 else 8) * peak, units(8) * most
    near(h.detach(), want_h, dtype, h_off, "h")
    near(last.detach(), want_last, torch.float32, h_off, "last state")
    near(dstate, want_dstate, torch.float32, s_off, "dstate")
    rest = torch.sigmoid(-gate.double())
    near(dx, want_dx, dtype, rest * s_off + 32 * U * want_dx.abs(), "dx")
    before = torch.cat([state.double()[None], want_h[:-1]])
    # h of the gradient's pass comes from runs of 8 steps whatever the forward pass did
    room = want_dx.abs() * units(8) * peak + rest * s_off * ((before - x.double()).abs() + units(8) * peak) + 32 * U * want_dgate.abs()
    near(dgate, want_dgate, dtype, room, "dgate")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_columns_take_narrow_workgroups(hip_ops, dtype):
    check(70, 40, 4096 if dtype == torch.float32 else 8192, dtype, "leaky", 7)      # 2560 waves of columns and more


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch_first", [False, True])
@pytest.mark.parametrize("with_state", [False, True])
def test_orders_in_memory_and_no_state(hip_ops, dtype, batch_first, with_state):
    check(150, 3, 136, dtype, "leaky", 8, batch_first=batch_first, with_state=with_state)
    check(5, 3, 136, dtype, "leaky", 9, batch_first=batch_first, with_state=with_state, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["leaky", "linear"])
@pytest.mark.parametrize("T,N,D", [(1, 4, 96), (16, 4, 96), (40, 4, 96), (700, 4, 96), (700, 4, 97)])
def test_starts_and_lengths(hip_ops, T, N, D, form):
    for dtype in DTYPES:
        g = gen(T + D)
        starts = torch.rand(T, N, generator=g) < 0.05
        starts[0, 0] = True
        starts[:, 3] = True                                                         # every step on its own
        lengths = torch.tensor([T, max(0, T // 2), 0, T - 1], dtype=torch.int32)
        check(T, N, D, dtype, form, 11, starts=starts.to(DEV))
        check(T, N, D, dtype, form, 12, lengths=lengths.to(DEV))
        check(T, N, D, dtype, form, 13, starts=starts.to(DEV), lengths=lengths.to(DEV), batch_first=True)
        check(T, N, D, dtype, form, 14, starts=starts.t().contiguous().to(DEV).t(), lengths=torch.tensor([-5, 1 << 40, 1, T]).to(DEV), grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20, 300])
def test_what_is_masked_may_hold_anything(hip_ops, T):
    """Padding full of NaN and infinities, and a state that overflowed in front of a start, change nothing."""
    N, D = 3, 130
    for dtype in DTYPES:
        for form in ("leaky", "linear"):
            x, gate, state, dh, dlast = operands(T, N, D, dtype, form, 15)
            lengths = torch.tensor([T, T // 2, 0], dtype=torch.int32, device=DEV)
            starts = torch.zeros(T, N, dtype=torch.bool, device=DEV)
            starts[T // 3, 0] = True
            outside = torch.arange(T, device=DEV)[:, None] >= lengths[None, :]
            dirty = [t.clone() for t in (x, gate, dh)]
            for t in dirty:
                t[outside] = float("nan")
                if T > 1:
                    t[-1, 2] = float("inf")
            dirty_state = state.clone()
            answers = []
            for xs, gs, ds in ((x, gate, dh), dirty):
                leaves = [t.clone().requires_grad_(True) for t in (xs, gs, state)]
                out = run(*leaves, form=form, starts=starts, lengths=lengths)
                answers.append([*out, *torch.autograd.grad(out, leaves, [ds, dlast])])
            for clean, got in zip(*answers):
                assert torch.equal(clean, got)
            # The first sequence's state is infinite before its start: from the start on it is as if it had been 0.
            dirty_state[0] = float("inf")
            after = run(x, gate, dirty_state, form=form, starts=starts)[0][T // 3:, 0]
            assert torch.equal(after, run(x, gate, state, form=form, starts=starts)[0][T // 3:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(20, 3), (700, 2), (700, 64)])
@pytest.mark.parametrize("form", ["leaky", "linear"])
def test_what_is_not_a_number_stays_until_a_start(hip_ops, T, N, form):
    """Decays whose product vanishes drop nothing: NaN lasts to the end of its sequence or to the next start, with starts given or not."""
    D = 130
    x, gate, state, _, _ = operands(T, N, D, torch.float32, form, 16)
    gate = torch.full_like(gate, -30.0 if form == "leaky" else 1e-9)
    x[3, 0, 5] = float("nan")
    starts = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    without, given = run(x, gate, state, form=form), run(x, gate, state, form=form, starts=starts)
    starts[T // 2, 0] = True
    dropped = run(x, gate, state, form=form, starts=starts)
    assert bool(without[0][3:, 0, 5].isnan().all()) and int(without[0].isnan().sum()) == T - 3 and int(without[1].isnan().sum()) == 1
    for a, b in zip(without, given):
        assert torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)
    assert bool(dropped[0][3:T // 2, 0, 5].isnan().all()) and int(dropped[0].isnan().sum()) == T // 2 - 3 and not bool(dropped[1].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(1, 3), (20, 3), (700, 2), (700, 64), (300, 200)])
@pytest.mark.parametrize("form,value", [("leaky", -30.0), ("linear", 1e-9), ("linear", -1e-9), ("linear", 0.0)])
def test_what_is_infinite_stays_until_a_start(hip_ops, T, N, form, value):
    """Decays whose product vanishes leave an infinite state, or gradient, infinite, of the sign that the steps give it; a decay of 0 makes it NaN."""
    D = 130
    x, gate, state, dh, dlast = operands(T, N, D, torch.float32, form, 19)
    gate = torch.full_like(gate, value)
    at = min(3, T - 1)
    x[at, 0, 5], dh[T - at - 1, 1, 7], state[1, 9], dlast[1, 9] = (float("inf"),) * 4
    starts = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    for mask in (None, starts, starts.clone().index_fill_(0, torch.tensor([T // 2], device=DEV), True)):
        leaves = [t.clone().requires_grad_(True) for t in (x, gate, state)]
        h, last = run(*leaves, form=form, starts=mask)
        dx, _, dstate = torch.autograd.grad([h, last], leaves, [dh, dlast])
        want = reference(x, gate, state, form, mask, dh=dh, dlast=dlast)
        for got, wanted in ((h, want[0]), (last, want[1]), (dx, want[3]), (dstate, want[5])):
            got = got.detach().double().cpu()
            assert torch.equal(got.isnan(), wanted.isnan())
            assert torch.equal(torch.where(got.isinf(), got.sign(), 0.0), torch.where(wanted.isinf(), wanted.sign(), 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(20, 3), (700, 2), (700, 64)])
def test_growth_of_nothing_is_nothing(hip_ops, T, N):
    """Gates of 2 grow past the range of float32 over a run, and 0 stays 0; with a start, what grew is gone."""
    D = 130
    leaves = [torch.zeros(T, N, D, device=DEV), torch.full((T, N, D), 2.0, device=DEV), torch.zeros(N, D, device=DEV)]
    starts = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    starts[T // 2] = True
    for mask in (None, starts):
        for t in leaves:
            t.requires_grad_(True)
        h, last = run(*leaves, form="linear", starts=mask)
        got = torch.autograd.grad([h, last], leaves, [torch.zeros_like(h), torch.zeros_like(last)])
        for t in (h, last, *got):
            assert bool((t == 0).all())
    x = torch.zeros(T, N, D, device=DEV)
    x[0] = 1.0
    h, last = run(x, leaves[1].detach(), form="linear", starts=starts)
    want = torch.exp2(torch.arange(T // 2, dtype=torch.float64)).to(torch.float32).to(DEV)          # infinite from 2^128 on
    assert torch.equal(h[:T // 2], want[:, None, None].expand(T // 2, N, D)) and bool((h[T // 2:] == 0).all()) and bool((last == 0).all())


GROWTH = [(20, 3, 130), (20, 3, 33), (700, 2, 130), (700, 2, 65), (700, 64, 130), (300, 200, 130), (40, 2000, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,N,D", GROWTH)
def test_growth_past_the_range_of_float32_and_back(hip_ops, T, N, D, dtype):
    """A state of 2^-110 that ten gates of 2^20 bring to 2^90, and four of 2^-10 to 2^50: every product is a power of two, so that nothing is
    rounded, and no state leaves the range, though the product of the gates does. The gradient goes the same way back."""
    gate = torch.ones(T, N, D)
    gate[3:13], gate[14:18] = 2.0 ** 20, -(2.0 ** -10)
    x, dh = torch.zeros(T, N, D), torch.zeros(T, N, D)
    state, dlast = torch.full((N, D), 2.0 ** -110), torch.full((N, D), 2.0 ** -100)
    want = reference(x, gate, state, "linear", dh=dh, dlast=dlast)
    for mask in (None, torch.zeros(T, N, dtype=torch.bool, device=DEV)):
        leaves = [t.to(DEV).requires_grad_(True) for t in (x.to(dtype), gate.to(dtype), state)]
        h, last = run(*leaves, form="linear", starts=mask)
        got = [h, last, *torch.autograd.grad([h, last], leaves, [dh.to(DEV, dtype), dlast.to(DEV)])]
        for a, b in zip(got, (want[0], want[1], *want[3:6])):
            assert torch.equal(a.detach().cpu(), b.to(a.dtype))         # a gradient of 2^-140 is 0 in bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,D", GROWTH)
def test_gates_beyond_one_are_walked_step_by_step(hip_ops, T, N, D):
    """Gates between -1.5 and 1.5: a prompt has the bits of the same prompt in single tokens, and gradients are as exact as a walk's, whose error is at
    most 2^-24 of |a| |h| + |x| a step (8 of them: the state, its sum and product, the gradient's), carried on by |a|."""
    g = gen(23)
    x, dh = torch.randn(T, N, D, generator=g), torch.randn(T, N, D, generator=g)
    gate = (torch.rand(T, N, D, generator=g) * 2 - 1) * 1.5
    state, dlast = torch.randn(N, D, generator=g), torch.randn(N, D, generator=g)
    starts, lengths = torch.rand(T, N, generator=g) < 0.02, torch.randint(0, T + 1, (N,), generator=g, dtype=torch.int32)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, gate, state)]
    with torch.no_grad():
        h, last = run(*leaves, form="linear")
        s = leaves[2]
        for t in range(T):
            token, s = run(leaves[0][t:t + 1], leaves[1][t:t + 1], s, form="linear")
            assert torch.equal(token[0], h[t]), t
        assert torch.equal(s, last)
    for masks in ({}, {"starts": starts, "lengths": lengths}):
        h, last = run(*leaves, form="linear", **{k: m.to(DEV) for k, m in masks.items()})
        got = [h, last, *torch.autograd.grad([h, last], leaves, [dh.to(DEV), dlast.to(DEV)])]
        want = reference(x, gate, state, "linear", dh=dh, dlast=dlast, **masks)
        a = gate.double().abs()
        limit, drop = masks.get("lengths", torch.full((N,), T)), masks.get("starts", torch.zeros(T, N, dtype=torch.bool))
        inside, keep = (torch.arange(T)[:, None] < limit[None, :])[:, :, None], (~drop)[:, :, None].double()
        size, off = state.double().abs(), torch.zeros(N, D, dtype=torch.float64)
        before, h_off = [], []
        for t in range(T):
            before.append((size * keep[t], off * keep[t]))
            new = a[t] * before[t][0] + x[t].double().abs()
            off = torch.where(inside[t], a[t] * before[t][1] + C * U * new, off)
            size = torch.where(inside[t], new, size)
            h_off.append(torch.where(inside[t], off, 0.0))
        near(got[0], want[0], torch.float32, torch.stack(h_off), "h")
        near(got[1], want[1], torch.float32, off, "last state")
        size, off = dlast.double().abs(), torch.zeros(N, D, dtype=torch.float64)
        x_off, gate_off = [None] * T, [None] * T
        for t in range(T - 1, -1, -1):
            new = size + dh[t].double().abs()
            s_off = off + C * U * new
            x_off[t] = torch.where(inside[t], s_off, 0.0)
            gate_off[t] = torch.where(inside[t], s_off * (before[t][0] + before[t][1]) + new * before[t][1] + C * U * new * before[t][0], 0.0)
            size, off = torch.where(inside[t], a[t] * new * keep[t], size), torch.where(inside[t], a[t] * s_off * keep[t], off)
        near(got[2], want[3], torch.float32, torch.stack(x_off), "dx")
        near(got[3], want[4], torch.float32, torch.stack(gate_off), "dgate")
        near(got[4], want[5], torch.float32, off, "dstate")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,D", [(1, 40, 3), (20, 33, 5), (300, 17, 24), (520, 2, 65), (40, 300, 1)])
def test_narrow_rows_side_by_side(hip_ops, T, N, D, dtype):
    """Sequences that lie next to each other run as one of more channels: the same bits as apart, whichever pass sees them so."""
    check(T, N, D, dtype, "leaky", 17)
    x, gate, state, dh, dlast = operands(T, N, D, dtype, "leaky", 18)
    apart = lambda t: torch.cat([t, t], 2)[:, :, :D] if t.dim() == 3 else t
    answers = []
    for inputs, outputs in ((lambda t: t, lambda t: t), (apart, apart), (lambda t: t, apart), (apart, lambda t: t)):
        leaves = [inputs(t).detach().requires_grad_(True) for t in (x, gate, state)]
        out = run(*leaves)
        answers.append([*out, *torch.autograd.grad(out, leaves, [outputs(dh), dlast])])
    alone = run(x, gate, state, lengths=torch.full((N,), T, dtype=torch.int32, device=DEV))
    for other in answers[1:]:
        assert all(torch.equal(a, b) for a, b in zip(answers[0], other))
    assert all(torch.equal(a, b) for a, b in zip(answers[0], alone))


@pytest.mark.gpu
def test_strided_operands_and_a_broadcast_gate(hip_ops):
    """Slices of one projection and a gate per channel go in without copies; the expanded gate's gradient is summed."""
    T, N, D = 90, 2, 96
    g = gen(21)
    wide = torch.randn(N, T, 2 * D + 1, generator=g).to(DEV, torch.bfloat16)
    leak = torch.randn(D, generator=g).to(DEV, torch.bfloat16).requires_grad_(True)
    x = wide[:, :, 1:D + 1].transpose(0, 1)                                         # odd offsets: no 4-byte accesses
    h, last = run(x, leak.expand(T, N, D), None)
    grad = torch.autograd.grad(h.float().sum(), leak)[0]
    want = reference(x, leak.detach().expand(T, N, D), None, "leaky", dh=torch.ones(T, N, D), dlast=None)
    near(h.detach(), want[0], torch.bfloat16, C * U * MEMORY * want[2], "h")
    total = want[4].sum((0, 1))
    # every element of the sum is rounded to bfloat16, and so is the sum, which autograd adds up in float32
    room = torch.finfo(torch.bfloat16).eps / 2 * (want[4].abs().sum((0, 1)) + total.abs()) + T * N * 2 * C * U * MEMORY * want[6] * 10
    assert bool(((grad.double().cpu() - total).abs() <= room).all())
    assert torch.equal(run(wide[:, ::2, :D].transpose(0, 1), wide[:, ::2, D:2 * D].transpose(0, 1))[0],
                       run(wide[:, ::2, :D].contiguous().transpose(0, 1), wide[:, ::2, D:2 * D].contiguous().transpose(0, 1))[0])


@pytest.mark.gpu
def test_gradient_against_differences(hip_ops):
    """One directional derivative per operand, float32, by central differences of the operator itself: truncation h^2 * third derivative
    and rounding 2^-24 * memory * |loss terms| / h at h = 2^-6 stay below 2e-3 of the sum of the terms' sizes."""
    T, N, D = 37, 2, 33
    x, gate, state, dh, dlast = operands(T, N, D, torch.float32, "leaky", 31)
    leaves = [t.requires_grad_(True) for t in (x, gate, state)]
    out = run(*leaves)
    grads = torch.autograd.grad(out, leaves, [dh, dlast])
    step = 2.0 ** -6
    for k in range(3):
        way = torch.randn(leaves[k].shape, generator=gen(40 + k)).to(DEV)

        def loss(sign):
            moved = [t.detach() + (sign * step * way if i == k else 0) for i, t in enumerate(leaves)]
            h, last = run(*moved)
            return (h.double() * dh.double()).sum() + (last.double() * dlast.double()).sum()
        slope = (loss(1) - loss(-1)) / (2 * step)
        want = (grads[k].double() * way.double()).sum()
        size = (grads[k].double() * way.double()).abs().sum()
        assert abs(float(slope - want)) <= 2e-3 * float(size)


@pytest.mark.gpu
def test_a_sequence_in_pieces_and_repeated_calls(hip_ops):
    """Handing the state over between pieces is the long call up to rounding, single tokens included; equal calls have equal bits."""
    T, N, D = 400, 2, 128
    x, gate, state, _, _ = operands(T, N, D, torch.float32, "leaky", 41)
    whole, last = run(x, gate, state)
    s, parts = state, []
    for a, b in ((0, 1), (1, 2), (2, 30), (30, 300), (300, 400)):
        h, s = run(x[a:b], gate[a:b], s)
        parts.append(h)
    err = 2 * C * U * MEMORY * float(whole.abs().max())
    assert float((torch.cat(parts) - whole).abs().max()) <= err and float((s - last).abs().max()) <= err
    for _ in range(3):
        again = run(x, gate, state)
        assert torch.equal(again[0], whole) and torch.equal(again[1], last)


@pytest.mark.gpu
def test_graph_replays_and_other_streams(hip_ops):
    T, N, D = 300, 2, 128
    x, gate, state, dh, dlast = operands(T, N, D, torch.bfloat16, "leaky", 51)
    leaves = [t.requires_grad_(True) for t in (x, gate, state)]

    def step():        # its autograd graph ends with it: none of the same leaves lives during a capture
        out = run(*leaves)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, [dh, dlast])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    want = [t.clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    del on_side
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(T, N, D, generator=gen(60 + k)).to(DEV, torch.bfloat16))
        want = [t.clone() for t in step()]
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_empty(hip_ops):
    for T, N, D in ((0, 2, 8), (3, 0, 8), (3, 2, 0)):
        x = torch.empty(T, N, D, device=DEV, requires_grad=True)
        state = torch.randn(N, D, device=DEV, requires_grad=True)
        h, last = run(x, x, state)
        assert h.shape == (T, N, D) and last.shape == (N, D)
        if T == 0:
            assert torch.equal(last, state)
            assert torch.equal(torch.autograd.grad(last.sum(), state)[0], torch.ones_like(state))


@pytest.mark.gpu
def test_refusals_on_the_gpu(hip_ops):
    x = torch.zeros(4, 2, 8, device=DEV)
    for args, kwargs, words in (((x, x[:3]), {}, "unsupported_shape"), ((x, x.half()), {}, "unsupported_dtype"), ((x, x, x[0].half()), {}, "unsupported_dtype"),
                                ((x, x, x[0, :1]), {}, "unsupported_shape"), ((x[0], x[0]), {}, "unsupported_rank"), ((x.double(), x.double()), {}, "unsupported_dtype"),
                                ((x, x), {"form": "other"}, "unsupported_form"), ((x, x), {"starts": torch.zeros(4, 2, device=DEV)}, "unsupported_dtype"),
                                ((x, x), {"lengths": torch.zeros(2)}, "unsupported_device"), ((x, x.cpu()), {}, "unsupported_device")):
        with pytest.raises(RuntimeError, match=words):
            run(*args, **kwargs)
    out = run(x.requires_grad_(True), x.detach() + 1)[0].sum()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(out, x, create_graph=True)[0].sum(), x)


def test_steps_too_far_apart_are_among_the_reasons():
    """What the kernels refuse of strides is listed beforehand, of the tensor that h_seq will be as well."""
    from torch._subclasses import FakeTensorMode
    from triton_snn_fusion_amd.runtime.hip_gated_recurrence_backend import check_gated_recurrence_support as reasons
    with FakeTensorMode():
        far = torch.empty(16, 65536, 2048, dtype=torch.bfloat16, device="cuda")
        near_by = torch.empty(65536, 16, 2048, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        assert len(reasons(far, far)) == 3 and all("unsupported_stride" in r for r in reasons(far, far))
        assert len(reasons(near_by, far)) == 1 and "unsupported_stride: gate_seq" in reasons(near_by, far)[0]
        one = torch.empty(1, 1, 2048, dtype=torch.bfloat16, device="cuda").expand(16, 65536, 2048)
        assert len(reasons(one, near_by)) == 1 and "unsupported_stride: h_seq" in reasons(one, near_by)[0]
        apart = torch.empty(2048, 16, 65536, dtype=torch.bfloat16, device="cuda").permute(1, 2, 0)     # channels apart: copied to steps outermost
        assert sum("unsupported_stride: gate_seq" in r for r in reasons(near_by, apart)) == 1
        assert reasons(near_by, near_by) == [] and reasons(far[:1], far[:1]) == [] and reasons(far[:, :1], far[:, :1]) != []


@pytest.mark.gpu
def test_a_gradient_whose_steps_lie_far_apart(hip_ops):
    """Sequences outermost go in whatever their size; a gradient with the steps outermost, 2 GiB within 16 steps, is brought into their order."""
    T, N, D = 16, 4096, 17600
    g = torch.Generator(device=DEV).manual_seed(5)
    draw = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    x, gate = (draw(N, T, D).transpose(0, 1).requires_grad_(True) for _ in range(2))
    dh = draw(T, N, D)
    h, _ = run(x, gate)
    got = torch.autograd.grad(h, [x, gate], dh, retain_graph=True)
    want = torch.autograd.grad(h, [x, gate], dh.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del x, gate, dh, h, got, want
    torch.cuda.empty_cache()


def test_refusals_without_a_gpu():
    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="unsupported_device"):
        run(x, x)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        run(None, x)


def test_entry_points_refuse_before_any_gpu_work(snnf_lib):
    f, b = snnf_lib.snnf_gated_recurrence, snnf_lib.snnf_gated_recurrence_backward

    def forward(x=16, T=4, N=2, D=8, dtype=0, form=0, state_out=16, workspace=None, nbytes=0):
        return f(x, 16, 8, 16, 16, 8, T, N, D, dtype, form, None, 0, 0, None, None, 16, 16, 8, state_out, None, workspace, nbytes, None)

    assert forward(T=0) == -1 and forward(N=-1) == -1 and forward(dtype=9) == -1 and forward(form=2) == -1
    assert forward(x=None) == -1 and b"non-null" in snnf_lib.snnf_last_error()
    assert forward(state_out=None) == -1 and forward(N=0, x=None) == 0 and forward(D=0, x=None) == 0
    assert f(16, 16, 8, 16, 16, 8, 4, 2, 8, 0, 0, None, 0, 0, None, 32, 16, 16, 8, 32, None, None, 0, None) == -1        # the state in place
    assert b"same memory" in snnf_lib.snnf_last_error()
    assert b(16, 16, 8, 16, 16, 8, 16, 16, 8, 4, 2, 8, 0, 0, None, 0, 0, None, 16, 32, 16, 16, 8, 16, 16, 8, 32, None, 0, None) == -1
    assert b"same memory" in snnf_lib.snnf_last_error()
    assert forward(T=(1 << 30) + 1) == -2
    assert snnf_lib.snnf_gated_recurrence_workspace_bytes(100000, 1, 64, 1, 0) > 0
    assert forward(T=100000, N=1, D=64, dtype=1) == -4 and b"workspace" in snnf_lib.snnf_last_error()
    assert b(16, 16, 8, 16, 16, 8, 16, 16, 8, 4, 2, 8, 0, 0, None, 0, 0, None, None, None, 16, 16, 8, 16, 16, 8, 16, None, 0, None) == -1    # no marks
    assert b"marks" in snnf_lib.snnf_last_error()
    assert snnf_lib.snnf_gated_recurrence_marks_bytes(0, 1, 1, 0) == 0 and snnf_lib.snnf_gated_recurrence_marks_bytes(1, 3, 5, 0) == 60
    assert f(16, 1 << 31, 8, 16, 16, 8, 4, 2, 8, 0, 0, None, 0, 0, None, None, 16, 16, 8, 16, None, None, 0, None) == -2
    assert b"unsupported_stride" in snnf_lib.snnf_last_error()


@pytest.mark.gpu
def test_python_implementation(hip_ops, monkeypatch):
    """What the dispatch module does not take runs in Python, on the same kernels: the same checks with the module out of the way, and equal bits."""
    from triton_snn_fusion_amd import _dispatch
    from triton_snn_fusion_amd.runtime import hip_gated_recurrence_backend as backend
    x, gate, state, dh, dlast = operands(300, 3, 130, torch.bfloat16, "leaky", 71)
    leaves = [t.requires_grad_(True) for t in (x, gate, state)]
    starts, lengths = (torch.rand(300, 3, generator=gen(1)) < 0.1).to(DEV), torch.tensor([300, 20, 299], dtype=torch.int32, device=DEV)

    def step():
        out = run(*leaves, starts=starts, lengths=lengths)
        return [*out, *torch.autograd.grad(out, leaves, [dh, dlast])]
    assert _dispatch.module().gated_recurrence(*leaves, starts, lengths, 0)[0].grad_fn is not None
    dispatched = step()
    monkeypatch.setattr(backend, "native", lambda t: None)
    assert all(torch.equal(a, b) for a, b in zip(step(), dispatched))
    for dtype in DTYPES:
        check(70, 3, 130, dtype, "leaky", 72, batch_first=True)
        check(300, 2, 65, dtype, "linear", 73, starts=starts[:, :2].contiguous(), lengths=lengths[:2].long())
    test_refusals_on_the_gpu(hip_ops)
    test_empty(hip_ops)


@pytest.mark.gpu
def test_one_output_used_and_one_input_differentiated(hip_ops):
    x, gate, state, dh, dlast = operands(40, 2, 70, torch.float32, "leaky", 74)
    for k, leaf in enumerate((x, gate, state)):
        args = [t.detach().requires_grad_(t is leaf) for t in (x, gate, state)]
        alone = torch.autograd.grad(run(*args), args[k], [dh, dlast])[0]
        every = [t.detach().requires_grad_(True) for t in (x, gate, state)]
        assert torch.equal(alone, torch.autograd.grad(run(*every), every[k], [dh, dlast])[0])
        for used, grads in ((0, [dh, torch.zeros_like(dlast)]), (1, [torch.zeros_like(dh), dlast])):
            got = torch.autograd.grad(run(*every)[used], every[k], grads[used])[0]
            assert torch.equal(got, torch.autograd.grad(run(*every), every[k], grads)[0])
