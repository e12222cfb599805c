"""Verification of drafted tokens against the definition in float64 on the CPU, request by request. Answers are whole numbers and have to be equal: the kernels decide as exact arithmetic
does wherever float32 cannot tell two numbers apart."""
import math

import pytest
import torch

from helpers import DEV, gen

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(logits, drafts, uniforms, noise, draft_logits=None, temperature=1.0, lengths=None):
    logits, drafts, uniforms, noise = logits.double().cpu(), drafts.cpu(), uniforms.double().cpu(), noise.double().cpu()
    N, K = drafts.shape
    V = logits.shape[2]
    each = temperature.double().cpu() if isinstance(temperature, torch.Tensor) else torch.full((N,), float(temperature), dtype=torch.float64)
    tokens, accepted = torch.full((N, K + 1), -100, dtype=torch.int64), torch.zeros(N, dtype=torch.int32)
    for n in range(N):
        t = float(each[n])

        def share(row):
            if not bool(torch.isfinite(row).any()) or bool((row.isnan() | (row == math.inf)).any()):
                return torch.zeros(V, dtype=torch.float64)
            if not t > 0:
                return (torch.arange(V) == int(row.argmax())).double()
            return torch.softmax(row / t, 0)

        count = K if lengths is None else min(max(int(lengths[n]), 0), K)
        j = 0
        while True:
            p = share(logits[n, j])
            r = p
            if j == count:
                break
            x = int(drafts[n, j])
            q = torch.zeros(V, dtype=torch.float64)
            if draft_logits is not None and t > 0:
                q = share(draft_logits[n, j].double().cpu())
            elif 0 <= x < V:
                q[x] = 1.0
            if not (0 <= x < V and float(uniforms[n, j]) * float(q[x]) < float(p[x])):
                r = (p - q).clamp(min=0)
                r = r if bool((r > 0).any()) else p
                break
            tokens[n, j] = x
            j += 1
        accepted[n] = j
        if bool((r > 0).any()):
            tokens[n, j] = int((r / noise[n]).argmax())
    return tokens, accepted


def operands(N, K, V, dtype, seed, draft=True, far=0.8):
    g = gen(seed)
    logits = torch.randn(N, K + 1, V, generator=g) * 2.0
    logits.scatter_add_(2, torch.randint(0, V, (N, K + 1, 2), generator=g), torch.full((N, K + 1, 2), 6.0))
    theirs = logits[:, :K] + far * torch.randn(N, K, V, generator=g)
    drafts = (theirs - (-torch.rand(N, K, V, generator=g).clamp(min=1e-9).log()).log()).argmax(2) if K else torch.zeros(N, 0, dtype=torch.int64)
    uniforms, noise = torch.rand(N, K, generator=g), torch.empty(N, V).exponential_(generator=g).clamp(min=1e-9)
    to = lambda t: t.to(DEV, dtype)
    return [to(logits), drafts.to(DEV), uniforms.to(DEV), noise.to(DEV)], to(theirs) if draft else None


def run(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_draft_verification_backend import run_hip_draft_verification
    return run_hip_draft_verification(*args, **kwargs)


def check(args, **options):
    want = reference(*args, **options)
    got = run(*args, **options)
    torch.cuda.synchronize()
    assert got.tokens.dtype == torch.int64 and got.accepted.dtype == torch.int32
    assert torch.equal(got.accepted.cpu(), want[1]), (got.accepted, want[1])
    assert torch.equal(got.tokens.cpu(), want[0]), (got.tokens, want[0])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K,V", [(1, 1, 1), (1, 0, 7), (3, 2, 2), (2, 4, 255), (5, 3, 1000), (1, 4, 40003), (40, 5, 1024), (3, 64, 300), (300, 2, 129), (2, 1, 200001)])
def test_sizes(hip_ops, N, K, V, dtype, draft):
    args, theirs = operands(N, K, V, dtype, 10 + N + V, draft)
    got = check(args, draft_logits=theirs)
    if N >= 40 and K > 1 and draft:
        assert 0 < float(got.accepted.float().mean()) < K          # the cases hold both answers


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_temperatures_and_lengths(hip_ops, dtype, draft):
    """Requests of their own temperature, greedy ones (0, below it, NaN) and numbers of drafts; what lies behind a request's drafts is NaN."""
    N, K, V = 24, 4, 3001
    args, theirs = operands(N, K, V, dtype, 21, draft)
    each = torch.rand(N, generator=gen(3)) + 0.3
    each[::4], each[1], each[2] = 0.0, -1.0, float("nan")
    args[1][::4] = args[0][::4, :K].float().argmax(2)              # greedy requests whose drafts stand
    args[1][4, 1] = (args[1][4, 1] + 1) % V
    lengths = torch.randint(-1, K + 2, (N,), generator=gen(4))
    want = reference(*args, draft_logits=theirs, temperature=each, lengths=lengths)
    for n in range(N):
        count = min(max(int(lengths[n]), 0), K)
        args[0][n, count + 1:] = float("nan")
        args[1][n, count:] = 1 << 40
        args[2][n, count:] = float("nan")
        if draft:
            theirs[n, count:] = float("nan")
    for wide in (torch.int32, torch.int64):
        got = run(*args, draft_logits=theirs, temperature=each.to(DEV), lengths=lengths.to(DEV, wide))
        assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])
    check(args[:1] + operands(N, K, V, dtype, 21, draft)[0][1:], draft_logits=operands(N, K, V, dtype, 21, draft)[1], temperature=0.7, lengths=torch.zeros(N, dtype=torch.int32, device=DEV))
    check(operands(N, K, V, dtype, 22, draft)[0], draft_logits=operands(N, K, V, dtype, 22, draft)[1], temperature=0)
    check(operands(N, K, V, dtype, 23, draft)[0], draft_logits=operands(N, K, V, dtype, 23, draft)[1], temperature=1e-3)
    check(operands(N, K, V, dtype, 24, draft)[0], draft_logits=operands(N, K, V, dtype, 24, draft)[1], temperature=50.0)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 9000, 70000])
def test_numbers_that_float32_cannot_tell_apart(hip_ops, V):
    """A uniform at the border of what stands, and the float32 below it; equal shares over equal noise, of which the lowest index is drawn."""
    logits = torch.full((4, 2, V), -math.inf, device=DEV)
    logits[..., 5] = logits[..., V - 3] = 1.25                       # p = 1/2 each
    drafts = torch.full((4, 1), 5, device=DEV)
    below = float(torch.nextafter(torch.tensor(0.5), torch.tensor(0.0)))
    uniforms = torch.tensor([[0.5], [below], [0.25], [0.75]], device=DEV)
    noise = torch.ones(4, V, device=DEV)
    got = run(logits, drafts, uniforms, noise)
    assert got.accepted.tolist() == [0, 1, 1, 0] and got.tokens[:, 0].tolist() == [V - 3, 5, 5, V - 3]
    assert got.tokens[1:3, 1].tolist() == [5, 5]
    # q(5) = 1/4: u q < p always; then q(5) = 1 - 2^-20 against p = 1/2
    theirs = torch.full((4, 1, V), -math.inf, device=DEV)
    theirs[..., [5, 6, 7, 8]] = 0.0
    assert run(logits, drafts, uniforms, noise, draft_logits=theirs).accepted.tolist() == [1, 1, 1, 1]
    # many equal shares
    flat = torch.zeros(3, 1, V, device=DEV, dtype=torch.bfloat16)
    noise = torch.full((3, V), 2.0, device=DEV)
    noise[1, [V // 2, V - 1]] = 0.5
    none = torch.zeros(3, 0, device=DEV)
    assert run(flat, none.long(), none, noise).tokens[:, 0].tolist() == [0, V // 2, 0]
    # shares that differ in the 30th bit
    near = torch.zeros(1, 1, V, device=DEV)
    noise = torch.full((1, V), 3.0, device=DEV)
    near[0, 0, V - 2] = 2.0 ** -30
    assert run(near, none[:1].long(), none[:1], noise).tokens[0, 0] == V - 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_drafts_of_the_same_model(hip_ops, dtype):
    """p = q: every draft stands, whatever the uniform, and nothing is left beside the draft's share. Up to a factor of 1 + 2^-10, the residual is small against both."""
    args, theirs = operands(30, 3, 5000, dtype, 31, True, far=0.0)
    args[2][:, 0] = 1.0 - 2.0 ** -24
    got = check(args, draft_logits=theirs)
    assert bool((got.accepted == 3).all())
    args, theirs = operands(60, 3, 5000, dtype, 32, True, far=2.0 ** -10)
    args[2][:] = 1.0 - 2.0 ** -24
    check(args, draft_logits=theirs)


@pytest.mark.gpu
def test_masked_and_broken_rows(hip_ops):
    V = 2500
    args, theirs = operands(8, 2, V, torch.float32, 41)
    mask = torch.rand(V, generator=gen(5)) < 0.9
    mask[7] = False
    args[0][:, :, mask.to(DEV)] = -math.inf
    args[0][1, 0] = -math.inf                                      # nothing left at the first draft
    args[0][2, 2] = -math.inf                                      # behind the last
    args[0][3, 0, 9] = math.nan
    args[0][4, 1, 9] = math.inf
    args[1][5, 0], args[1][6, 1] = -1, V
    args[1][7], args[2][7] = 7, 0.0
    args[0][2, :2, 7], theirs[2, :, 7] = 20.0, 20.0
    args[1][2], args[2][2] = 7, 0.1
    for options in ({"draft_logits": theirs}, {}):
        got = check(args, **options)
        assert got.tokens[1].tolist() == [-100] * 3 and got.tokens[3].tolist() == [-100] * 3
        assert got.tokens[2].tolist() == [7, 7, -100] and int(got.accepted[2]) == 2 and int(got.accepted[5]) == 0
    got = run(*args, temperature=0.0)
    assert got.tokens[1].tolist() == [-100] * 3 and int(got.accepted[1]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [777, 30001])
def test_layouts_give_the_same_answers(hip_ops, V):
    args, theirs = operands(6, 3, V, torch.bfloat16, 51)
    want = run(*args, draft_logits=theirs)

    def apart(t):                                                   # rows an odd number of elements apart, places outermost
        out = torch.zeros(t.shape[1], t.shape[0], t.shape[2] + 5, dtype=t.dtype, device=DEV)[..., 3:-2]
        return out.transpose(0, 1).copy_(t)
    moved = [apart(args[0]), args[1].to(torch.int32).t().contiguous().t(), args[2].t().contiguous().t(), torch.zeros(6, V + 3, device=DEV)[:, 1:-2].copy_(args[3])]
    for other in (run(*moved, draft_logits=apart(theirs)), run(torch.stack([args[0]] * 2, -1)[..., 0], *args[1:3], args[3].t().contiguous().t(), draft_logits=theirs)):
        assert torch.equal(want.tokens, other.tokens) and torch.equal(want.accepted, other.accepted)
    assert torch.equal(run(args[0], args[1], args[2], args[3][:1].expand(6, V)).tokens, run(args[0], args[1], args[2], args[3][:1].repeat(6, 1)).tokens)


@pytest.mark.gpu
def test_tokens_are_distributed_as_the_target(hip_ops):
    """20000 requests of the same row: the first token's frequencies, each within 5 standard deviations of p (a chance of 1 in 10^5 for 16 tokens; the numbers are seeded)."""
    N, V = 20000, 16
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    p, q = torch.randn(V, generator=gen(1)).to(DEV), torch.randn(V, generator=gen(2)).to(DEV)
    drafts = torch.multinomial(torch.softmax(q, 0).expand(N, V), 1, generator=g)
    uniforms, noise = torch.rand(N, 1, generator=g, device=DEV), torch.empty(N, V, device=DEV).exponential_(generator=g).clamp(min=1e-9)
    got = run(p.expand(N, 2, V), drafts, uniforms, noise, draft_logits=q.expand(N, 1, V))
    share = torch.softmax(p.double().cpu(), 0)
    seen = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double() / N
    assert bool(((seen - share).abs() <= 5 * (share * (1 - share) / N).sqrt()).all())
    assert 0.2 < float(got.accepted.float().mean()) < 0.95


@pytest.mark.gpu
def test_captured_and_on_two_streams(hip_ops):
    """Replays on new numbers, with eager calls of other sizes on another stream between: each call's scratch memory is its own."""
    args, theirs = operands(2, 4, 60000, torch.bfloat16, 61)
    other, other_theirs = operands(9, 2, 33000, torch.bfloat16, 62)
    want_other = run(*other, draft_logits=other_theirs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*args, draft_logits=theirs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        answer = run(*args, draft_logits=theirs)
    for seed in range(5):
        new, new_theirs = operands(2, 4, 60000, torch.bfloat16, 70 + seed)
        for a, b in zip((*args, theirs), (*new, new_theirs)):
            a.copy_(b)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            got = [run(*other, draft_logits=other_theirs) for _ in range(3)]
        torch.cuda.synchronize()
        want = reference(*args, draft_logits=theirs)
        assert torch.equal(answer.tokens.cpu(), want[0]) and torch.equal(answer.accepted.cpu(), want[1])
        for one in got:
            assert torch.equal(one.tokens, want_other.tokens) and torch.equal(one.accepted, want_other.accepted)


@pytest.mark.gpu
def test_no_requests(hip_ops):
    got = run(torch.zeros(0, 3, 10, device=DEV), torch.zeros(0, 2, dtype=torch.int64, device=DEV), torch.zeros(0, 2, device=DEV), torch.zeros(0, 10, device=DEV))
    assert got.tokens.shape == (0, 3) and got.accepted.shape == (0,)


def test_refusals_on_the_cpu():
    t = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="unsupported_device"):
        run(t, torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2), torch.zeros(2, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("change,match", [
    ({"logits": lambda t: t[0]}, "unsupported_rank"), ({"logits": lambda t: t[:, :0]}, "unsupported_rank"), ({"logits": lambda t: t.double()}, "unsupported_dtype"),
    ({"logits": lambda t: t[..., :0]}, "logits, got"), ({"logits": lambda t: t[:, :1].expand(2, 66, 8)}, "at most 64 drafts"),
    ({"drafts": lambda t: t[:, :1]}, "drafts must be"), ({"drafts": lambda t: t.float()}, "drafts must be"), ({"uniforms": lambda t: t.double()}, "uniforms must be"),
    ({"noise": lambda t: t[:, :4]}, "noise must be"), ({"noise": lambda t: t.half()}, "noise must be"), ({"draft_logits": lambda t: t.half()}, "draft_logits must be"),
    ({"draft_logits": lambda t: t[:, :1]}, "draft_logits must be"), ({"temperature": lambda t: torch.ones(3, device=DEV)}, "temperature must be"),
    ({"temperature": lambda t: "hot"}, "temperature must be"), ({"lengths": lambda t: torch.zeros(2, device=DEV)}, "lengths must be"),
    ({"lengths": lambda t: torch.zeros(2, dtype=torch.int32)}, "unsupported_device"), ({"drafts": lambda t: None}, "drafts must be a tensor")])
def test_refusals(hip_ops, change, match):
    call = {"logits": torch.zeros(2, 3, 8, device=DEV), "drafts": torch.zeros(2, 2, dtype=torch.int64, device=DEV), "uniforms": torch.zeros(2, 2, device=DEV),
            "noise": torch.ones(2, 8, device=DEV), "draft_logits": torch.zeros(2, 2, 8, device=DEV), "temperature": 1.0, "lengths": None}
    for name, f in change.items():
        call[name] = f(call[name])
    with pytest.raises(RuntimeError, match=match):
        run(**call)
