"""Scores of given tokens and their gradient against the formulas in float64 on the CPU.

Tolerances, in float32 roundings u = 2^-24. z = (x - M) log2 e is off by 3 u |z|, 2^z by that times ln 2 and 2 u: terms of the sums by
(3 |x - M| + 2) u, and those that matter have |x - M| < 16 or so; chains of at most V / threads terms and a tree add 40 u. So log s is off by
C = 96 u, logprob by C u + 2 u (|x| + |M| + log s), entropy by C u (1 + entropy + mean |x - M|), probabilities by C u relative for |x - M| < 16
and 3 u |x - M| beyond. A gradient in a 16-bit type is rounded once more."""
import math

import pytest
import torch

from helpers import DEV, gen

U = 2.0 ** -24
C = 96.0
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def run(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_token_scores_backend import run_hip_token_scores
    return run_hip_token_scores(*args, **kwargs)


def reference(x, tokens, k):
    x = x.double().cpu()
    V = x.shape[-1]
    M = x.max(-1, keepdim=True).values
    none = M == -math.inf
    y = torch.where(none, torch.full_like(x, -math.inf), x - M)
    e = torch.exp(y)
    s = e.sum(-1, keepdim=True)
    logp = torch.where(none, torch.full_like(x, -math.inf), y - torch.log(s))
    p = torch.where(none, torch.zeros_like(x), e / s)
    entropy = -(p * torch.where(p > 0, logp, torch.zeros_like(x))).sum(-1)
    given = (tokens >= 0) & (tokens < V)
    logprob = torch.where(given, logp.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0], torch.zeros_like(entropy))
    best = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :k]
    return logprob, entropy, logp.gather(-1, best), best, logp, p, given


def check(x, tokens, k, what=""):
    """x on the CPU in its dtype."""
    dtype = x.dtype
    dev = x.to(DEV).requires_grad_(True)
    got = run(dev, tokens.to(DEV), top_k=k)
    rows = tokens.numel()
    g = gen(rows + x.shape[-1])
    dl, de = torch.randn(tokens.shape, generator=g), torch.randn(tokens.shape, generator=g)
    grad = torch.autograd.grad([got.logprob, got.entropy], dev, [dl.to(DEV), de.to(DEV)])[0]
    with torch.no_grad():
        plain = run(dev, tokens.to(DEV), top_k=k)
    torch.cuda.synchronize()
    logprob, entropy, top, best, logp, p, given = reference(x, tokens, k)
    assert torch.equal(plain.logprob, got.logprob) and torch.equal(plain.entropy, got.entropy)
    x64 = x.double()
    M = x64.max(-1).values
    reach = torch.where(p > 0, (x64 - M[..., None]).abs(), torch.zeros_like(p))
    mean_reach = (p * reach).sum(-1)
    log_s = torch.log((p.max(-1).values.clamp(min=1e-300)) ** -1)

    def near(a, b, room, name):
        a, b = a.detach().double().cpu(), b.double()
        same = (a == b) | ((a - b).abs() <= room)
        assert bool(same.all()), f"{what} {name}: off by {float((a - b).abs().nan_to_num(nan=math.inf).max()):.3g}"
    size = torch.where(given, x64.gather(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None])[..., 0].abs().nan_to_num(posinf=0.0), torch.zeros_like(M))
    near(got.logprob, logprob, C * U + 2 * U * (size + M.abs().nan_to_num(posinf=0.0) + log_s), "logprob")
    near(got.entropy, entropy, C * U * (1 + entropy + mean_reach), "entropy")
    if k:
        assert torch.equal(got.top_token.cpu(), best), f"{what} top_token"
        near(got.top_logprob, top, C * U + 2 * U * (top.abs().nan_to_num(posinf=0.0) + 2 * M.abs().nan_to_num(posinf=0.0)[..., None] + log_s[..., None]), "top_logprob")
    else:
        assert got.top_token is None and got.top_logprob is None
    pull = torch.where(given, dl.double(), torch.zeros_like(logprob))
    finite = torch.where(p > 0, logp, torch.zeros_like(logp))
    inner = pull[..., None] + de.double()[..., None] * (finite + entropy[..., None])
    want = -p * inner
    left = (M > -math.inf).double()
    want.scatter_add_(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None], (pull * left)[..., None])
    spread = pull.abs()[..., None] + de.double().abs()[..., None] * (finite.abs() + entropy[..., None] + 1)
    room = p * spread * (C + 4 * reach) * U
    room = room + torch.zeros_like(p).scatter_(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None], (2 * U * pull.abs())[..., None])
    if dtype != torch.float32:
        room = room + torch.finfo(dtype).eps / 2 * want.abs()
    room = room + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
    near(grad, want, room, "gradient")


def logits(lead, V, dtype, seed, std=2.5):
    g = gen(seed)
    x = torch.randn(*lead, V, generator=g) * std
    tokens = torch.randint(0, V, lead, generator=g)
    x.scatter_add_(-1, tokens[..., None], 6 * torch.rand(*lead, 1, generator=g))
    return x.to(dtype), tokens


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 63, 5), (5, 64, 64), (4, 65, 1), (7, 513, 20), (64, 1000, 5), (2, 8193, 64),
                                      (3, 32000, 8), (3, 50021, 20), (1, 100003, 20), (2, 131072, 64), (600, 2050, 3), (1100, 37, 10)])
def test_sizes(hip_ops, rows, V, k, dtype):
    x, tokens = logits((rows,), V, dtype, rows + V)
    check(x, tokens, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,rows", [(1000, 4), (33000, 4), (200000, 4)])
def test_masks_and_tokens_that_are_not_given(hip_ops, dtype, V, rows):
    x, tokens = logits((rows,), V, dtype, V)
    x[:, torch.rand(V, generator=gen(3)) < 0.4] = -math.inf
    x[1] = -math.inf                                            # nothing is left
    x[2] = -math.inf
    x[2, [5, 700]] = torch.tensor([1.0, 2.0], dtype=dtype)      # two are: fewer than the alternatives asked for
    x[3] = torch.finfo(dtype).min                               # masked with the type's lowest value instead
    x[3, 17] = 3.0
    tokens[0] = -100
    tokens[-1] = V
    check(x, tokens, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_values_go_by_the_lower_index(hip_ops, dtype):
    for V, rows in ((1000, 3), (40000, 3), (140000, 2)):
        x = torch.zeros(rows, V, dtype=dtype)                   # all equal: more than can be ranked at once
        x[0, ::7] = 2.0
        x[1] = torch.randint(0, 5, (V,), generator=gen(V)).to(dtype)
        x[-1, 100] = -0.0
        check(x, torch.randint(0, V, (rows,), generator=gen(4)), 20, what=str(V))
    # one thread holds many of the largest
    x = torch.zeros(2, 65536, dtype=dtype)
    x[0, ::2048] = 5.0
    x[1, 8::8192] = torch.arange(8).to(dtype) + 1
    check(x, torch.tensor([0, 8]), 30)


FILLS = {"few": lambda x, g: x.masked_fill(torch.rand(x.shape, generator=g) >= 5.0 / x.shape[-1], -math.inf),
         "lowest": lambda x, g: x.masked_fill(torch.rand(x.shape, generator=g) >= 5.0 / x.shape[-1], torch.finfo(x.dtype).min),
         "neighbours": lambda x, g: torch.where((torch.arange(x.shape[-1]) >= 100) & (torch.arange(x.shape[-1]) < 290), x, torch.full_like(x, -math.inf)),
         "same": lambda x, g: torch.full_like(x, 1.5),
         "end": lambda x, g: torch.where(torch.arange(x.shape[-1]) < x.shape[-1] - 50, torch.full_like(x, -3.0), x.abs()),
         "signs": lambda x, g: torch.where(torch.rand(x.shape, generator=g) < 0.5, torch.zeros_like(x), -torch.zeros_like(x)),
         "first": lambda x, g: torch.where(torch.arange(x.shape[-1]) == 0, x, torch.full_like(x, -math.inf)),
         "last": lambda x, g: torch.where(torch.arange(x.shape[-1]) == x.shape[-1] - 1, x, torch.full_like(x, -math.inf)),
         "nan": lambda x, g: torch.full_like(x, -math.inf).masked_fill(torch.rand(x.shape, generator=g) < 0.9, math.nan)}


@pytest.mark.gpu
@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("rows,V", [(3, 70), (5, 300), (3, 1000), (2, 9001), (600, 5003), (2, 33000), (2, 150001)])
def test_alternatives_where_few_elements_count(hip_ops, rows, V, fill):
    """Masks that leave fewer than top_k, masks of the type's lowest value, rows of one value: the lower index first, NaN behind everything."""
    g = gen(31)
    for dtype in (torch.bfloat16, torch.float32):
        x = FILLS[fill](logits((rows,), V, dtype, 32)[0], g)
        order = torch.sort(torch.where(x.isnan(), torch.full_like(x.double(), -math.inf), x.double()), dim=-1, descending=True, stable=True).indices
        if fill == "nan":         # minus infinity first, then the others, each by the index
            order = torch.sort(x.isnan().double(), dim=-1, stable=True).indices
        for k in (1, 5, 20, 64):
            got = run(x.to(DEV), top_k=k)
            assert torch.equal(got.top_token.cpu(), order[:, :k]), (dtype, k)


@pytest.mark.gpu
def test_far_values(hip_ops):
    """Logits far from each other and far from 0: differences are what counts."""
    for dtype, top in ((torch.float32, 1e6), (torch.bfloat16, 1e6), (torch.float16, 3e4)):
        g = gen(6)
        x = (torch.randn(4, 3000, generator=g) + torch.tensor([top, -top, 0.0, 0.0])[:, None])
        x[2] *= 200.0
        check(x.to(dtype), torch.randint(0, 3000, (4,), generator=g), 5)


@pytest.mark.gpu
def test_nan_and_infinity(hip_ops):
    for V in (100, 70000):
        x, tokens = logits((4,), V, torch.float32, V)
        clean = run(x.to(DEV), tokens.to(DEV), top_k=5)
        dirty = x.clone()
        dirty[1, 3] = math.nan
        dirty[2, 4] = math.inf
        dirty[3] = math.nan
        got = run(dirty.to(DEV), tokens.to(DEV), top_k=5)
        assert torch.equal(got.logprob[0], clean.logprob[0]) and torch.equal(got.top_token[:2], clean.top_token[:2])
        assert bool(got.logprob[1:].isnan().all()) and bool(got.entropy[1:].isnan().all())
        assert int(got.top_token[2, 0]) == 4 and got.top_token[3].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.gpu
def test_shapes_strides_and_types_of_tokens(hip_ops):
    g = gen(8)
    wide = torch.randn(3, 5, 2051, generator=g).to(DEV, torch.bfloat16)
    x = wide[:, :, 1:1501]
    tokens = torch.randint(0, 1500, (3, 5), generator=g).to(DEV)
    a, b = run(x, tokens, top_k=4), run(x.contiguous(), tokens.int(), top_k=4)
    assert a.logprob.shape == (3, 5) and a.top_token.shape == (3, 5, 4)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    turned = run(x.transpose(0, 1), tokens.t(), top_k=4)
    assert torch.equal(turned.logprob, a.logprob.t()) and torch.equal(turned.top_token, a.top_token.transpose(0, 1))
    none = run(x, None, top_k=0)
    assert float(none.logprob.abs().max()) == 0.0 and torch.equal(none.entropy, a.entropy)
    one = run(x[0, 0], tokens[0, 0], top_k=2)
    assert one.logprob.shape == () and one.top_token.shape == (2,) and torch.equal(one.logprob, a.logprob[0, 0])
    # gradients of one of the two, and an expanded one
    leaf = x.contiguous().requires_grad_(True)
    for k in range(2):
        out = run(leaf, tokens)
        lone = torch.autograd.grad(out[k].sum(), leaf)[0]
        out = run(leaf, tokens)
        ones = [torch.zeros_like(out[0]), torch.zeros_like(out[0])]
        ones[k] += 1
        assert torch.equal(lone, torch.autograd.grad(out[:2], leaf, ones)[0])
    assert not run(leaf, tokens, top_k=3).top_logprob.requires_grad


@pytest.mark.gpu
def test_gradient_against_differences(hip_ops):
    """Central differences, float32, step 2^-6 along a random direction: truncation and rounding stay below 1e-2 of the terms' sizes."""
    x, tokens = logits((4,), 300, torch.float32, 9, std=1.0)
    leaf, tokens = x.to(DEV).requires_grad_(True), tokens.to(DEV)
    dl, de = torch.randn(4, generator=gen(1)).to(DEV), torch.randn(4, generator=gen(2)).to(DEV)
    grad = torch.autograd.grad(run(leaf, tokens)[:2], leaf, [dl, de])[0]
    way = torch.randn(4, 300, generator=gen(3)).to(DEV)

    def loss(step):
        out = run(leaf.detach() + step * way, tokens)
        return (out.logprob.double() * dl).sum() + (out.entropy.double() * de).sum()
    slope = (loss(2.0 ** -6) - loss(-2.0 ** -6)) * 32
    assert abs(float(slope - (grad.double() * way).sum())) <= 1e-2 * float((grad.double() * way).abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(40, 3000), (2, 150000)])
def test_graph_replays_and_other_streams(hip_ops, rows, V):
    x, tokens = logits((rows,), V, torch.bfloat16, 10)
    leaf, tokens = x.to(DEV).requires_grad_(True), tokens.to(DEV)
    ones = torch.ones(rows, device=DEV)

    def step():        # its autograd graph ends with it: none of the same leaves lives during a capture
        out = run(leaf, tokens, top_k=6)
        return [*(t.detach() for t in out), torch.autograd.grad(out[:2], leaf, [ones, ones])[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
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
            leaf.copy_(logits((rows,), V, torch.bfloat16, 20 + k)[0])
        want = [t.clone() for t in step()]
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_empty_and_refusals(hip_ops):
    x = torch.zeros(0, 8, device=DEV)
    out = run(x, torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert out.logprob.shape == (0,) and out.top_token.shape == (0, 2)
    x = torch.zeros(2, 8, device=DEV)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    for args, kwargs, words in (((x, t[:1]), {}, "unsupported_shape"), ((x.double(), t), {}, "unsupported_dtype"), ((x, t.float()), {}, "unsupported_dtype"),
                                ((x, t.cpu()), {}, "unsupported_device"), ((x, t), {"top_k": 9}, "unsupported_top_k"), ((x, t), {"top_k": -1}, "unsupported_top_k"),
                                ((torch.zeros(2, 100, device=DEV), t), {"top_k": 65}, "unsupported_top_k"), ((x[0, 0], None), {}, "unsupported_shape"),
                                ((torch.zeros(2, 0, device=DEV), t), {}, "unsupported_shape")):
        with pytest.raises(RuntimeError, match=words):
            run(*args, **kwargs)


@pytest.mark.gpu
def test_python_implementation(hip_ops, monkeypatch):
    """What the dispatch module does not take runs in Python, on the same kernels: the same checks with the module out of the way, and equal bits."""
    from triton_snn_fusion_amd import _dispatch
    from triton_snn_fusion_amd.runtime import hip_token_scores_backend as backend
    x, tokens = logits((5,), 3001, torch.bfloat16, 31)
    leaf, on_gpu, ones = x.to(DEV).requires_grad_(True), tokens.to(DEV), torch.ones(5, device=DEV)

    def step():
        out = run(leaf, on_gpu, top_k=6)
        return [*out, torch.autograd.grad(out[:2], leaf, [ones, ones])[0]]
    assert _dispatch.module().token_scores(leaf, on_gpu, 6)[0].grad_fn is not None
    dispatched = step()
    monkeypatch.setattr(backend, "native", lambda t: None)
    assert all(torch.equal(a, b) for a, b in zip(step(), dispatched))
    for dtype in DTYPES:
        check(*logits((3,), 1001, dtype, 32), 7)
        check(*logits((2,), 90000, dtype, 33), 0)
    test_empty_and_refusals(hip_ops)


@pytest.mark.gpu
def test_differentiated_once(hip_ops):
    x = torch.randn(3, 16, device=DEV, requires_grad=True)
    out = run(x).entropy.sum()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(out, x, create_graph=True)[0].sum(), x)


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="unsupported_device"):
        run(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="must be a tensor"):
        run(None)


def test_entry_points_refuse_before_any_gpu_work(snnf_lib):
    def forward(rows=2, V=8, dtype=0, k=0, logits=16, top=None, logprob=16):
        return snnf_lib.snnf_token_scores(logits, 8, rows, V, dtype, None, k, logprob, 16, top, top, None, None, 0, None)
    assert forward(rows=-1) == -1 and forward(V=0) == -1 and forward(k=-1) == -1 and forward(dtype=4) == -1 and forward(logits=None) == -1
    assert forward(k=9, top=16) == -2 and forward(V=100, k=65, top=16) == -2 and forward(k=2) == -1 and forward(logprob=None) == -1
    assert forward(rows=0, logits=None) == 0
    assert snnf_lib.snnf_token_scores_workspace_bytes(1, 1 << 20, 4) > 0 and forward(rows=1, V=1 << 20, k=4, top=16) == -4
    assert snnf_lib.snnf_token_scores_workspace_bytes(0, 8, 0) == 0
    assert snnf_lib.snnf_token_scores_backward(16, 8, 2, 8, 0, None, None, 16, None, None, 16, None) == -1
    assert snnf_lib.snnf_token_scores_backward(16, 8, 2, 8, 7, None, 16, 16, None, None, 16, None) == -1
