"""Verdicts and draws that are close, on rows whose shares and sums float32 rounds the same way again and again: equal tails, slopes of many small steps, near-flat rows in many pieces. Against
float64 on the CPU, on the same numbers; the uniforms lie 2^-20 to 2^-16 of a share around it, where float64 leaves no doubt."""
import math

import pytest
import torch

from helpers import DEV, gen
from test_gpu_draft_verification import run


def verdicts(row, token, temperature=1.0, requests=1200):
    """`requests` at a time (many: a workgroup to a row; few: a row in pieces) with uniforms around the token's share."""
    V = row.numel()
    wide = row.double() / temperature
    p = float(torch.exp(wide[token] - wide.max()) / torch.exp(wide - wide.max()).sum())
    offsets = torch.cat([s * torch.logspace(-20, -16, 600, base=2.0, dtype=torch.float64) for s in (-1.0, 1.0)])
    uniforms = (p * (1.0 + offsets)).float()
    want = uniforms.double() < p
    on, noise = row.to(DEV), torch.ones(1, V, device=DEV)
    for at in range(0, len(uniforms), requests):
        u = uniforms[at:at + requests]
        n = len(u)
        got = run(on.expand(n, 2, V), torch.full((n, 1), token, device=DEV), u[:, None].to(DEV), noise.expand(n, V), temperature=temperature)
        assert torch.equal(got.accepted.cpu().bool(), want[at:at + requests]), (got.accepted.cpu().bool() != want[at:at + requests]).nonzero().flatten()[:8]


def tails(V, dtype, g):
    """A maximum over equal rest, which together weighs a half to twice as much."""
    for _ in range(3):
        row = torch.full((V,), -math.log(V) + float(torch.rand((), generator=g)) * 1.4 - 0.7).to(dtype)
        row[V // 3] = 0.0
        yield row


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1200, 100])
@pytest.mark.parametrize("temperature", [1.0, 0.7000000476837158, 1.2999999523162842])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [32000, 131072, 1 << 20])
def test_equal_tails(hip_ops, V, dtype, temperature, requests):
    for row in tails(V, dtype, gen(V)):
        verdicts((row.float() * temperature).to(dtype), V // 3, temperature, requests)


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1200, 100])
@pytest.mark.parametrize("step", [2.0 ** -11, 3e-4, 1e-3, 0.01, 0.3])
@pytest.mark.parametrize("V", [50000, 1 << 20])
def test_logits_that_rise(hip_ops, V, step, requests):
    """Each round of a workgroup sees a new maximum; with falling ones, none."""
    for each in (1024, 2048, 4096):
        row = (torch.arange(V) // each).float() * step
        verdicts(row, V - 1, requests=requests)
        verdicts(row.flip(0).contiguous(), 0, requests=requests)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(1, 1 << 18), (1, 300001), (12, 131072)])
def test_draws_beside_a_draft_of_nearly_the_same(hip_ops, N, V, dtype):
    """Near-flat rows, with residuals down to 2^-15 of the shares."""
    for seed in range(6):
        g = gen(100 * seed + N)
        logits = (torch.randn(N, 2, V, generator=g) * 2.0 ** -(2 * seed)).to(dtype).to(DEV)
        theirs = (logits[:, :1].float() + 2.0 ** -(4 + 2 * seed) * torch.randn(N, 1, V, generator=g).to(DEV)).to(dtype)
        drafts, noise = torch.randint(0, V, (N, 1), generator=g).to(DEV), torch.empty(N, V).exponential_(generator=g).to(DEV)
        p, q = torch.softmax(logits[:, 0].double(), -1), torch.softmax(theirs[:, 0].double(), -1)
        # turned down wherever q is the larger; else the draw is from the second row
        uniforms = torch.full((N, 1), 1.0 - 2.0 ** -24, device=DEV)
        stands = uniforms[:, 0].double() * q.gather(1, drafts)[:, 0] < p.gather(1, drafts)[:, 0]
        r = torch.where(stands[:, None], torch.softmax(logits[:, 1].double(), -1), (p - q).clamp(min=0))
        got = run(logits, drafts, uniforms, noise, draft_logits=theirs)
        assert torch.equal(got.accepted.bool(), stands)
        assert torch.equal(got.tokens.gather(1, stands.long()[:, None])[:, 0], (r / noise.double()).argmax(1))


@pytest.mark.gpu
def test_shares_that_vanish_in_float32(hip_ops):
    """Drafts of 2^-150 to 2^-900 in both distributions, a factor of 2^-4 to 2^4 apart: verdicts by float64."""
    V, N = 3000, 60
    logits, theirs = torch.randn(N, 2, V, generator=gen(1)), torch.randn(N, 1, V, generator=gen(2))
    at = torch.linspace(-610.0, -100.0, N)
    logits[:, 0, 7], theirs[:, 0, 7] = at, at + torch.rand(N, generator=gen(3)) * 4 - 2
    p, q = torch.softmax(logits[:, 0].double(), -1)[:, 7], torch.softmax(theirs[:, 0].double(), -1)[:, 7]
    uniforms = torch.rand(N, 1, generator=gen(4))
    want = uniforms[:, 0].double() * q < p
    got = run(logits.to(DEV), torch.full((N, 1), 7, device=DEV), uniforms.to(DEV), torch.ones(N, V, device=DEV), draft_logits=theirs.to(DEV))
    assert 10 < int(want.sum()) < 50 and torch.equal(got.accepted.cpu().bool(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logits_of_any_size(hip_ops, dtype):
    """The type's lowest value as a mask, rows of nothing else, the largest values, and a large number beside which float32 has no small differences."""
    V, low, high = 5000, torch.finfo(dtype).min, torch.finfo(dtype).max
    logits = torch.randn(9, 2, V, generator=gen(5)).to(dtype)
    logits[0, :, 10:], logits[1], logits[2], logits[3, :, 3:9] = low, low, high, high
    logits[4], logits[5, :, ::2] = (logits[4].float() + 50000).to(dtype), high
    logits[6, 0, 9], logits[7, 0], logits[8, 1] = math.nan, math.inf, -math.inf
    drafts, uniforms, noise = torch.full((9, 1), 4), torch.full((9, 1), 1.0 - 2.0 ** -24), torch.empty(9, V).exponential_(generator=gen(6))
    uniforms[8] = 0.0
    got = run(logits.to(DEV), drafts.to(DEV), uniforms.to(DEV), noise.to(DEV))
    r = torch.softmax(logits[:, 0].double(), -1)
    r[:, 4] = 0.0
    assert got.accepted[:8].tolist() == [0] * 8 and torch.equal(got.tokens[:6, 0].cpu(), (r / noise.double())[:6].argmax(1))
    assert got.tokens[6:].tolist() == [[-100] * 2] * 2 + [[4, -100]]


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1.0, 2.0 ** -10])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_around_the_largest_that_float32_takes(hip_ops, sign, temperature):
    """2^22 powers of two, where rows are left to float64: numbers on both sides of it weigh as they are."""
    V, N = 6000, 40
    g = gen(8)
    logits = (sign * 2.0 ** 22 * math.log(2.0) + torch.cat([torch.linspace(-10.0, 10.0, N - 8), torch.linspace(-1200.0, 1200.0, 8)])[:, None, None] + torch.randn(N, 2, V, generator=g) * 2).mul(temperature).float()
    drafts, uniforms, noise = torch.randint(0, V, (N, 1), generator=g), torch.rand(N, 1, generator=g) * 2e-4, torch.empty(N, V).exponential_(generator=g)
    p = torch.softmax(logits.double() / temperature, -1)
    want = (uniforms.double() < p[:, 0].gather(1, drafts))[:, 0]
    r = torch.where(want[:, None], p[:, 1], p[:, 0].scatter(1, drafts, 0.0))
    got = run(logits.to(DEV), drafts.to(DEV), uniforms.to(DEV), noise.to(DEV), temperature=temperature)
    assert 5 < int(want.sum()) < 35 and torch.equal(got.accepted.cpu().bool(), want)
    assert torch.equal(got.tokens.cpu().gather(1, want.long()[:, None])[:, 0], (r / noise.double()).argmax(1))
