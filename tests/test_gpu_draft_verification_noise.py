"""The draw of the verification of drafted tokens over noise that is not exponential: the argmax of r / noise is taken as it is written, an entry of r = 0 having 0 whatever its noise is,
and one of r > 0 over noise that is NaN being left out. Against the definition in float64 on the CPU; answers are whole numbers and have to be equal."""
import math

import pytest
import torch

from helpers import DEV, gen
from test_gpu_draft_verification import DTYPES, operands, run


def reference(logits, drafts, uniforms, noise, draft_logits=None, temperature=1.0):
    logits, drafts, uniforms, noise = logits.double().cpu(), drafts.cpu(), uniforms.double().cpu(), noise.double().cpu()
    N, K = drafts.shape
    V = logits.shape[2]
    each = temperature.double().cpu() if isinstance(temperature, torch.Tensor) else torch.full((N,), float(temperature), dtype=torch.float64)
    tokens, accepted = torch.full((N, K + 1), -100, dtype=torch.int64), torch.zeros(N, dtype=torch.int32)
    for n in range(N):
        t = float(each[n])
        share = lambda row: torch.softmax(row / t, 0) if t > 0 else (torch.arange(V) == int(row.argmax())).double()
        j = 0
        while True:
            r = p = share(logits[n, j])
            if j == K:
                break
            x = int(drafts[n, j])
            q = (torch.arange(V) == x).double() if draft_logits is None or not t > 0 else share(draft_logits[n, j].double().cpu())
            if not float(uniforms[n, j]) * float(q[x]) < float(p[x]):
                r = (p - q).clamp(min=0)
                r = r if bool((r > 0).any()) else p
                break
            tokens[n, j] = x
            j += 1
        accepted[n] = j
        value = torch.where(r > 0, r / noise[n], 0.0)
        tokens[n, j] = int((value == value.nan_to_num(-math.inf, math.inf, -math.inf).max()).nonzero()[0]) if not bool(value.isnan().all()) else -100
    return tokens, accepted


def check(args, **options):
    want = reference(*args, **options)
    got = run(*args, **options)
    torch.cuda.synchronize()
    assert torch.equal(got.accepted.cpu(), want[1]), (got.accepted, want[1])
    assert torch.equal(got.tokens.cpu(), want[0]), (got.tokens, want[0])


def noises(N, V, g):
    e = torch.empty(N, V).exponential_(generator=g).clamp(min=1e-9)
    at = lambda share: torch.rand(N, V, generator=g) < share
    yield "one number below 0", torch.full((N, V), -1e-12)
    yield "below 0", -e
    yield "both signs", torch.where(at(0.5), e, -e)
    yield "few above 0", torch.where(at(2.0 / V), e, -e)
    yield "zeros", torch.where(at(1.0 / V), 0.0, e)
    yield "zeros of both signs", torch.where(at(0.5), 0.0, -0.0)
    yield "infinities", torch.where(at(0.5), math.inf, -e)
    yield "NaN", torch.where(at(0.3), math.nan, torch.where(at(0.5), e, -e))
    yield "subnormal", e * 2.0 ** -135
    yield "next to the largest", e.clamp(max=10.0) * 2.0 ** 124


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 300, 9001, 70000])
def test_noise_that_is_not_exponential(hip_ops, V, dtype, draft):
    N = 6
    for i, (what, noise) in enumerate(noises(N, V, gen(V))):
        for temperature in (0.8, 0.0):
            args, theirs = operands(N, 2, V, dtype, 70 + i, draft)
            args[3] = noise.to(DEV)
            print(what, temperature, flush=True)
            check(args, draft_logits=theirs, temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3, 5000, 40000])
def test_masked_entries_over_noise_below_zero(hip_ops, V, dtype):
    """Of entries of r = 0, masked ones and a draft that was turned down among them, the lowest index; entries whose shares are too small for float32 have more than 0."""
    args, theirs = operands(8, 1, V, dtype, 81)
    args[2][:] = 1.0 - 2.0 ** -24
    masked = torch.rand(8, 1, V, generator=gen(1)) < 0.05
    masked[:, :, 0] = False
    masked[:, :, 1] = True
    args[0][masked.expand(8, 2, V).to(DEV)] = -math.inf
    args[0][4:, :, 0], theirs[4:, :, 0] = -90.0, -math.inf
    args[1][:] = 2
    args[3] = -args[3]
    for options in ({"draft_logits": theirs}, {}):
        check(args, **options)
        check(args, temperature=0.9, **options)


@pytest.mark.gpu
def test_a_draft_distribution_of_which_nothing_is_left(hip_ops):
    """Masked whole, or not finite: its draft does not stand, and the token comes from the target alone."""
    args, theirs = operands(6, 1, 3000, torch.float32, 91)
    theirs[0], theirs[1, 0, 5], theirs[2, 0, 7], theirs[3] = -math.inf, math.nan, math.inf, math.nan
    got = run(*args, draft_logits=theirs)
    p = torch.softmax(args[0][:4, 0].double(), -1) / args[3][:4].double()
    assert got.accepted[:4].tolist() == [0] * 4 and torch.equal(got.tokens[:4, 0], p.argmax(-1))
