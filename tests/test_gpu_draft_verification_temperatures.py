"""Verification of drafted tokens at the ends of what a temperature may be, against the definition in float64 on the CPU: whole numbers, which have to be equal."""
import math

import pytest
import torch

from helpers import DEV
from test_gpu_draft_verification import DTYPES, operands, run
from test_gpu_draft_verification_noise import reference


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [3, 3000, 70000])
@pytest.mark.parametrize("temperature", [2.0 ** -149, 1e-39, 4e-39, 1.2e-38, 1e-31, 1e-29, 1e-10, 1e10, 1e29, 1e31, 3e38])
def test_very_low_and_very_high_ones(hip_ops, V, dtype, draft, temperature):
    args, theirs = operands(6, 2, V, dtype, 31, draft)
    args[0][:, :, 1] = -math.inf
    if draft:
        theirs[:, :, 2] = -math.inf
    each = torch.full((6,), temperature)
    want = reference(*args, draft_logits=theirs, temperature=each)
    got = run(*args, draft_logits=theirs, temperature=each.to(DEV))
    assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])
    got = run(*args, draft_logits=theirs, temperature=float(each[0]))
    assert torch.equal(got.tokens.cpu(), want[0]) and torch.equal(got.accepted.cpu(), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [4, 3000, 70000])
def test_an_infinite_one(hip_ops, V, dtype):
    """What is not masked is equal: the largest of 1 / noise is drawn, with the first draft turned down (uniform 1 - 2^-24, masked in the target) or standing (uniform 0)."""
    args, _ = operands(4, 1, V, dtype, 41)
    args[0][:, :, 1] = -math.inf
    args[1][:], args[2][:] = 1, 1.0 - 2.0 ** -24
    args[1][2:], args[2][2:] = 2, 0.0
    for temperature in (math.inf, torch.full((4,), math.inf, device=DEV)):
        got = run(*args, temperature=temperature)
        shares = (args[0][:, 0] > -math.inf).double() / args[3].double()
        assert got.accepted.tolist() == [0, 0, 1, 1] and torch.equal(got.tokens[:2, 0], shares.argmax(1)[:2]) and torch.equal(got.tokens[2:, 1], shares.argmax(1)[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-42, math.inf])
def test_rows_of_which_nothing_is_left(hip_ops, temperature):
    args, theirs = operands(5, 2, 2500, torch.float32, 51)
    args[0][0, 0], args[0][1, 0, 9], args[0][2, 0, 9], theirs[3, 0] = -math.inf, math.nan, math.inf, -math.inf
    got = run(*args, draft_logits=theirs, temperature=temperature)
    assert got.accepted[:4].tolist() == [0] * 4 and got.tokens[:3].tolist() == [[-100] * 3] * 3 and int(got.tokens[3, 0]) >= 0
