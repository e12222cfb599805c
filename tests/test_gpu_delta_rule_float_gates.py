"""Gradients of float32 gates beside heads of 16 bits: they are float32's own, though heads' products are of bfloat16 terms.

Tolerance, of the root mean square of the error relative to that of the gradient. Three terms leave 2^-24 of a product, as float32 does. A gate's gradient sums over the steps of a chunk what a
step's queries, keys, values and corrections give, each some 16 roundings of u = 2^-24 off by its products, decays and the inverse; over at most 64 steps and with signs at random those are 8 times 16 / 2: 64 u.
Two terms (2^-17, 128 u a product) do not pass, nor do decays whose logarithm is rounded to float32 at sums of 64 gates."""
import pytest
import torch

from helpers import DEV, gen
from test_gpu_delta_rule import NAMES, U, check, operands, reference, run


def errors(shape, dtype, seed, starts=None, lengths=None):
    leaves, dout, dlast = operands(*shape, dtype, seed, torch.float32)
    want, _ = reference(*leaves, shape[4] ** -0.5, starts, lengths, dout, dlast)
    leaves = [t.requires_grad_(True) for t in leaves]
    out, last = run(*leaves, starts=None if starts is None else starts.to(DEV), lengths=None if lengths is None else lengths.to(DEV))
    grads = torch.autograd.grad([out, last], leaves, [dout, dlast])
    rms = lambda t: float((t.double() ** 2).mean().sqrt())
    return {name: rms(got.double().cpu() - to) / rms(to) for name, got, to in zip(NAMES[5:7], grads[3:5], want[5:7])}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(100, 2, 1, 2, 64, 64), (512, 1, 1, 1, 128, 128), (300, 3, 2, 4, 33, 70), (70, 130, 1, 1, 24, 48), (66, 260, 1, 1, 72, 72), (1300, 1, 1, 2, 96, 40), (1250, 2, 1, 1, 128, 128)])
def test_are_as_exact_as_float32(hip_ops, shape, dtype):
    found = errors(shape, dtype, 600 + shape[0])
    print(found, flush=True)
    assert max(found.values()) <= 64 * U, found


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [90, 1200])
def test_with_starts_and_lengths(hip_ops, T, dtype):
    N = 4
    lengths, starts = torch.tensor([T, T // 2, 0, T - 1], dtype=torch.int32), torch.rand(T, N, generator=gen(T)) < 0.01
    found = errors((T, N, 1, 2, 64, 64), dtype, 700 + T, starts, lengths)
    print(found, flush=True)
    assert max(found.values()) <= 64 * U, found


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(70, 2, 1, 2, 64, 64), (130, 1, 2, 2, 128, 128), (1200, 1, 1, 2, 40, 24), (66, 256, 1, 1, 24, 24)])
def test_everything_else_beside_them(hip_ops, shape, dtype):
    check(shape, dtype, 800 + shape[0], gates=torch.float32)
    check(shape, dtype, 810 + shape[0], gates=torch.float32, batch_first=True, without=(3,))
    check(shape, dtype, 820 + shape[0], gates=torch.float32, without=(4, 5))
