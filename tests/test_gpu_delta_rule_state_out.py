"""A state that is written in place is a write that autograd sees, from the dispatch module and from Python."""
import pytest
import torch

from helpers import DEV, gen
from test_gpu_delta_and_drafts import run_delta, without_module


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("T", [0, 3, 70])
def test_a_graph_that_kept_the_state_notices(hip_ops, monkeypatch, T, python):
    if python:
        without_module(monkeypatch)
    x = torch.randn(T, 2, 1, 8, generator=gen(1)).to(DEV)
    state, weight = torch.randn(2, 1, 8, 8, generator=gen(2)).to(DEV), torch.ones(8, device=DEV, requires_grad=True)
    for given in (state, state.clone()):
        loss, version = (weight * state).sum(), state._version
        run_delta(x, x, x, state=given, state_out=state)
        assert state._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    other = torch.empty_like(state)
    loss = (weight * state).sum()
    run_delta(x, x, x, state=state, state_out=other)
    loss.backward()
    assert torch.equal(weight.grad, state.sum((0, 1, 2)))


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True])
def test_states_of_inference_mode(hip_ops, monkeypatch, python):
    if python:
        without_module(monkeypatch)
    x = torch.randn(3, 2, 1, 8, generator=gen(1)).to(DEV)
    with torch.inference_mode():
        state = torch.zeros(2, 1, 8, 8, device=DEV)
        want = run_delta(x, x, x, state=state)[1]
        run_delta(x, x, x, state=state, state_out=state)
    assert torch.equal(state, want)
    with torch.inference_mode():
        again = run_delta(x, x, x, state=state)[1]
    with torch.no_grad():
        run_delta(x, x, x, state=state, state_out=state)
    assert torch.equal(state, again)
