"""RecurrentStack.step refuses before any layer's state has moved on: layers without a step (GRU has none), too few
states."""
import pytest
import torch
import torch.nn as nn

from rnn_kernel_b200 import GRU, RecurrentStack


class Counter(nn.Module):
    """A layer whose state counts its tokens, in place."""

    def step(self, x, state):
        state += 1
        return x


@pytest.fixture
def plain_norms(monkeypatch):
    monkeypatch.setattr("rnn_kernel_b200.norm.layer_norm", lambda x, w, b, eps, residual: x if residual is None else (x, x + residual))


def stack(*layers):
    return RecurrentStack(layers, 8)


def test_steps_move_every_state(plain_norms):
    states = [torch.zeros(()), torch.zeros(())]
    stack(Counter(), Counter()).step(torch.zeros(2, 8), states)
    assert states == [1, 1]


@pytest.mark.parametrize("where", [0, 1, 2])
def test_a_layer_without_a_step(plain_norms, where):
    layers = [Counter(), Counter()]
    layers.insert(where, GRU(8, 8))
    states = [torch.zeros(()) for _ in layers]
    with pytest.raises(RuntimeError, match="GRU has no step"):
        stack(*layers).step(torch.zeros(2, 8), states)
    assert states == [0, 0, 0]


@pytest.mark.parametrize("given", [0, 1])
def test_too_few_states(plain_norms, given):
    states = [torch.zeros(()) for _ in range(given)]
    with pytest.raises(ValueError, match="2 states"):
        stack(Counter(), Counter()).step(torch.zeros(2, 8), states)
    assert states == [0] * given
