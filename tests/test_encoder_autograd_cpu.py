"""CPU: what the differentiable forms of the encoder's operators ask of the kernels and keep (the kernels stand in as plain
torch operations: these tests are about the autograd logic around them)."""
import pytest
import torch

from two_towers_overlords_amd import encoder, ops


@pytest.fixture
def linear_calls(monkeypatch):
    calls = []

    def linear_act(x, w, bias=None, residual=None, activation="none", save_preact=False, out=None):
        calls.append(save_preact)
        z = x @ w.t() + (0 if bias is None else bias)
        y = torch.relu(z) + (0 if residual is None else residual)
        return (y, z) if save_preact else y

    monkeypatch.setattr(ops, "linear_act", linear_act)
    return calls


def test_linear_keeps_a_pre_activation_only_for_a_backward_pass(linear_calls):
    x, w, b = torch.randn(5, 4), torch.randn(3, 4, requires_grad=True), torch.randn(3, requires_grad=True)
    r = torch.randn(5, 3, requires_grad=True)
    with torch.no_grad():
        y = encoder.linear(x, w, b, activation="relu")
    assert linear_calls == [False] and not y.requires_grad
    assert encoder.linear(x, w, b, activation="relu").requires_grad and linear_calls[-1]
    assert encoder.linear(x, w.detach(), None, r, "relu").requires_grad and not linear_calls[-1]  # the residual's gradient is dy
    with torch.inference_mode():
        encoder.linear(x, w, b, activation="relu")
    assert not linear_calls[-1]
