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


@pytest.fixture
def attention_calls(monkeypatch):
    monkeypatch.setattr(ops, "packed_attention", lambda q, k, v, cu, **kw: (q * 1, q[:, :, 0].t().contiguous()))
    seen = []

    def bwd(dout, q, k, v, out, lse, cu, grads=None, **kw):
        seen.append(kw)
        grads = [torch.empty_like(t) for t in (q, k, v)] if grads is None else grads
        for t in grads:
            t.fill_(1.0)
        return tuple(grads)

    monkeypatch.setattr(ops, "packed_attention_bwd", bwd)
    return seen


def both(q, k, v, cu, **kw):
    yield lambda: encoder.attention(q, k, v, cu, **kw), q
    qkv = torch.cat([q, k, v], 1).detach().requires_grad_(True)
    yield lambda: encoder.attention_qkv(qkv, q.shape[1], cu, **kw), qkv


@pytest.mark.parametrize("name", ["key_mask", "prefix", "slopes", "cu"])
def test_a_mask_changed_before_the_backward_pass_is_noticed(attention_calls, name):
    """The gradients are formed again from the masks: ones changed in place in between would silently give others."""
    q, k, v = (torch.randn(6, 2, 8, requires_grad=True) for _ in range(3))
    cu = torch.tensor([0, 6], dtype=torch.int32)
    given = dict(key_mask=torch.ones(6, dtype=torch.bool), prefix=torch.zeros(1, dtype=torch.int32), slopes=torch.rand(2))
    for run, leaf in both(q, k, v, cu, **given):
        run().sum().backward()
        assert leaf.grad is not None and all(attention_calls[-1][n] is not None for n in given)
        out = run()
        (cu if name == "cu" else given[name]).zero_()
        with pytest.raises(RuntimeError, match="inplace"):
            out.sum().backward()


def test_slopes_that_want_a_gradient_are_refused(attention_calls):
    q, k, v = (torch.randn(6, 2, 8, requires_grad=True) for _ in range(3))
    slopes = torch.rand(2, requires_grad=True)
    for run, _ in both(q, k, v, torch.tensor([0, 6], dtype=torch.int32), slopes=slopes):
        with pytest.raises(ValueError, match="no gradient"):
            run()
        with torch.no_grad():
            run()
