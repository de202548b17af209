"""CPU: the rows that InBatchSoftmaxLoss hands to the kernel (which stands in as a plain torch operation)."""
import pytest
import torch

from two_towers_overlords_amd import model


@pytest.fixture
def seen(monkeypatch):
    seen = []

    def softmax_loss(x, candidates, target, *, scale=1.0, row_ids=None, cand_ids=None, ignore_index=-100):
        seen.append((x.detach(), candidates.detach()))
        return torch.logsumexp(x.float() @ candidates.float().t() * scale, 1) - scale * (x.float() * candidates[target].float()).sum(1)

    monkeypatch.setattr(model, "softmax_loss", softmax_loss)
    return seen


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_zero_rows_and_long_rows_are_normalised_in_every_type(seen, dt):
    q = torch.randn(5, 8).to(dt)
    q[1] = 0
    q[2] = 30000.0  # its square is beyond fp16
    loss = model.InBatchSoftmaxLoss()(q, torch.randn(5, 8).to(dt))
    (x, w), = seen
    assert x.dtype == w.dtype == dt and bool(torch.isfinite(loss)) and bool((x[1] == 0).all())
    norms = x.float().norm(dim=1)
    # every entry is rounded once, so the norm is off by at most that
    assert bool(((norms[[0, 2, 3, 4]] - 1).abs() <= torch.finfo(dt).eps / 2 + 8 * 2.0 ** -24).all())


def test_rows_of_a_transposed_matrix_are_taken(seen):
    q, d = torch.randn(8, 5).t(), torch.randn(5, 8)
    model.InBatchSoftmaxLoss()(q, d)
    assert all(t.is_contiguous() for t in seen[0])
