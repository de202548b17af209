"""GPU: packed_attention with caps far below and above the scores, rows whose scores are all 0 among them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap", [1e-15, 1e-7, 1e-6, 1e-4, 1.0, 1e6, 1e15])
def test_any_cap_gives_finite_results(dt, cap):
    from two_towers_overlords_amd import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    n, Dh = 70, 32
    q, k, v, do = (torch.randn(n, 1, Dh, generator=g, device="cuda").to(dt) for _ in range(4))
    q[:32] = 0  # the first wave's scores are all 0
    q[40] = 0
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    o, lse = ops.packed_attention(q, k, v, cu, softcap=cap)
    grads = ops.packed_attention_bwd(do, q, k, v, o, lse, cu, softcap=cap)
    s = cap * torch.tanh(q[:, 0].double() @ k[:, 0].double().t() / math.sqrt(Dh) / cap)
    want = torch.softmax(s, 1) @ v[:, 0].double()
    u, E = torch.finfo(dt).eps / 2, 2.0 ** -23
    # a score is at most 8 here and off by (32 + 8) E of it (or of the cap, if that is smaller); 70 terms; P and o are rounded
    top = min(cap, float(s.abs().max()) + 1)
    tol = (2 * (32 + 16) * E * top + 2 * u + (n + 16) * E) * (torch.softmax(s, 1) @ v[:, 0].double().abs()) + 2 * torch.finfo(dt).smallest_normal * u
    assert bool(((o[:, 0].double() - want).abs() <= tol).all())
    assert all(bool(torch.isfinite(t).all()) for t in grads)
