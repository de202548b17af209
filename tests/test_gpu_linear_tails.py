"""GPU: linear_act's activations where their values are small: the error is relative to the value, not to 1."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def values_and_slopes(act, z):
    """act(z) and act'(z) in 64 bits without cancellation, the sum of the slope's terms' magnitudes, and what the slope multiplies
    the exponential's factor (the density, or the logistic function) by."""
    if act == "gelu":
        cdf, pdf = torch.erfc(-z / math.sqrt(2.0)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, cdf + z.abs() * pdf, 1 + z.abs()
    u = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    du = torch.ones_like(z) if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s, r = torch.sigmoid(u), torch.sigmoid(-u)
    return z * s, s + z * s * r * du, s + z.abs() * s * r * du, 1 + z.abs() * du


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [50, 4000])
def test_small_values_are_good_to_the_types_rounding(dt, act, rows):
    """K = 1 and a weight of 1: z is the input itself.  rows: the form for few rows and the tiled one.

    Beside the result's own rounding (u, or half a subnormal step): the exponential's argument is at most 123 (e^-85 = 2^-123) and
    carries three roundings of 2^-24: 123 ln 2 * 3 * 2^-24 = 1.6e-5 relative; the 16-bit error function is fitted to 1e-5 more,
    and ten further operations of 2^-23 are 1.2e-6: 2^-15 in all.  Values below float's normal range may be flushed to 0, the exponential's factor too, before it is
    multiplied by |z| (the value) or by 1 + |z| u'(z) (the slope: up to 265 for gelu_tanh, whose factor leaves the range at -10.3)."""
    from two_towers_overlords_amd import ops

    z = torch.cat([-torch.logspace(-3, math.log10(13), rows - rows // 4), torch.logspace(-3, math.log10(13), rows // 4)])
    z = z.to(dt).cuda().unsqueeze(1)
    # columns enough that the second form is the tiled one; every column is the same
    w = torch.ones(24 if rows < 100 else 160, 1, dtype=dt, device="cuda")
    y, kept = ops.linear_act(z, w, None, None, act, save_preact=True)
    assert torch.equal(kept, z.expand_as(kept))
    Y, D, mag, times = values_and_slopes(act, z.double())
    info = torch.finfo(dt)
    u, floor = info.eps / 2, info.smallest_normal * info.eps / 2 + 2.0 ** -126
    rel = 2.0 ** -15
    worst = ((y.double() - Y).abs() - ((u + (1 + u) * rel) * Y.abs() + floor + z.double().abs() * 2.0 ** -126)).max()
    assert float(worst) <= 0
    one = torch.ones(1, 1, dtype=dt, device="cuda")
    dz, _, _ = ops.linear_act_bwd(torch.ones_like(z), z, one, z, act)  # = act'(z)
    worst = ((dz.double() - D).abs() - (u * D.abs() + (1 + u) * rel * mag + floor + times * 2.0 ** -126)).max()
    assert float(worst) <= 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("odd", [False, True])
def test_each_gradient_alone_in_the_workspace_that_it_asks_for(dt, act, odd):
    """The C entry with dx, dw and dbias in every combination: the same bits as together, nothing written behind the workspace."""
    import two_towers_overlords_amd as pkg
    from two_towers_overlords_amd import _lib, ops

    lib = pkg.load()
    code = {torch.float32: _lib.TT_F32, torch.bfloat16: _lib.TT_BF16, torch.float16: _lib.TT_F16}[dt]
    M, N, K = 3001, 72, 40 + odd
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w, dy = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((M, K), (N, K), (M, N)))
    _, z = ops.linear_act(x, w, None, None, act, save_preact=True)
    want = ops.linear_act_bwd(dy, x, w, z, act)
    for need in range(1, 8):
        outs = [torch.empty_like(t) if need >> i & 1 else None for i, t in enumerate(want)]
        ptr = [None if o is None else o.data_ptr() for o in outs]
        n = lib.tt_linear_act_bwd_workspace_bytes(dy.data_ptr(), N, x.data_ptr() if need & 2 else None, K, w.data_ptr() if need & 1 else None, K,
                                                  M, N, K, code, _lib.ACTIVATIONS[act])
        ws = torch.full((n + 4096,), 77, dtype=torch.uint8, device="cuda")
        rc = lib.tt_linear_act_bwd(dy.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, None if z is None else z.data_ptr(), *ptr, M, N, K, code,
                                   _lib.ACTIVATIONS[act], ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert bool((ws[n:] == 77).all())
        assert all(o is None or torch.equal(o, t) for o, t in zip(outs, want))
