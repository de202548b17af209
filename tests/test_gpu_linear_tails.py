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
