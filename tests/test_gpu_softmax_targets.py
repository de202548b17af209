"""GPU: gradients of softmax_loss where many targets are likely (p > 1/4: the target's entry is minus the sum of the row's
others), over tile shapes whose last tile ends far behind the last candidate, and whatever the workspace held before the call.

Tolerances as in test_gpu_encoder_ops: u = half a step of the type, E = 2^-23 per fp32 result and term of a sum, F = 8 units
for the exponentials; elementwise bounds evaluated in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -23
F = 8
HALF = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def lib():
    import two_towers_overlords_amd as pkg

    return pkg.load()


def rows_near_targets(dt, N, V, D, groups=False):
    """Unit rows, scale 20: a row is its target plus noise that grows along the rows, so p falls from nearly 1 to nearly 0."""
    g = torch.Generator(device="cuda").manual_seed(N + 3 * V + 5 * D)
    w = torch.randn(V, D, generator=g, device="cuda")
    w /= w.norm(dim=1, keepdim=True)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[-1] = V - 1
    x = w[t] + torch.linspace(0.0, 2.0, N, device="cuda")[:, None] * torch.randn(N, D, generator=g, device="cuda") * D ** -0.5
    x /= x.norm(dim=1, keepdim=True)
    t[5::50] = -100
    cid = torch.randint(0, max(1, V // 2), (V,), generator=g, device="cuda") if groups else None
    rid = cid[t.clamp(min=0)] if groups else None
    c = (torch.rand(N, generator=g, device="cuda") + 0.1) / N
    return x.to(dt), w.to(dt), t, rid, cid, c


def gradients(lib, fill, c, x, w, t, lse, scale, rid, cid):
    """tt_softmax_loss_bwd in a workspace that holds `fill` everywhere."""
    from two_towers_overlords_amd import _lib

    N, D = x.shape
    V = w.shape[0]
    dt = {torch.float32: _lib.TT_F32, torch.bfloat16: _lib.TT_BF16, torch.float16: _lib.TT_F16}[x.dtype]
    n = lib.tt_softmax_loss_bwd_workspace_bytes(x.data_ptr(), D, w.data_ptr(), D, N, V, D, dt)
    ws = torch.full((n // 4 + 4,), fill, dtype=torch.float32, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ptr = lambda a: None if a is None else a.data_ptr()
    rc = lib.tt_softmax_loss_bwd(c.data_ptr(), x.data_ptr(), D, w.data_ptr(), D, t.data_ptr(), ptr(rid), ptr(cid), lse.data_ptr(), N, V, D, dt,
                                 scale, -100, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    return dx, dw


def check(lib, dt, N, V, D, groups=False, scale=20.0):
    from two_towers_overlords_amd import ops

    x, w, t, rid, cid, c = rows_near_targets(dt, N, V, D, groups)
    loss, lse = ops.softmax_loss(x, w, t, scale=scale, row_ids=rid, cand_ids=cid)
    dx, dw = gradients(lib, 1e4, c, x, w, t, lse, scale, rid, cid)
    for fill in (-3e38, math.nan):
        again = gradients(lib, fill, c, x, w, t, lse, scale, rid, cid)
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]), f"the workspace's old contents ({fill}) reach the gradients"

    on = t != -100
    at = t.clamp(min=0)[:, None]
    X, W, C = x.double(), w.double(), (c.double() * on)[:, None]
    l = X @ W.t() * scale
    el = (D + F) * E * (X.abs() @ W.t().abs()) * scale + F * E * l.abs()
    if groups:
        out = rid[:, None] == cid[None]
        out.scatter_(1, at, False)
        l.masked_fill_(out, -math.inf)
        el.masked_fill_(out, 0.0)
    lse64 = torch.logsumexp(l, 1, keepdim=True)
    p = torch.exp(l - lse64)
    near = float((p.gather(1, at).squeeze(1)[on] > 0.25).double().mean())
    assert 0.2 < near < 0.99, near  # both forms of the target's entry
    lm = float(l[l > -math.inf].abs().max())
    rel = el + el.amax(1, keepdim=True) + (V + 4 * F + 8 * lm) * E  # of p: its logit's, lse's, the exponentials'
    del l, el
    G = p.clone()
    G.scatter_add_(1, at, torch.full_like(lse64, -1.0))
    G *= C
    u = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).smallest_normal * u
    stored = float(c.abs().max()) * 2.0 ** -39 if dt == torch.float16 else tiny  # fp16's G is kept 2^14 up, relative to max |c|
    rG = (C.abs() * p * rel + F * E * G.abs()) * (1 + u) + (0 if dt == torch.float32 else u) * G.abs() + stored * on[:, None]
    del p, rel
    for name, got, want, mag, terms in (("dx", dx, G @ W, (rG @ W.abs(), G.abs() @ W.abs()), V),
                                        ("dw", dw, G.t() @ X, (rG.t() @ X.abs(), G.t().abs() @ X.abs()), N)):
        want = want * scale
        tol = u * want.abs() + (1 + u) * scale * (mag[0] + (terms + F) * E * (mag[0] + mag[1])) + tiny
        got = got.double()
        assert bool(torch.isfinite(got).all()), f"{name}: not finite"
        worst = ((got - want).abs() / tol).max()
        assert float(worst) <= 1, f"{name}: {float(worst):.3g} of the bound"


@pytest.mark.parametrize("dt", HALF + [torch.float32])
@pytest.mark.parametrize("groups", [False, True])
@pytest.mark.parametrize("N,V,D", [(300, 700, 72), (1499, 2297, 72), (3700, 3700, 72), (2048, 7000, 40)])
def test_gradients_of_likely_targets(lib, N, V, D, groups, dt):
    check(lib, dt, N, V, D, groups)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("N,V", [(4096, 3968), (1024, 16000), (512, 30522), (8192, 30522)])
def test_gradients_of_likely_targets_among_many_candidates(lib, N, V, dt):
    check(lib, dt, N, V, 64)
