"""GPU: linear_act, packed_attention and softmax_loss with their gradients against plain 64-bit evaluations of their formulas.

Tolerances are elementwise bounds of the arithmetic, evaluated in 64 bits beside the reference:

    u   half a step of the type (finfo.eps / 2): every value that is rounded to the type
    e   2^-23: every fp32 result and every term of an fp32 sum, twice fp32's half step — the exponentials, reciprocals and error
        functions in fp32 are good to a few units, which F counts
    A sum of n products carries at most (n + F) e of the sum of its terms' magnitudes, in any order."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -23
F = 8
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the spacing of the type's subnormals: what rounding costs below its normal range."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


@pytest.fixture(scope="module")
def ops():
    import two_towers_overlords_amd as pkg
    from two_towers_overlords_amd import ops

    pkg.load()
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0, dt=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)


def within(name, got, want, tol):
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if got.numel() == 0:
        return
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    bad = (got - want).abs() - tol
    assert float(bad.max()) <= 0, f"{name}: {float((got - want).abs().flatten()[bad.argmax()]):.3e} beyond {float(tol.expand_as(want).flatten()[bad.argmax()]):.3e}"


# ------------------------------------------------------------------------------------------------ linear_act
def act64(z, name):
    z = z.detach().requires_grad_(True)
    y = {"none": lambda t: t * 1, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"), "silu": torch.nn.functional.silu}[name](z)
    (d,) = torch.autograd.grad(y.sum(), z)
    return y.detach(), d


# |act'| and |act''| are at most these over the real line (gelu: 1.13 and 0.80 = 2 / sqrt(2 pi); silu: 1.10 and 0.5)
D1, D2 = 1.13, 0.80


def check_linear(ops, dt, M, K, N, act, bias=True, res=True, seed=0, x=None, w=None, r=None):
    g = gen(seed + M + 7 * K + 13 * N)
    x = randn(g, M, K, dt=dt) if x is None else x
    w = randn(g, N, K, std=K ** -0.5, dt=dt) if w is None else w
    b = randn(g, N, std=0.3, dt=dt) if bias else None
    r = (randn(g, M, N, dt=dt) if r is None else r) if res else None
    dy = randn(g, M, N, dt=dt)
    y, z = ops.linear_act(x, w, b, r, act, save_preact=True)
    y2 = ops.linear_act(x, w, b, r, act)
    assert torch.equal(y, y2) and (z is None) == (act == "none")
    X, W, DY = x.double(), w.double(), dy.double()
    Z = X @ W.t() + (0 if b is None else b.double())
    mag = X.abs() @ W.t().abs() + (0 if b is None else b.double().abs())
    Y, D = act64(Z, act)
    ez = (K + F) * E * mag  # of the fp32 z
    u = half(dt)
    fast = 0.0 if dt == torch.float32 else 2.0 ** -22  # the 1.5e-7 of the 16-bit types' error function
    ey = D1 * ez + (F * E + fast) * (Z.abs() + 1)
    R = 0 if r is None else r.double()
    within("y", y, Y + R, u * (Y + R).abs() + (1 + u) * (ey + E * (Y.abs() + (0 if r is None else R.abs()))) + tiny(dt))
    dx, dw, db = ops.linear_act_bwd(dy, x, w, z, act, bias=bias)
    zerr = 0 if act == "none" else ez + u * Z.abs() + tiny(dt)
    kink = 0
    if act == "relu":  # the derivative jumps: where z is within its error of 0 either side is right
        kink = (Z.abs() <= zerr).double() * DY.abs()
        d2 = 0
    else:
        d2 = 0 if act == "none" else D2
    DZ = DY * D
    edz = DY.abs() * (d2 * zerr + F * E + (0 if act in ("none", "relu") else fast * (1 + Z.abs()))) + kink
    rdz = edz + u * (DZ.abs() + edz) + tiny(dt)  # after its rounding to the type
    dz_mag = DZ.abs() + rdz
    DX, DW, DB = DZ @ W, DZ.t() @ X, DZ.sum(0)
    within("dx", dx, DX, u * DX.abs() + (1 + u) * (rdz @ W.abs() + (N + F) * E * (dz_mag @ W.abs())) + tiny(dt))
    within("dw", dw, DW, u * DW.abs() + (1 + u) * (rdz.t() @ X.abs() + (M + F) * E * (dz_mag.t() @ X.abs())) + tiny(dt))
    if bias:
        within("db", db, DB, u * DB.abs() + (1 + u) * (edz.sum(0) + (M + F) * E * dz_mag.sum(0)) + tiny(dt))
    else:
        assert db is None


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,N,act", [
    (1, 1, 1, "none"), (1, 384, 1536, "gelu"), (11, 384, 384, "none"), (7, 8, 5, "relu"), (64, 64, 64, "silu"),
    (65, 72, 129, "gelu_tanh"), (130, 100, 36, "gelu"), (33, 17, 31, "silu"), (257, 384, 1152, "none"), (1000, 136, 264, "gelu"),
    (2049, 96, 512, "relu")])
def test_linear_act_and_gradients(ops, dt, M, K, N, act):
    check_linear(ops, dt, M, K, N, act)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1499, 72, 2296), (72, 1499, 2296), (1499, 2296, 72), (4095, 72, 4088), (72, 4088, 4088), (4095, 4088, 72)])
def test_linear_act_tile_shapes(ops, dt, M, K, N):
    """Outputs large enough for 128- and 256-wide tiles, in the forward and in either gradient product, ragged at both edges."""
    check_linear(ops, dt, M, K, N, "gelu")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True)])
def test_linear_act_without_bias_or_residual(ops, dt, bias, res):
    check_linear(ops, dt, 50, 40, 24, "gelu", bias=bias, res=res)


@pytest.mark.parametrize("dt", DTYPES)
def test_linear_act_long_contraction_over_rows(ops, dt):
    """dw sums over the rows: split and joined when the output is small."""
    check_linear(ops, dt, 9001, 64, 40, "gelu")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("off,extra", [(0, 8), (0, 3), (1, 8), (2, 5)])
def test_linear_act_row_strided_views(ops, dt, off, extra):
    g = gen(3)
    M, K, N = 37, 48, 56
    x = randn(g, M, K + extra, dt=dt)[:, off:off + K] if off + K <= K + extra else None
    w = randn(g, N, K + extra, std=0.2, dt=dt)[:, off:off + K]
    r = randn(g, M, N + extra, dt=dt)[:, off:off + N]
    check_linear(ops, dt, M, K, N, "gelu", x=x, w=w, r=r)
    buf = torch.full((M + 2, N + extra), 7.0, device="cuda", dtype=dt)
    out = buf[1:M + 1, off:off + N]
    got = ops.linear_act(x, w, None, r, "relu", out=out)
    assert got is out and torch.equal(out, ops.linear_act(x, w, None, r, "relu"))
    buf[1:M + 1, off:off + N] = 7.0
    assert bool((buf == 7.0).all())  # nothing around the view was written


def test_linear_act_no_rows(ops):
    x, w = torch.empty(0, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    y, z = ops.linear_act(x, w, None, None, "gelu", save_preact=True)
    assert y.shape == (0, 8)
    dx, dw, db = ops.linear_act_bwd(y, x, w, z, "gelu")
    assert dx.shape == (0, 16) and not bool(dw.any()) and not bool(db.any())


def test_linear_act_adds_into_its_residual(ops):
    g = gen(4)
    x, w, r = randn(g, 70, 32), randn(g, 48, 32), randn(g, 70, 48)
    want = ops.linear_act(x, w, None, r)
    assert torch.equal(ops.linear_act(x, w, None, r, out=r), want)


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", DTYPES)
def test_linear_act_far_values(ops, dt, act):
    """Pre-activations far out on both sides, infinities and NaN: value and derivative are their limits, NaN stays NaN."""
    z = torch.tensor([-60000.0, -100.0, -41.0, -39.0, 0.0, 39.0, 41.0, 100.0, 60000.0], device="cuda", dtype=dt).unsqueeze(1)
    one = torch.ones(1, 1, device="cuda", dtype=dt)
    y, zz = ops.linear_act(z, one, None, None, act, save_preact=True)
    assert torch.equal(zz, z)
    Y, D = act64(z.double(), act)
    within("y", y, Y, half(dt) * Y.abs() + F * E * (1 + Y.abs()))
    dx, _, _ = ops.linear_act_bwd(torch.ones_like(y), z, one, zz, act)
    within("dx", dx, D, half(dt) * D.abs() + 2 * F * E)
    bad = torch.tensor([[float("nan")], [float("inf")], [1.0]], device="cuda", dtype=dt)
    y, zz = ops.linear_act(bad, one, None, None, act, save_preact=True)
    assert bool(y[0].isnan()) and float(y[1]) == float("inf") and float(y[2]) > 0
    dz, _, _ = ops.linear_act_bwd(torch.ones_like(y), bad, one, zz, act)
    assert bool(dz[0].isnan()) and abs(float(dz[1]) - 1) < 1e-2


def test_linear_act_relu_keeps_the_sign_below_fp16s_range(ops):
    x = torch.full((4, 8), 2.0 ** -14, device="cuda", dtype=torch.float16)
    w = torch.full((8, 8), 2.0 ** -14, device="cuda", dtype=torch.float16)  # z = 2^-25: rounds to 0 in fp16
    _, z = ops.linear_act(x, w, None, None, "relu", save_preact=True)
    dx, _, db = ops.linear_act_bwd(torch.ones(4, 8, device="cuda", dtype=torch.float16), x, w, z, "relu")
    assert bool((z > 0).all()) and bool((db == 4).all())


# ------------------------------------------------------------------------------------------------ packed_attention
def attention64(q, k, v, do, lens, scale, causal, prefix, cap, slopes, keep):
    """Per document and head in 64 bits: outputs, gradients and elementwise bounds' ingredients."""
    T, H, Dh = q.shape
    Hkv = k.shape[1]
    rep = H // Hkv
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
    res = dict(o=z(q), lse=torch.full((H, T), -math.inf, dtype=torch.float64, device="cuda"), dq=z(q), dk=z(k), dv=z(v))
    tol = dict(o=z(q), lse=torch.zeros((H, T), dtype=torch.float64, device="cuda"), dq=z(q), dk=z(k), dv=z(v))
    dt, u = q.dtype, half(q.dtype)
    up = 0.0 if dt == torch.float32 else u   # P and dS are rounded to the type before the second products
    tp = tiny(dt)
    at = 0
    for b, n in enumerate(lens):
        s_ = slice(at, at + n)
        at += n
        if n == 0:
            continue
        pos = torch.arange(n, device="cuda")
        see = torch.ones(n, n, dtype=torch.bool, device="cuda")
        if causal:
            see = pos[None] <= pos[:, None]
        elif prefix is not None:
            see = (pos[None] <= pos[:, None]) | (pos[None] < int(prefix[b]))
        if keep is not None:
            see = see & keep[s_].bool()[None]
        for h in range(H):
            Q, K, V, DO = q[s_, h].double(), k[s_, h // rep].double(), v[s_, h // rep].double(), do[s_, h].double()
            if keep is not None:  # masked keys may hold anything
                K, V = torch.where(keep[s_].bool()[:, None], K, 0.0), torch.where(keep[s_].bool()[:, None], V, 0.0)
            raw = Q @ K.t() * scale
            es = (Dh + F) * E * (Q.abs() @ K.t().abs()) * scale
            s, der = raw, torch.ones_like(raw)
            if cap > 0:
                th = torch.tanh(raw / cap)
                s, der = cap * th, 1 - th * th
                es = es + F * E * cap
            if slopes is not None:
                bias = float(slopes[h]) * (pos[:, None] - pos[None]).abs()
                s = s - bias
                es = es + F * E * (raw.abs() + bias)
            s = torch.where(see, s, -math.inf)
            any_ = see.any(1, keepdim=True)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(see & any_, torch.exp(s - torch.where(any_, lse, 0.0)), 0.0)
            # relative error of p: its score's, the row's worst (through the sum), the exponent's rounding, n additions
            es = torch.where(see, es, 0.0)
            smag = torch.where(see, s.abs(), 0.0).amax(1, keepdim=True)
            rp = es + es.amax(1, keepdim=True) + (n + 2 * F + 4 * smag) * E
            O = p @ V
            eo = ((rp + up) * p + tp) @ V.abs() + (n + F) * E * (p @ V.abs())
            res["o"][s_, h], tol["o"][s_, h] = O, u * O.abs() + (1 + u) * eo + tp
            res["lse"][h, s_] = lse.squeeze(1)
            tol["lse"][h, s_] = (es.amax(1) + (n + F + 4 * smag.squeeze(1)) * E)
            # gradients: P and delta come from the stored lse and the stored (rounded) o
            dp = DO @ V.t()
            edp = (Dh + F) * E * (DO.abs() @ V.t().abs())
            delta = (DO * O).sum(1, keepdim=True)
            edel = (DO.abs() * (u * O.abs() + (1 + u) * eo + tp)).sum(1, keepdim=True) + (Dh + F) * E * (DO * O).abs().sum(1, keepdim=True)
            rp2 = es + tol["lse"][h, s_].unsqueeze(1) + (2 * F + 8 * smag) * E
            ds = p * (dp - delta) * der
            # the derivative of the cap moves by at most 2 |error of tanh| + the score's error over cap
            eder = (2 * es / cap + F * E) if cap > 0 else 0
            eds = p * ((rp2 * (dp - delta).abs() + edp + edel) + (dp - delta).abs() * eder) + F * E * p * (dp - delta).abs()
            rds = eds * (1 + up) + up * ds.abs() + tp
            res["dq"][s_, h] = ds @ K * scale
            tol["dq"][s_, h] = u * res["dq"][s_, h].abs() + (1 + u) * scale * (rds @ K.abs() + (n + F) * E * ((ds.abs() + rds) @ K.abs())) + tp
            kv = h // rep
            dk, dv = ds.t() @ Q * scale, p.t() @ DO
            res["dk"][s_, kv] += dk
            res["dv"][s_, kv] += dv
            tol["dk"][s_, kv] += scale * (rds.t() @ Q.abs() + (n * rep + F) * E * ((ds.abs() + rds).t() @ Q.abs()))
            ep = (rp2 + up) * p + tp
            tol["dv"][s_, kv] += ep.t() @ DO.abs() + (n * rep + F) * E * ((p + ep).t() @ DO.abs())
    for name in ("dk", "dv"):
        tol[name] = u * res[name].abs() + (1 + u) * tol[name] + tp
    return res, tol


def make_attention(dt, lens, H, Hkv, Dh, seed=0, tail=0, std=1.0):
    g = gen(seed + sum(lens) + 31 * H + Dh)
    T = sum(lens) + tail
    qkv = randn(g, T, H + 2 * Hkv, Dh, std=std, dt=dt)
    cu = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    return qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:], randn(g, T, H, Dh, dt=dt), cu


def check_attention(ops, dt, lens, H, Hkv, Dh, causal=False, prefix=None, cap=0.0, alibi=False, keep=None, tail=0, seed=0, scale=None):
    q, k, v, do, cu = make_attention(dt, lens, H, Hkv, Dh, seed, tail)
    slopes = torch.tensor([2.0 ** (-(h + 1)) for h in range(H)], device="cuda") if alibi else None
    pre = torch.tensor(prefix, dtype=torch.int32, device="cuda") if prefix is not None else None
    kw = dict(scale=scale, causal=causal, prefix=pre, softcap=cap, slopes=slopes, key_mask=keep)
    o, lse = ops.packed_attention(q, k, v, cu, **kw)
    grads = ops.packed_attention_bwd(do, q, k, v, o, lse, cu, **kw)
    again = ops.packed_attention_bwd(do, q, k, v, *ops.packed_attention(q, k, v, cu, **kw), cu, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))  # no atomics: the same bits
    res, tol = attention64(q, k, v, do, lens, Dh ** -0.5 if scale is None else scale, causal, prefix, cap, slopes, keep)
    T = sum(lens)
    if tail:
        assert not bool(o[T:].any()) and bool((lse[:, T:] == -math.inf).all()) and not any(bool(t[T:].any()) for t in grads)
    empty = res["lse"][:, :T] == -math.inf
    assert torch.equal(lse[:, :T] == -math.inf, empty)
    within("lse", torch.where(empty, 0.0, lse[:, :T].double()), torch.where(empty, 0.0, res["lse"][:, :T]), tol["lse"][:, :T])
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(name, t, res[name], tol[name])
    return o, lse, grads


LENS = [[1], [11], [32], [33], [64, 1, 0, 65], [128, 127, 129], [7, 300, 0, 0, 2], [200, 200]]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lens", LENS, ids=lambda l: "-".join(map(str, l)))
def test_attention_document_lengths(ops, dt, lens):
    check_attention(ops, dt, lens, 2, 2, 32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Dh", [8, 16, 24, 32, 40, 64, 72, 96, 128])
def test_attention_head_dims(ops, dt, Dh):
    check_attention(ops, dt, [70, 33], 3, 1, Dh, alibi=True)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2), (8, 1), (12, 12)])
def test_attention_shared_heads(ops, dt, H, Hkv):
    check_attention(ops, dt, [90, 5], H, Hkv, 64, causal=True)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kw", [dict(causal=True), dict(prefix=[0, 40, 500]), dict(prefix=[64, 1, 129]), dict(cap=5.0), dict(alibi=True),
                                dict(causal=True, cap=2.0, alibi=True), dict(prefix=[100, 32, 0], alibi=True, cap=30.0), dict(scale=0.3)],
                         ids=lambda k: "+".join(k))
@pytest.mark.parametrize("Dh", [32, 128])
def test_attention_masks_and_scores(ops, dt, kw, Dh):
    check_attention(ops, dt, [129, 70, 260], 2, 2, Dh, **kw)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_key_mask_leaves_rows_empty(ops, dt, causal):
    """Holes, a document whose keys are all taken out, and a causal start that sees nothing: those rows give 0."""
    lens = [100, 40, 65]
    keep = torch.rand(205, generator=gen(1), device="cuda") > 0.4
    keep[100:140] = False
    keep[140:150] = False
    o, lse, (dq, dk, dv) = check_attention(ops, dt, lens, 2, 1, 64, causal=causal, keep=keep)
    dead = torch.zeros(205, dtype=torch.bool, device="cuda")
    dead[100:140] = True
    if causal:
        dead[140:150] = True
    assert not bool(o[dead].any()) and not bool(dq[dead].any()) and not bool(dk[~keep].any()) and not bool(dv[~keep].any())
    assert torch.equal(ops.packed_attention(*make_attention(dt, lens, 2, 1, 64)[:3], make_attention(dt, lens, 2, 1, 64)[4],
                                            causal=causal, key_mask=keep.to(torch.uint8) * 255)[0], o)


@pytest.mark.parametrize("dt", DTYPES)
def test_attention_masked_keys_may_hold_anything(ops, dt):
    q, k, v, do, cu = make_attention(dt, [70, 50], 2, 2, 32)
    keep = torch.rand(120, generator=gen(2), device="cuda") > 0.3
    o, lse = ops.packed_attention(q, k, v, cu, key_mask=keep)
    g = ops.packed_attention_bwd(do, q, k, v, o, lse, cu, key_mask=keep)
    for bad in (float("nan"), float("inf"), torch.finfo(dt).min):
        k2, v2 = k.clone(), v.clone()
        k2[~keep], v2[~keep] = bad, bad
        o2, lse2 = ops.packed_attention(q, k2, v2, cu, key_mask=keep)
        g2 = ops.packed_attention_bwd(do, q, k2, v2, o2, lse2, cu, key_mask=keep)
        assert torch.equal(o, o2) and torch.equal(lse, lse2) and all(torch.equal(a, b) for a, b in zip(g, g2))


@pytest.mark.parametrize("dt", DTYPES)
def test_attention_documents_do_not_touch(ops, dt):
    """A document's results do not depend on its neighbours, NaN in them included; tokens behind the last get 0."""
    q, k, v, do, cu = make_attention(dt, [50, 77, 40], 2, 2, 32, tail=9)
    o, lse = ops.packed_attention(q, k, v, cu)
    g = ops.packed_attention_bwd(do, q, k, v, o, lse, cu)
    q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
    for t in (q2, k2, v2, do2):
        t[:50] = float("nan")
        t[127:] = float("nan")
    o2, lse2 = ops.packed_attention(q2, k2, v2, cu)
    g2 = ops.packed_attention_bwd(do2, q2, k2, v2, o2, lse2, cu)
    assert torch.equal(o[50:127], o2[50:127]) and all(torch.equal(a[50:127], b[50:127]) for a, b in zip(g, g2))
    assert not bool(o2[167:].any()) and not any(bool(t[167:].any()) for t in g2)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_long_document(ops, dt):
    check_attention(ops, dt, [1500, 3], 1, 1, 64, causal=True, alibi=True)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kw", [dict(causal=True), dict(prefix=[300, 0, 700, 5, 64]), dict()], ids=["causal", "prefix", "full"])
def test_attention_long_documents_in_sorted_order(ops, dt, kw):
    """Few long documents: their tiles run longest first.  An empty one, one short one and rows behind the last among them."""
    check_attention(ops, dt, [701, 0, 1030, 64, 300], 2, 1, 64, tail=150, **kw)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_more_long_documents_than_lanes(ops, dt):
    check_attention(ops, dt, [257 + i % 5 for i in range(67)], 1, 1, 32, causal=True)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_many_documents(ops, dt):
    """More documents than the 64-wide search takes in one step."""
    lens = [(7 * i) % 23 for i in range(4500)]
    q, k, v, do, cu = make_attention(dt, lens, 1, 1, 32)
    o, lse = ops.packed_attention(q, k, v, cu)
    pick = list(range(0, 4500, 97)) + [4499]
    ends = torch.tensor(lens).cumsum(0).tolist()
    for b in pick:
        n, e = lens[b], ends[b]
        if n == 0:
            continue
        s = slice(e - n, e)
        one, _ = ops.packed_attention(q[s], k[s], v[s], torch.tensor([0, n], dtype=torch.int32, device="cuda"))
        assert torch.equal(one, o[s]), b


@pytest.mark.parametrize("dt", DTYPES)
def test_attention_gradients_into_one_buffer_and_token_major_views(ops, dt):
    T, H, Dh = 77, 3, 32
    q, k, v, do, cu = make_attention(dt, [30, 47], H, H, Dh)
    o, lse = ops.packed_attention(q, k, v, cu)
    g = ops.packed_attention_bwd(do, q, k, v, o, lse, cu)
    buf = torch.full((T + 2, 3 * H, Dh), 3.0, device="cuda", dtype=dt)
    views = tuple(buf[1:T + 1, i * H:(i + 1) * H] for i in range(3))
    ops.packed_attention_bwd(do, q, k, v, o, lse, cu, grads=views)
    assert all(torch.equal(a, b) for a, b in zip(g, views)) and bool((buf[0] == 3).all()) and bool((buf[-1] == 3).all())
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]  # head-major storage
    assert torch.equal(ops.packed_attention(*hm, cu)[0], o)


def test_attention_no_tokens(ops):
    z = torch.empty(0, 2, 32, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    o, lse = ops.packed_attention(z, z, z, cu)
    assert o.shape == (0, 2, 32) and lse.shape == (2, 0)
    assert all(t.shape == (0, 2, 32) for t in ops.packed_attention_bwd(o, z, z, z, o, lse, cu))


def test_attention_large_scores_do_not_overflow(ops):
    for dt in DTYPES:
        q, k, v, do, cu = make_attention(dt, [80], 1, 1, 32, std=30.0)
        o, lse = ops.packed_attention(q, k, v, cu)
        g = ops.packed_attention_bwd(do, q, k, v, o, lse, cu)
        assert all(bool(torch.isfinite(t).all()) for t in (o, lse, *g))


# ------------------------------------------------------------------------------------------------ softmax_loss
def check_softmax(ops, dt, N, V, D, scale=1.0, groups=False, ignore=(), unit=False, seed=0, x=None, w=None, coef=None):
    g = gen(seed + N + 3 * V + 5 * D)
    if x is None:
        x, w = randn(g, N, D), randn(g, V, D, std=2 * D ** -0.5)
        if unit:
            x, w = x / x.norm(dim=1, keepdim=True), w / w.norm(dim=1, keepdim=True)
        x, w = x.to(dt), w.to(dt)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    for i in ignore:
        t[i] = -100
    rid = cid = None
    if groups:
        cid = torch.randint(0, max(1, V // 3), (V,), generator=g, device="cuda")
        rid = cid[t.clamp(min=0)]
    c = (torch.rand(N, generator=g, device="cuda") + 0.1) / N if coef is None else coef
    kw = dict(scale=scale, row_ids=rid, cand_ids=cid)
    loss, lse = ops.softmax_loss(x, w, t, **kw)
    dx, dw = ops.softmax_loss_bwd(c, x, w, t, lse, **kw)
    on = t != -100
    X, W, C = x.double(), w.double(), c.double() * on
    l = X @ W.t() * scale
    el = (D + F) * E * (X.abs() @ W.t().abs()) * scale + F * E * l.abs()
    at = t.clamp(min=0).unsqueeze(1)
    out = torch.zeros_like(l, dtype=torch.bool)
    if groups:
        out = rid[:, None] == cid[None]
        out &= torch.arange(V, device="cuda")[None] != at
    l = torch.where(out, -math.inf, l)
    el = torch.where(out, 0.0, el)
    LSE = torch.logsumexp(l, 1)
    fin = LSE > -math.inf
    lm = torch.where(out, 0.0, l.abs()).amax(1)
    elb = el.amax(1) + (V + 2 * F + 4 * lm) * E * 1.0
    assert torch.equal(lse > -math.inf, fin)
    within("lse", torch.where(fin, lse.double(), 0.0), torch.where(fin, LSE, 0.0), elb + E * torch.where(fin, LSE.abs(), 0.0))
    LOSS = torch.where(on, LSE - l.gather(1, at).squeeze(1), 0.0)
    within("loss", loss, LOSS, (2 * elb + E * lm * 4) * on)
    p = torch.where(out | ~fin[:, None], 0.0, torch.exp(l - torch.where(fin, LSE, 0.0)[:, None]))
    hot = torch.zeros_like(p)
    hot.scatter_(1, at, 1.0)
    G = C[:, None] * (p - hot)
    u = half(dt)
    tp = float(c.abs().max()) * 2.0 ** -39 if dt == torch.float16 else tiny(dt)  # fp16's G is stored 2^14 up, relative to max |c|
    eG = C[:, None].abs() * p * (el + elb[:, None] + (2 * F + 4 * lm[:, None]) * E) + F * E * G.abs()
    rG = eG * (1 + u) + (0 if dt == torch.float32 else u) * G.abs() + tp * on[:, None]
    DX, DW = G @ W * scale, G.t() @ X * scale
    within("dx", dx, DX, u * DX.abs() + (1 + u) * scale * (rG @ W.abs() + (V + F) * E * ((G.abs() + rG) @ W.abs())) + tiny(dt))
    within("dw", dw, DW, u * DW.abs() + (1 + u) * scale * (rG.t() @ X.abs() + (N + F) * E * ((G.abs() + rG).t() @ X.abs())) + tiny(dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 2, 8), (3, 5, 7), (64, 64, 64), (65, 129, 40), (5, 3001, 100), (300, 1000, 384),
                                   (1030, 33, 72), (2, 70001, 64)])
def test_softmax_loss_and_gradients(ops, dt, N, V, D):
    check_softmax(ops, dt, N, V, D)
    check_softmax(ops, dt, N, V, D, scale=20.0, unit=True, groups=True, ignore=(0,) if N > 1 else ())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V", [(1499, 2297), (4095, 4089)])
def test_softmax_loss_tile_shapes(ops, dt, N, V):
    """128- and 256-wide tiles, ragged at both edges."""
    check_softmax(ops, dt, N, V, 72, scale=20.0, unit=True, groups=True, ignore=(0, 17, N - 1))


@pytest.mark.parametrize("dt", DTYPES)
def test_softmax_loss_rows_without_a_target(ops, dt):
    check_softmax(ops, dt, 40, 90, 32, ignore=tuple(range(0, 40, 3)))
    x, w = torch.randn(6, 16, device="cuda").to(dt), torch.randn(9, 16, device="cuda").to(dt)
    t = torch.full((6,), -100, device="cuda")
    loss, lse = ops.softmax_loss(x, w, t)
    dx, dw = ops.softmax_loss_bwd(torch.ones(6, device="cuda"), x, w, t, lse)
    assert not any(bool(a.any()) for a in (loss, dx, dw))
    loss, lse = ops.softmax_loss(x, w, torch.zeros(6, dtype=torch.int64, device="cuda"), row_ids=torch.zeros(6, dtype=torch.int64, device="cuda"),
                                 cand_ids=torch.zeros(9, dtype=torch.int64, device="cuda"))
    assert float(loss.abs().max()) <= 16 * E * float(lse.abs().max())  # the target is the only candidate


@pytest.mark.parametrize("dt", DTYPES)
def test_softmax_loss_uneven_upstream(ops, dt):
    c = torch.tensor([2.0 ** -i for i in range(50)], device="cuda") * 100
    check_softmax(ops, dt, 50, 300, 64, coef=c)
    check_softmax(ops, dt, 50, 300, 64, coef=torch.zeros(50, device="cuda"))
    check_softmax(ops, dt, 50, 300, 64, coef=-c)


def test_softmax_loss_bad_targets_are_nan(ops):
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(5, 8, device="cuda")
    for bad in (5, -1, 2 ** 40):
        t = torch.tensor([0, bad, 2, 3], device="cuda")
        loss, lse = ops.softmax_loss(x, w, t)
        assert loss.isnan().tolist() == [False, True, False, False]
        dx, _ = ops.softmax_loss_bwd(torch.ones(4, device="cuda"), x, w, t, lse)
        assert dx.isnan().any(1).tolist() == [False, True, False, False]


@pytest.mark.parametrize("dt", DTYPES)
def test_softmax_loss_row_strided_views(ops, dt):
    g = gen(9)
    for off, extra in ((0, 8), (8, 16), (1, 3)):
        x = randn(g, 30, 48 + off + extra, std=0.3, dt=dt)[:, off:off + 48]
        w = randn(g, 70, 48 + off + extra, std=0.3, dt=dt)[:, off:off + 48]
        check_softmax(ops, dt, 30, 70, 48, x=x, w=w)


def test_softmax_loss_no_rows(ops):
    x, w = torch.empty(0, 16, device="cuda"), torch.randn(9, 16, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = ops.softmax_loss(x, w, t)
    dx, dw = ops.softmax_loss_bwd(loss, x, w, t, lse)
    assert loss.shape == (0,) and dx.shape == (0, 16) and not bool(dw.any())


def test_softmax_loss_in_several_pieces(ops):
    """More gradient entries than one piece holds: 16-bit types sum dx over pieces of the candidates, float sums dw over pieces
    of the rows."""
    check_softmax(ops, torch.float32, 4099, 17003, 24, groups=True, ignore=(0, 4098))
    check_softmax(ops, torch.float32, 4099, 40003, 24, groups=True, ignore=(0, 4098))
    check_softmax(ops, torch.bfloat16, 4099, 70003, 16)
    check_softmax(ops, torch.float16, 4099, 33001, 24)


@pytest.mark.parametrize("scale", [20.0, 60.0])
def test_softmax_loss_of_nearly_certain_targets_keeps_its_digits(ops, scale):
    """float: loss and gradient of rows whose target takes all but 1e-6 .. 1e-20 of the probability are good to a relative error,
    not to the rounding of an lse of 20 or 60."""
    g = gen(5)
    w = randn(g, 300, 64)
    w /= w.norm(dim=1, keepdim=True)
    x = w[:200] + 0.02 * randn(g, 200, 64)
    x /= x.norm(dim=1, keepdim=True)
    t = torch.arange(200, device="cuda")
    loss, lse = ops.softmax_loss(x, w, t, scale=scale)
    dx, _ = ops.softmax_loss_bwd(torch.ones(200, device="cuda"), x, w, t, lse, scale=scale)
    l = x.double() @ w.double().t() * scale
    d = l - l.gather(1, t[:, None])
    d.scatter_(1, t[:, None], -math.inf)
    rest = torch.exp(d).sum(1)  # loss = log(1 + rest)
    # the differences of two logits carry (64 + F) e scale 2 absolute; the target's own term is 1, and after it come at most 4 + 2
    # additions in its lane, 1 between lanes, 1 between waves, 5 of tiles and 15 of their lanes: 28 roundings of 2^-24
    rel = 2 * (64 + F) * E * scale
    within("loss", loss, torch.log1p(rest), rel * rest + 28 * E / 2 + E * torch.log1p(rest))
    p = torch.exp(d - torch.log1p(rest)[:, None])
    p.scatter_(1, t[:, None], 0.0)
    G = p.clone()
    G.scatter_(1, t[:, None], -p.sum(1, keepdim=True))
    DX = G @ w.double() * scale
    # the row's common factor exp(-lse) carries lse's rounding, 2^-24 of |lse| <= scale + log 300, once
    rg = rel + E * (scale + 8) + (300 + F) * E
    within("dx", dx, DX, 4 * rg * scale * (G.abs() @ w.double().abs()) + tiny(torch.float32))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Dh", [32, 128])
@pytest.mark.parametrize("kw", [dict(), dict(softcap=30.0, slopes=True), dict(causal=True), dict(prefix=True)], ids=["full", "cap", "causal", "prefix"])
def test_attention_single_key_has_exactly_no_gradient_of_scores(ops, dt, Dh, kw):
    """A query that sees one key has p = 1 whatever q and k are: dq and dk are 0, dv = dO."""
    docs, H = 37, 4
    g = gen(Dh)
    q, k, v, do = (randn(g, docs, H, Dh).to(dt) for _ in range(4))
    cu = torch.arange(docs + 1, dtype=torch.int32, device="cuda")
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = torch.full((H,), 0.5, device="cuda")
    if "prefix" in kw:
        kw["prefix"] = torch.ones(docs, dtype=torch.int32, device="cuda")
    o, lse = ops.packed_attention(q, k, v, cu, **kw)
    dq, dk, dv = ops.packed_attention_bwd(do, q, k, v, o, lse, cu, **kw)
    assert not bool(dq.any()) and not bool(dk.any())
    within("dv", dv, do.double(), 2 * half(dt) * do.double().abs() + (64 * E) * do.double().abs())  # p and dv are rounded
    if "causal" in kw or "prefix" in kw:  # the first query of longer documents
        cu = torch.tensor([0, 5, docs], dtype=torch.int32, device="cuda")
        if "prefix" in kw:
            kw["prefix"] = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        o, lse = ops.packed_attention(q, k, v, cu, **kw)
        dq, dk, dv = ops.packed_attention_bwd(do, q, k, v, o, lse, cu, **kw)
        assert not bool(dq[0].any()) and not bool(dq[5].any()) and bool(dq[1].any())


@pytest.mark.parametrize("dt", DTYPES)
def test_softmax_loss_of_a_single_candidate_is_exactly_nothing(ops, dt):
    """The target is the row's only candidate, by itself or because its group's others are left out: loss and gradients are 0."""
    N, D = 300, 72
    g = gen(5)
    x = randn(g, N, D).to(dt)
    for V in (1, 2, 700):
        w = randn(g, V, D).to(dt)
        t = torch.randint(0, V, (N,), generator=g, device="cuda")
        kw = dict(row_ids=torch.full((N,), 3, device="cuda"), cand_ids=torch.full((V,), 3, device="cuda")) if V > 1 else {}
        loss, lse = ops.softmax_loss(x, w, t, scale=1.7, **kw)
        dx, dw = ops.softmax_loss_bwd(torch.ones(N, device="cuda"), x, w, t, lse, scale=1.7, **kw)
        assert not any(bool(a.any()) for a in (loss, dx, dw)), V


@pytest.mark.parametrize("dt", DTYPES)
def test_softmax_loss_rows_without_a_target_keep_candidate_0(ops, dt):
    """All candidates in one group: a row's sum holds its target alone, or candidate 0 where it has none."""
    g = gen(11)
    x, w = randn(g, 9, 16).to(dt), randn(g, 300, 16).to(dt)
    t = torch.tensor([5, -100, 299, -100, 0, 1, 2, -100, 3], device="cuda")
    one = torch.ones(300, dtype=torch.int64, device="cuda")
    loss, lse = ops.softmax_loss(x, w, t, row_ids=one[:9], cand_ids=one)
    l = (x.double() * w[t.clamp(min=0)].double()).sum(1)
    within("lse", lse, l, (16 + 3 * F) * E * (x.double().abs() * w[t.clamp(min=0)].double().abs()).sum(1) + 4 * E)
    assert not bool(loss.any())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("c", [0.0, 1e-44, 1e-39, 1e-20, 1e20])
def test_softmax_loss_coefficients_of_any_size(ops, dt, c):
    """16-bit gradients of the logits are relative to the largest coefficient, whatever its size."""
    g = gen(3)
    x, w = randn(g, 33, 24).to(dt), randn(g, 70, 24).to(dt)
    t = torch.randint(0, 70, (33,), generator=g, device="cuda")
    _, lse = ops.softmax_loss(x, w, t)
    dx, dw = ops.softmax_loss_bwd(torch.full((33,), c, device="cuda"), x, w, t, lse)
    if c <= 1e-39:
        assert all(bool((a.abs() <= 1e-36).all()) for a in (dx, dw))
    elif dt != torch.float16:  # beyond fp16's range
        one = ops.softmax_loss_bwd(torch.ones(33, device="cuda"), x, w, t, lse)
        for a, b in zip((dx, dw), one):  # each G and each result rounded once on either side
            within("scaled", a.double() / c, b.double(), 4 * half(dt) * (b.double().abs() + b.double().abs().amax()) + 64 * E * b.double().abs().amax())
