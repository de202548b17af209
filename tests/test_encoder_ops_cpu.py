"""CPU: argument checks of linear_act, packed_attention and softmax_loss — at the C entry (no launch happens) and in ops."""
import ctypes as C

import pytest
import torch

import two_towers_overlords_amd as pkg
from two_towers_overlords_amd import _lib, ops

NULL, SHAPE, DTYPE, ALIGN, WS, UNSUPPORTED = -1, -2, -3, -4, -5, -7
P = 4096  # a 16-byte aligned address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    return pkg.load()


def linear(lib, x=P, ldx=8, w=P, ldw=8, bias=None, res=None, ldr=0, y=P, ldy=8, z=None, M=4, N=8, K=8, dt=1, act=0, ws=None, n=0):
    return lib.tt_linear_act(x, ldx, w, ldw, bias, res, ldr, y, ldy, z, M, N, K, dt, act, ws, n, None)


def test_linear_act_refusals(lib):
    assert linear(lib, dt=0) == DTYPE and linear(lib, dt=4) == DTYPE
    assert linear(lib, act=5) == UNSUPPORTED and linear(lib, act=-1) == UNSUPPORTED
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(ldx=7), dict(ldw=7), dict(ldy=7), dict(res=P, ldr=7), dict(M=2 ** 31)):
        assert linear(lib, **bad) == SHAPE, bad
    for bad in (dict(x=None), dict(w=None), dict(y=None)):
        assert linear(lib, **bad) == NULL, bad
    assert linear(lib, M=0, x=None, y=None) == 0
    # rows that are not whole 16-byte chunks need a workspace
    need = lib.tt_linear_act_workspace_bytes(P, 9, P, 8, 4, 8, 8, 1)
    assert need > 0 and lib.tt_linear_act_workspace_bytes(P, 8, P, 8, 4, 8, 8, 1) == 0
    assert lib.tt_linear_act_workspace_bytes(P + 4, 8, P, 8, 4, 8, 8, 1) > 0
    assert linear(lib, ldx=9) == NULL and linear(lib, ldx=9, ws=P, n=need - 1) == WS and linear(lib, ldx=9, ws=P + 4, n=need) == ALIGN


def test_linear_act_bwd_refusals(lib):
    def bwd(dy=P, lddy=8, x=P, ldx=8, w=P, ldw=8, z=None, dx=P, dw=P, db=P, M=4, N=8, K=8, dt=1, act=0, ws=P, n=1 << 20):
        return lib.tt_linear_act_bwd(dy, lddy, x, ldx, w, ldw, z, dx, dw, db, M, N, K, dt, act, ws, n, None)

    assert bwd(dt=7) == DTYPE and bwd(act=9) == UNSUPPORTED
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(lddy=7), dict(ldx=7), dict(ldw=7)):
        assert bwd(**bad) == SHAPE, bad
    for bad in (dict(dy=None), dict(x=None), dict(w=None), dict(ws=None), dict(act=2)):
        assert bwd(**bad) == NULL, bad
    assert bwd(n=0) == WS and bwd(ws=P + 8) == ALIGN


def attention_args(**kw):
    a = _lib.TTAttentionArgs()
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, n, _lib.TTHeadView(P, 64, 32))
    a.lse = a.delta = a.cu_seqlens = P
    a.T, a.docs, a.heads, a.kv_heads, a.head_dim, a.dtype, a.scale = 10, 1, 2, 2, 32, 1, 0.5
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("fn", ["tt_packed_attention", "tt_packed_attention_bwd"])
def test_attention_refusals(lib, fn):
    def go(**kw):
        return getattr(lib, fn)(attention_args(**kw), None)

    assert getattr(lib, fn)(None, None) == NULL
    assert go(dtype=0) == DTYPE
    for bad in (dict(T=-1), dict(docs=0), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(head_dim=0), dict(head_dim=12),
                dict(head_dim=136), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(softcap=-1.0)):
        assert go(**bad) == SHAPE, bad
    assert go(causal=1, prefix=P) == UNSUPPORTED
    for bad in ("q", "k", "v", "out"):
        assert go(**{bad: _lib.TTHeadView(None, 64, 32)}) == NULL
        assert go(**{bad: _lib.TTHeadView(P + 4, 64, 32)}) == ALIGN
        assert go(**{bad: _lib.TTHeadView(P, 66, 32)}) == ALIGN
        assert go(**{bad: _lib.TTHeadView(P, 64, 34)}) == ALIGN
    assert go(lse=None) == NULL and go(cu_seqlens=None) == NULL
    assert go(T=0, lse=None) == 0
    if fn.endswith("bwd"):
        assert go(delta=None) == NULL
        for bad in ("dout", "dq", "dk", "dv"):
            assert go(**{bad: _lib.TTHeadView(None, 64, 32)}) == NULL and go(**{bad: _lib.TTHeadView(P + 8, 64, 32)}) == ALIGN


def test_softmax_loss_refusals(lib):
    def fwd(x=P, ldx=8, w=P, ldw=8, t=P, rid=None, cid=None, N=4, V=9, D=8, dt=1, scale=1.0, loss=P, lse=P, ws=P, n=1 << 22):
        return lib.tt_softmax_loss(x, ldx, w, ldw, t, rid, cid, N, V, D, dt, scale, -100, loss, lse, ws, n, None)

    def bwd(c=P, x=P, ldx=8, w=P, ldw=8, t=P, rid=None, cid=None, lse=P, N=4, V=9, D=8, dt=1, scale=1.0, dx=P, dw=P, ws=P, n=1 << 22):
        return lib.tt_softmax_loss_bwd(c, x, ldx, w, ldw, t, rid, cid, lse, N, V, D, dt, scale, -100, dx, dw, ws, n, None)

    for f in (fwd, bwd):
        assert f(dt=0) == DTYPE
        for bad in (dict(N=-1), dict(V=0), dict(D=0), dict(ldx=7), dict(ldw=7), dict(scale=0.0), dict(scale=float("nan"))):
            assert f(**bad) == SHAPE, bad
        for bad in (dict(x=None), dict(w=None), dict(t=None), dict(lse=None), dict(ws=None), dict(rid=P), dict(cid=P)):
            assert f(**bad) == NULL, bad
        assert f(n=0) == WS and f(ws=P + 4) == ALIGN
    assert fwd(loss=None) == NULL and bwd(c=None) == NULL and fwd(N=0, x=None) == 0


def test_workspaces_hold_no_logits(lib):
    """8192 rows x a million candidates: 32 GiB of fp32 logits; both passes work in a small part of that."""
    N, V, D = 8192, 1 << 20, 384
    logits = 4 * N * V
    assert lib.tt_softmax_loss_workspace_bytes(P, D, P, D, N, V, D, 1) < logits / 50
    assert lib.tt_softmax_loss_bwd_workspace_bytes(P, D, P, D, N, V, D, 1) < logits / 50


def test_sizes_beyond_a_tiles_offsets_are_refused(lib):
    """A tile's 32-bit offsets reach 256 packed rows of 2^22 elements."""
    big = 1 << 23
    assert linear(lib, K=big, ldx=big, ldw=big) == SHAPE and linear(lib, N=big, ldy=big) == SHAPE and linear(lib, M=(1 << 30) + 1) == SHAPE
    assert lib.tt_linear_act_bwd(P, big, P, 8, P, 8, None, P, P, P, 4, big, 8, 1, 0, P, 1 << 40, None) == SHAPE
    args = (P, big, P, big, P, None, None, 4, 9, big, 1, 1.0, -100)
    assert lib.tt_softmax_loss(*args, P, P, P, 1 << 40, None) == SHAPE
    assert lib.tt_softmax_loss_bwd(P, P, 8, P, 8, P, None, None, P, 4, (1 << 28) + 1, 8, 1, 1.0, -100, P, P, P, 1 << 60, None) == SHAPE
    assert lib.tt_packed_attention(attention_args(T=(1 << 30) + 1), None) == SHAPE
    assert lib.tt_packed_attention(attention_args(k=_lib.TTHeadView(P, 1 << 22, 32)), None) == ALIGN


@pytest.mark.parametrize("V", [8_400_000, 30_000_000, 1 << 28])
def test_float_gradient_rows_stay_within_a_tiles_offsets(lib, V):
    """Rows of float G as long as all candidates: no block of them is larger than a tile's 32-bit offsets reach."""
    D, N = 8, 1000
    need = lib.tt_softmax_loss_bwd_workspace_bytes(P, D, P, D, N, V, D, _lib.TT_F32)
    parts = 2 * ((V + 127) // 128 * 128 // 64)
    assert 0 < need <= 2 ** 32 * (1 + 1 / 32) + 2 ** 22 and need > 4 * V + parts  # G, its rows' partial sums, dx in parts


def test_struct_matches_the_header():
    assert C.sizeof(_lib.TTAttentionArgs) == 280 and C.sizeof(_lib.TTHeadView) == 24


@pytest.mark.parametrize("call", [
    lambda t: ops.linear_act(t, t), lambda t: ops.linear_act_bwd(t, t, t), lambda t: ops.softmax_loss(t, t, t),
    lambda t: ops.packed_attention(t.view(1, 4, 4), t.view(1, 4, 4), t.view(1, 4, 4), t)])
def test_no_cpu_fallback(call):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        call(torch.zeros(4, 4, dtype=torch.float64))


def test_ops_refuse_unknown_activations():
    with pytest.raises(ValueError, match="activation"):
        ops.linear_act(torch.zeros(4, 4), torch.zeros(4, 4), activation="swish")
