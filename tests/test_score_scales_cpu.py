"""CPU: scales and caps of scores that leave float32's range are refused, at the C entry (no launch happens)."""
import pytest

import two_towers_overlords_amd as pkg
from two_towers_overlords_amd import _lib, ops

SHAPE, WS, NULL = -2, -5, -1
P = 4096


@pytest.mark.parametrize("scale,ok", [(1e39, False), (float("inf"), False), (2e15, False), (1e15, True), (1.0, True), (1e-15, True), (9e-16, False),
                                      (1e-46, False), (0.0, False), (-1.0, False), (float("nan"), False)])
def test_scales(scale, ok):
    lib = pkg.load()
    args = (P, 8, P, 8, P, None, None, 4, 9, 8, 1, scale, -100)
    assert lib.tt_softmax_loss(*args, P, P, P, 0, None) == (WS if ok else SHAPE)
    assert lib.tt_softmax_loss_bwd(P, P, 8, P, 8, P, None, None, P, 4, 9, 8, 1, scale, -100, P, P, P, 0, None) == (WS if ok else SHAPE)
    for name in ("scale", "softcap"):
        a = _lib.TTAttentionArgs()
        a.T, a.docs, a.heads, a.kv_heads, a.head_dim, a.dtype, a.scale = 10, 1, 2, 2, 32, 1, 0.5
        setattr(a, name, scale)
        want = NULL if ok or (name == "softcap" and a.softcap == 0.0) else SHAPE  # what comes next is refused for its null pointers
        assert lib.tt_packed_attention(a, None) == want and lib.tt_packed_attention_bwd(a, None) == want
    assert ops._scale_ok(scale) == ok
