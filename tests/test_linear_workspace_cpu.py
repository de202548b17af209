"""CPU: the workspace of linear_act_bwd holds what the wanted gradients need, at the C entry (no launch happens)."""
import two_towers_overlords_amd as pkg
from two_towers_overlords_amd import _lib

P = 4096  # a 16-byte aligned address that no refused call touches
WS = -5


def test_only_the_wanted_gradients_are_counted():
    lib = pkg.load()
    M, N, K = 8192, 512, 256

    def need(x, w, ld=K, act=0):
        return lib.tt_linear_act_bwd_workspace_bytes(P, N, x, ld, w, ld, M, N, K, _lib.TT_F32, act)

    def call(dx, dw, db, n, ld=K, act=0):
        return lib.tt_linear_act_bwd(P, N, P, ld, P, ld, P, dx, dw, db, M, N, K, _lib.TT_F32, act, P, n, None)

    slab = 4 * N * K  # dw's contraction over 8192 rows is split: parts of N x K
    assert need(P, P) >= need(None, P) + 2 * slab
    # rows that are not whole 16-byte chunks are copied, for the product that reads them
    odd = K + 1
    assert need(None, P, odd) == need(None, P) + 4 * N * K and need(P, None, odd) == need(P, None) + 4 * M * K
    # dz is formed for the products, not for dbias
    assert need(None, None, act=2) == need(None, None) and need(None, P, act=2) == need(None, P) + 4 * M * N
    for dx, dw, x, w in ((P, None, None, P), (None, P, P, None), (P, P, P, P), (None, None, None, None)):
        for ld, act in ((K, 0), (odd, 0), (K, 2)):
            assert call(dx, dw, P, need(x, w, ld, act) - 1, ld, act) == WS
