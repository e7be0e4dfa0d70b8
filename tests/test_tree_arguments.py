"""CPU checks of the refusals of the trees' and pages' entry points: the C ones return their status
before anything is launched (the pointers are never dereferenced), the Python ones refuse CPU
tensors; the oracles on cases worked by hand."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import tree as OT

OK, EINVAL, EUNSUP, EWS = 0, -1, -2, -4
F32, BF16 = 0, 1
FAKE = ctypes.c_void_p(4096)
OFF = ctypes.c_void_p(4104)


def test_tree_statuses():
    from specdec import _lib
    L = _lib.lib()

    def layout(B=2, nodes=26, table=FAKE, mb=4, bs=16, T=9, slots=FAKE, parents=FAKE, mask=FAKE):
        return L.sdx_tree_layout(parents, B, FAKE, FAKE, nodes, table, mb, bs, T, -1, mask, FAKE, slots, None,
                                 None)

    assert layout(T=0) == OK
    for bad in (dict(B=-1), dict(B=0), dict(nodes=0), dict(mb=0), dict(bs=0), dict(T=-1), dict(parents=None),
                dict(mask=None), dict(slots=None), dict(table=None)):
        assert layout(**bad) == EINVAL, bad
    for bad in (dict(nodes=513), dict(B=1 << 24), dict(mb=1 << 32), dict(T=1 << 32)):
        assert layout(**bad) == EUNSUP, bad

    def accept(B=2, T=9, P=4, tokens=FAKE, path=FAKE):
        return L.sdx_tree_accept(tokens, FAKE, FAKE, B, FAKE, T, None, P, path, FAKE, FAKE, None, None)

    assert accept(B=0) == OK
    for bad in (dict(B=-1), dict(T=-1), dict(P=0), dict(tokens=None), dict(path=None)):
        assert accept(**bad) == EINVAL, bad
    assert accept(P=513) == EUNSUP and accept(B=1 << 24) == EUNSUP


def test_page_statuses():
    from specdec import _lib
    L = _lib.lib()

    def compact(pool=FAKE, dtype=BF16, layers=2, re=64, nb=8, bs=16, table=FAKE, B=2, mb=4, P=4, stride=4096):
        return L.sdx_compact_paged(pool, 2 * stride, stride, dtype, layers, re, nb, bs, table, B, mb, FAKE,
                                   FAKE, P, FAKE, None, None, None)

    def copy(pool=FAKE, dtype=BF16, layers=2, re=64, nb=8, bs=16, n=3, copies=FAKE, stride=4096):
        return L.sdx_copy_pages(pool, 2 * stride, stride, dtype, layers, re, nb, bs, copies, n, None, None)

    assert compact(B=0) == OK and copy(n=0) == OK
    shared = (dict(pool=None), dict(dtype=5), dict(layers=0), dict(re=0), dict(re=4), dict(nb=0), dict(bs=0),
              dict(pool=OFF), dict(stride=4100))
    for bad in shared + (dict(table=None), dict(B=-1), dict(mb=0), dict(P=0)):
        assert compact(**bad) == EINVAL, bad
    for bad in shared + (dict(copies=None), dict(n=-1)):
        assert copy(**bad) == EINVAL, bad
    for bad in (dict(layers=40000), dict(re=1 << 30), dict(P=513), dict(B=1 << 24)):
        assert compact(**bad) == EUNSUP, bad
    assert copy(n=1 << 24) == EUNSUP and copy(re=1 << 30) == EUNSUP

    def free(table=FAKE, B=2, mb=4, bs=16, nb=100, out=FAKE, ws=FAKE, nbytes=None):
        need = L.sdx_free_pages_workspace(B, mb, nb)
        return L.sdx_free_pages(table, B, mb, FAKE, bs, nb, out, FAKE, ws, need if nbytes is None else nbytes,
                                None, None)

    for bad in (dict(table=None), dict(B=-1), dict(mb=0), dict(bs=0), dict(nb=0), dict(out=None)):
        assert free(**bad) == EINVAL, bad
    assert free(nb=1 << 31) == EUNSUP and free(B=1 << 20, mb=1 << 20) == EUNSUP
    assert L.sdx_free_pages_workspace(2, 4, 100) >= 16
    assert free(nbytes=3) == EWS and free(ws=None) == EWS and free(ws=OFF) == EWS

    def fork(table=FAKE, B=2, mb=4, N=3, bs=16, fb=FAKE, nf=8, out=ctypes.c_void_p(8192), copies=FAKE, ws=FAKE,
             nbytes=None):
        need = L.sdx_fork_block_tables_workspace(N)
        return L.sdx_fork_block_tables(table, B, mb, FAKE, FAKE, FAKE, N, bs, fb, nf, None, out, copies, FAKE,
                                       ws, need if nbytes is None else nbytes, None, None)

    assert fork(N=0) == OK
    for bad in (dict(table=None), dict(B=-1), dict(N=-1), dict(mb=0), dict(bs=0), dict(fb=None), dict(nf=-1),
                dict(out=None), dict(copies=None), dict(out=FAKE)):
        assert fork(**bad) == EINVAL, bad
    assert fork(N=1 << 24) == EUNSUP and fork(mb=1 << 28) == EUNSUP
    assert fork(nbytes=3) == EWS and fork(ws=None) == EWS


def test_entry_points_refuse_cpu_tensors():
    from specdec import kvcache as K
    from specdec import tree as R
    z, i = torch.zeros(2, dtype=torch.long), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 2, 1, 1, 8)
    for call in (lambda: R.tree_layout(i, z, z[:1]),
                 lambda: R.tree_accept(z, i, z, z, 4),
                 lambda: K.compact_paged(pool, i.view(1, 2), z[:1], z.view(1, 2), z[:1]),
                 lambda: K.free_page_list(i.view(1, 2), 4),
                 lambda: K.fork_block_tables(i.view(1, 2), z[:1], z, z, i, 16),
                 lambda: K.copy_pages(pool, torch.zeros(3, 1, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_oracles_by_hand():
    #      0          two children of the root, one of which has a child; a row of one node
    #     / \.
    #    1   2 - 3
    parents, cu = [-1, 0, 0, 2, -1], [0, 4, 5]
    table = np.array([[3, 1], [0, 2]])
    sees, pos, slots, ok = OT.tree_layout(parents, cu, [18, 1], table, 16, 1, 6)
    assert ok and sees == [{0}, {0, 1}, {0, 2}, {0, 2, 3}, {0}, set()]
    assert pos.tolist() == [14, 15, 15, 16, 0, 0]
    assert slots.tolist() == [3 * 16 + 14, 3 * 16 + 15, 16, 17, 0, -1]
    path, keep, y = OT.tree_accept([9, 5, 7, 8, 4], parents, [7, 1, 8, 6, 2], cu, 4)
    assert path.tolist() == [[0, 2, 3, -1], [0, -1, -1, -1]]
    assert keep.tolist() == [3, 1] and y.tolist() == [6, 2]
    pool = torch.arange(4 * 16.).view(1, 1, 4, 16, 1).expand(1, 2, 4, 16, 1).clone()
    assert OT.compact(pool, table, [14, 0], path, keep)
    assert pool[0, 0, 3, 14:, 0].tolist() == [62.0, 16.0] and pool[0, 0, 1, :2, 0].tolist() == [17.0, 17.0]
    assert OT.free_pages(np.array([[1, 5], [1, -1]]), 6, [20, 3], 16) == ([0, 2, 3, 4], True)
    # row 0 branches in two and row 1 ends: the branch takes a copy of 4 tokens of page 5
    out, copies, used, ok = OT.fork(np.array([[1, 5], [2, -1]]), [20, 3], [0, 0, -1], [21, 32, 0], [7, 8], 16)
    assert ok and used == 1 and out.tolist() == [[1, 5], [1, 7], [-1, -1]]
    assert copies.tolist() == [[-1, 5, -1], [-1, 7, -1], [0, 4, 0]]


def test_penalty_statuses():
    from specdec import _lib
    L = _lib.lib()
    far = ctypes.c_void_p(1 << 30)

    def call(logits=FAKE, dtype=BF16, R=4, V=100, ld=100, out=far, old=100, B=2, cu=FAKE, hist=FAKE, hld=50, H=50,
             hlen=FAKE, bi=FAKE, nb=3, al=FAKE, ald=4, tok=FAKE, mask=FAKE, words=1):
        return L.sdx_penalize_logits(logits, dtype, R, V, ld, out, old, B, cu, hist, hld, H, hlen, None, None, None,
                                     None, bi, FAKE, nb, al, ald, tok, mask, words, None, None)

    assert call(R=0) == OK
    for bad in (dict(logits=None), dict(out=None), dict(dtype=4), dict(R=-1), dict(V=0), dict(ld=99), dict(old=99),
                dict(B=-1), dict(B=0), dict(cu=None), dict(hlen=None), dict(hld=49), dict(bi=None), dict(nb=-1),
                dict(ald=3), dict(tok=None), dict(words=0), dict(words=-1), dict(logits=ctypes.c_void_p(4097)),
                dict(out=ctypes.c_void_p(4098)), dict(out=ctypes.c_void_p(4096), old=101)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(nb=1025), dict(H=1 << 20, hld=1 << 20), dict(R=(1 << 21) + 1, cu=FAKE),
                dict(V=(1 << 30) + 1, ld=1 << 31, old=1 << 31, ald=1 << 30, R=1)):
        assert call(**{"out": ctypes.c_void_p(1 << 50), **bad}) == EUNSUP, bad


def test_penalties_refuse_cpu_tensors():
    from specdec import sampling as S
    with pytest.raises(RuntimeError, match="ROCm device"):
        S.penalize_logits(torch.zeros(2, 8))


def test_penalty_oracle_by_hand():
    from oracle import penalties as PN
    x = np.array([[2.0, -2.0, 1.0, 0.5], [2.0, -2.0, 1.0, 0.5]])
    out, _, touched = PN.penalize(x, np.array([[0, 1, 1, 3]]), [3], [0, 2], prompt_len=[1], repetition=[2.0],
                                  frequency=[0.25], presence=[1.0], bias_ids=np.array([[2, 2, 9]]),
                                  bias=np.array([[1.0, 0.5, 7.0]]), node_tokens=[0, 3],
                                  allowed=np.array([[15], [13]], dtype=np.int32))
    # row 0 saw 0 (prompt and path), 1 twice; row 1 token 3 too, and may not go on with 1
    assert out[0].tolist() == [1.0 - 0.25 - 1.0, -4.0 - 0.5 - 1.0, 2.5, 0.5]
    assert out[1].tolist() == [-0.25, -np.inf, 2.5, 0.25 - 0.25 - 1.0]
    assert touched.tolist() == [[True, True, True, False], [True] * 4]


def test_tree_attention_statuses():
    from specdec import _lib
    L = _lib.lib()

    def call(T=3, B=2, hq=4, hkv=2, d=64, dtype=BF16, nb=8, bs=16, mb=4, words=1, scale=0.1, q=FAKE, pool=FAKE,
             mask=FAKE, out=FAKE, ws=FAKE, nbytes=None):
        need = L.sdx_tree_attention_workspace(max(T, 1), max(B, 1), max(hq, 1), max(hkv, 1), d)
        return L.sdx_tree_attention_paged(q, dtype, T, B, FAKE, hq, hkv, d, pool, FAKE, nb, bs, FAKE, mb, FAKE,
                                          mask, words, scale, ws, need if nbytes is None else nbytes, out, None,
                                          None)

    assert call(T=0) == OK
    for bad in (dict(T=-1), dict(B=-1), dict(B=0), dict(hq=0), dict(hq=3), dict(hkv=0), dict(bs=0), dict(mb=0),
                dict(nb=0), dict(words=0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(scale=3e38), dict(q=None), dict(mask=None), dict(out=None), dict(q=OFF), dict(pool=OFF),
                dict(out=OFF)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(d=96), dict(d=256), dict(dtype=F32), dict(mb=1 << 28), dict(nb=1 << 29), dict(T=1 << 24)):
        assert call(**bad) == EUNSUP, bad
    need = L.sdx_tree_attention_workspace(3, 2, 4, 2, 64)
    assert call(nbytes=need - 1) == EWS and call(ws=None) == EWS and call(ws=OFF) == EWS
    assert L.sdx_tree_attention_workspace(0, 2, 4, 2, 64) == 0
    assert L.sdx_tree_attention_workspace(3, 2, 4, 3, 64) == 0
    # two parts a workgroup, however many nodes there are
    assert L.sdx_tree_attention_workspace(1 << 16, 2048, 32, 8, 128) <= 80 << 20
