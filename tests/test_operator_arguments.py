"""CPU checks of the refusals of the log probabilities and the batch layout: the C entry
points return their status before anything is launched (the pointers are never
dereferenced), the Python ones refuse CPU tensors; the oracles on cases worked by hand."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from oracle import paged as OP

OK, EINVAL, EUNSUP, EWS = 0, -1, -2, -4
F32, BF16 = 0, 1
FAKE = ctypes.c_void_p(4096)


def test_token_logprobs_statuses():
    from specdec import _lib
    L = _lib.lib()

    def call(rows=2, V=1000, ld=1000, T=1.0, n=1, top=5, dtype=BF16, logits=FAKE, ws=FAKE, nbytes=None):
        need = L.sdx_token_logprobs_workspace(max(rows, 1), V, max(top, 0))
        return L.sdx_token_logprobs(logits, dtype, rows, V, ld, T, FAKE, n, top, FAKE, FAKE, FAKE,
                                    FAKE, ws, need if nbytes is None else nbytes, None)

    assert call(rows=0) == OK
    for bad in (dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")),
                dict(T=1e-44), dict(ld=999), dict(V=0), dict(top=-1), dict(V=4, ld=4, top=5),
                dict(dtype=7), dict(logits=None), dict(rows=-1),
                dict(logits=ctypes.c_void_p(4097))):
        assert call(**bad) == EINVAL, bad
    assert call(top=65) == EUNSUP and b"top_n" in L.sdx_last_error()
    assert call(rows=(1 << 23) + 1) == EUNSUP
    V = 151936
    need = L.sdx_token_logprobs_workspace(2, V, 5)
    assert need > 0
    assert call(V=V, ld=V, nbytes=need - 1) == EWS and call(V=V, ld=V, ws=None) == EWS
    assert L.sdx_token_logprobs_workspace(4096, V, 20) == 0  # a workgroup per row
    assert L.sdx_token_logprobs_workspace(0, V, 20) == 0


def test_layout_statuses():
    from specdec import _lib
    L = _lib.lib()

    def tables(batch=4, free=FAKE, nfree=8, bs=16, mb=4, cu=None, pre=None, G=0, out=FAKE):
        return L.sdx_build_block_tables(FAKE, batch, free, nfree, bs, mb, cu, pre, G, out, None,
                                        None, None)

    assert tables(batch=0) == OK
    for bad in (dict(batch=-1), dict(free=None), dict(bs=0), dict(mb=0), dict(out=None),
                dict(cu=FAKE, pre=None, G=1), dict(cu=FAKE, pre=FAKE, G=0), dict(nfree=-1)):
        assert tables(**bad) == EINVAL, bad
    assert tables(batch=1 << 24) == EUNSUP and tables(mb=1 << 28) == EUNSUP

    def slots(batch=4, mb=4, bs=16, T=3, pos=FAKE):
        return L.sdx_paged_slot_mapping(FAKE, batch, mb, FAKE, FAKE, bs, T, -1, pos, FAKE, None, None)

    assert slots(T=0) == OK
    for bad in (dict(batch=0), dict(mb=0), dict(bs=0), dict(T=-1), dict(pos=None)):
        assert slots(**bad) == EINVAL, bad
    assert slots(T=1 << 32) == EUNSUP

    def append(pool=FAKE, staged=FAKE, dtype=BF16, layers=2, T=3, re=64, ns=64, stride=4096):
        return L.sdx_append_slots(pool, 2 * stride, stride, staged, dtype, layers, T, re, ns, FAKE,
                                  None, None)

    assert append(T=0) == OK
    for bad in (dict(pool=None), dict(staged=None), dict(dtype=9), dict(layers=0), dict(T=-1),
                dict(re=0), dict(re=4), dict(ns=0), dict(staged=ctypes.c_void_p(4104)),
                dict(stride=4100)):
        assert append(**bad) == EINVAL, bad
    assert append(layers=40000) == EUNSUP and append(T=1 << 40) == EUNSUP


def test_prefix_attention_statuses():
    from specdec import _lib
    L = _lib.lib()

    def call(T=3, B=2, hq=4, hkv=2, d=64, dtype=BF16, nb=8, bs=16, mb=4, G=1, scale=0.1, q=FAKE,
             pool=FAKE, out=FAKE, ws=FAKE, nbytes=None):
        need = L.sdx_prefix_attention_workspace(max(T, 1), max(B, 1), max(G, 1), max(hq, 1),
                                                max(hkv, 1), d)
        return L.sdx_prefix_attention_paged(q, dtype, T, B, FAKE, hq, hkv, d, pool, FAKE, nb, bs, FAKE,
                                            mb, FAKE, FAKE, FAKE, G, scale, ws,
                                            need if nbytes is None else nbytes, out, None, None)

    assert call(T=0) == OK
    off = ctypes.c_void_p(4104)
    for bad in (dict(T=-1), dict(B=-1), dict(B=0), dict(G=0), dict(hq=0), dict(hq=3), dict(hkv=0),
                dict(bs=0), dict(mb=0), dict(nb=0), dict(scale=0.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(q=None), dict(out=None), dict(q=off), dict(pool=off),
                dict(out=off)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(d=96), dict(d=256), dict(dtype=F32), dict(mb=1 << 28), dict(nb=1 << 29),
                dict(T=1 << 24)):
        assert call(**bad) == EUNSUP, bad
    need = L.sdx_prefix_attention_workspace(3, 2, 1, 4, 2, 64)
    assert call(nbytes=need - 1) == EWS and call(ws=None) == EWS and call(ws=off) == EWS
    assert L.sdx_prefix_attention_workspace(0, 2, 1, 4, 2, 64) == 0
    assert L.sdx_prefix_attention_workspace(3, 2, 1, 4, 3, 64) == 0
    # two parts at least, and no more room than for two where queries are many
    assert L.sdx_prefix_attention_workspace(1 << 16, 9, 1, 32, 8, 128) >= 2 * (1 << 21) * 130 * 4
    assert L.sdx_prefix_attention_workspace(640, 128, 1, 32, 8, 128) <= 200 << 20


def test_entry_points_refuse_cpu_tensors():
    from specdec import attention as A
    from specdec import kvcache as K
    from specdec import sampling as S
    z = torch.zeros(2, dtype=torch.long)
    for call in (lambda: S.token_logprobs(torch.zeros(2, 8), z),
                 lambda: K.build_block_tables(z, z, 16, 2),
                 lambda: K.paged_slot_mapping(z.view(1, 2), z, z[:1], 16, 1),
                 lambda: A.shared_prefix_attention_paged(*[z] * 8),
                 lambda: K.append_paged_slots(torch.zeros(1, 2, 1, 1, 8), torch.zeros(1, 2, 2, 8), z)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_oracles_by_hand():
    # two groups: rows 0-2 share 20 tokens (one page of 16), row 3 alone
    t, used, ok = OP.build_block_tables([40, 20, 10, 17], [9, 8, 7, 6, 5, 4, 3], 16, 3, [0, 3, 4],
                                        [20, 0])
    assert ok and used == 6
    assert t.tolist() == [[9, 8, 7], [9, 6, -1], [9, -1, -1], [5, 4, -1]]
    pos, slots, ok = OP.slot_mapping(t, [0, 2, 2, 3, 5], [40, 20, 10, 17], 16, 6)
    assert ok and pos.tolist() == [38, 39, 9, 15, 16, 0]
    assert slots.tolist() == [7 * 16 + 6, 7 * 16 + 7, 9 * 16 + 9, 5 * 16 + 15, 4 * 16, -1]
    x = np.log(np.array([[0.5, 0.25, 0.25]]))
    logp, ent, top, ids = OL.token_logprobs(x, np.array([[1, 3]]), 1.0, 3)
    assert np.allclose(logp[0, 0], np.log(0.25)) and logp[0, 1] == -np.inf
    assert np.allclose(ent, 1.5 * np.log(2)) and ids.tolist() == [[0, 1, 2]]
