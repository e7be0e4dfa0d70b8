"""Block tables of batches of more rows than one round of workgroups: each takes several rows. The
tables are whole values, equal to those of the same formula in numpy; the time is in proportion to
the rows, not to their square."""
import numpy as np
import pytest
import torch

from oracle import paged as OP
from specdec.kvcache import build_block_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int64), device=DEV)


def tables(kv, free, bs, mb, cu, pre):
    """oracle.paged.build_block_tables of batches that fit, over whole arrays."""
    B = len(kv)
    first = np.repeat(cu[:-1], np.diff(cu))
    need = -(-kv // bs)
    shared = np.where(first == np.arange(B), 0, np.minimum(np.repeat(pre, np.diff(cu)) // bs, need))
    own = need - shared
    at = np.cumsum(own) - own
    col = np.arange(mb)
    src = np.where(col < shared[:, None], at[first][:, None] + col, (at - shared)[:, None] + col)
    return np.where(col < need[:, None], free[np.clip(src, 0, len(free) - 1)], -1), int(own.sum())


def batch(rng, B, per, prefix, own):
    cuts = np.sort(rng.integers(0, B + 1, B // per))     # groups of any size, empty ones too
    cu = np.concatenate([[0], cuts, [B]])
    pre = rng.integers(0, prefix + 1, len(cu) - 1)
    first = np.repeat(cu[:-1], np.diff(cu))
    kv = np.repeat(pre, np.diff(cu)) + rng.integers(0, own + 1, B)
    cut = (rng.random(B) < 0.2) & (first != np.arange(B))  # rows shorter than the prefix
    kv[cut] = rng.integers(0, kv.max() + 1, cut.sum())
    return cu, pre, kv


@pytest.mark.parametrize("B,per,prefix,own,bs", [
    (2047, 5, 60, 30, 16), (2048, 3, 60, 30, 16), (2049, 3, 60, 30, 16), (4097, 700, 60, 30, 8),
    (6145, 1, 20, 30, 16), (9001, 4000, 300, 30, 7), (20000, 5000, 40, 9, 1),
])
def test_several_rows_of_a_workgroup(B, per, prefix, own, bs):
    rng = np.random.default_rng(B)
    cu, pre, kv = batch(rng, B, per, prefix, own)
    mb = int(-(-kv.max() // bs)) + 1
    free = rng.permutation(int(np.sum(-(-kv // bs)))).astype(np.int32)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for grouped in (True, False):
        g = (cu, pre) if grouped else (None, None)
        want, used, ok = OP.build_block_tables(kv, free, bs, mb, *g)
        assert ok
        if grouped:
            assert np.array_equal(tables(kv, free, bs, mb, cu, pre)[0], want)
        args = (dev(cu), dev(pre)) if grouped else (None, None)
        for n in (used, used - 1):                       # enough pages, and one too few
            t, u = build_block_tables(dev(kv), torch.as_tensor(free[:n], device=DEV), bs, mb, *args,
                                      error=err)
            assert np.array_equal(t.cpu().numpy(), want if n == used else np.full_like(want, -1))
            assert u.item() == (used if n == used else 0) and err.item() == (n != used)
        err.zero_()
    # a bad row at the end of some workgroup's
    kv[B - 2] = -1
    t, u = build_block_tables(dev(kv), torch.as_tensor(free, device=DEV), bs, mb, dev(cu), dev(pre), error=err)
    assert (t == -1).all() and u.item() == 0 and err.item() == 1


def test_a_million_rows_in_proportion():
    """2^20 rows. With every row's workgroup adding up all rows, 131,072 took 92 ms and these would
    take 64 times that; a tenth of a second is a sixtieth."""
    rng = np.random.default_rng(1)
    B = 1 << 20
    cu, pre, kv = batch(rng, B, 8, 40, 20)
    mb = int(-(-kv.max() // 16)) + 1
    free = rng.permutation(int(np.sum(-(-kv // 16)))).astype(np.int32)
    want, used = tables(kv, free, 16, mb, cu, pre)
    args = (dev(kv), torch.as_tensor(free, device=DEV), 16, mb, dev(cu), dev(pre))
    t, u = build_block_tables(*args)
    assert torch.equal(t.cpu(), torch.as_tensor(want.astype(np.int32))) and u.item() == used
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    build_block_tables(*args)
    b.record()
    torch.cuda.synchronize()
    assert a.elapsed_time(b) < 100, a.elapsed_time(b)
