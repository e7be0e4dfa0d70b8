"""GPU parity of the cache's page operators with the row-by-row oracle: copies and whole numbers,
equal bit for bit."""
import numpy as np
import pytest
import torch

from oracle import tree as OT
from specdec.kvcache import (PagedKVCache, compact_paged, copy_pages, fork_block_tables,
                             free_page_list)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x, dtype=None):
    return torch.as_tensor(np.asarray(x), device=DEV, dtype=dtype)


def new_error():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def make_pool(seed, L, nb, bs, re, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((L, 2, nb, bs, re), generator=g, device=DEV).to(dtype)


def paths(rng, ns, P):
    """Ascending paths of nodes, with how many are kept."""
    path = np.full((len(ns), P), -7, dtype=np.int64)     # behind keep: anything
    keep = np.zeros(len(ns), dtype=np.int64)
    for b, n in enumerate(ns):
        k = int(rng.integers(0, min(n, P) + 1))
        keep[b] = k
        path[b, :k] = np.sort(rng.permutation(n)[:k])
        if b % 3 == 0 and k:
            path[b, :k] += -path[b, 0]                   # from node 0
    return path, keep


@pytest.mark.parametrize("L,ns,P,bs,re,dtype", [
    (1, [1], 1, 16, 8, torch.bfloat16),
    (3, [26, 0, 64, 5], 16, 16, 256, torch.bfloat16),
    (5, [512, 300, 9], 512, 16, 64, torch.float16),
    (4, [30] * 40, 30, 1, 24, torch.float32),
    (2, [40, 17, 64, 3, 12], 9, 7, 1032, torch.float16),
    (7, [64, 50, 33], 64, 32, 1024, torch.bfloat16),
])
def test_compact(L, ns, P, bs, re, dtype):
    rng = np.random.default_rng(sum(ns) + L)
    B = len(ns)
    start = rng.integers(0, 3 * bs, B)
    mb = int(max(-(-(start + np.asarray(ns)) // bs))) + 1
    nb = B * mb + 2
    table = rng.permutation(nb)[:B * mb].reshape(B, mb)
    path, keep = paths(rng, ns, P)
    pool = make_pool(1, L, nb, bs, re, dtype)
    want = pool.cpu().clone()
    assert OT.compact(want, table, start, path, keep)
    err = new_error()
    compact_paged(pool, dev(table, torch.int32), dev(start), dev(path), dev(keep), error=err)
    assert torch.equal(pool.cpu(), want) and err.item() == 0


def test_compact_refuses_rows():
    """Rows out of range stay as they are, whole; the others move."""
    rng = np.random.default_rng(5)
    bs, mb, B, P = 16, 3, 9, 4
    table = rng.permutation(B * mb).reshape(B, mb)
    start = np.full(B, 20)
    path = np.tile([0, 2, 5, 9], (B, 1))
    keep = np.full(B, 4)
    path[1] = [0, 2, 2, 3]
    path[2] = [-1, 2, 3, 4]
    path[3] = [0, 1, 2, mb * bs]
    keep[4] = P + 1
    keep[5] = -1
    start[6] = -3
    table[7, 1] = -1
    table[8, 1] = B * mb
    pool = make_pool(2, 2, B * mb, bs, 64, torch.bfloat16)
    before, want = pool.clone(), pool.cpu().clone()
    assert not OT.compact(want, table, start, path, keep)
    err, kept = new_error(), dev([9] * B)
    compact_paged(pool, dev(table, torch.int32), dev(start), dev(path), dev(keep), kept=kept, error=err)
    assert err.item() == 1 and torch.equal(pool.cpu(), want) and not torch.equal(pool, before)
    assert kept.tolist() == [4] + [0] * 8
    # without an error word nothing else happens either
    pool2 = before.clone()
    compact_paged(pool2, dev(table, torch.int32), dev(start), dev(path), dev(keep))
    assert torch.equal(pool2, pool)


def test_cache_method_moves_and_commits():
    c = PagedKVCache(2, 2, 8, 16, 1, 64, 4)
    c.pool.normal_()
    c.block_table.copy_(dev([[5, 1, 0, -1], [2, 7, -1, -1]], torch.int32))
    c.lengths.copy_(dev([30, 3]))
    want = c.pool.clone()
    path, keep = dev([[0, 3, 4], [0, 1, -1]]), dev([3, 2])
    assert OT.compact(want, c.block_table.cpu().numpy(), [30, 3], path.cpu().numpy(), [3, 2])
    c.compact(path, keep)
    assert torch.equal(c.pool, want) and c.lengths.tolist() == [33, 5] and c.error.item() == 0
    c.compact(dev([[0, 1, 2], [0, 1, 1]]), dev([0, 3]))       # nothing of row 0, row 1 is refused
    assert torch.equal(c.pool, want) and c.lengths.tolist() == [33, 5] and c.error.item() == 1


@pytest.mark.parametrize("B,mb,nb,bs,lengths", [
    (1, 1, 1, 16, True), (1, 1, 1, 16, False), (3, 5, 31, 16, True), (3, 5, 33, 7, False),
    (64, 300, 20011, 16, True), (700, 90, 63001, 8, True), (5, 40, 8192, 16, False),
    (2, 3, 8193, 16, True), (4, 2000, 600007, 16, True), (0, 4, 40, 16, True),
    # the ends of the form of one kernel
    (23, 89, 16384, 16, True), (23, 89, 16385, 16, True), (32, 64, 16384, 16, False), (1, 5, 16383, 16, False),
])
def test_free_pages(B, mb, nb, bs, lengths):
    rng = np.random.default_rng(B + nb)
    table = rng.integers(0, nb, (B, mb))                # pages may be held several times
    kv = rng.integers(0, mb * bs + 1, B)
    if B > 2:
        kv[1] = 0
    col = np.arange(mb)
    table = np.where(col < (-(-kv // bs))[:, None], table, rng.choice([-1, -5, nb + 3], (B, mb))
                     if lengths else -1)
    ids, ok = OT.free_pages(table, nb, kv if lengths else None, bs)
    assert ok
    err = new_error()
    free, num = free_page_list(dev(table, torch.int32), nb, kv_len=dev(kv) if lengths else None,
                               block_size=bs if lengths else None, error=err)
    assert num.tolist() == [len(ids)] and err.item() == 0
    assert free.tolist() == ids + [-1] * (nb - len(ids))


def test_free_pages_reports():
    kv = dev([20, 3])
    for table, kvl in (([[1, 9], [0, -1]], kv), ([[1, -1], [0, -1]], kv),
                       ([[1, 2], [0, -1]], dev([20, 33])), ([[1, 2], [0, -1]], dev([20, -1]))):
        err = new_error()
        free_page_list(dev(table, torch.int32), 4, kv_len=kvl, block_size=16, error=err)
        assert err.item() == 1


def random_tables(rng, B, mb, nb, bs, kv):
    """Rows that share their first pages in runs, each page at one column."""
    ids = iter(rng.permutation(nb))
    table = np.full((B, mb), -1)
    for b in range(B):
        need = -(-int(kv[b]) // bs)
        same = 0
        if b and rng.random() < 0.7:                    # as deep as both have whole pages
            same = int(rng.integers(0, min(int(kv[b]), int(kv[b - 1])) // bs + 1))
            table[b, :same] = table[b - 1, :same]
        for c in range(same, need):
            table[b, c] = next(ids)
    return table


@pytest.mark.parametrize("B,N,mb,bs", [(1, 1, 1, 16), (1, 9, 4, 16), (6, 6, 5, 7), (40, 33, 12, 16),
                                       (3, 200, 9, 1), (130, 300, 30, 32), (5, 0, 3, 16),
                                       # the ends of the form of one workgroup
                                       (9, 16, 512, 3), (9, 17, 512, 3), (9, 16, 513, 3), (30, 15, 40, 16)])
def test_fork(B, N, mb, bs):
    rng = np.random.default_rng(B + N)
    kv = rng.integers(0, mb * bs + 1, B)
    kv[0] = min(kv[0] | 1, mb * bs)
    nb = B * mb + N * mb + 1
    table = random_tables(rng, B, mb, nb, bs, kv)
    parent = rng.integers(-1, B, N)
    old = np.where(parent >= 0, kv[np.maximum(parent, 0)], 0)
    room = np.minimum(old + rng.integers(0, 2 * bs + 1, N), mb * bs)
    ids, ok = OT.free_pages(table, nb, kv, bs)
    assert ok
    want, copies, used, ok = OT.fork(table, kv, parent, room, ids, bs)
    assert ok
    err = new_error()
    bt = dev(table, torch.int32)
    free, num = free_page_list(bt, nb, kv_len=dev(kv), block_size=bs)
    got, gc, gu = fork_block_tables(bt, dev(kv), dev(parent), dev(room), free, bs, num_free=num, error=err)
    assert err.item() == 0 and gu.tolist() == [used]
    assert got.tolist() == want.tolist() and gc.tolist() == copies.tolist()
    assert bt.tolist() == table.tolist()
    # the pages exactly, without a count on the device, into given tables
    out = torch.full((N, mb), 9, dtype=torch.int32, device=DEV)
    got, gc, gu = fork_block_tables(bt, dev(kv), dev(parent), dev(room), dev(ids[:used], torch.int32), bs,
                                    out=out, error=err)
    assert err.item() == 0 and got is out and got.tolist() == want.tolist() and gu.tolist() == [used]
    if used:                                             # one page short
        got, gc, gu = fork_block_tables(bt, dev(kv), dev(parent), dev(room),
                                        dev(ids[:used - 1], torch.int32), bs, error=err)
        assert err.item() == 1 and gu.tolist() == [0] and (got == -1).all()
        assert (gc[:2] == -1).all() and (gc[2] == 0).all()
        err.zero_()
        fork_block_tables(bt, dev(kv), dev(parent), dev(room), free, bs, num_free=num * 0 + used - 1,
                          error=err)
        assert err.item() == 1


def test_fork_of_a_page_that_another_row_holds_whole():
    """Two old rows share a page that one of them fills in part only (it was rolled back): the row
    that goes on from it takes a copy, wherever it stands."""
    table = np.array([[4, 2, -1], [4, 9, -1]])
    kv = np.array([10, 20])                              # row 0 ends inside page 4, row 1 holds it
    for parent in ([0, 1], [1, 0]):
        old = kv[parent]
        want, copies, used, ok = OT.fork(table, kv, parent, old + 1, [7, 8], 16)
        assert ok and used == 1 and copies[0].max() == 4
        got, gc, gu = fork_block_tables(dev(table, torch.int32), dev(kv), dev(parent), dev(old + 1),
                                        dev([7, 8], torch.int32), 16)
        assert got.tolist() == want.tolist() and gc.tolist() == copies.tolist() and gu.item() == 1


def test_fork_refuses():
    table, kv = np.array([[0, 1], [2, -1]]), np.array([20, 5])
    good = dict(kv=kv, parent=[0, 1, -1], room=[21, 5, 3], table=table)
    bad = [dict(parent=[0, 2, -1]), dict(parent=[0, -2, -1]), dict(room=[19, 5, 3]),
           dict(room=[33, 5, 3]), dict(room=[21, 5, -1]), dict(kv=np.array([33, 5])),
           dict(kv=np.array([20, -5])), dict(table=np.array([[0, -1], [2, -1]])),
           dict(table=np.array([[-1, 1], [2, -1]]))]
    for change in [{}] + bad:
        c = {**good, **change}
        want, copies, used, ok = OT.fork(c["table"], c["kv"], c["parent"], c["room"], [7, 8, 9], 16)
        assert ok == (not change)
        err = new_error()
        got, gc, gu = fork_block_tables(dev(c["table"], torch.int32), dev(c["kv"]), dev(c["parent"]),
                                        dev(c["room"]), dev([7, 8, 9], torch.int32), 16, error=err)
        assert err.item() == (0 if ok else 1) and got.tolist() == want.tolist()
        assert gc.tolist() == copies.tolist() and gu.item() == used


@pytest.mark.parametrize("L,nb,bs,re,dtype", [(1, 5, 16, 8, torch.bfloat16), (3, 40, 7, 264, torch.float16),
                                              (9, 64, 16, 1024, torch.float32), (5, 30, 1, 16, torch.bfloat16)])
def test_copy_pages(L, nb, bs, re, dtype):
    rng = np.random.default_rng(L)
    pages = rng.permutation(nb)
    n = nb // 2
    copies = np.stack([rng.choice(pages[n:], n), pages[:n], rng.integers(0, bs + 1, n)])  # a source twice
    copies[0, rng.random(n) < 0.3] = -1
    pool = make_pool(3, L, nb, bs, re, dtype)
    want = pool.clone()
    for s, d, t in copies.T:
        if s >= 0 and d >= 0:
            want[:, :, d, :t] = want[:, :, s, :t]
    err = new_error()
    copy_pages(pool, dev(copies, torch.int32), error=err)
    assert torch.equal(pool, want) and err.item() == 0
    for entry in ([nb, 0, 1], [0, nb, 1], [0, 1, bs + 1], [0, 1, -1]):
        err = new_error()
        copy_pages(pool, dev([[x] for x in entry], torch.int32), error=err)
        assert torch.equal(pool, want) and err.item() == 1


def test_beams_as_a_graph():
    """Free pages, tables and copies of a beam step, captured and replayed with other parents; what
    the new rows read is what their parents held."""
    rng = np.random.default_rng(4)
    B, mb, bs, L, re = 12, 6, 16, 3, 64
    nb = 3 * B * mb
    kv = rng.integers(1, (mb - 1) * bs, B)
    table = random_tables(rng, B, mb, nb, bs, kv)
    bt, dkv = dev(table, torch.int32), dev(kv)
    parent, room = dev(np.arange(B)), dev(kv + 1)
    pool = make_pool(6, L, nb, bs, re, torch.bfloat16)
    err = new_error()

    def step():
        free, num = free_page_list(bt, nb, kv_len=dkv, block_size=bs, error=err)
        new, copies, used = fork_block_tables(bt, dkv, parent, room, free, bs, num_free=num, error=err)
        copy_pages(pool, copies, error=err)
        return free, num, new, copies, used

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    flat = lambda: pool.view(L, 2, nb * bs, re)  # noqa: E731
    for seed in range(3):
        p = np.random.default_rng(seed).integers(0, B, B)
        parent.copy_(dev(p))
        room.copy_(dev(kv[p] + 1))
        pos = lambda n: np.arange(n)  # noqa: E731
        held = [flat()[:, :, dev(table[q][pos(kv[q]) // bs] * bs + pos(kv[q]) % bs)].clone() for q in p]
        g.replay()
        torch.cuda.synchronize()
        new = out[2].cpu().numpy()
        for i, q in enumerate(p):
            got = flat()[:, :, dev(new[i][pos(kv[q]) // bs] * bs + pos(kv[q]) % bs)]
            assert torch.equal(got, held[i])
        # the pages that rows write next are theirs alone
        last = [new[i][kv[q] // bs] for i, q in enumerate(p)]
        assert len(set(last)) == B and err.item() == 0
        for x, y in zip(out, step()):
            assert torch.equal(x, y)


def test_more_items_than_a_grid_holds():
    """2.2 million entries and rows, of which those at the ends do something, in one layer: more
    workgroups than a launch takes."""
    n, bs, re = 2_200_000, 4, 8
    pool = make_pool(3, 1, 40, bs, re, torch.bfloat16)
    want = pool.clone()
    copies = torch.full((3, n), -1, dtype=torch.int32, device=DEV)
    at = dev([0, 1_048_575, 1_048_576, 2_097_151, 2_097_152, n - 1])
    copies[:, at] = dev([np.arange(6), np.arange(10, 16), [4, 1, 2, 3, 4, 1]], torch.int32)
    for i, t in enumerate([4, 1, 2, 3, 4, 1]):
        want[:, :, 10 + i, :t] = want[:, :, i, :t]
    err = new_error()
    copy_pages(pool, copies, error=err)
    assert torch.equal(pool, want) and err.item() == 0
    table = torch.full((n, 1), -1, dtype=torch.int32, device=DEV)
    start, keep = (torch.zeros(n, dtype=torch.int64, device=DEV) for _ in range(2))
    path = torch.full((n, 1), 2, dtype=torch.int64, device=DEV)
    table[at, 0] = dev(np.arange(20, 26), torch.int32)
    start[at] = 1
    keep[at] = 1
    want[:, :, 20:26, 1] = want[:, :, 20:26, 3]
    kept = torch.full((n,), -9, dtype=torch.int64, device=DEV)
    compact_paged(pool, table, start, path, keep, kept=kept, error=err)
    assert torch.equal(pool, want) and torch.equal(kept, keep) and err.item() == 0
