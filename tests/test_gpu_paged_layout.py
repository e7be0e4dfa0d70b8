"""GPU checks of the batch layout in the paged cache against the row-by-row oracle
(oracle/paged.py): block tables with shared prefix pages, slots of packed tokens, append by
slot. Whole values and copies: everything is equal."""
import numpy as np
import pytest
import torch

from oracle import paged as OP
from specdec.kvcache import (PagedKVCache, append_paged_slots, build_block_tables,
                             paged_slot_mapping)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _dev(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int64), device=DEV)


def _batch(rng, G, per, prefix, own, empty=0.2):
    """cu_group, prefix_len, kv_len: groups of 0 .. per rows, rows shorter than the prefix too."""
    n = rng.integers(0 if G > 1 else 1, per + 1, G)
    cu = np.concatenate([[0], np.cumsum(n)])
    pre = rng.integers(0, prefix + 1, G)
    kv = np.repeat(pre, n) + rng.integers(0, own + 1, cu[-1])
    first = np.repeat(cu[:-1], n)
    cut = (rng.random(cu[-1]) < empty) & (first != np.arange(cu[-1]))
    kv[cut] = rng.integers(0, kv.max() + 1, cut.sum()) if cut.any() else 0
    return cu, pre, kv


@pytest.mark.parametrize("G,per,prefix,own,bs", [
    (1, 1, 0, 0, 16), (1, 1, 5, 1, 16), (1, 4, 600, 40, 16), (5, 3, 64, 7, 16), (7, 9, 33, 20, 1),
    (40, 6, 1000, 300, 16), (1500, 2, 50, 9, 8), (3, 900, 300, 60, 7), (2, 3, 20000, 9000, 2),
])
def test_block_tables_match_oracle(G, per, prefix, own, bs):
    rng = np.random.default_rng(G * 100 + per)
    cu, pre, kv = _batch(rng, G, per, prefix, own)
    if cu[-1] == 0:
        pytest.skip("no rows")
    mb = int(-(-kv.max() // bs)) + int(rng.integers(0, 3)) or 1
    free = rng.permutation(int(np.sum(-(-kv // bs))) + 2).astype(np.int32)
    want, used, ok = OP.build_block_tables(kv, free, bs, mb, cu, pre)
    assert ok
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    t, u = build_block_tables(_dev(kv), torch.as_tensor(free, device=DEV), bs, mb, _dev(cu),
                              _dev(pre), error=err)
    assert np.array_equal(t.cpu().numpy(), want) and u.item() == used and err.item() == 0
    # just enough pages, and one too few
    t, u = build_block_tables(_dev(kv), torch.as_tensor(free[:used], device=DEV), bs, mb, _dev(cu),
                              _dev(pre), error=err)
    assert np.array_equal(t.cpu().numpy(), want) and err.item() == 0
    if used:
        t, u = build_block_tables(_dev(kv), torch.as_tensor(free[:used - 1], device=DEV), bs, mb,
                                  _dev(cu), _dev(pre), error=err)
        assert (t == -1).all() and u.item() == 0 and err.item() == 1


def test_block_tables_without_groups_and_given_output():
    kv = np.array([0, 1, 16, 17, 0, 40])
    free = np.arange(20, 0, -1).astype(np.int32)
    out = torch.full((6, 5), 77, dtype=torch.int32, device=DEV)
    t, u = build_block_tables(_dev(kv), torch.as_tensor(free, device=DEV), 16, 5, out=out)
    want, used, _ = OP.build_block_tables(kv, free, 16, 5)
    assert t is out and np.array_equal(t.cpu().numpy(), want) and u.item() == used == 7


@pytest.mark.parametrize("case", ["negative", "long", "offsets", "descending", "short", "prefix"])
def test_block_tables_refuse_whole_batches(case):
    """A length, offset or prefix that does not fit: nothing is handed out, the error is set."""
    kv, cu, pre = np.array([40, 33, 20, 50]), np.array([0, 2, 4]), np.array([32, 16])
    if case == "negative":
        kv[3] = -1
    elif case == "long":
        kv[2] = 16 * 4 + 1
    elif case == "offsets":
        cu[2] = 3
    elif case == "descending":
        cu = np.array([0, 5, 4])
    elif case == "short":
        cu[0] = 1
    else:
        pre[1] = 21          # longer than the group's first row
    free = torch.arange(64, dtype=torch.int32, device=DEV)
    assert not OP.build_block_tables(kv, np.arange(64), 16, 4, cu, pre)[2]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    t, u = build_block_tables(_dev(kv), free, 16, 4, _dev(cu), _dev(pre), error=err)
    assert (t == -1).all() and u.item() == 0 and err.item() == 1


def test_block_tables_arguments():
    kv, free = _dev([3]), torch.arange(4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="together"):
        build_block_tables(kv, free, 16, 4, cu_group=_dev([0, 1]))
    with pytest.raises(ValueError, match="offsets"):
        build_block_tables(kv, free, 16, 4, cu_group=_dev([0, 1, 1]), prefix_len=_dev([0]))
    with pytest.raises(ValueError, match="out must be"):
        build_block_tables(kv, free, 16, 4, out=torch.zeros((1, 5), dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="bad arguments"):
        build_block_tables(kv, free, 0, 4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        build_block_tables(kv.cpu(), free, 16, 4)
    t, u = build_block_tables(_dev([]), free, 16, 4)
    assert t.shape == (0, 4) and u.item() == 0


@pytest.mark.parametrize("B,q_hi,own,bs,pad", [
    (1, 1, 0, 16, 0), (1, 700, 30, 16, 3), (64, 9, 900, 16, 0), (500, 3, 100, 7, 11),
    (1025, 2, 40, 16, 5), (3000, 2, 40, 1, 0), (9, 4000, 100, 32, 0),
])
def test_slots_match_oracle(B, q_hi, own, bs, pad):
    rng = np.random.default_rng(B)
    q = rng.integers(0, q_hi + 1, B)
    q[rng.integers(B)] = q_hi
    kv = q + rng.integers(0, own + 1, B)
    cu = np.concatenate([[0], np.cumsum(q)])
    mb = int(-(-kv.max() // bs)) + 1
    table = rng.permutation(B * mb).reshape(B, mb)
    T = int(cu[-1]) + pad
    wp, ws, ok = OP.slot_mapping(table, cu, kv, bs, T, padding=-7)
    assert ok
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    p, s = paged_slot_mapping(_dev(table).to(torch.int32), _dev(cu), _dev(kv), bs, T,
                              padding_slot_id=-7, error=err)
    assert np.array_equal(p.cpu().numpy(), wp) and np.array_equal(s.cpu().numpy(), ws)
    assert err.item() == 0


def test_slots_of_rows_out_of_range():
    """A row shorter than its tokens, one past its table, one with a missing page: padding
    and the error; the other rows are served."""
    table = np.array([[3, 1], [0, 2], [-1, 4], [5, 6]])
    kv, q = np.array([1, 9, 6, 8]), np.array([2, 2, 4, 3])
    cu = np.concatenate([[0], np.cumsum(q)])
    wp, ws, ok = OP.slot_mapping(table, cu, kv, 4, 11)
    assert not ok and (ws[8:] >= 0).all()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    p, s = paged_slot_mapping(_dev(table).to(torch.int32), _dev(cu), _dev(kv), 4, 11, error=err)
    assert np.array_equal(p.cpu().numpy(), wp) and np.array_equal(s.cpu().numpy(), ws)
    assert err.item() == 1
    with pytest.raises(ValueError, match="block_table must be"):
        paged_slot_mapping(_dev(table).to(torch.int32), _dev(cu[:-1]), _dev(kv), 4, 11)


def test_far_positions_pass_32_bits():
    """Slots past 2^32: page ids times the block size in 64 bits, and table rows whose
    positions need them."""
    bs = 1 << 20
    table = torch.tensor([[2**31 - 1, 2**31 - 2], [7, 2**31 - 5]], dtype=torch.int32, device=DEV)
    kv, cu = _dev([bs + 3, 2 * bs]), _dev([0, 4, 6])
    p, s = paged_slot_mapping(table, cu, kv, bs, 6)
    wp, ws, _ = OP.slot_mapping(table.cpu().numpy().astype(np.int64), cu.cpu().numpy(),
                                kv.cpu().numpy(), bs, 6)
    assert np.array_equal(p.cpu().numpy(), wp) and np.array_equal(s.cpu().numpy(), ws)
    assert ws.max() > 2**32
    big = torch.full((1, 5000), -1, dtype=torch.int32, device=DEV)
    big[0, 4500] = 3
    p, s = paged_slot_mapping(big, _dev([0, 1]), _dev([4500 * bs + 1]), bs, 1)
    assert p.item() == 4500 * bs and s.item() == 3 * bs


@pytest.mark.parametrize("bs,shift", [(1 << 30, 30), ((1 << 31) - 1, 31), (1 << 28, 28)])
def test_block_tables_of_lengths_past_32_bits(bs, shift):
    kv = np.array([7 * bs, 3 * bs + 5, 3 * bs + 6, 0, 1, (5 << shift) + 1])
    cu, pre, free = np.array([0, 3, 3, 6]), np.array([3 * bs + 5, 0, 0]), np.arange(40, 0, -1)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    want, used, ok = OP.build_block_tables(kv, free, bs, 8, cu, pre)
    t, u = build_block_tables(_dev(kv), torch.as_tensor(free.astype(np.int32), device=DEV), bs, 8,
                              _dev(cu), _dev(pre), error=err)
    assert ok and np.array_equal(t.cpu().numpy(), want) and u.item() == used and err.item() == 0
    kv[4] = 8 * bs + 1  # a page more than the table has
    t, u = build_block_tables(_dev(kv), torch.as_tensor(free.astype(np.int32), device=DEV), bs, 8,
                              _dev(cu), _dev(pre), error=err)
    assert (t == -1).all() and u.item() == 0 and err.item() == 1


@pytest.mark.parametrize("L,T,hkv,d,dtype", [
    (1, 1, 1, 64, torch.bfloat16), (3, 5, 2, 64, torch.float16), (2, 257, 8, 128, torch.bfloat16),
    (64, 33, 8, 128, torch.bfloat16), (2, 100, 1, 40, torch.float16), (1, 70, 3, 28, torch.float32),
])
def test_append_slots(L, T, hkv, d, dtype):
    """Every (layer, side) gets its vectors; padded and outside slots leave the pool alone."""
    g = torch.Generator(device=DEV).manual_seed(T)
    nb, bs = T // 4 + 2, 5
    cache = PagedKVCache(L, 1, nb, bs, hkv, d, nb, dtype=dtype, device=DEV)
    cache.pool.copy_(torch.randn(cache.pool.shape, generator=g, device=DEV))
    slots = torch.randperm(nb * bs, generator=g, device=DEV)[:T].contiguous()
    if T > 4:
        slots[1::4] = -1
    staged = torch.randn((L, 2, T, hkv * d), generator=g, device=DEV).to(dtype)
    want = cache.pool.clone()
    at = (slots >= 0).nonzero().squeeze(1)
    want.view(L, 2, nb * bs, -1)[:, :, slots[at]] = staged[:, :, at]
    cache.append_slots(staged, slots)
    assert torch.equal(cache.pool, want) and cache.error.item() == 0
    # a slot past the pool is skipped and reported; strided staged rows are taken as they are
    slots[0] = nb * bs
    wide = torch.randn((L, 2, T, 2 * hkv * d), generator=g, device=DEV).to(dtype)[..., hkv * d:]
    at = ((slots >= 0) & (slots < nb * bs)).nonzero().squeeze(1)
    want.view(L, 2, nb * bs, -1)[:, :, slots[at]] = wide[:, :, at]
    cache.append_slots(wide, slots)
    assert torch.equal(cache.pool, want) and cache.error.item() == 1


def test_append_slots_equals_the_uniform_append():
    """The same tokens through PagedKVCache.append and through slots from the lengths."""
    B, q, hkv, d, bs, mb = 6, 4, 2, 64, 8, 9
    g = torch.Generator(device=DEV).manual_seed(1)
    a = PagedKVCache(3, B, B * mb, bs, hkv, d, mb, device=DEV)
    b = PagedKVCache(3, B, B * mb, bs, hkv, d, mb, device=DEV)
    a.block_table.copy_(torch.randperm(B * mb, generator=g, device=DEV).view(B, mb))
    a.lengths.copy_(torch.randint(0, 60, (B,), generator=g, device=DEV))
    staged = torch.randn((3, 2, B, q, hkv * d), generator=g, device=DEV).to(torch.bfloat16)
    a.append(staged)
    cu = torch.arange(B + 1, device=DEV) * q
    _, slots = paged_slot_mapping(a.block_table, cu, a.lengths + q, bs, B * q)
    b.append_slots(staged.view(3, 2, B * q, hkv * d), slots)
    assert torch.equal(a.pool, b.pool)


def test_append_slots_arguments():
    pool = torch.zeros((2, 2, 3, 4, 64), dtype=torch.bfloat16, device=DEV)
    st, sl = torch.zeros((2, 2, 5, 64), dtype=torch.bfloat16, device=DEV), _dev(range(5))
    with pytest.raises(ValueError, match="staged must be"):
        append_paged_slots(pool, st[:, :, :4], sl)
    with pytest.raises(ValueError, match="pool must be"):
        append_paged_slots(pool[..., :32], st, sl)
    with pytest.raises(RuntimeError, match="16-byte"):
        append_paged_slots(torch.zeros((1, 2, 3, 4, 4), dtype=torch.bfloat16, device=DEV),
                           torch.zeros((1, 2, 5, 4), dtype=torch.bfloat16, device=DEV), sl)
    append_paged_slots(pool, st[:, :, :0], sl[:0])
    with pytest.raises(TypeError, match="error must be"):
        append_paged_slots(pool, st, sl, error=torch.zeros(1, device=DEV))


def test_layout_in_graphs_and_on_a_side_stream():
    rng = np.random.default_rng(5)
    cu, pre, kv = _batch(rng, 6, 5, 300, 80)
    free = torch.as_tensor(rng.permutation(2000).astype(np.int32), device=DEV)
    kvd, cud, pred = _dev(kv), _dev(cu), _dev(pre)
    q = np.minimum(rng.integers(0, 6, len(kv)), kv)
    cuq = _dev(np.concatenate([[0], np.cumsum(q)]))
    T = int(q.sum())

    def call():
        t, u = build_block_tables(kvd, free, 16, 40, cud, pred)
        return (t, u, *paged_slot_mapping(t, cuq, kvd, 16, T))

    want = [x.clone() for x in call()]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        got = call()
    for _ in range(3):
        g.replay()
        call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = call()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want))
