"""Calls at the edges of the operators around steps over trees: what cannot be right is refused or
reported, never cut, skipped or taken for something else."""
import numpy as np
import pytest
import torch

from oracle import tree as OT
from specdec.attention import tree_attention_paged, tree_attention_workspace
from specdec.kvcache import compact_paged, copy_pages, fork_block_tables, free_page_list
from specdec.sampling import penalize_logits
from specdec.tree import tree_accept, tree_layout

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x, dtype=None):
    return torch.as_tensor(np.asarray(x), device=DEV, dtype=dtype)


def new_error():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def attention_case(n, start, d=64, pad=0, bs=16):
    """n: nodes per row, start: keys in front of them."""
    g = torch.Generator(device=DEV).manual_seed(3)
    n, start = np.asarray(n), np.asarray(start)
    cu, kv = np.concatenate([[0], np.cumsum(n)]), n + start
    mb = int(-(-kv.max() // bs)) + 1
    B, T = len(n), int(cu[-1]) + pad
    table = np.arange(B * mb).reshape(B, mb)
    parents = [max(i // 2 - 1, -1) for m in n for i in range(m)] + [-1] * pad
    mask = tree_layout(dev(parents, torch.int32), dev(cu), dev(kv),
                       max_nodes=max(64, -(-int(n.max()) // 64) * 64))[0]
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV).half()  # noqa: E731
    return dict(q=rnd(T, 8, d), cu_q=dev(cu), k_pool=rnd(B * mb, bs, 2 * d), v_pool=rnd(B * mb, bs, 2 * d),
                block_table=dev(table, torch.int32), kv_len=dev(kv), tree_mask=mask)


# ---- free pages that are none

@pytest.mark.parametrize("N,mb,bs", [(3, 4, 16), (16, 512, 3), (17, 40, 16), (300, 9, 4), (5, 700, 2)])
def test_a_fork_takes_pages_in_front_of_the_first_that_is_none(N, mb, bs):
    """The list of free_page_list, -1 behind its pages, without their number or with a number that is
    too large; a negative entry among the pages. What fits in front of it is given, else nothing."""
    rng = np.random.default_rng(N)
    B = N
    kv = rng.integers(1, mb * bs + 1, B)
    need = -(-kv // bs)
    ids = rng.permutation(int(need.sum()))
    table = np.full((B, mb), -1)
    at = 0
    for b in range(B):
        table[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
    parent = rng.integers(0, B, N)                       # some twice: copies
    room = np.minimum(kv[parent] + rng.integers(0, 3 * bs + 1, N), mb * bs)
    most = N * mb
    _, _, used, ok = OT.fork(table, kv, parent, room, list(range(at, at + most)), bs)
    assert ok and used > 0
    bt, rest = dev(table, torch.int32), (dev(kv), dev(parent), dev(room))
    for have in (used, used - 1):                        # pages that are free
        pages = np.arange(at, at + have)
        nb = at + have
        want, copies, u, ok = OT.fork(table, kv, parent, room, pages, bs)
        assert ok == (have == used)
        free, num = free_page_list(bt, nb, kv_len=rest[0], block_size=bs)
        assert num.item() == have and free.numel() > have
        for n in (None, num, num + 1, num * 0 + nb):
            err = new_error()
            got, gc, gu = fork_block_tables(bt, *rest, free, bs, num_free=n, error=err)
            assert got.tolist() == want.tolist() and gc.tolist() == copies.tolist()
            assert gu.item() == u and err.item() == (0 if ok else 1)
    pages = np.arange(at, at + used)
    for hole in {0, used // 2, used - 1}:
        p = pages.copy()
        p[hole] = -1
        err = new_error()
        got, gc, gu = fork_block_tables(bt, *rest, dev(p, torch.int32), bs, error=err)
        assert (got == -1).all() and (gc[:2] == -1).all() and (gc[2] == 0).all()
        assert gu.item() == 0 and err.item() == 1


# ---- masks without columns

def test_a_mask_of_no_columns_is_no_chain():
    x = torch.randn((4, 100), device=DEV)
    c = dict(cu_rows=dev([0, 4]), frequency=torch.ones(1, device=DEV), node_tokens=dev([1, 2, 3, 4]))
    for R in (4, 0):
        y, tok = x[:R], c["node_tokens"][:R]
        with pytest.raises(ValueError, match="words"):
            penalize_logits(y, **{**c, "cu_rows": dev([0, R]), "node_tokens": tok},
                            tree_mask=torch.zeros((R, 0), dtype=torch.int64, device=DEV))


# ---- histories without columns

def test_lengths_of_a_history_of_no_columns():
    x = torch.randn((3, 100), device=DEV)
    h = torch.zeros((3, 0), dtype=torch.int64, device=DEV)
    rep = torch.full((3,), 2.0, device=DEV)
    tok = dev([1, 2, 3])
    err = new_error()
    got = penalize_logits(x, h, dev([0, 0, 0]), repetition=rep, node_tokens=tok, error=err)
    assert err.item() == 0 and torch.equal(got, penalize_logits(x, repetition=rep, node_tokens=tok))
    for lens, prompt in (([0, 1, 0], None), ([0, -1, 0], None), ([0, 0, 0], [0, 1, 0])):
        err = new_error()
        out = penalize_logits(x, h, dev(lens), prompt_len=None if prompt is None else dev(prompt), repetition=rep,
                              node_tokens=tok, error=err)
        assert err.item() == 1 and torch.equal(out[1], x[1])
        assert torch.equal(out[0::2], got[0::2])


# ---- whole numbers that 32 bits do not hold

@pytest.mark.parametrize("far", [1 << 32, (1 << 32) + 1, -(1 << 32), (1 << 40) - 1, -(1 << 33) - 1])
def test_numbers_past_32_bits_are_out_of_range(far):
    up = dev([-1, 0, far, 0])
    table = dev([[2, 1]], torch.int32)
    err = new_error()
    mask, pos, slots = tree_layout(up, dev([0, 4]), dev([9]), table, 16, error=err)
    assert err.item() == 1 and (mask == 0).all() and (pos == 0).all() and (slots == -1).all()
    path, keep, _ = tree_accept(dev([5, 6, 7, 8]), up, dev([7, 7, 7, 7]), dev([0, 4]), 4)
    assert path.tolist() == [[0, -1, -1, -1]] and keep.tolist() == [1]     # node 2 is nobody's child
    # pages
    wide = torch.tensor([[2, far]], device=DEV)
    err = new_error()
    free_page_list(wide, 4, kv_len=dev([20]), block_size=16, error=err)
    assert err.item() == 1
    pool = torch.randn((1, 2, 4, 16, 8), device=DEV).half()
    before = pool.clone()
    err = new_error()
    compact_paged(pool, wide, dev([14]), dev([[1, 3]]), dev([2]), error=err)
    assert err.item() == 1 and torch.equal(pool, before)
    for row in range(3):                                   # a source, a target, a number of tokens
        copies = dev([[1], [2], [3]])
        copies[row] = far
        err = new_error()
        copy_pages(pool, copies, error=err)
        # negative pages are entries that are skipped
        assert torch.equal(pool, before) and err.item() == (0 if row < 2 and far < 0 else 1)
    q = torch.randn((4, 1, 64), device=DEV).half()
    kp = torch.randn((4, 16, 64), device=DEV).half()
    err = new_error()
    tree_attention_paged(q, dev([0, 4]), kp, kp, wide, dev([20]), torch.full((4, 1), 15, device=DEV), error=err)
    assert err.item() == 1
    if far < 0:                                            # a new table without holes
        err = new_error()
        got, _, used = fork_block_tables(table, dev([20]), dev([0]), dev([32]), dev([far]), 16,
                                         error=err)
        assert used.item() == 0 and err.item() == 0 and got.tolist() == [[2, 1]]
        got, _, used = fork_block_tables(table, dev([16]), dev([0]), dev([17]), dev([far]), 16, error=err)
        assert used.item() == 0 and err.item() == 1 and (got == -1).all()


# ---- numbers that are not whole

def test_only_whole_numbers_are_taken_for_whole_numbers():
    i64 = lambda *x: dev(x, torch.int64)  # noqa: E731
    pool = torch.zeros((1, 2, 4, 16, 8), dtype=torch.half, device=DEV)
    table = dev([[0, 1], [2, -1]], torch.int32)
    q = torch.zeros((3, 1, 64), dtype=torch.half, device=DEV)
    kp = torch.zeros((4, 16, 64), dtype=torch.half, device=DEV)
    x = torch.zeros((3, 10), device=DEV)
    cu, kv = i64(0, 2, 3), i64(20, 3)
    calls = [
        (tree_layout, dict(parents=dev([-1, 0, -1], torch.int32), cu_q=cu, kv_len=kv, block_table=table,
                           block_size=16), ("parents", "cu_q", "kv_len", "block_table")),
        (tree_accept, dict(tokens=i64(1, 2, 3), parents=dev([-1, 0, -1], torch.int32), choice=i64(2, 5, 6), cu_q=cu,
                           max_path=4), ("tokens", "parents", "choice", "cu_q")),
        (compact_paged, dict(pool=pool, block_table=table, kv_start=kv - 2, path=dev([[0, 1], [0, 1]]), keep=i64(2, 1)),
         ("block_table", "kv_start", "path", "keep")),
        (free_page_list, dict(block_table=table, num_blocks=4, kv_len=kv, block_size=16),
         ("block_table", "kv_len")),
        (fork_block_tables, dict(block_table=table, kv_len=kv, parent=i64(0, 1), room=i64(21, 4),
                                 free_blocks=dev([3], torch.int32), block_size=16, num_free=i64(1)),
         ("block_table", "kv_len", "parent", "room", "free_blocks", "num_free")),
        (copy_pages, dict(pool=pool, copies=dev([[0], [3], [5]], torch.int32)), ("copies",)),
        (tree_attention_paged, dict(q=q, cu_q=cu, k_pool=kp, v_pool=kp, block_table=table, kv_len=kv,
                                    tree_mask=torch.ones((3, 1), dtype=torch.int64, device=DEV)),
         ("cu_q", "kv_len", "block_table")),
        (penalize_logits, dict(logits=x, history=i64(1, 2).view(2, 1), history_len=i64(1, 1), cu_rows=cu,
                               prompt_len=i64(0, 1), node_tokens=i64(1, 2, 3), bias_ids=i64(1, 2).view(2, 1),
                               bias=torch.ones((2, 1), device=DEV)),
         ("history", "history_len", "cu_rows", "prompt_len", "node_tokens", "bias_ids")),
    ]
    for call, args, names in calls:
        call(**args)
        for name in names:
            for dtype in (torch.float32, torch.bool, torch.bfloat16):
                with pytest.raises(TypeError, match=name):
                    call(**{**args, name: args[name].to(dtype)})


# ---- outputs that nothing is computed for

def call_over_nan(c, **more):
    """The call, with NaN in all memory that it allocates."""
    torch.use_deterministic_algorithms(True, warn_only=True)
    try:
        assert torch.empty_like(c["q"]).isnan().all()
        return tree_attention_paged(**c, **more)
    finally:
        torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,start", [([5, 9, 4], [100, 20, 0]), ([3] * 70, [5] * 70), ([1] * 600, [7] * 600),
                                     ([0, 0], [4, 4]), ([300], [50])])
def test_an_allocated_output_is_0_where_nothing_is_computed(n, start, d):
    c = attention_case(n, start, d=d, pad=37)
    T = int(c["cu_q"][-1])
    want = torch.full_like(c["q"], 7.0)
    tree_attention_paged(**c, out=want)
    assert (want[T:] == 7).all()                          # a given one is left as it was
    want[T:] = 0
    assert torch.equal(call_over_nan(c), want)
    if T == 0:
        return
    # a row that is refused, a token in front of the first row
    b = len(n) - 1
    a, e = c["cu_q"].tolist()[b:b + 2]
    bad = dict(c, kv_len=c["kv_len"].clone())
    bad["kv_len"][b] = -3
    err = new_error()
    got = call_over_nan(bad, error=err)
    assert err.item() == 1 and (got[a:e] == 0).all() and (got[T:] == 0).all()
    given = torch.full_like(c["q"], 7.0)
    tree_attention_paged(**bad, out=given)
    assert (given[a:e] == 7).all() and torch.equal(given[:a], got[:a])
    if n[0] > 1:
        assert (call_over_nan(dict(c, cu_q=c["cu_q"].clamp(min=1)))[0] == 0).all()


def test_an_allocated_output_of_rows_that_share_nodes_is_0():
    c = shared_nodes(40)
    assert (call_over_nan(c) == 0).all()


def test_padding_of_an_allocated_output_in_a_graph():
    c = attention_case([5, 9], [100, 20], pad=9)
    call_over_nan(c)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tree_attention_paged(**c)
    for last in (14, 11, 5, 14):
        c["cu_q"][2] = last
        c["kv_len"][1] = 20 + last - 5
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert (out[last:] == 0).all() and torch.equal(out, tree_attention_paged(**c))


# ---- rows that share their nodes

def shared_nodes(B):
    """Offsets 0, 256, 0, 256, ...: every row with nodes has all of them."""
    c = attention_case([64] * 4, [30] * 4)
    cu = torch.zeros(B + 1, dtype=torch.int64, device=DEV)
    cu[1::2] = 256
    return dict(c, cu_q=cu, kv_len=torch.full((B,), 350, device=DEV),
                block_table=c["block_table"][:1].repeat(B, 4), tree_mask=c["tree_mask"].repeat(1, 4))


@pytest.mark.parametrize("B", [40, 64, 70, 600, 1100])
def test_rows_that_share_their_nodes_compute_nothing(B):
    """More items than the workspace has records for, laid out by each wave (to 64 rows), by the
    workgroup, and in several rounds of it: no output, and nothing behind the workspace."""
    c = shared_nodes(B)
    T, hq, d = c["q"].shape
    hkv = c["k_pool"].shape[2] // d
    need = tree_attention_workspace(T, B, hq, hkv, d).numel()
    room = torch.full((need + (1 << 20),), 0x5A, dtype=torch.uint8, device=DEV)
    items = hkv * sum(-(-256 * (hq // hkv) // 256) for b in range(0, B, 2))
    assert items > hkv * (T * (hq // hkv) // 256 + min(B, T))
    err, out = new_error(), torch.full_like(c["q"], 7.0)
    tree_attention_paged(**c, out=out, workspace=room[:need], error=err)
    assert err.item() == 1 and (out == 7).all() and (room[need:] == 0x5A).all()


# ---- counts written over counts

def test_kept_may_be_keep_itself():
    """Rows that are refused have 0 in it then, and move nothing."""
    L, B, mb, bs = 9, 40, 3, 16
    g = torch.Generator(device=DEV).manual_seed(2)
    pool = torch.randn((L, 2, B * mb, bs, 64), generator=g, device=DEV).half()
    table = np.arange(B * mb).reshape(B, mb)
    start, path, keep = np.full(B, 20), np.tile([1, 2, 5, 9], (B, 1)), np.full(B, 4)
    path[::3, 2] = 2                                     # does not ascend
    keep[5] = 0
    want = pool.cpu().clone()
    assert not OT.compact(want, table, start, path, keep)
    k, err = dev(keep), new_error()
    compact_paged(pool, dev(table, torch.int32), dev(start), dev(path), k, kept=k, error=err)
    assert torch.equal(pool.cpu(), want) and err.item() == 1
    assert k.tolist() == [0 if b % 3 == 0 else int(keep[b]) for b in range(B)]
    s = dev(start)
    with pytest.raises(RuntimeError, match="apart"):
        compact_paged(pool, dev(table, torch.int32), s, dev(path), dev(keep), kept=s)
    assert torch.equal(pool.cpu(), want) and s.tolist() == start.tolist()


# ---- lists of many pages

@pytest.mark.parametrize("nb,B,mb", [(1 << 17, 8, 40), ((1 << 17) + 1, 8, 40), (20_000, 70, 300), (3_000_017, 40, 100),
                                     (1_300_000, 900, 300), (20_000_003, 5, 7)])
def test_free_pages_of_large_pools(nb, B, mb):
    """At the ends of the forms: segments that are added up page by page, and by their counts."""
    g = torch.Generator(device=DEV).manual_seed(nb)
    table = torch.randint(0, nb, (B, mb), generator=g, device=DEV)
    table[0, 0], table[-1, -1], table[0, 1:3] = nb - 1, 0, 8191
    kv = torch.randint(0, mb * 16 + 1, (B,), generator=g, device=DEV)
    kv[0], kv[-1] = mb * 16, mb * 16
    held = torch.zeros(nb, dtype=torch.bool, device=DEV)
    at = torch.arange(mb, device=DEV) < ((kv + 15) // 16)[:, None]
    held[table[at]] = True
    want = (~held).nonzero().view(-1)
    err = new_error()
    free, num = free_page_list(table.int(), nb, kv_len=kv, block_size=16, error=err)
    assert err.item() == 0 and num.item() == want.numel()
    assert torch.equal(free[:want.numel()].long(), want) and (free[want.numel():] == -1).all()


# ---- sizes past 32 bits

def test_pages_past_32_bits_are_moved_and_copied():
    """Sides of 2.6 GB, a pool of 10 GB: pages at its ends and where 2^32 and 2^33 bytes lie."""
    L, nb, bs, re = 2, 40000, 16, 2048
    pool = torch.zeros((L, 2, nb, bs, re), dtype=torch.bfloat16, device=DEV)
    page = bs * re * 2
    assert pool.numel() * 2 > 2 ** 33
    near = sorted({p for e in (31, 32, 33) for s in range(4) for p in range((2 ** e - s * nb * page) // page - 1,
                                                                            (2 ** e - s * nb * page) // page + 2)
                   if 0 <= p < nb} | {0, 1, nb - 2, nb - 1})
    assert len(near) >= 8
    small = torch.randn((L, 2, len(near), bs, re), device=DEV).bfloat16()
    pool[:, :, near] = small
    n = len(near) // 2
    table = np.arange(2 * n).reshape(n, 2)[:, ::-1]        # rows of two pages, in the small pool and in the large
    start, path, keep = np.full(n, 10), np.tile([0, 3, 4, 7, 20], (n, 1)), np.full(n, 5)
    want = small.cpu()
    assert OT.compact(want, table, start, path, keep)
    err = new_error()
    compact_paged(pool, dev(np.asarray(near)[table], torch.int32), dev(start), dev(path), dev(keep), error=err)
    assert torch.equal(pool[:, :, near].cpu(), want) and err.item() == 0
    half = len(near) // 2
    copies = np.stack([np.arange(half), np.arange(half, 2 * half), 1 + np.arange(half) % bs])
    for s, d, t in copies.T:
        want[:, :, d, :t] = want[:, :, s, :t]
    copies[:2] = np.asarray(near)[copies[:2]]
    copy_pages(pool, dev(copies, torch.int32), error=err)
    assert torch.equal(pool[:, :, near].cpu(), want) and err.item() == 0
    pool[:, :, near] = 0
    assert not pool.any()                                 # nothing else


def test_logits_past_32_bits_of_elements():
    R, V = 17000, 131071                                  # 2.2e9 logits, rows off alignment
    assert R * V > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(1)
    line = torch.randn(V, generator=g, device=DEV).bfloat16()
    x = line.repeat(R, 1)
    hist = torch.randint(0, V, (R, 4), generator=g, device=DEV)
    c = dict(history_len=torch.full((R,), 4, device=DEV), repetition=torch.full((R,), 1.3, device=DEV),
             presence=torch.full((R,), 0.5, device=DEV))
    err = new_error()
    assert penalize_logits(x, hist, **c, out=x, error=err) is x and err.item() == 0
    rows = [0, 1, R // 2, 2 ** 31 // V - 1, 2 ** 31 // V, 2 ** 31 // V + 1, R - 2, R - 1]
    few = penalize_logits(line.repeat(len(rows), 1), hist[rows], **{k: v[rows] for k, v in c.items()})
    assert torch.equal(x[rows], few)
    changed = torch.zeros(R, dtype=torch.int64, device=DEV)
    for r0 in range(0, R, 1000):
        changed[r0:r0 + 1000] = (x[r0:r0 + 1000] != line).sum(1)
    assert (changed <= 4).all() and (changed > 0).all()


# ---- arguments that hold nothing

def test_an_empty_list_lies_over_nothing():
    """No free pages, as an empty slice of the memory that the new table is written to."""
    out = torch.full((2, 4), 9, dtype=torch.int32, device=DEV)
    err = new_error()
    got, copies, used = fork_block_tables(dev([[5, 6, -1, -1]], torch.int32), dev([20]), dev([0, -1]), dev([32, 0]),
                                          out.view(-1)[3:3], 16, out=out, error=err)
    assert err.item() == 0 and used.item() == 0 and got.tolist() == [[5, 6, -1, -1], [-1] * 4]
    with pytest.raises(RuntimeError, match="lie over"):
        fork_block_tables(dev([[5, 6, -1, -1]], torch.int32), dev([20]), dev([0, -1]), dev([32, 0]),
                          out.view(-1)[3:4], 16, out=out, error=err)
