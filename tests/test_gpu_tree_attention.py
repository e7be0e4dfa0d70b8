"""GPU parity of tree_attention_paged with softmax(q k^T scale) v in float64, row by row.

Tolerance, elementwise: with u half a step of the type (2^-8 bf16, 2^-11 fp16) the output's
own rounding is u |out|; every weight is rounded once, which moves the output by at most
u A, A = sum p |v| / sum p; and the fp32 part (scores over d products, the exponential's
argument, sums over chains of n / 64 + 64 keys, the joins of up to 512 parts) moves weights by at
most e = 2^-24 (4 (d + 8) S + n / 32 + 1024) relative, numerator and denominator, S the largest
scale sum |q k|: u |out| + (u + e) A (1 + u).
"""
import math
import threading

import numpy as np
import pytest
import torch

from specdec._lib import SpecdecError
from specdec.attention import (tree_attention_paged, tree_attention_workspace,
                               verify_attention_paged)
from specdec.tree import tree_layout

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(seed, n, start, hq, hkv, d, bs=16, dtype=torch.bfloat16, pad=0, words=None, kind="tree"):
    """n: nodes per row, start: keys in front of them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    n, start = np.asarray(n), np.asarray(start)
    cu, kv = np.concatenate([[0], np.cumsum(n)]), n + start
    need = -(-kv // bs)
    B, mb, nb = len(n), max(1, int(need.max()) + 1), int(need.sum()) + 3
    ids = iter(rng.permutation(nb))
    table = np.full((B, mb), -1)
    for b in range(B):
        table[b, :need[b]] = [next(ids) for _ in range(need[b])]
    T = int(cu[-1]) + pad
    if kind == "chain":
        parents = [i - 1 for m in n for i in range(m)]
    else:
        parents = [int(rng.integers(0, i)) if i else -1 for m in n for i in range(m)]
    dev = lambda x, t=None: torch.as_tensor(np.asarray(x), device=DEV, dtype=t)  # noqa: E731
    words = words or -(-max(1, int(n.max())) // 64)
    mask = tree_layout(dev(parents + [-1] * pad, torch.int32), dev(cu), dev(kv), max_nodes=64 * words)[0]
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    return dict(q=rnd(T, hq, d), cu_q=dev(cu), k_pool=rnd(nb, bs, hkv * d), v_pool=rnd(nb, bs, hkv * d),
                block_table=dev(table, torch.int32), kv_len=dev(kv), tree_mask=mask)


def reference(c, scale=None):
    """(out, A, S) in float64; rows without nodes leave zeros."""
    q, kp, vp = c["q"].double(), c["k_pool"], c["v_pool"]
    T, hq, d = q.shape
    bs, hkv = kp.shape[1], kp.shape[2] // d
    scale = 1 / math.sqrt(d) if scale is None else scale
    cu, kv = c["cu_q"].tolist(), c["kv_len"].tolist()
    out, A = torch.zeros_like(q), torch.zeros_like(q)
    S = 0.0
    for b in range(len(kv)):
        n, m = kv[b], cu[b + 1] - cu[b]
        if m == 0:
            continue
        pos = torch.arange(n, device=DEV)
        page = c["block_table"][b, pos // bs].long()
        k = kp[page, pos % bs].double().view(n, hkv, d).permute(1, 2, 0).contiguous()
        v = vp[page, pos % bs].double().view(n, hkv, d).permute(1, 0, 2).contiguous()
        x = q[cu[b]:cu[b + 1]].view(m, hkv, hq // hkv, d).permute(1, 2, 0, 3)
        j = torch.arange(m, device=DEV)
        sees = torch.ones((m, n), dtype=torch.bool, device=DEV)
        sees[:, n - m:] = (c["tree_mask"][cu[b]:cu[b + 1]][:, j // 64] >> (j % 64)) & 1 == 1
        w = (torch.matmul(x, k.unsqueeze(1)) * scale).masked_fill(~sees, -math.inf)
        S = max(S, float((torch.matmul(x.abs(), k.abs().unsqueeze(1)) * scale).max()))
        p = torch.nan_to_num(torch.softmax(w, -1))            # a node that sees nothing: 0
        o, a = torch.matmul(p, v.unsqueeze(1)), torch.matmul(p, v.abs().unsqueeze(1))
        out[cu[b]:cu[b + 1]] = o.permute(2, 0, 1, 3).reshape(m, hq, d)
        A[cu[b]:cu[b + 1]] = a.permute(2, 0, 1, 3).reshape(m, hq, d)
    return out, A, S


def check(c, scale=None, got=None, rows=None, ref=None, **more):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    if got is None:
        got = tree_attention_paged(**c, scale=scale, error=err, **more)
    want, A, S = ref or reference(c, scale)
    u = torch.finfo(got.dtype).eps / 2
    e = 2.0 ** -24 * (4 * (got.shape[2] + 8) * S + int(c["kv_len"].max()) / 32 + 1024)
    off = (got.double() - want).abs() - (u * want.abs() + (u + e) * A * (1 + u))
    T = int(c["cu_q"][-1])
    off = off[:T] if rows is None else off[rows]
    assert torch.isfinite(got[:T] if rows is None else got[rows]).all()
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()
    assert err.item() == 0
    return got


@pytest.mark.parametrize("n,start,heads,bs,dtype", [
    ([1], [0], (1, 1, 64), 16, torch.bfloat16),                       # one key
    ([1], [1], (4, 4, 128), 16, torch.float16),
    ([2], [0], (8, 2, 128), 16, torch.bfloat16),                      # nothing in the cache
    ([26], [2011], (32, 8, 128), 16, torch.bfloat16),
    ([64, 1, 0, 33, 63], [64, 63, 100, 65, 128], (32, 8, 128), 16, torch.bfloat16),
    ([31, 32, 5], [500, 7, 0], (14, 2, 64), 16, torch.float16),
    ([65, 64, 129], [30, 700, 1], (8, 2, 128), 16, torch.bfloat16),   # masks of several words
    ([512], [100], (4, 4, 64), 16, torch.bfloat16),
    ([300, 2], [0, 900], (5, 1, 128), 7, torch.float16),              # a token's heads in two tiles
    ([40, 17, 9], [1, 2, 3], (10, 2, 128), 1, torch.bfloat16),
    ([9] * 40, [13 * i for i in range(40)], (6, 3, 64), 32, torch.bfloat16),
    ([1 + i % 64 for i in range(300)], [i % 130 for i in range(300)], (8, 2, 64), 16, torch.float16),
    ([1] * 700, [5] * 700, (2, 1, 128), 8, torch.bfloat16),           # more rows than threads
    ([16, 3], [300, 200], (128, 1, 128), 16, torch.bfloat16),         # a wide group
])
def test_matches_float64(n, start, heads, bs, dtype):
    check(make(len(n) + sum(n), n, start, *heads, bs=bs, dtype=dtype))


@pytest.mark.parametrize("n,start,heads,dtype", [
    ([3], [60000], (8, 1, 128), torch.bfloat16),      # one row over the whole grid
    ([60], [30001], (32, 8, 128), torch.float16),
    ([64, 2, 40], [9000, 20000, 3], (16, 4, 64), torch.bfloat16),
    ([48] * 24, [3000 + 77 * i for i in range(24)], (32, 8, 128), torch.bfloat16),
])
def test_long_keys(n, start, heads, dtype):
    check(make(sum(n), n, start, *heads, dtype=dtype))


@pytest.mark.parametrize("scale", [1e-4, 0.5, 3.0])
def test_scales(scale):
    check(make(5, [26, 7], [300, 40], 8, 2, 128), scale=scale)
    check(make(6, [26, 7], [300, 40], 8, 2, 64, dtype=torch.float16), scale=scale)


def test_a_chain_is_the_verify_attention():
    c = make(7, [5, 9, 1, 4], [700, 64, 0, 31], 32, 8, 128, kind="chain")
    want = verify_attention_paged(c["q"], c["cu_q"], c["k_pool"], c["v_pool"], c["block_table"],
                                  c["kv_len"], 9)
    got = check(c)
    ref, A, S = reference(c)
    assert ((got.double() - want.double()).abs() <= 2 * (2.0 ** -8 * (ref.abs() + A) * 1.1 + 1e-3 * A)).all()


def test_the_mask_is_what_counts():
    """Bits past a row's nodes are not looked at; nodes without any bit see the cache, or nothing."""
    c = make(8, [20, 70, 3], [100, 0, 0], 8, 2, 64, words=3)
    c["tree_mask"][2] = 0                     # sees the cache alone
    c["tree_mask"][25] = 0                    # sees nothing
    c["tree_mask"][26] = torch.tensor([0, 0, -1], device=DEV)      # bits of no node
    c["tree_mask"][90:, 0] |= ~7
    g = torch.Generator(device=DEV).manual_seed(3)
    c["tree_mask"][30:60] = torch.randint(-2 ** 63, 2 ** 63 - 1, (30, 3), generator=g, device=DEV)
    c["tree_mask"][:19] |= -1 << 20
    got = check(c)
    assert (got[25] == 0).all() and (got[26] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hidden_keys_hold_anything(dtype):
    """Infinities and NaN in nodes that a query does not see, behind the row's keys, and in pages
    of nobody do not reach its output; those that it sees do."""
    d = 128
    c = make(9, [30, 70, 5], [100, 31, 64], 8, 2, d, dtype=dtype)
    ref = reference(c)
    used = torch.zeros(c["k_pool"].shape[:2], dtype=torch.bool, device=DEV)
    kv, bs = c["kv_len"].tolist(), 16
    for b, n in enumerate(kv):
        pos = torch.arange(n, device=DEV)
        used[c["block_table"][b, pos // bs].long(), pos % bs] = True
    for p, bad in ((c["k_pool"], float("nan")), (c["v_pool"], float("inf"))):
        p[~used] = bad
    check(c, ref=ref)
    # node 1 of row 0 and node 2 of row 1 hold infinities and NaN: those that see them are left out
    hit = torch.zeros(c["q"].shape[0], dtype=torch.bool, device=DEV)
    for b, node, t0 in ((0, 1, 0), (1, 2, 30)):
        pos = kv[b] - (30, 70)[b] + node
        page, at = int(c["block_table"][b, pos // bs]), pos % bs
        c["v_pool"][page, at, ::3] = float("nan")
        c["v_pool"][page, at, 1::3] = float("-inf")
        c["k_pool"][page, at, 5] = float("inf")
        n = (30, 70)[b]
        hit[t0:t0 + n] = (c["tree_mask"][t0:t0 + n, node // 64] >> (node % 64)) & 1 == 1
    got = tree_attention_paged(**c)
    check(c, got=got, ref=ref, rows=~hit)
    assert hit.any() and not torch.isfinite(got[hit]).any(-1).all()


def test_seen_infinite_values_reach_the_output():
    c = make(10, [6], [10], 4, 2, 64)
    pos = 10 + 3
    page, at = int(c["block_table"][0, pos // 16]), pos % 16
    c["v_pool"][page, at, 7] = float("inf")          # dim 7 of KV head 0
    c["v_pool"][page, at, 64 + 9] = float("nan")     # dim 9 of KV head 1
    sees = (c["tree_mask"][:, 0] >> 3) & 1 == 1
    got = tree_attention_paged(**c)
    assert sees.any() and not sees.all()
    assert (got[sees][:, :2, 7] == float("inf")).all() and got[sees][:, 2:, 9].isnan().all()
    assert torch.isfinite(got[~sees]).all()
    rest = got.clone()
    rest[:, :2, 7] = 0
    rest[:, 2:, 9] = 0
    assert torch.isfinite(rest).all()


def test_rows_out_of_range_are_left_as_they_were():
    n, start = [5, 9, 4, 6, 3], [100, 20, 0, 40, 50]
    good = make(11, n, start, 8, 2, 64, pad=4)
    cu = good["cu_q"].tolist()
    ref = reference(good)
    for change in ("kv small", "kv large", "kv negative", "offset"):
        c = dict(good, kv_len=good["kv_len"].clone(), cu_q=good["cu_q"].clone())
        lost = [3]
        if change == "kv small":
            c["kv_len"][3] = 5
        elif change == "kv large":
            c["kv_len"][3] = c["block_table"].shape[1] * 16 + 1
        elif change == "kv negative":
            c["kv_len"][3] = -7
        else:
            c["cu_q"][4] = cu[3] - 1                      # row 3 has -1 nodes, row 4 more than its own
            lost = [3, 4]
            c["kv_len"][4] = 2
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full_like(c["q"], 7.0)
        tree_attention_paged(**c, out=out, error=err)
        assert err.item() == 1
        keep = torch.ones(out.shape[0], dtype=torch.bool, device=DEV)
        keep[cu[-1]:] = False
        for b in lost:
            keep[cu[b]:cu[b + 1]] = False
        assert (out[~keep] == 7).all()
        check(good, got=out, ref=ref, rows=keep)
    # more nodes than the mask has words for
    c = make(12, [65, 3], [5, 6], 8, 2, 64)
    c["tree_mask"] = c["tree_mask"][:, :1].contiguous()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(c["q"], 7.0)
    tree_attention_paged(**c, out=out, error=err)
    assert err.item() == 1 and (out[:65] == 7).all() and (out[65:] != 7).any()


def test_rows_that_share_their_nodes_are_refused():
    """Offsets that go back and forth name more nodes than there are: nothing is computed."""
    c = make(13, [64] * 4, [30] * 4, 8, 1, 64)
    B = 40
    c["cu_q"] = torch.tensor([0, 64] * (B // 2) + [256], device=DEV)
    c["kv_len"] = torch.full((B,), 94, device=DEV)
    c["block_table"] = c["block_table"][:1].repeat(B, 1)
    c["cu_q"][::2] = 0
    c["cu_q"][1::2] = 256
    c["tree_mask"] = c["tree_mask"].repeat(1, 4)
    c["kv_len"] += 256
    c["block_table"] = c["block_table"].repeat(1, 4)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(c["q"], 7.0)
    tree_attention_paged(**c, out=out, error=err)
    assert err.item() == 1


def test_pages_outside_the_pool_are_reported():
    for page in (-1, 10 ** 6):
        c = make(14, [5, 9], [100, 20], 8, 2, 64)
        ref = reference(c)
        c["block_table"][0, 2] = page
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = tree_attention_paged(**c, error=err)
        assert err.item() == 1
        check(c, got=out, ref=ref, rows=slice(5, 14))


def test_arguments():
    c = make(15, [5, 9], [100, 20], 8, 2, 64)
    want = tree_attention_paged(**c)
    for bad in (dict(q=c["q"].float()), dict(q=c["q"].half()), dict(k_pool=c["k_pool"][:, :, :64]),
                dict(cu_q=c["cu_q"][:-1]), dict(block_table=c["block_table"][0]), dict(scale=0.0),
                dict(scale=float("nan")), dict(tree_mask=c["tree_mask"].int()), dict(tree_mask=c["tree_mask"][:3]),
                dict(tree_mask=c["tree_mask"][:, :0]), dict(out=want.float()), dict(out=want[:5]),
                dict(error=torch.zeros(1, device=DEV)), dict(kv_len=c["kv_len"].cpu()),
                dict(workspace=torch.empty(64, dtype=torch.uint8, device=DEV)), dict(scale=3e38)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            tree_attention_paged(**{**c, **bad})
    with pytest.raises(SpecdecError, match="head_dim"):
        e = make(15, [5], [10], 2, 1, 32)
        tree_attention_paged(**e)
    with pytest.raises(ValueError):
        tree_attention_workspace(0, 1, 8, 2, 64)
    ws = tree_attention_workspace(14, 2, 8, 2, 64)
    ws.fill_(255)                                          # no initial contents
    assert torch.equal(tree_attention_paged(**c, workspace=ws), want)
    wide = torch.zeros((14, 9, 8, 64), dtype=c["q"].dtype, device=DEV)
    wide[:, 4] = c["q"]
    assert torch.equal(tree_attention_paged(**{**c, "q": wide[:, 4]}), want)      # strided queries
    odd = torch.zeros(14 * 512 + 1, dtype=c["q"].dtype, device=DEV)[1:].view(14, 8, 64)
    odd.copy_(c["q"])
    assert torch.equal(tree_attention_paged(**{**c, "q": odd}), want)             # unaligned ones
    two = c["tree_mask"].repeat(1, 2)
    assert torch.equal(tree_attention_paged(**{**c, "tree_mask": two[:, :1]}), want)
    empty = {**c, "q": c["q"][:0], "tree_mask": c["tree_mask"][:0], "cu_q": c["cu_q"] * 0}
    assert tree_attention_paged(**empty).shape == (0, 8, 64)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes a side: pages at its end."""
    nb, bs, hkv, d = 70000, 16, 16, 128                    # 4.6 GB a side
    c = make(16, [9, 30], [200, 77], 32, hkv, d)
    for k in ("k_pool", "v_pool"):
        small = c[k]
        big = torch.zeros((nb, bs, hkv * d), dtype=small.dtype, device=DEV)
        big[nb - small.shape[0]:] = small
        c[k] = big
    ref = reference({**c, "block_table": torch.where(c["block_table"] >= 0, c["block_table"] + nb - small.shape[0],
                                                     -1)})
    c["block_table"] = torch.where(c["block_table"] >= 0, c["block_table"] + nb - small.shape[0], -1)
    check(c, ref=ref)


def test_streams_threads_and_a_graph():
    cs = [make(20 + i, [26, 5 + i, 40], [900 + 50 * i, 64, 10], 16, 4, 128) for i in range(3)]
    want = [tree_attention_paged(**c) for c in cs]
    torch.cuda.synchronize()
    got, streams = [None] * 3, [torch.cuda.Stream() for _ in range(3)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i] = tree_attention_paged(**cs[i])
        streams[i].synchronize()

    for where in (streams, [torch.cuda.default_stream()] * 3):
        streams = where
        threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs = []
    for c in cs[:2]:                                       # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = tree_attention_paged(**c)
        graphs.append((g, out, c))
    for seed in range(3):
        for i, (g, out, c) in enumerate(graphs):
            new = make(40 + seed, [26, 5 + i, 40], [800 + seed + 50 * i, 60, 10 + seed], 16, 4, 128)
            for k in ("q", "tree_mask", "kv_len"):
                c[k].copy_(new[k])
            g.replay()
        torch.cuda.synchronize()
        for g, out, c in graphs:
            assert torch.equal(out, tree_attention_paged(**c))
