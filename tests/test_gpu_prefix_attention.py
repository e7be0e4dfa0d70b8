"""GPU parity of shared_prefix_attention_paged with softmax(q k^T scale) v in float64, row by
row.

Tolerance, elementwise: with u half a step of the type (2^-8 bf16, 2^-11 fp16) the output's
own rounding is u |out|; every weight is rounded once, which moves the output by at most
u A, A = sum p |v| / sum p; and the fp32 part (scores over d products, the exponential's
argument, sums over chains of n / 64 + 64 keys, the joins) moves weights by at most
e = 2^-24 (4 (d + 8) S + n / 32 + 256) relative, numerator and denominator, S the largest
scale sum |q k|: u |out| + (u + e) A (1 + u).
"""
import math

import numpy as np
import pytest
import torch

from specdec._lib import SpecdecError
from specdec.attention import (shared_attention_workspace, shared_prefix_attention_paged,
                               verify_attention_paged)
from specdec.kvcache import build_block_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(seed, n, prefix, own, q, hq, hkv, d, bs=16, dtype=torch.bfloat16, pad=0, kv=None):
    """n: rows per group; prefix: per group; own, q: per row (own keys before the new ones)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, prefix, own, q = (np.asarray(x, dtype=np.int64) for x in (n, prefix, own, q))
    cu_g = np.concatenate([[0], np.cumsum(n)])
    cu_q = np.concatenate([[0], np.cumsum(q)])
    kv = np.repeat(prefix, n) + own + q if kv is None else np.asarray(kv)
    need = -(-kv // bs)
    mb = int(need.max()) + 1
    dev = lambda x: torch.as_tensor(x, device=DEV)  # noqa: E731
    free = torch.randperm(int(need.sum()) + 3, generator=g, device=DEV).to(torch.int32)
    table, used = build_block_tables(dev(kv), free, bs, mb, dev(cu_g), dev(prefix))
    T, nb = int(cu_q[-1]) + pad, free.numel()
    rnd = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    return dict(q=rnd(T, hq, d), cu_q=dev(cu_q), k_pool=rnd(nb, bs, hkv * d), v_pool=rnd(nb, bs, hkv * d),
                block_table=table, kv_len=dev(kv), cu_group=dev(cu_g), prefix_len=dev(prefix))


def reference(c, scale=None):
    """(out, A, S) in float64; rows without tokens leave zeros."""
    q, kp, vp = c["q"].double(), c["k_pool"], c["v_pool"]
    T, hq, d = q.shape
    bs, hkv = kp.shape[1], kp.shape[2] // d
    scale = 1 / math.sqrt(d) if scale is None else scale
    cu, kv, cg, pre = (c[k].tolist() for k in ("cu_q", "kv_len", "cu_group", "prefix_len"))
    out, A = torch.zeros_like(q), torch.zeros_like(q)
    S = 0.0
    for g in range(len(pre)):
        for b in range(cg[g], cg[g + 1]):
            n, m = kv[b], cu[b + 1] - cu[b]
            if m == 0:
                continue
            pos = torch.arange(n, device=DEV)
            row = torch.where(pos < pre[g], cg[g], b)
            page = c["block_table"][row, pos // bs].long()
            k = kp[page, pos % bs].double().view(n, hkv, d).permute(1, 2, 0).contiguous()
            v = vp[page, pos % bs].double().view(n, hkv, d).permute(1, 0, 2).contiguous()
            x = q[cu[b]:cu[b + 1]].view(m, hkv, hq // hkv, d).permute(1, 2, 0, 3)
            sees = pos <= (n - m + torch.arange(m, device=DEV)).unsqueeze(1)
            w = (torch.matmul(x, k.unsqueeze(1)) * scale).masked_fill(~sees, -math.inf)
            S = max(S, float((torch.matmul(x.abs(), k.abs().unsqueeze(1)) * scale).max()))
            p = torch.softmax(w, -1)
            o, a = torch.matmul(p, v.unsqueeze(1)), torch.matmul(p, v.abs().unsqueeze(1))
            out[cu[b]:cu[b + 1]] = o.permute(2, 0, 1, 3).reshape(m, hq, d)
            A[cu[b]:cu[b + 1]] = a.permute(2, 0, 1, 3).reshape(m, hq, d)
    return out, A, S


def check(c, scale=None, got=None, rows=None):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    if got is None:
        got = shared_prefix_attention_paged(**c, scale=scale, error=err)
    want, A, S = reference(c, scale)
    u = torch.finfo(got.dtype).eps / 2
    e = 2.0 ** -24 * (4 * (got.shape[2] + 8) * S + int(c["kv_len"].max()) / 32 + 256)
    off = (got.double() - want).abs() - (u * want.abs() + (u + e) * A * (1 + u))
    T = int(c["cu_q"][-1])
    off = off[:T] if rows is None else off[rows]
    assert torch.isfinite(got[:T] if rows is None else got[rows]).all()
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()
    assert err.item() == 0
    return got


@pytest.mark.parametrize("n,prefix,own,q,heads,bs,dtype", [
    ([1], [0], [0], [1], (1, 1, 64), 16, torch.bfloat16),           # one key
    ([1], [5], [0], [1], (4, 4, 128), 16, torch.float16),           # a group of one row
    ([2], [1], [0, 0], [1, 1], (8, 2, 128), 16, torch.bfloat16),
    ([4], [64], [0, 1, 63, 64], [1, 1, 1, 1], (32, 8, 128), 16, torch.bfloat16),
    ([4], [63], [5, 70, 0, 130], [3, 1, 5, 2], (32, 8, 128), 16, torch.float16),
    ([3], [65], [200, 127, 128], [9, 1, 4], (16, 2, 64), 7, torch.bfloat16),
    ([5], [129], [3, 0, 9, 1, 4], [1, 0, 2, 0, 3], (14, 2, 64), 1, torch.float16),
    ([6], [1000], [30, 0, 500, 2, 9, 77], [2, 5, 1, 4, 9, 3], (32, 8, 128), 16, torch.bfloat16),
    ([2, 0, 3, 1], [300, 40, 17, 90], [8, 2, 0, 31, 5, 64], [1, 4, 2, 2, 0, 3], (8, 1, 128), 32,
     torch.bfloat16),                                               # groups, an empty and a single one
    ([3, 2], [0, 250], [90, 700, 3, 1, 2], [1, 2, 3, 1, 1], (10, 2, 128), 16, torch.float16),
    ([2], [40], [10, 20], [70, 33], (4, 2, 128), 16, torch.bfloat16),  # own rows of the shared form
    ([2], [500], [0, 7], [300, 1], (8, 8, 64), 16, torch.float16),
    ([40], [777], [13] * 40, [1] * 40, (8, 2, 128), 16, torch.bfloat16),
    ([64], [2000], list(range(64)), [1 + i % 9 for i in range(64)], (32, 8, 128), 16, torch.bfloat16),
    ([9] * 20, [50 + 7 * i for i in range(20)], [i % 50 for i in range(180)],
     [i % 4 for i in range(180)], (6, 3, 64), 16, torch.bfloat16),
])
def test_matches_float64(n, prefix, own, q, heads, bs, dtype):
    check(make(len(own) + sum(prefix), n, prefix, own, q, *heads, bs=bs, dtype=dtype))


@pytest.mark.parametrize("P,own,q,rows,heads", [
    (40000, 3, 1, 1, (8, 8, 128)),     # one row: its keys over the whole grid, many parts
    (40000, 3, 1, 2, (8, 1, 128)),     # a prefix over the whole grid
    (10, 30000, 2, 3, (8, 2, 64)),     # long rows behind a short prefix
    (9000, 1500, 7, 16, (16, 4, 128)),
])
def test_long_keys(P, own, q, rows, heads):
    check(make(P + own, [rows], [P], [own + i for i in range(rows)], [q] * rows, *heads))


def test_many_rows_and_groups():
    """More segments than threads: several per thread."""
    rng = np.random.default_rng(3)
    n = rng.integers(0, 5, 400)
    B = int(n.sum())
    check(make(5, n, rng.integers(0, 80, 400), rng.integers(0, 90, B), rng.integers(0, 3, B), 4, 2, 64))


def test_equals_the_attention_without_sharing():
    """The same tables read by verify_attention_paged, whose rows read the prefix each."""
    c = make(11, [5, 3], [96, 160], [9, 30, 0, 7, 200, 1, 2, 64], [3, 1, 2, 5, 4, 1, 1, 9], 32, 8, 128)
    got = check(c)
    other = verify_attention_paged(c["q"], c["cu_q"], c["k_pool"], c["v_pool"], c["block_table"],
                                   c["kv_len"], 9)
    assert (got.float() - other.float()).abs().max() < 3e-2


def test_prefix_that_ends_inside_a_page():
    """Of the page with the prefix's end, a row's own page holds other bytes before it: they
    are not read."""
    c = make(2, [4], [37], [20, 3, 0, 8], [2, 1, 3, 1], 8, 2, 128)
    own_pages = c["block_table"][1:, 2].long()
    c["k_pool"][own_pages, :5] = float("nan")
    c["v_pool"][own_pages, :5] = float("nan")
    check(c)


def test_queries_inside_the_prefix():
    """Rows whose keys end inside the prefix see their part of it, their new positions one
    key more each; a row that is shorter than one page too."""
    for heads in ((8, 2, 128), (4, 4, 64)):
        for q in ([4, 3, 9, 1, 2], [40, 17, 3, 1, 2]):
            kv = [200, 150, 64, 7, 260]
            check(make(8, [5], [200], [0] * 5, q, *heads, kv=kv))


def test_keys_that_no_query_sees():
    """NaN and infinities in every slot that is not a visible key: page tails behind a row's
    end, pages of nobody."""
    for dtype, heads in ((torch.bfloat16, (32, 8, 128)), (torch.float16, (8, 2, 64))):
        for q in (1, 20):
            c = make(4, [6], [333], [0, 5, 70, 130, 64, 1], [q] * 6, *heads, dtype=dtype)
            bs, nb = 16, c["k_pool"].shape[0]
            used = torch.zeros((nb, bs), dtype=torch.bool, device=DEV)
            for b in range(6):
                pos = torch.arange(int(c["kv_len"][b]), device=DEV)
                row = torch.where(pos < 333, 0, b)
                used[c["block_table"][row, pos // bs].long(), pos % bs] = True
            c["k_pool"][~used] = float("nan")
            c["v_pool"][~used] = float("inf")
            check(c)


@pytest.mark.parametrize("dtype,heads,q", [
    (torch.bfloat16, (32, 8, 128), [6, 3, 8, 1]),   # a wave's keys each
    (torch.bfloat16, (16, 1, 128), [9, 70, 40, 3]),  # tiles that the waves share
    (torch.float16, (8, 2, 64), [5, 8, 2, 7]),
    (torch.float16, (8, 1, 64), [9, 80, 20, 30]),
])
def test_keys_that_some_queries_see(dtype, heads, q):
    """NaN and infinities in K and V of one of a row's new tokens: the row's tokens before it
    are as without them, it and those after it as the formula has it."""
    for seed, prefix, kv in ((21, 100, None), (22, 200, [200, 150, 70, 260])):
        own = [0, 150, 64, 7]
        c = make(seed, [4], [prefix], own, q, *heads, dtype=dtype, kv=kv)
        plain = shared_prefix_attention_paged(**c)
        for b in range(4):
            end, at = int(c["kv_len"][b]), q[b] // 2  # the at-th new token's position
            pos = end - q[b] + at
            page = int(c["block_table"][0 if pos < prefix else b, pos // 16])
            rows = slice(int(c["cu_q"][b]), int(c["cu_q"][b]) + at)
            for name, value, dims in (("v_pool", float("nan"), slice(3, 5)),
                                      ("v_pool", float("inf"), slice(0, None)),
                                      ("v_pool", -float("inf"), slice(17, 50)),
                                      ("k_pool", float("nan"), slice(1, 2))):
                d = dict(c, **{name: c[name].clone()})
                d[name][page, pos % 16, dims] = value
                got = shared_prefix_attention_paged(**d)
                if name == "v_pool":
                    assert torch.equal(got[rows], plain[rows])
                else:  # other rows' scores move the running maximum's steps
                    check(c, got=got, rows=torch.arange(rows.start, rows.stop, device=DEV))
                if pos >= prefix and name == "v_pool":  # of this row alone
                    keep = torch.ones(got.shape[0], dtype=torch.bool, device=DEV)
                    keep[rows.stop:int(c["cu_q"][b + 1])] = False
                    assert torch.equal(got[keep], plain[keep])
                after = got[rows.stop:int(c["cu_q"][b + 1])].view(-1, heads[0], heads[2])
                if name == "k_pool":  # the first KV head's scores
                    assert after[:, :heads[0] // heads[1]].isnan().all()
                else:  # the formula's value in the dims set, and finite values in the others
                    want = torch.zeros(heads[1] * heads[2], dtype=dtype, device=DEV)
                    want[dims] = value
                    want = want.view(heads[1], heads[2]).repeat_interleave(heads[0] // heads[1], 0)
                    odd = ~want.isfinite()
                    assert after.isfinite().logical_not().equal(odd.expand_as(after))
                    assert after[odd.expand_as(after)].nan_to_num(7, 8, 9).eq(
                        want.nan_to_num(7, 8, 9)[odd].repeat(after.shape[0])).all()


def test_extreme_scores():
    """Scores far apart (one key takes all), equal everywhere, and rising along the keys, so
    that the running maximum moves by more and by less than its slack."""
    for dtype in (torch.bfloat16, torch.float16):
        c = make(6, [3], [700], [90, 0, 300], [3, 30, 1], 8, 2, 128, dtype=dtype)
        check(c, scale=6.0)
        check(c, scale=1e-6)
        ramp = torch.linspace(0, 3, c["k_pool"].shape[0], device=DEV).view(-1, 1, 1)
        c["k_pool"] = (ramp.expand_as(c["k_pool"])).to(dtype).contiguous()
        c["q"] = c["q"].abs()
        check(c)
        c["k_pool"] = -c["k_pool"]
        check(c)


def test_rows_out_of_range_are_left_alone():
    """Rows with impossible lengths and groups with impossible offsets: the error is set,
    their output stays, the others are served; tokens behind the last row stay as they were."""
    def run(c):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full_like(c["q"], 7.0)
        got = shared_prefix_attention_paged(**c, out=out, error=err)
        assert got is out
        return out, err.item()

    c = make(3, [3, 2], [64, 40], [9, 3, 30, 8, 1], [2, 1, 3, 4, 2], 8, 2, 128, pad=5)
    out, e = run(c)
    assert e == 0 and (out[12:] == 7).all()
    good = check(c, got=out)
    for row, kv in ((1, 0), (4, 10 ** 6), (3, -5)):
        d = dict(c, kv_len=c["kv_len"].clone())
        d["kv_len"][row] = kv
        out, e = run(d)
        a, b = int(c["cu_q"][row]), int(c["cu_q"][row + 1])
        assert e == 1 and (out[a:b] == 7).all()
        keep = torch.ones(12, dtype=torch.bool, device=DEV)
        keep[a:b] = False
        check(c, got=out, rows=keep.nonzero().squeeze(1))
    d = dict(c, prefix_len=torch.tensor([64, -1], device=DEV))
    out, e = run(d)
    assert e == 1 and (out[6:] == 7).all()
    check(c, got=out, rows=torch.arange(6, device=DEV))
    for cu in ([0, 3, 4], [1, 3, 5], [0, 9, 5]):
        out, e = run(dict(c, cu_group=torch.tensor(cu, device=DEV)))
        assert e == 1
    out, e = run(dict(c, cu_q=torch.tensor([0, 2, 3, 6, 10, 400], device=DEV)))
    assert e == 1 and (out[10:] == 7).all()
    d = dict(c, block_table=c["block_table"].clone())
    d["block_table"][4, 3 if int(c["kv_len"][4]) > 48 else 2] = 10 ** 6
    out, e = run(d)
    assert e == 1
    check(c, got=out, rows=torch.arange(10, device=DEV))
    assert torch.equal(run(c)[0], good)


def test_pool_offsets_past_32_bits():
    """Pages at the end of a pool of more than 2^32 elements."""
    hkv, d, bs = 8, 128, 64
    nb = (1 << 32) // (hkv * d * bs) + 70
    c = make(9, [3], [150], [70, 3, 0], [2, 1, 4], 8, hkv, d, bs=bs)
    small = c["k_pool"].shape[0]
    for name in ("k_pool", "v_pool"):
        big = torch.empty((nb, bs, hkv * d), dtype=torch.bfloat16, device=DEV)
        big[:4] = float("nan")
        big[nb - small:] = c[name]
        c[name] = big
    t = c["block_table"]
    c["block_table"] = torch.where(t >= 0, t + (nb - small), t).contiguous()
    check(c)


def test_a_long_prompt_in_one_call():
    """33,000 new tokens of a group's first row and none of the others': 132,000 query rows of
    a KV head; some of them checked."""
    T, hq, hkv, d = 33000, 8, 2, 64
    c = make(31, [3], [T], [0, 0, 0], [T, 0, 0], hq, hkv, d, kv=[T, T, T], dtype=torch.float16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = shared_prefix_attention_paged(**c, error=err)
    assert err.item() == 0 and torch.isfinite(got).all()
    pos = torch.arange(T, device=DEV)
    page = c["block_table"][0, pos // 16].long()
    k, v = (c[n][page, pos % 16].double().view(T, hkv, d) for n in ("k_pool", "v_pool"))
    for t in (0, 1, 63, 64, 127, 128, 5000, 16383, 16384, 32767, 32768, T - 1):
        x = c["q"][t].double().view(hkv, hq // hkv, d)
        kt = k[:t + 1].permute(1, 2, 0).contiguous()
        vt = v[:t + 1].permute(1, 0, 2).contiguous()
        w = torch.softmax(torch.matmul(x, kt) / math.sqrt(d), -1)
        S = float(torch.matmul(x.abs(), kt.abs()).max()) / math.sqrt(d)
        want, A = torch.matmul(w, vt), torch.matmul(w, vt.abs())
        u = 2.0 ** -11
        e = 2.0 ** -24 * (4 * (d + 8) * S + T / 32 + 256)
        off = (got[t].double().view_as(want) - want).abs() - (u * want.abs() + (u + e) * A * (1 + u))
        assert off.max().item() <= 0, (t, off.max().item())


def test_arguments():
    c = make(1, [2], [20], [3, 4], [1, 2], 4, 2, 64)

    def bad(**kw):
        return shared_prefix_attention_paged(**dict(c, **kw))

    with pytest.raises(TypeError):
        bad(q=c["q"].float())
    with pytest.raises(TypeError):
        bad(q=c["q"].half())
    with pytest.raises(ValueError, match="contiguous"):
        bad(k_pool=c["k_pool"].transpose(0, 1).contiguous().transpose(0, 1),
            v_pool=c["v_pool"].transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError, match="query heads"):
        bad(q=torch.zeros((3, 3, 64), dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="lengths need"):
        bad(cu_q=c["cu_q"][:-1])
    with pytest.raises(ValueError, match="lengths need"):
        bad(cu_group=c["cu_group"][:-1])
    with pytest.raises(ValueError, match="scale"):
        bad(scale=0.0)
    with pytest.raises(ValueError, match="scale"):
        bad(scale=float("nan"))
    with pytest.raises(ValueError, match="out must be"):
        bad(out=torch.zeros((3, 4, 128), dtype=torch.bfloat16, device=DEV))
    with pytest.raises(SpecdecError, match="workspace"):
        bad(workspace=torch.zeros(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(SpecdecError, match="head_dim"):
        shared_prefix_attention_paged(**make(1, [2], [20], [3, 4], [1, 2], 4, 2, 96))
    with pytest.raises(RuntimeError, match="ROCm device"):
        bad(kv_len=c["kv_len"].cpu())
    with pytest.raises(ValueError):
        shared_attention_workspace(3, 2, 1, 4, 3, 64)
    assert bad(q=c["q"][:0], cu_q=torch.zeros(3, dtype=torch.long, device=DEV)).shape == (0, 4, 64)


def test_strided_queries_and_given_workspace():
    c = make(12, [3], [90], [3, 40, 4], [1, 2, 9], 8, 2, 128)
    want = check(c)
    qkv = torch.cat([c["q"], c["q"][:, :4]], 1)
    ws = shared_attention_workspace(12, 3, 1, 8, 2, 128)
    got = shared_prefix_attention_paged(**dict(c, q=qkv[:, :8]), workspace=ws)
    assert torch.equal(got, want)
    ws.fill_(255)                       # no initial contents
    assert torch.equal(shared_prefix_attention_paged(**c, workspace=ws), want)
    flat = torch.zeros(c["q"].numel() + 1, dtype=torch.bfloat16, device=DEV)
    flat[1:] = c["q"].flatten()         # two bytes past a 16-byte boundary
    assert torch.equal(shared_prefix_attention_paged(**dict(c, q=flat[1:].view_as(c["q"]))), want)


def test_graphs_and_streams():
    """Two captured calls of different batches replayed in turn with eager calls between, and
    calls on two streams at once, each give the eager bits; lengths may change between
    replays."""
    a = make(21, [8], [800], [9] * 8, [2] * 8, 32, 8, 128)
    b = make(22, [3, 2], [100, 900], [5, 70, 1, 2, 3], [1, 4, 2, 1, 1], 32, 8, 128)
    want = [check(a).clone(), check(b).clone()]
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(shared_prefix_attention_paged(**c))
        graphs.append(g)
    for turn in range(4):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        eager = shared_prefix_attention_paged(**(a, b)[turn % 2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(eager, want[turn % 2])
    a["kv_len"] -= 4                    # a rollback in place
    graphs[0].replay()
    torch.cuda.synchronize()
    check(a, got=outs[0])
    a["kv_len"] += 4
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(shared_prefix_attention_paged(**(a, b)[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
