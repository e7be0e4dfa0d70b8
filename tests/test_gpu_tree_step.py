"""Steps over trees of drafted tokens as a serving loop runs them, on a small model: layout, append,
tree attention, penalties, choices, the walk, and the accepted path's compaction, eagerly and as one
replayed graph. With greedy choices the rows have to go on exactly as a loop that knows no trees and
no cache pages does, token by token, whatever was drafted; the keys that stay in the cache are those
of the tokens that were accepted. Rows then branch and end by forked tables and copied pages.
"""
import numpy as np
import pytest
import torch

from specdec.attention import tree_attention_paged
from specdec.kvcache import (PagedKVCache, build_block_tables, copy_pages, fork_block_tables,
                             free_page_list)
from specdec.proposer_ops import greedy_draft_tokens
from specdec.sampling import penalize_logits, sample_from_probs, to_probs
from specdec.tree import tree_accept, tree_layout

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HKV, D, BS, V, P = 8, 2, 64, 16, 211, 6


def dev(x, dtype=None):
    return torch.as_tensor(np.asarray(x), device=DEV, dtype=dtype)


class Model:
    """One attention layer; logits so far apart that roundings decide nothing."""

    def __init__(self, seed=1, max_pos=400):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
        self.emb, self.pos = rnd(V, 96), rnd(max_pos, 96)
        self.w = {n: rnd(96, m * D) / 10 for n, m in (("q", HQ), ("k", HKV), ("v", HKV))}
        self.out = rnd(HQ * D, V)

    def qkv(self, tokens, positions):
        h = self.emb[tokens] + self.pos[positions]
        return [(h @ self.w[n]).to(torch.bfloat16) for n in "qkv"]

    def logits(self, att):
        return (att.float().reshape(att.shape[0], -1) @ self.out).to(torch.bfloat16)

    def greedy(self, tokens, prompt, new, pen):
        """The same row without a cache, a tree or a kernel of this package."""
        toks = list(tokens)
        for _ in range(new):
            t = dev(toks)
            q, k, v = self.qkv(t, torch.arange(len(toks), device=DEV))
            q = q[-1].double().view(HKV, HQ // HKV, D)
            k, v = (x.double().view(-1, HKV, D).transpose(0, 1) for x in (k, v))
            w = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / 8.0, -1)
            x = self.logits(torch.matmul(w, v).to(torch.bfloat16).view(1, HQ, D))[0].double()
            if pen:
                rep, freq, pres = pen
                c = torch.bincount(t[prompt:], minlength=V)
                seen = torch.bincount(t, minlength=V) > 0
                x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x) - freq * c - pres * (c > 0)
            toks.append(int(x.argmax()))
        return toks


def close(got, want):
    """The same products summed by library calls of other shapes: in fp32 apart by at most 96 2^-24
    sum |h w| < 2^-11 (the sum is below 80), then both rounded to bf16, one step of 2^-7 |x| more."""
    assert ((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() * 1.01 + 2.0 ** -10).all()


class Loop:
    def __init__(self, lens, room, pen, seed=3):
        self.m, self.pen, self.B = Model(), pen, len(lens)
        self.rng = np.random.default_rng(seed)
        self.rows = [list(self.rng.integers(0, V, n)) for n in lens]
        self.prompt = list(lens)
        mb, pages = -(-room // BS), len(lens) * -(-room // BS) + 3
        self.c = PagedKVCache(1, self.B, pages, BS, HKV, D, mb)
        self.c.pool.fill_(float("nan"))          # what was never written is never read
        free = torch.randperm(pages, device=DEV).to(torch.int32)
        build_block_tables(dev([room] * self.B), free, BS, mb, out=self.c.block_table, error=self.c.error)
        self.step([[-1] + list(range(n - 2)) for n in lens], [r[:-1] for r in self.rows], accept=False)
        self.c.lengths.copy_(dev([n - 1 for n in lens]))

    def forward(self, tokens, parents, cu, start, history, hlen, prompt, N, choose):
        """One step; all that a graph of it holds."""
        c = self.c
        kv = start + (cu[1:] - cu[:-1])
        mask, pos, slots = tree_layout(parents, cu, kv, c.block_table, BS, max_nodes=N, error=c.error)
        q, k, v = self.m.qkv(tokens, pos)
        c.append_slots(torch.stack([k, v])[None], slots)
        att = tree_attention_paged(q.view(-1, HQ, D), cu, c.pool[0, 0], c.pool[0, 1], c.block_table, kv,
                                   mask, error=c.error)
        x = self.m.logits(att)
        if self.pen:
            r, f, p = (torch.full((self.B,), z, device=DEV) for z in self.pen)
            x = penalize_logits(x, history, hlen, cu, prompt_len=prompt, repetition=r, frequency=f, presence=p,
                                node_tokens=tokens, tree_mask=mask, error=c.error)
        choice = choose(x)
        path, keep, y = tree_accept(tokens, parents, choice, cu, P, error=c.error)
        return choice, path, keep, y

    def step(self, parents, tokens, accept=True, choose=greedy_draft_tokens):
        n = [len(p) for p in parents]
        cu = dev(np.concatenate([[0], np.cumsum(n)]))
        H = max(len(r) for r in self.rows)
        hist = np.zeros((self.B, H), dtype=np.int64)
        for b, r in enumerate(self.rows):
            hist[b, :len(r)] = r
        # the history ends in front of the pending token, the tree's node 0
        args = (dev(sum(tokens, [])), dev(sum(parents, []), torch.int32), cu, self.c.lengths.clone(), dev(hist),
                dev([len(r) - 1 for r in self.rows]),
                dev(np.minimum(self.prompt, [len(r) - 1 for r in self.rows])), max(n))
        choice, path, keep, y = self.forward(*args, choose)
        if accept:
            self.c.compact(path, keep)
            for b, (k, p) in enumerate(zip(keep.tolist(), path.tolist())):
                if n[b]:
                    self.rows[b] += [tokens[b][i] for i in p[1:k]] + [int(y[b])]
        assert self.c.error.item() == 0
        return args, choice, path, keep, y

    def draft(self, n, hit):
        """Trees of n[b] nodes; some of their paths are what the row says next."""
        parents, tokens = [], []
        for b, m in enumerate(n):
            if m == 0:
                parents.append([]), tokens.append([])
                continue
            p = [-1] + [int(self.rng.integers(0, i)) for i in range(1, m)]
            t = [self.rows[b][-1]] + list(self.rng.integers(0, V, m - 1))
            nxt = self.m.greedy(self.rows[b], self.prompt[b], hit[b], self.pen)[len(self.rows[b]):]
            at = 0
            for i in range(1, m):               # the right tokens along some path
                if p[i] == at and nxt and self.rng.random() < 0.8:
                    t[i], at = nxt.pop(0), i
            parents.append(p), tokens.append([int(x) for x in t])
        return parents, tokens


@pytest.mark.parametrize("pen", [None, (1.2, 0.3, 0.5)])
def test_greedy_rows_go_on_as_without_trees(pen):
    s = Loop([20, 3, 33, 17], 200, pen)
    start = [list(r) for r in s.rows]
    accepted = 0
    for k in range(5):
        n = [[26, 64, 1, 7], [5, 0, 30, 64], [70, 9, 9, 9], [12, 40, 3, 0], [1, 1, 1, 1]][k]
        *_, keep, _ = s.step(*s.draft(n, [3, 4, 2, 1]))
        accepted += int((keep - 1).clamp(min=0).sum())
    assert accepted > 8                          # trees with nothing to accept would test little
    for b, r in enumerate(s.rows):
        assert r == s.m.greedy(start[b], s.prompt[b], len(r) - len(start[b]), pen)
        # the cache holds the keys of the row's tokens but the pending one
        L = len(r) - 1
        assert int(s.c.lengths[b]) == L
        _, k, v = s.m.qkv(dev(r[:-1]), torch.arange(L, device=DEV))
        for side, want in ((0, k), (1, v)):
            close(s.c.gather(0, side, b, L), want)


def test_sampled_choices_and_a_replayed_graph():
    """A step as one graph: the same tokens, paths and keys as eagerly, replay after replay."""
    s = Loop([20, 3, 33], 160, (1.1, 0.2, 0.1))
    u = torch.rand(26 + 9 + 40, device=DEV)
    choose = lambda x: sample_from_probs(to_probs(x, 0.9, 0.95), u=u)  # noqa: E731
    n = [26, 9, 40]
    args, *_ = s.step(*s.draft(n, [2, 2, 2]), choose=choose)
    args = (*(torch.nn.functional.pad(a, (0, 60)) if i == 4 else a.clone() if torch.is_tensor(a) else a
              for i, a in enumerate(args)),)
    lengths, pool = s.c.lengths.clone(), s.c.pool.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = s.forward(*args, choose)
        s.c.compact(out[1], out[2])
    s.c.lengths.copy_(lengths), s.c.pool.copy_(pool)
    for k in range(3):
        parents, tokens = s.draft(n, [3, 3, 3])
        u.copy_(torch.rand(75, device=DEV))
        lengths, pool, rows = s.c.lengths.clone(), s.c.pool.clone(), [list(r) for r in s.rows]
        eager_args, *eager = s.step(parents, tokens, choose=choose)
        after = (s.c.lengths.clone(), s.c.pool.clone())
        s.c.lengths.copy_(lengths), s.c.pool.copy_(pool)
        for a, e in zip(args, eager_args):
            if torch.is_tensor(a):
                a[tuple(slice(0, x) for x in e.shape)].copy_(e)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager))
        assert torch.equal(s.c.lengths, after[0])
        assert torch.equal(s.c.pool.nan_to_num(7.0), after[1].nan_to_num(7.0))
        assert rows != s.rows


def test_rows_branch_and_end():
    """Row 0 goes on as two rows and row 1 as one, row 2 ends: both branches go on by themselves."""
    s = Loop([20, 30, 9, 5], 96, None)
    s.step(*s.draft([9, 9, 9, 9], [2, 2, 2, 2]))
    c, kv = s.c, s.c.lengths.clone()
    par = dev([0, 1, 0, 3])
    free, num = free_page_list(c.block_table, c.num_blocks, kv_len=kv, block_size=BS, error=c.error)
    table, copies, used = fork_block_tables(c.block_table, kv, par, kv[par] + 40, free, BS, num_free=num,
                                            error=c.error)
    copy_pages(c.pool, copies, error=c.error)
    c.block_table.copy_(table), c.lengths.copy_(kv[par])
    s.rows = [list(s.rows[b]) for b in (0, 1, 0, 3)]
    s.prompt = [s.prompt[b] for b in (0, 1, 0, 3)]
    s.rows[2][-1] = (s.rows[2][-1] + 1) % V      # the second branch's pending token is another
    start = [list(r) for r in s.rows]
    for _ in range(3):
        s.step(*s.draft([12, 5, 12, 30], [2, 2, 2, 2]))
    assert c.error.item() == 0 and s.rows[0] != s.rows[2]
    for b, r in enumerate(s.rows):
        assert r == s.m.greedy(start[b], s.prompt[b], len(r) - len(start[b]), None)
