"""Several answers of one prompt, as a serving step runs them: block tables laid out once, the
prompt run through each group's first row, then steps of ragged new tokens - slots, append,
attention over the shared prompt, log probabilities - with tokens taken back in between,
eagerly and as a replayed graph. Every step's attention is compared with float64 over the keys
and values that each answer was given, kept apart from the cache, its scores with the float64
oracle. Tolerances: those of the attention's and the log probabilities' own tests, for the
attention u |out| + (u + e) A (1 + u) with u = 2^-8, A = sum p |v| / sum p and
e = 2^-24 (4 (d + 8) S + n / 32 + 256), S the largest scale sum |q k|.
"""
import math

import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from specdec.attention import shared_prefix_attention_paged
from specdec.kvcache import (PagedKVCache, build_block_tables, paged_slot_mapping)
from specdec.sampling import token_logprobs
from specdec.tinylm import HEAD, TinyLM

pytestmark = pytest.mark.gpu
DEV = "cuda"
T_LOGITS, TOP = 0.8, 5


class Answers:
    def __init__(self, prompts, answers, room, hq=8, hkv=2, vocab=1009, bs=16):
        """prompts: tokens per group; answers: rows per group; room: new tokens per row."""
        self.lm = TinyLM(vocab, hq=hq, hkv=hkv, max_pos=512, seed=7)
        self.hq, self.hkv, self.V, self.bs = hq, hkv, vocab, bs
        self.g = torch.Generator(device=DEV).manual_seed(9)
        self.cu_group = np.concatenate([[0], np.cumsum(answers)])
        self.group = np.repeat(np.arange(len(prompts)), answers)
        self.prompts = prompts
        B = len(self.group)
        self.len = np.asarray(prompts)[self.group]
        full = torch.as_tensor(self.len + room, device=DEV)
        self.dcu, self.dpre = (torch.as_tensor(x, device=DEV) for x in (self.cu_group, prompts))
        mb = int(-(-(max(prompts) + room) // bs))
        pages = int((-(-(self.len + room) // bs)).sum())
        self.cache = PagedKVCache(1, B, pages, bs, hkv, HEAD, mb)
        self.cache.pool.fill_(float("nan"))  # slots that were never written are never read
        free = torch.randperm(pages, generator=self.g, device=DEV).to(torch.int32)
        build_block_tables(full, free, bs, mb, self.dcu, self.dpre, out=self.cache.block_table,
                           error=self.cache.error)
        # what each answer was given: K and V of its positions, the prompt's of its first row's
        self.kv = [torch.zeros((2, 0, hkv * HEAD), dtype=torch.bfloat16, device=DEV) for _ in range(B)]

    def step(self, tok, nxt, cu_q, kv_len):
        """One forward of packed tokens; all that a graph of it would hold."""
        p, c = self.lm.p, self.cache
        pos, slots = paged_slot_mapping(c.block_table, cu_q, kv_len, self.bs, tok.numel(), error=c.error)
        h = p["emb"][tok] + p["pos"][pos]
        q, k, v = (torch.mm(h, p[n]) for n in ("wq", "wk", "wv"))
        staged = torch.stack([k, v]).unsqueeze(0)
        c.append_slots(staged, slots)
        att = shared_prefix_attention_paged(q.view(-1, self.hq, HEAD), cu_q, c.pool[0, 0], c.pool[0, 1],
                                            c.block_table, kv_len, self.dcu, self.dpre, error=c.error)
        logits = torch.mm(h + torch.mm(att.view(-1, self.hq * HEAD), p["wo"]), p["wlm"])
        return (staged, q, att, logits, *token_logprobs(logits, nxt, T_LOGITS, TOP))

    def inputs(self, n, pad):
        """Random tokens, n[b] for row b, padded to `pad`: (tokens, next ids, cu_q, kv_len)."""
        self.len = self.len + n
        cu = np.concatenate([[0], np.cumsum(n)])
        tok, nxt = torch.randint(0, self.V, (2, pad), generator=self.g, device=DEV)
        return tok, nxt, torch.as_tensor(cu, device=DEV), torch.as_tensor(self.len, device=DEV)

    def check(self, n, out, nxt):
        staged, q, att, logits, logp, ent, top_logp, top_ids = out
        assert self.cache.error.item() == 0
        u, at, group = 2.0 ** -8, 0, self.hq // self.hkv
        for b, m in enumerate(n):
            if m == 0:
                continue
            new = staged[0, :, at:at + m]
            self.kv[b] = torch.cat([self.kv[b], new], 1)
            L = self.kv[b].shape[1]
            assert L == self.len[b]
            k, v = self.kv[b].double().view(2, L, self.hkv, HEAD).permute(0, 2, 1, 3).unbind(0)
            x = q[at:at + m].double().view(m, self.hkv, group, HEAD).permute(1, 2, 0, 3)
            kt = k.transpose(1, 2).contiguous().unsqueeze(1)
            sees = torch.arange(L, device=DEV) <= (L - m + torch.arange(m, device=DEV)).unsqueeze(1)
            w = torch.softmax((torch.matmul(x, kt) / math.sqrt(HEAD)).masked_fill(~sees, -math.inf), -1)
            S = float(torch.matmul(x.abs(), kt.abs()).max()) / math.sqrt(HEAD)
            want, A = torch.matmul(w, v.unsqueeze(1)), torch.matmul(w, v.abs().unsqueeze(1))
            got = att[at:at + m].double().view(m, self.hkv, group, HEAD).permute(1, 2, 0, 3)
            e = 2.0 ** -24 * (4 * (HEAD + 8) * S + L / 32 + 256)
            off = (got - want).abs() - (u * want.abs() + (u + e) * A * (1 + u))
            assert off.max().item() <= 0, (b, off.max().item())
            at += m
        rl, re, rt, ri = OL.token_logprobs(logits[:at].double().cpu().numpy(),
                                           nxt[:at, None].cpu().numpy(), T_LOGITS, TOP)
        U = 2.0 ** -24
        base = U * (self.V / 256 + 32 + 24 + 2 * (re + np.log(self.V)))
        cpu = lambda t: t[:at].double().cpu().numpy()  # noqa: E731
        assert (np.abs(cpu(logp)[:, None] - rl) <= base[:, None] + 3 * U * np.abs(rl)).all()
        assert (np.abs(cpu(ent) - re) <= 2 * base * (1 + np.abs(re))).all()
        assert (np.abs(cpu(top_logp) - rt) <= base[:, None] + 3 * U * np.abs(rt)).all()
        assert np.array_equal(top_ids[:at].cpu().numpy(), ri)

    def prefill(self):
        """Each group's prompt through its first row; the other rows have it thereby."""
        n = np.zeros(len(self.group), dtype=np.int64)
        n[self.cu_group[:-1]] = self.prompts
        before = self.len
        self.len = before - n
        args = self.inputs(n, int(n.sum()))
        self.check(n, self.step(*args), args[1])
        for b in range(len(n)):
            self.kv[b] = self.kv[self.cu_group[self.group[b]]]

    def take_back(self, n):
        self.len = self.len - n
        for b in range(len(n)):
            self.kv[b] = self.kv[b][:, :self.len[b]]


@pytest.mark.parametrize("prompts,answers,heads", [
    ([37, 5, 150], [4, 1, 3], (8, 2)),
    ([64], [6], (4, 1)),
    ([1, 333], [2, 5], (4, 4)),
])
def test_answers_of_a_prompt(prompts, answers, heads):
    a = Answers(prompts, answers, 90, *heads)
    a.prefill()
    B, rng = len(a.group), np.random.default_rng(len(prompts))
    for _ in range(4):
        n = rng.integers(0, 6, B)
        n[0] += n.sum() == 0
        args = a.inputs(n, int(n.sum()))
        a.check(n, a.step(*args), args[1])
        a.take_back(rng.integers(0, n + 1))
    # the same step as a graph over buffers that the steps fill, padded to a fixed size
    pad = 6 * B
    static = [t.clone() for t in a.inputs(np.zeros(B, dtype=np.int64), pad)]
    static[2].zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.step(*static)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step(*static)
    for i in range(6):
        n = rng.integers(0, 7, B) if i != 2 else np.zeros(B, dtype=np.int64)
        args = a.inputs(n, pad)
        for t, x in zip(static, args):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        if n.sum():
            a.check(n, out, args[1])
        a.take_back(rng.integers(0, n + 1))
