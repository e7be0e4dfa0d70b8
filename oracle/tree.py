"""Trees of drafted tokens and the cache's pages after them, row by row.

TEST INFRASTRUCTURE ONLY (see `oracle/__init__.py`). The chain forms are the slot formula of
`vllm_draft_spec/proposer.py:295-314` and the accept loop of `specdec/engine.py:285-303`.
"""
import numpy as np


def tree_layout(parents, cu_q, kv_len, table, block_size, words, num_tokens, padding=-1):
    """-> (mask as sets of nodes per token, positions, slots, ok)."""
    sees = [set() for _ in range(num_tokens)]
    pos = np.zeros(num_tokens, dtype=np.int64)
    slots = np.full(num_tokens, padding, dtype=np.int64)
    ok = cu_q[0] == 0 and cu_q[-1] <= num_tokens
    for b in range(len(kv_len)):
        q0, q1, kv = int(cu_q[b]), int(cu_q[b + 1]), int(kv_len[b])
        n = q1 - q0
        good = 0 <= q0 <= q1 <= num_tokens and n <= 64 * words and kv >= n
        good = good and (table is None or kv <= table.shape[1] * block_size)
        good = good and all(-1 <= parents[q0 + i] < i for i in range(n))
        if not good:
            ok = False
            continue
        for i in range(n):
            p = int(parents[q0 + i])
            sees[q0 + i] = {i} | (sees[q0 + p] if p >= 0 else set())
            pos[q0 + i] = kv - n + len(sees[q0 + i]) - 1
            if table is None:
                continue
            at = kv - n + i
            page = int(table[b, at // block_size])
            if page < 0:
                ok = False
            else:
                slots[q0 + i] = page * block_size + at % block_size
    return sees, pos, slots, ok


def tree_accept(tokens, parents, choice, cu_q, max_path, active=None):
    """-> (path [B, max_path], keep, y)."""
    B = len(cu_q) - 1
    path = np.full((B, max_path), -1, dtype=np.int64)
    keep, y = np.zeros(B, dtype=np.int64), np.full(B, -1, dtype=np.int64)
    for b in range(B):
        q0, n = int(cu_q[b]), int(cu_q[b + 1] - cu_q[b])
        if n == 0 or (active is not None and not active[b]):
            continue
        cur = 0
        while cur is not None:
            path[b, keep[b]] = cur
            keep[b] += 1
            c = int(choice[q0 + cur])
            y[b] = max(c, -1)
            if c < 0 or keep[b] == max_path:
                break
            cur = next((j for j in range(cur + 1, n) if parents[q0 + j] == cur and
                        tokens[q0 + j] == c), None)
    return path, keep, y


def compact(pool, table, start, path, keep):
    """pool [L, 2, num_blocks, bs, re], in place -> ok."""
    nb, bs = pool.shape[2:4]
    ok = True
    for b in range(len(keep)):
        k, s, cap = int(keep[b]), int(start[b]), table.shape[1] * bs
        p = [int(x) for x in path[b, :max(k, 0)]]
        if not (0 <= k <= path.shape[1] and 0 <= s <= cap) or \
                any(x < 0 or s + x >= cap for x in p) or any(x >= y for x, y in zip(p, p[1:])):
            ok = False
            continue
        where = [(int(table[b, (s + x) // bs]), (s + x) % bs) for x in p]
        to = [(int(table[b, (s + i) // bs]), (s + i) % bs) for i in range(k)]
        if any(not 0 <= g < nb for g, _ in where + to):
            ok = False
            continue
        kept = [pool[:, :, g, o].clone() for g, o in where]
        for (g, o), x in zip(to, kept):
            pool[:, :, g, o] = x
    return ok


def free_pages(table, num_blocks, kv_len=None, block_size=None):
    """-> (ids, ok)."""
    held, ok = set(), True
    B, mb = table.shape
    for b in range(B):
        if kv_len is None:
            pages = [int(p) for p in table[b] if p >= 0]
        else:
            kv = int(kv_len[b])
            ok = ok and 0 <= kv <= mb * block_size
            pages = [int(p) for p in table[b, :max(0, -(-kv // block_size))]]
        ok = ok and all(0 <= p < num_blocks for p in pages)
        held |= set(pages)
    return [p for p in range(num_blocks) if p not in held], ok


def fork(table, kv_len, parent, room, free, block_size):
    """-> (table [N, mb], copies [3, N], used, ok)."""
    (B, mb), N, bs = table.shape, len(parent), block_size
    out = np.full((N, mb), -1, dtype=np.int64)
    copies = np.stack([np.full(N, -1), np.full(N, -1), np.zeros(N, dtype=np.int64)])
    refused = (out.copy(), copies.copy(), 0, False)
    rows = []
    for i in range(N):
        p = int(parent[i])
        if p < -1 or p >= B:
            return refused
        n = int(kv_len[p]) if p >= 0 else 0
        if n < 0 or n > mb * bs or int(room[i]) < n or int(room[i]) > mb * bs:
            return refused
        if p >= 0 and any(int(g) < 0 for g in table[p, :-(-n // bs)]):
            return refused
        rows.append((p, n // bs, n % bs))
    used = 0
    for i, (p, whole, part) in enumerate(rows):
        kept = whole
        if p >= 0:
            out[i, :whole] = table[p, :whole]
        copy = False
        if part:
            page = int(table[p, whole])
            for j, (o, w, r) in enumerate(rows):
                if j != i and o >= 0 and (w > whole or (w == whole and r and j < i)) and \
                        int(table[o, whole]) == page:
                    copy = True
            if not copy:
                out[i, whole] = page
                kept += 1
        take = -(-int(room[i]) // bs) - kept
        if used + take > len(free):
            return refused
        out[i, kept:kept + take] = free[used:used + take]
        if copy:
            copies[:, i] = page, free[used], part
        used += take
    return out, copies, used, True
