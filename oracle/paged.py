"""The layout of a batch in a paged cache, row by row: block tables from lengths with the
pages that a group's rows share, and the slots of packed new tokens
(`vllm_draft_spec/proposer.py:295-314` at a count per row)."""
import numpy as np


def build_block_tables(kv_len, free_blocks, block_size, max_blocks, cu_group=None, prefix_len=None):
    """-> (table [B, max_blocks], used, ok); not ok: all -1 and 0."""
    B = len(kv_len)
    table = np.full((B, max_blocks), -1, dtype=np.int64)
    refused = (np.full_like(table, -1), 0, False)
    cu = [0, B] if cu_group is None else [int(c) for c in cu_group]
    pre = [0] if cu_group is None else [int(p) for p in prefix_len]
    if cu[0] != 0 or cu[-1] != B or any(a > b for a, b in zip(cu, cu[1:])):
        return refused
    used = 0
    for g, p in enumerate(pre):
        for b in range(cu[g], cu[g + 1]):
            n = int(kv_len[b])
            if n < 0 or n > max_blocks * block_size or p < 0 or p > kv_len[cu[g]]:
                return refused
            need = -(-n // block_size)
            shared = min(p // block_size, need) if b != cu[g] else 0
            table[b, :shared] = table[cu[g], :shared]
            if used + need - shared > len(free_blocks):
                return refused
            table[b, shared:need] = free_blocks[used:used + need - shared]
            used += need - shared
    return table, used, True


def slot_mapping(table, cu_q, kv_len, block_size, num_tokens, padding=-1):
    """-> (positions, slots, ok)."""
    pos = np.zeros(num_tokens, dtype=np.int64)
    slots = np.full(num_tokens, padding, dtype=np.int64)
    ok = True
    for b in range(len(kv_len)):
        n, m = int(kv_len[b]), int(cu_q[b + 1] - cu_q[b])
        for j in range(m):
            t, p = int(cu_q[b]) + j, n - m + j
            if t >= num_tokens:
                break
            if n < m or n > table.shape[1] * block_size or table[b, p // block_size] < 0:
                ok = False
                continue
            pos[t] = p
            slots[t] = int(table[b, p // block_size]) * block_size + p % block_size
    return pos, slots, ok
