"""Trees of drafted tokens: several continuations of a row in one pass of the target.

The reference drafts a chain per row (`specdec/engine.py:246-258`) and accepts its longest
prefix (`engine.py:285-303`). A tree's nodes branch: row b's nodes are cu_q[b] .. cu_q[b+1] - 1
of the step's packed ones, node 0 the row's pending token, every node behind its parent, and
their K/V lie in the cache in that order. A step runs

    mask, pos, slots = tree_layout(parents, cu_q, kv_len, block_table, block_size)
    append_paged_slots(pool, staged, slots)                     # `specdec.kvcache`, every layer's K/V
    o = tree_attention_paged(q, cu_q, k, v, block_table, kv_len, mask)   # `specdec.attention`
    x = penalize_logits(logits, history, history_len, cu_q, ..., node_tokens=tokens, tree_mask=mask)
    choice = greedy_draft_tokens(x)                             # or sample_from_probs(to_probs(x))
    path, keep, y = tree_accept(tokens, parents, choice, cu_q, max_path)
    compact_paged(pool, block_table, kv_len - n, path, keep)    # `specdec.kvcache`

and row b goes on with its start + keep[b] keys and the pending token y[b]. With draws for
choices the kept tokens are distributed as draws from the target alone: every one of them is one.
"""
import torch

from . import _lib

__all__ = ["tree_layout", "tree_accept", "MAX_NODES"]

MAX_NODES = 512   # of a row


def _offsets(cu_q, batch, T):
    if cu_q.numel() != batch + 1:
        raise ValueError(f"{batch} rows need cu_q [{batch + 1}], got {cu_q.numel()} offsets")
    return _lib.as_int64("cu_q", cu_q)


def tree_layout(parents, cu_q, kv_len, block_table=None, block_size=None, max_nodes=64,
                padding_slot_id=-1, error=None):
    """Which nodes each node sees, its position and its cache slot.

    parents [T] int32: the index in its row of every node's parent, below its own, -1 for a
    root; cu_q [B+1] int64 offsets of the rows' nodes; kv_len [B] int64 keys per row, the nodes
    included; max_nodes >= every row's (a mask has ceil(max_nodes / 64) words, 512 nodes at most).
    Returns (mask [T, words] int64: bit j % 64 of word j / 64 where node j of the row is the node
    itself or an ancestor; positions [T] int64: kv_len[b] - n_b + depth, what a rotation goes by;
    slots [T] int64 of node i at cache position kv_len[b] - n_b + i, or None without a
    block_table [B, max_blocks] int32). Nodes behind cu_q[B] are padding (mask 0, position 0,
    slot padding_slot_id), and so are those of a row whose parents, lengths or offsets are out of range
    and slots without a page, which set `error` (an int32 [1] device tensor) when given.
    """
    _lib.one_gpu(parents, cu_q, kv_len, block_table, error)
    if error is not None and (error.dtype != torch.int32 or error.numel() < 1):
        raise TypeError("error must be an int32 device tensor of one element")
    if parents.dim() != 1:
        raise ValueError(f"parents must be [T], got {tuple(parents.shape)}")
    if (block_table is None) != (block_size is None):
        raise ValueError("block_table and block_size go together")
    max_nodes = int(max_nodes)
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes must lie in [1, {MAX_NODES}], got {max_nodes}")
    T, B = parents.numel(), kv_len.numel()
    up = _lib.as_int32("parents", parents)
    cu = _offsets(cu_q, B, T)
    kl = _lib.as_int64("kv_len", kv_len)
    bt = None
    if block_table is not None:
        if block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError(f"block_table must be [{B}, max_blocks], got {tuple(block_table.shape)}")
        bt = _lib.as_int32("block_table", block_table)
    mask, pos = kl.new_empty((T, (max_nodes + 63) // 64)), kl.new_empty(T)
    slots = None if bt is None else kl.new_empty(T)
    if T:
        with _lib.on_device(up):
            rc = _lib.lib().sdx_tree_layout(
                _lib.ptr(up), B, _lib.ptr(cu), _lib.ptr(kl), max_nodes, _lib.ptr(bt),
                0 if bt is None else bt.shape[1], 0 if bt is None else int(block_size), T,
                int(padding_slot_id), _lib.ptr(mask), _lib.ptr(pos), _lib.ptr(slots), _lib.ptr(error),
                _lib.stream_of(up))
        _lib.check(rc, "tree_layout")
    return mask, pos, slots


def tree_accept(tokens, parents, choice, cu_q, max_path, active=None, error=None):
    """The nodes that the target's choices accept.

    tokens [T] int64 of the nodes, parents and cu_q as `tree_layout`, choice [T] int64: the target's
    next token behind every node. The walk starts at node 0 of each row and goes to the lowest
    child whose token is the choice at the node, as far as there is one, max_path (at most 512)
    nodes in all. active [B] (None: all) leaves rows out. Returns (path [B, max_path] int64, the
    nodes of the walk, -1 behind them; keep [B] int64, how many; y [B] int64, the choice at the
    last of them). Rows without nodes or out of range and rows left out keep 0 and have y -1; those out of
    range set `error` (an int32 [1] device tensor) when given.
    """
    _lib.one_gpu(tokens, parents, choice, cu_q, active, error)
    if error is not None and (error.dtype != torch.int32 or error.numel() < 1):
        raise TypeError("error must be an int32 device tensor of one element")
    T, B = tokens.numel(), cu_q.numel() - 1
    if B < 0 or parents.numel() != T or choice.numel() != T:
        raise ValueError(f"{T} tokens need parents [{T}] and choice [{T}], got {parents.numel()} and "
                         f"{choice.numel()}, and cu_q an offset at least")
    max_path = int(max_path)
    if not 1 <= max_path <= MAX_NODES:
        raise ValueError(f"max_path must lie in [1, {MAX_NODES}], got {max_path}")
    tk, ch = _lib.as_int64("tokens", tokens), _lib.as_int64("choice", choice)
    up, cu = _lib.as_int32("parents", parents), _lib.as_int64("cu_q", cu_q)
    act = None
    if active is not None:
        if active.numel() != B:
            raise ValueError(f"active must be [{B}], got {active.numel()} rows")
        act = (active != 0).to(torch.uint8).contiguous()
    path, keep, y = tk.new_empty((B, max_path)), tk.new_empty(B), tk.new_empty(B)
    if B:
        with _lib.on_device(tk):
            rc = _lib.lib().sdx_tree_accept(
                _lib.ptr(tk), _lib.ptr(up), _lib.ptr(ch), B, _lib.ptr(cu), T, _lib.ptr(act), max_path,
                _lib.ptr(path), _lib.ptr(keep), _lib.ptr(y), _lib.ptr(error), _lib.stream_of(tk))
        _lib.check(rc, "tree_accept")
    return path, keep, y
