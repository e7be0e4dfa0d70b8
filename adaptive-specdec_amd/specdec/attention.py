"""Verify attention over the paged KV cache (one layer), on MFMA.

`verify_attention_paged` reads every row's keys; `shared_prefix_attention_paged`
reads the keys that a group's rows share once for all of them; `tree_attention_paged` is for
rows whose new tokens are a tree (`specdec.tree`).

The attention of the target's verify forward: every batch row's k_b + 1 new
positions against the row's cached keys, under the mask of
`specdec/kvcache.py:138-162` (query j of row b sees slot s iff
s <= lengths[b] + j) with grouped-query heads (`repeat_kv`). The reference runs
it as HF SDPA inside the target forward (`bench/bench_engine.py:170-174`,
`specdec/engine.py:273-275`); here it reads the pool that
`PagedKVCache.append` writes, so the new positions' K/V must be appended first.
"""
import math

import torch

from . import _lib

__all__ = ["verify_attention_paged", "attention_workspace", "shared_prefix_attention_paged",
           "shared_attention_workspace", "tree_attention_paged", "tree_attention_workspace"]


def attention_workspace(B, max_q, hq, hkv, block_size, max_blocks, chunk_tokens=0,
                        device="cuda"):
    """A workspace for verify_attention_paged at these sizes (uint8 device tensor)."""
    need = _lib.lib().sdx_verify_attention_workspace(B, int(max_q), hq, hkv, block_size,
                                                     max_blocks, int(chunk_tokens))
    if need == 0:
        _lib.check(-1, "verify_attention workspace query")
    return torch.empty(need, dtype=torch.uint8, device=device)


def verify_attention_paged(q, cu_q, k_pool, v_pool, block_table, kv_len, max_q, scale=None,
                           out=None, error=None, chunk_tokens=0, workspace=None):
    """q [T, Hq, d] bf16 (T = cu_q[-1], head dim d of 64 or 128); cu_q [B+1]
    int64; k_pool / v_pool [num_blocks, block_size, Hkv * d] bf16 (one layer's K
    and V sides of a PagedKVCache pool); block_table [B, max_blocks] int32;
    kv_len [B] int64 (keys per row, the new positions included); max_q >= every
    row's q_b. Returns out [T, Hq, d] bf16. Rows whose shape or pages are out of range are
    skipped and set `error` (an int32 [1] device tensor) when given. Each row's
    keys are split in chunks of `chunk_tokens` (0: the library's default) on
    separate workgroups; rows of several chunks merge fp32 partials held in
    `workspace` (a uint8 device tensor, allocated here when None); the chunks
    are launched longest first."""
    _lib.require_gpu(q, cu_q, k_pool, v_pool, block_table, kv_len)
    if q.dtype != torch.bfloat16 or k_pool.dtype != torch.bfloat16 or v_pool.dtype != torch.bfloat16:
        raise TypeError("verify_attention_paged: bf16 q and pools")
    T, hq, d = q.shape
    nb, bs, re = k_pool.shape
    if v_pool.shape != k_pool.shape or re % d != 0:
        raise ValueError("verify_attention_paged: k_pool / v_pool must be [num_blocks, bs, Hkv*d]")
    hkv = re // d
    B = cu_q.numel() - 1
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("verify_attention_paged: pools must be contiguous")
    q = q.contiguous()
    cu = _lib.as_dtype(cu_q, torch.int64)
    kl = _lib.as_dtype(kv_len, torch.int64)
    bt = _lib.as_dtype(block_table, torch.int32)
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = attention_workspace(B, max_q, hq, hkv, bs, bt.shape[1], chunk_tokens, q.device)
    rc = _lib.lib().sdx_verify_attention_paged(
        _lib.ptr(q), _lib.BF16, B, _lib.ptr(cu), int(max_q), hq, hkv, d,
        _lib.ptr(k_pool), _lib.ptr(v_pool), nb, bs, _lib.ptr(bt),
        bt.shape[1], _lib.ptr(kl), scale, int(chunk_tokens),
        _lib.ptr(workspace), workspace.numel(), _lib.ptr(out), _lib.ptr(error), _lib.stream_of(q))
    _lib.check(rc, "verify_attention_paged")
    return out


def shared_attention_workspace(num_tokens, batch, num_groups, hq, hkv, head_dim, device="cuda"):
    """A workspace for shared_prefix_attention_paged at these sizes (uint8 device tensor)."""
    need = _lib.lib().sdx_prefix_attention_workspace(int(num_tokens), int(batch), int(num_groups), hq,
                                                     hkv, head_dim)
    if need == 0:
        raise ValueError("shared_attention_workspace: tokens, rows, groups and heads of at least 1, "
                         "query heads a multiple of KV heads, head_dim 64 or 128")
    return torch.empty(need, dtype=torch.uint8, device=device)


def shared_prefix_attention_paged(q, cu_q, k_pool, v_pool, block_table, kv_len, cu_group, prefix_len,
                                  scale=None, out=None, error=None, workspace=None):
    """`verify_attention_paged` for a batch whose groups of rows share a prefix, the prefix's
    keys read once per group.

    q [T, Hq, d] bf16 or fp16 (head dim d of 64 or 128), row b's new positions at cu_q[b] ..
    cu_q[b+1] - 1 (cu_q [B+1] int64, any number per row); k_pool / v_pool [num_blocks,
    block_size, Hkv * d] of q's type; block_table [B, max_blocks] int32; kv_len [B] int64, keys
    per row with the prefix and the new positions. The rows of group g, cu_group[g] ..
    cu_group[g+1] - 1 (cu_group [G+1] int64), share their first prefix_len[g] (int64 [G])
    keys, which are read through the table of the group's first row; the keys behind them come
    from the row's own table. Query j of row b sees keys s <= kv_len[b] - q_b + j. Returns out
    [T, Hq, d] of q's type. Rows or groups out of range are skipped and set `error` (an int32
    [1] device tensor) when given, and so do page ids outside the pool. `workspace` (uint8,
    `shared_attention_workspace`) holds fp32 parts and serves one call at a time; None: the
    calling thread's own for the current stream, kept for its next calls up to 512 MiB. Its size is
    8 T Hq (d + 2) bytes at least (1.1 GB for 33,000 tokens of 32 heads of 128)."""
    _lib.one_gpu(q, cu_q, k_pool, v_pool, block_table, kv_len, cu_group, prefix_len, out, error,
                 workspace)
    if q.dtype not in (torch.bfloat16, torch.float16) or k_pool.dtype != q.dtype or \
            v_pool.dtype != q.dtype:
        raise TypeError("shared_prefix_attention_paged: q and pools all bf16 or all fp16")
    if q.dim() != 3 or k_pool.dim() != 3 or k_pool.shape != v_pool.shape:
        raise ValueError("shared_prefix_attention_paged: q [T, Hq, d], k_pool / v_pool [num_blocks, "
                         "bs, Hkv*d]")
    T, hq, d = q.shape
    nb, bs, re = k_pool.shape
    hkv = re // d
    if re % d or hkv < 1 or hq % hkv:
        raise ValueError(f"shared_prefix_attention_paged: {hq} query heads of {d} over rows of {re}")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("shared_prefix_attention_paged: pools must be contiguous")
    if error is not None and error.dtype != torch.int32:
        raise TypeError("shared_prefix_attention_paged: error must be int32")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("shared_prefix_attention_paged: workspace must be contiguous")
    B, G = kv_len.numel(), prefix_len.numel()
    if cu_q.numel() != B + 1 or cu_group.numel() != G + 1 or block_table.dim() != 2 or \
            block_table.shape[0] != B:
        raise ValueError(f"shared_prefix_attention_paged: {B} lengths need cu_q [{B + 1}] and "
                         f"block_table [{B}, max_blocks], {G} prefixes cu_group [{G + 1}]")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("shared_prefix_attention_paged: out must be contiguous, of q's shape and type")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("shared_prefix_attention_paged: scale must be positive and finite")
    if T == 0:
        return out
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    cu = _lib.as_dtype(cu_q, torch.int64)
    kl = _lib.as_dtype(kv_len, torch.int64)
    cg = _lib.as_dtype(cu_group, torch.int64)
    pl = _lib.as_dtype(prefix_len, torch.int64)
    bt = _lib.as_dtype(block_table, torch.int32)
    with _lib.on_device(q):
        if workspace is None:
            need = _lib.workspace_bytes("sdx_prefix_attention_workspace", T, B, G, hq, hkv, d)
            workspace = _lib.cached_workspace(need, q.device, "prefix_attn")
        rc = _lib.lib().sdx_prefix_attention_paged(
            _lib.ptr(q), _lib.dtype_code(q), T, B, _lib.ptr(cu), hq, hkv, d, _lib.ptr(k_pool),
            _lib.ptr(v_pool), nb, bs, _lib.ptr(bt), bt.shape[1], _lib.ptr(kl), _lib.ptr(cg),
            _lib.ptr(pl), G, scale, _lib.ptr(workspace), workspace.numel(), _lib.ptr(out),
            _lib.ptr(error), _lib.stream_of(q))
    _lib.check(rc, "shared_prefix_attention_paged")
    return out


def tree_attention_workspace(num_tokens, batch, hq, hkv, head_dim, device="cuda"):
    """A workspace for tree_attention_paged at these sizes (uint8 device tensor)."""
    need = _lib.lib().sdx_tree_attention_workspace(int(num_tokens), int(batch), hq, hkv, head_dim)
    if need == 0:
        raise ValueError("tree_attention_workspace: nodes, rows and heads of at least 1, query heads a "
                         "multiple of KV heads, head_dim 64 or 128")
    return torch.empty(need, dtype=torch.uint8, device=device)


def tree_attention_paged(q, cu_q, k_pool, v_pool, block_table, kv_len, tree_mask, scale=None, out=None,
                         error=None, workspace=None):
    """`verify_attention_paged` for rows whose new tokens are the nodes of a tree.

    q [T, Hq, d] bf16 or fp16 (head dim d of 64 or 128), row b's n_b nodes at cu_q[b] ..
    cu_q[b+1] - 1 (cu_q [B+1] int64); k_pool / v_pool [num_blocks, block_size, Hkv * d] of q's
    type; block_table [B, max_blocks] int32; kv_len [B] int64, keys per row, the nodes, which are
    its last, included; tree_mask [T, words] int64 of `specdec.tree.tree_layout` (n_b up to 64
    words and 512). Node i sees the kv_len[b] - n_b keys in front of the nodes and every node
    j whose bit j % 64 of word j / 64 is set. Returns out [T, Hq, d] of q's type, 0 for a node that
    sees nothing. Rows out of range are skipped and set `error` (an int32 [1] device tensor) when
    given, and so do page ids outside the pool. The nodes of such rows and those behind cu_q[B] are left
    as they were in an `out` that is given, and are 0 in one that is allocated here (where offsets that
    descend skip all rows). `workspace` (uint8, `tree_attention_workspace`) holds fp32 parts and serves
    one call at a time; None: the calling thread's own for the current stream, kept for its next calls."""
    _lib.one_gpu(q, cu_q, k_pool, v_pool, block_table, kv_len, tree_mask, out, error, workspace)
    if q.dtype not in (torch.bfloat16, torch.float16) or k_pool.dtype != q.dtype or \
            v_pool.dtype != q.dtype:
        raise TypeError("tree_attention_paged: q and pools all bf16 or all fp16")
    if q.dim() != 3 or k_pool.dim() != 3 or k_pool.shape != v_pool.shape:
        raise ValueError("tree_attention_paged: q [T, Hq, d], k_pool / v_pool [num_blocks, bs, Hkv*d]")
    T, hq, d = q.shape
    nb, bs, re = k_pool.shape
    hkv = re // d
    if re % d or hkv < 1 or hq % hkv:
        raise ValueError(f"tree_attention_paged: {hq} query heads of {d} over rows of {re}")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("tree_attention_paged: pools must be contiguous")
    if error is not None and (error.dtype != torch.int32 or error.numel() < 1):
        raise TypeError("tree_attention_paged: error must be an int32 device tensor of one element")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("tree_attention_paged: workspace must be contiguous")
    B = kv_len.numel()
    if cu_q.numel() != B + 1 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"tree_attention_paged: {B} lengths need cu_q [{B + 1}] and block_table [{B}, "
                         f"max_blocks]")
    if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != T or \
            tree_mask.shape[1] < 1:
        raise ValueError(f"tree_attention_paged: tree_mask must be int64 [{T}, words], got "
                         f"{tree_mask.dtype} {tuple(tree_mask.shape)}")
    call = _lib.lib().sdx_tree_attention_paged
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        call = _lib.lib().sdx_tree_attention_paged_whole
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("tree_attention_paged: out must be contiguous, of q's shape and type")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("tree_attention_paged: scale must be positive and finite")
    if T == 0:
        return out
    q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    cu = _lib.as_int64("cu_q", cu_q)
    kl = _lib.as_int64("kv_len", kv_len)
    bt = _lib.as_int32("block_table", block_table)
    tm = tree_mask.contiguous()
    with _lib.on_device(q):
        if workspace is None:
            need = _lib.workspace_bytes("sdx_tree_attention_workspace", T, B, hq, hkv, d)
            workspace = _lib.cached_workspace(need, q.device, "tree_attn")
        rc = call(
            _lib.ptr(q), _lib.dtype_code(q), T, B, _lib.ptr(cu), hq, hkv, d, _lib.ptr(k_pool),
            _lib.ptr(v_pool), nb, bs, _lib.ptr(bt), bt.shape[1], _lib.ptr(kl), _lib.ptr(tm), tm.shape[1],
            scale, _lib.ptr(workspace), workspace.numel(), _lib.ptr(out), _lib.ptr(error),
            _lib.stream_of(q))
    _lib.check(rc, "tree_attention_paged")
    return out
