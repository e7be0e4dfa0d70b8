"""Penalties, biases and grammar masks on logits in float64, row by row.

TEST INFRASTRUCTURE ONLY (see `oracle/__init__.py`). They come before the transforms of
`specdec/sampling.py:34-67`.
"""
import numpy as np


def penalize(logits, history, history_len, cu_rows, prompt_len=None, repetition=None, frequency=None,
             presence=None, bias_ids=None, bias=None, allowed=None, node_tokens=None, sees=None):
    """logits [R, V] float64; sees: per row the nodes on its path (None: a chain's). Returns
    (out, size, touched): size bounds every intermediate value, touched where anything applies."""
    R, V = logits.shape
    out, size = logits.copy(), np.abs(logits)
    touched = np.zeros((R, V), dtype=bool)
    for b in range(len(cu_rows) - 1):
        ids = np.asarray([] if history is None else history[b, :int(history_len[b])], dtype=np.int64)
        P = 0 if prompt_len is None else int(prompt_len[b])
        inside = lambda x: x[(x >= 0) & (x < V)]  # noqa: E731
        for r in range(int(cu_rows[b]), int(cu_rows[b + 1])):
            i = r - int(cu_rows[b])
            path = np.asarray([], dtype=np.int64)
            if node_tokens is not None:
                nodes = range(i + 1) if sees is None else sorted(sees[r])
                path = np.asarray([node_tokens[int(cu_rows[b]) + j] for j in nodes], dtype=np.int64)
            count = np.bincount(inside(np.concatenate([ids[P:], path])), minlength=V)
            seen = (np.bincount(inside(ids), minlength=V) > 0) | (count > 0)
            x = out[r]
            with np.errstate(all="ignore"):
                rep = 1.0 if repetition is None else float(repetition[b])
                f = 0.0 if frequency is None else float(frequency[b])
                p = 0.0 if presence is None else float(presence[b])
                x = np.where(seen, np.where(x > 0, x / rep, x * rep), x)
                x = np.where(count > 0, x - f * count - p, x)
                size[r] = np.maximum(size[r], np.abs(x)) * max(1.0, rep) + abs(f) * count + abs(p)
                touched[r] = seen
                if bias_ids is not None:
                    for v, y in zip(bias_ids[b], bias[b]):
                        if 0 <= v < V:
                            x[v] += y
                            size[r, v] += abs(y)
                            touched[r, v] = True
                if allowed is not None:
                    v = np.arange(V)
                    no = (allowed[r, v // 32] >> (v % 32)) & 1 == 0
                    x = np.where(no, -np.inf, x)
                    touched[r] |= no
            out[r] = x
    return out, size, touched
