"""token_logprobs in float64 (what `specdec/sampling.py:34-67,93-95` would be composed
for): log softmax at given ids, entropy, and the likeliest tokens by value then id."""
import numpy as np


def token_logprobs(logits, ids, temperature=1.0, top_n=0):
    """logits [rows, V], ids [rows, n] -> (logp [rows, n], entropy [rows], top_logp, top_ids)."""
    x = np.asarray(logits, dtype=np.float64)
    rows, V = x.shape
    with np.errstate(all="ignore"):
        m = x.max(axis=1, keepdims=True)
        d = (x - m) / temperature
        e = np.exp(d)
        z = e.sum(axis=1, keepdims=True)
        y = d - np.log(z)
        p = e / z
        entropy = -np.where(p > 0, p * y, np.where(np.isnan(p), p, 0.0)).sum(axis=1)
    ok = (ids >= 0) & (ids < V)
    logp = np.take_along_axis(y, np.where(ok, ids, 0), axis=1)
    nan_row = np.isnan(y).any(axis=1, keepdims=True)
    logp = np.where(nan_row, np.nan, np.where(ok, logp, -np.inf))
    # by value, then by lowest id; NaN after everything
    order = np.lexsort((np.broadcast_to(np.arange(V), x.shape),
                        -np.where(np.isnan(x), -np.inf, x), np.isnan(x)), axis=1)[:, :top_n]
    top = np.where(nan_row, np.nan, np.take_along_axis(y, order, axis=1))
    return logp, np.where(nan_row[:, 0], np.nan, entropy), top, order
