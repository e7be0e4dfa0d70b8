"""Batches whose groups, or rows, or both are more than the plan's threads, with empty groups and rows
without tokens among them, against float64 (bounds: those of the attention's own test)."""
import numpy as np
import pytest
import torch

from specdec.attention import shared_prefix_attention_paged
from test_gpu_prefix_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,empty,per,tokens", [
    (700, 0.85, 2, 3),      # fewer rows than threads
    (513, 0.0, 1, 2), (1300, 0.3, 3, 1), (30, 0.0, 60, 1), (2100, 0.5, 2, 1),
])
def test_more_groups_or_rows_than_threads(groups, empty, per, tokens):
    rng = np.random.default_rng(groups)
    n = rng.integers(1, per + 1, groups)
    n[rng.random(groups) < empty] = 0
    B = int(n.sum())
    q = rng.integers(0, tokens + 1, B)
    q[rng.integers(B)] = tokens
    c = make(groups, n, rng.integers(0, 90, groups), rng.integers(0, 70, B), q, 4, 2, 64)
    got = check(c)
    assert torch.equal(shared_prefix_attention_paged(**c), got)


def test_one_row_in_error_among_many():
    """A row past its table in a batch of more rows than threads: it alone keeps its output."""
    rng = np.random.default_rng(2)
    n = rng.integers(1, 4, 600)
    B = int(n.sum())
    c = make(3, n, rng.integers(0, 60, 600), rng.integers(0, 50, B), np.ones(B, dtype=np.int64), 4, 2, 64)
    c["kv_len"][B - 3] = 10 ** 7
    out, err = torch.full_like(c["q"], 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    shared_prefix_attention_paged(**c, out=out, error=err)
    assert err.item() == 1 and (out[B - 3] == 7).all()
    c["kv_len"][B - 3] = 1
    keep = torch.arange(B, device="cuda")
    keep = keep[keep != B - 3]
    # the row's own length is no concern of the others': compared with a length in range
    check(c, got=out, rows=keep)
