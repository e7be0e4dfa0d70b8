"""fp16 weights of shared_prefix_attention_paged far below the largest: they are below the least
normal number, so their rounding is absolute and adds up over the keys.

With the largest weight 2^7 the rounding of a weight below 2^-14 is at most 2^-25, that is
2^-32 of the largest: over n keys at most n 2^-32 max |v| of the output (the sum of the
weights is no less than the largest), beside the bound of the attention's own test,
u |out| + (u + e) A (1 + u), u = 2^-11.
"""
import math

import pytest
import torch

from specdec.attention import shared_prefix_attention_paged

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("first", [0, 70, 131071])
@pytest.mark.parametrize("below", [17.5, 20.0, 24.5])
def test_many_keys_far_below_one(below, first):
    """One token over 131,072 keys, one of them `below` nats above all others, beside so many
    other tokens that its keys are one part."""
    n, others, hq, d, bs = 131072, 6100, 32, 64, 16
    T = 1 + others
    pages = n // bs + others // bs + 1
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.zeros((T, hq, d), dtype=torch.float16, device=DEV)
    q[:, :, 0] = 1.0
    k = torch.zeros((pages, bs, d), dtype=torch.float16, device=DEV)
    v = (torch.rand((pages, bs, d), generator=g, device=DEV) + 0.5).half()
    table = torch.zeros((2, n // bs), dtype=torch.int32, device=DEV)
    table[0] = torch.arange(n // bs, device=DEV)
    table[1, :pages - n // bs] = torch.arange(n // bs, pages, device=DEV)
    k[:n // bs, :, 0] = -below
    k[first // bs, first % bs, 0] = 0.0
    dev = lambda *x: torch.tensor(x, device=DEV)  # noqa: E731
    got = shared_prefix_attention_paged(q, dev(0, 1, T), k, v, table, dev(n, others), dev(0, 1, 2),
                                        dev(0, 0), scale=1.0)[0].double()
    p = torch.exp(k[:n // bs].view(n, d)[:, 0].double())
    x = v[:n // bs].reshape(n, d).double()
    A = (p[:, None] * x).sum(0) / p.sum()     # the output too: v is positive
    u, e = 2.0 ** -11, 2.0 ** -24 * (4 * (d + 8) * below + n / 32 + 256)
    off = (got - A).abs() - (u * A + (u + e) * A * (1 + u) + n * 2.0 ** -32 * float(x.max()))
    assert off.max().item() <= 0, off.max().item()


def test_rising_scores_in_half_precision():
    """Scores that rise by less than the running maximum's slack from tile to tile, then by more:
    no weight passes the type's largest number."""
    n, hq, d, bs = 4096, 4, 64, 16
    q = torch.zeros((1, hq, d), dtype=torch.float16, device=DEV)
    q[:, :, 0] = 1.0
    v = torch.ones((n // bs, bs, d), dtype=torch.float16, device=DEV)
    pos = torch.arange(n, device=DEV)
    table = torch.arange(n // bs, device=DEV, dtype=torch.int32).view(1, -1)
    dev = lambda *x: torch.tensor(x, device=DEV)  # noqa: E731
    for rise in (1.0, 5.5, 10.0, 10.4, 11.0, 30.0, 700.0):    # nats a tile of 64 keys
        k = torch.zeros((n // bs, bs, d), dtype=torch.float16, device=DEV)
        k.view(n, d)[:, 0] = (pos // 64 * rise).half()
        got = shared_prefix_attention_paged(q, dev(0, 1), k, v, table, dev(n), dev(0, 1), dev(0),
                                            scale=1.0).double()
        # all values 1: the weights' rounding alone, u of each, moves the output
        assert (got - 1).abs().max().item() <= 3 * 2.0 ** -11, rise
    assert math.isfinite(float(got.sum()))
