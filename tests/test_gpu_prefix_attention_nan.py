"""Scores that are no number in shared_prefix_attention_paged: a NaN in a query vector, or in a
key that a query sees, makes that query's output NaN in the heads that it concerns, in
whichever part of the keys it stands and however the call was cut into parts; the other
outputs are those of the same call without it (within the bound of the attention's own test,
which is derived there)."""
import math

import pytest
import torch

from specdec.attention import shared_prefix_attention_paged
from test_gpu_prefix_attention import make, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def slot_of(c, row, pos):
    """(page, place in it) of the key that row `row` reads at `pos`; one group."""
    row = 0 if pos < int(c["prefix_len"][0]) and c["kv_len"].numel() > 1 else row
    return int(c["block_table"][row, pos // 16]), pos % 16


def check(c, odd):
    """c: finite inputs; odd: the same with NaN."""
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = shared_prefix_attention_paged(**odd, error=err)
    want, A, S = reference(c)
    nan = reference(odd)[0].isnan()
    assert err.item() == 0 and nan.any()
    assert torch.equal(got.isnan(), nan)
    u = torch.finfo(got.dtype).eps / 2
    e = 2.0 ** -24 * (4 * (got.shape[2] + 8) * S + int(c["kv_len"].max()) / 32 + 256)
    off = (got.double() - want).abs() - (u * want.abs() + (u + e) * A * (1 + u))
    assert off[~nan].numel() == 0 or off[~nan].max().item() <= 0


# rows, prefix, own keys before the new ones, new tokens per row
WHOLE = ([1], [0], [40], [2])                      # one part, written directly
LONG = ([1], [0], [30000], [2])                    # a row over many parts
SHARED = ([3], [100], [0, 0, 5], [1, 2, 1])        # prefix and own keys
WIDE = ([3], [40000], [0, 3, 9], [1, 1, 2])        # a prefix over many parts
INSIDE = ([2], [64], [0, 0], [3, 40])              # no own keys: rows that end with the prefix
KV = {id(INSIDE): [64, 64]}


@pytest.mark.parametrize("heads,dtype", [((8, 2, 128), torch.bfloat16), ((4, 4, 64), torch.float16),
                                         ((16, 2, 64), torch.bfloat16)])
@pytest.mark.parametrize("shape", [WHOLE, LONG, SHARED, WIDE, INSIDE])
def test_nan_query(shape, heads, dtype):
    c = make(5, *shape, *heads, dtype=dtype, kv=KV.get(id(shape)))
    for t, h in ((0, 0), (c["q"].shape[0] - 1, heads[0] - 1)):
        odd = dict(c, q=c["q"].clone())
        odd["q"][t, h, 7] = math.nan
        check(c, odd)


@pytest.mark.parametrize("heads,dtype", [((8, 2, 128), torch.bfloat16), ((4, 4, 64), torch.float16)])
@pytest.mark.parametrize("shape,row,pos", [
    (WHOLE, 0, 0), (WHOLE, 0, 41),
    (LONG, 0, 17000), (LONG, 0, 30001),
    (SHARED, 0, 100),   # the row's only own key
    (SHARED, 1, 101),   # seen by the last of two new tokens
    (SHARED, 2, 105), (SHARED, 0, 0), (SHARED, 0, 99),
    (WIDE, 0, 40000), (WIDE, 0, 20000), (WIDE, 1, 40003),
])
def test_nan_key(shape, row, pos, heads, dtype):
    c = make(6, *shape, *heads, dtype=dtype)
    odd = dict(c, k_pool=c["k_pool"].clone())
    page, at = slot_of(c, row, pos)
    odd["k_pool"][page, at, heads[2] + 3] = math.nan   # of the second KV head
    check(c, odd)


@pytest.mark.parametrize("heads,dtype", [((8, 2, 128), torch.bfloat16), ((4, 4, 64), torch.float16)])
def test_parts_without_a_number_beside_others(heads, dtype):
    """All of a prefix's keys, or all own keys of a row, are NaN, the others are not: every part of
    that range has no maximum."""
    c = make(7, [3], [3000], [200, 0, 9], [1, 2, 1], *heads, dtype=dtype)
    odd = dict(c, k_pool=c["k_pool"].clone())
    for pos in range(3000, 3201):
        page, at = slot_of(c, 0, pos)
        odd["k_pool"][page, at] = math.nan
    check(c, odd)
    odd = dict(c, k_pool=c["k_pool"].clone())
    pages = c["block_table"][0, :3000 // 16].long()
    odd["k_pool"][pages] = math.nan
    check(c, odd)


def test_keys_that_are_minus_infinity_alone_give_zeros():
    """Every visible score -inf: no weight is left, and the output is 0, as that of
    verify_attention_paged."""
    for own in ([0, 3], [5000, 3]):
        c = make(8, [2], [200], own, [1, 1], 8, 2, 128)
        c["q"] = c["q"].abs() + 0.5
        c["k_pool"] = torch.full_like(c["k_pool"], -math.inf)
        assert (shared_prefix_attention_paged(**c) == 0).all()
