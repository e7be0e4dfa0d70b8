"""The list of token_logprobs for every row, those without finite scores among them: by value, NaN
last, the lowest id first among equals, as oracle/logprobs.py orders them."""
import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from specdec.sampling import token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN, INF = float("nan"), float("inf")


def rows_of(V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn((14, V), generator=g, device=DEV) * 3).to(dtype)
    x[1, V - 1] = INF                         # one infinity
    x[2, ::3] = INF                           # many
    x[3, V // 2] = NAN
    x[4] = NAN
    x[5, 1:] = NAN                            # fewer numbers than the list is long
    x[6, :V - 2] = NAN
    x[7, :] = NAN
    x[7, V // 2:V // 2 + 3] = 1.5
    x[8, :3] = NAN                            # in the first and last elements
    x[8, V - 3:] = NAN
    x[9] = -INF                               # no number that is finite, some that are none
    x[9, V // 3] = NAN
    x[10, ::2] = NAN
    x[10, 1] = INF
    x[11] = -INF
    x[11, V - 1] = INF
    x[12, :] = -x[12, :].abs()                # NaN with the sign bit
    x[12, 5:V // 2] = torch.tensor(NAN, device=DEV).neg().to(dtype)
    x[13, V // 4:] = NAN
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,at", [(64, 0), (101, 0), (101, 3), (2500, 1), (5003, 5), (40000, 0), (70001, 7)])
@pytest.mark.parametrize("top_n", [1, 5, 20, 64])
def test_lists_of_all_rows(V, at, dtype, top_n):
    """Rows at offset `at` of a wider buffer, few of them (split over workgroups where they are long)
    and, for short ones, so many that each is one workgroup's."""
    base = rows_of(V, dtype)
    want = OL.token_logprobs(base.double().cpu().numpy(), np.zeros((14, 1), dtype=np.int64), 1.0, top_n)
    for times in (1, 170) if V < 6000 else (1,):
        buf = torch.zeros((14 * times, V + 9), dtype=dtype, device=DEV)
        x = buf[:, at:at + V]
        x.copy_(base.repeat(times, 1))
        ids = torch.zeros((14 * times, 1), dtype=torch.long, device=DEV)
        logp, ent, tl, ti = token_logprobs(x, ids, top_n=top_n)
        got = ti.cpu().numpy().reshape(times, 14, top_n)
        assert (got == want[3]).all(), np.argwhere((got != want[3]).any(-1))[:5]
        assert np.array_equal(tl.isnan().cpu().numpy().reshape(times, 14, top_n),
                              np.broadcast_to(np.isnan(want[2]), got.shape))
        assert np.array_equal(ent.isnan().cpu().numpy().reshape(times, 14),
                              np.broadcast_to(np.isnan(want[1]), got.shape[:2]))
