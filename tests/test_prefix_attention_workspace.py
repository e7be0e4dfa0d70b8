"""CPU checks of the shared attention's workspace and refusals: its size at the accepted limits,
room for every list of units that valid offsets give, and arguments that the C entry point or
the wrapper turn down before anything is launched."""
import ctypes
import random

import pytest

FAKE = ctypes.c_void_p(4096)


def _lib():
    from specdec import _lib
    return _lib.lib()


def test_rows_without_tokens_take_no_room():
    """A token in a batch of 2^22 rows and groups: a list of its own two segments, not of all."""
    L = _lib()
    one = L.sdx_prefix_attention_workspace(1, 1, 1, 1, 1, 64)
    most = L.sdx_prefix_attention_workspace(1, 1 << 22, 1 << 22, 1, 1, 64)
    assert most - one <= 8 * (1 << 22) + 256    # the groups' sizes, 8 bytes each


def test_room_for_every_list_of_units():
    """Entries that any split of the tokens over rows and groups needs: tiles of 128 query rows in
    every chunk, no more chunks than parts, 32 bytes each; the query allows for them."""
    L, rng = _lib(), random.Random(5)
    for _ in range(300):
        hkv = rng.choice([1, 2, 8])
        group, d = rng.choice([1, 2, 4, 7, 16]), rng.choice([64, 128])
        rows = rng.randint(1, 60)
        q = [rng.choice([0, 0, 1, 1, 2, rng.randint(1, 700)]) for _ in range(rows)]
        T = sum(q)
        if T == 0:
            continue
        cuts = sorted(rng.sample(range(rows + 1), rng.randint(0, min(rows, 9))))
        cuts = [0] + cuts + [rows]
        groups = [sum(q[a:b]) for a, b in zip(cuts, cuts[1:])]
        tiles = sum(-(-m * group // 128) for m in q + groups)
        hq = hkv * group
        one = T * hq * (d + 2) * 4
        parts = max(2, min(512, 2 * -(-512 // hkv), (192 << 20) // one) // 2 * 2)
        need = 32 * tiles * (parts // 2) + parts * one
        assert L.sdx_prefix_attention_workspace(T, rows, len(groups), hq, hkv, d) >= need


def test_scales_that_overflow_in_base_two_are_refused():
    """The kernels multiply by scale log2(e) in fp32: infinite from 2.4e38 on, and 0 times it is no
    score."""
    L = _lib()

    def call(scale):
        need = L.sdx_prefix_attention_workspace(3, 2, 1, 4, 2, 64)
        # no workspace: a scale that is taken ends there
        return L.sdx_prefix_attention_paged(FAKE, 1, 3, 2, FAKE, 4, 2, 64, FAKE, FAKE, 8, 16, FAKE, 4,
                                            FAKE, FAKE, FAKE, 1, scale, None, need, FAKE, None, None)

    assert call(2.3e38) == -4 and call(0.125) == -4
    for bad in (2.4e38, 3.4e38, float("inf"), float("nan"), 0.0, -1.0):
        assert call(bad) == -1, bad


def test_workspaces_that_are_not_whole_are_refused(monkeypatch):
    """A view whose elements do not lie one after another covers fewer bytes than it counts."""
    import torch

    from specdec import attention as A
    from specdec import _lib as B
    monkeypatch.setattr(B, "one_gpu", lambda *t: None)
    z = torch.zeros
    args = (z((3, 4, 64), dtype=torch.half), z(3).long(), z((8, 16, 128), dtype=torch.half),
            z((8, 16, 128), dtype=torch.half), z((2, 4), dtype=torch.int32), z(2).long(), z(2).long(),
            z(1).long())
    for ws in (z(1, dtype=torch.uint8).expand(1 << 30), z(1 << 20, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            A.shared_prefix_attention_paged(*args, workspace=ws)
