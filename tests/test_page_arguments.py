"""CPU checks of arguments of the page operators that lie over one another, and of the attention that
writes its output whole: the C entry points return their status before anything is launched (the
pointers are never dereferenced)."""
import ctypes

OK, EINVAL, EUNSUP, EWS = 0, -1, -2, -4


def test_compact_does_not_write_what_it_reads():
    """Other workgroups of a row read its start while one writes kept: the tokens would be looked for at
    the wrong place."""
    from specdec import _lib
    L = _lib.lib()
    B, mb, P = 3, 4, 5
    table, start, path, keep = 1 << 20, 2 << 20, 3 << 20, 4 << 20

    def call(kept):
        p = ctypes.c_void_p
        return L.sdx_compact_paged(p(1 << 30), 8192, 4096, 1, 0x7FFF, 64, 8, 16, p(table), B, mb, p(start), p(path), P,
                                   p(keep), p(kept), None, None)

    for at, size in ((table, 4 * B * mb), (start, 8 * B), (path, 8 * B * P), (keep, 8 * B)):
        for kept in (at, at + 8, at + size - 8, at - 8, at - 8 * B + 8):
            if kept != keep:
                assert call(kept) == EINVAL, (at, kept)
                assert b"kept may be keep itself" in L.sdx_last_error()


def test_forked_tables_do_not_lie_over_what_is_read():
    """Every row reads the old tables, the parents and the number of free pages while others write theirs."""
    from specdec import _lib
    L = _lib.lib()
    B, mb, N, free = 6, 4, 5, 7
    base = dict(table=(1 << 20, 4 * B * mb), kv=(2 << 20, 8 * B), parent=(3 << 20, 8 * N), room=(4 << 20, 8 * N),
                free=(5 << 20, 4 * free), num=(6 << 20, 8))
    apart = dict(out=7 << 20, copies=8 << 20, used=9 << 20)
    p = ctypes.c_void_p
    ws = L.sdx_fork_block_tables_workspace(N)

    def call(**over):
        w = {**apart, **over}
        at = {k: p(v[0]) for k, v in base.items()}
        return L.sdx_fork_block_tables(at["table"], B, mb, at["kv"], at["parent"], at["room"], N, 16, at["free"], free,
                                       at["num"], p(w["out"]), p(w["copies"]), p(w["used"]), p(10 << 20), ws, None,
                                       None)

    for name, size in (("out", 4 * N * mb), ("copies", 12 * N), ("used", 8)):
        for at, n in base.values():
            for where in (at, at + n - 4, at - size + 4):
                assert call(**{name: where}) == EINVAL, (name, at, where)
                assert b"may not lie over" in L.sdx_last_error()


def test_the_attention_that_writes_its_output_whole_refuses_alike():
    from specdec import _lib
    L = _lib.lib()
    fake, off = ctypes.c_void_p(4096), ctypes.c_void_p(4104)

    def call(T=3, B=2, hq=4, hkv=2, d=64, mb=4, scale=0.1, out=fake, nbytes=None):
        need = L.sdx_tree_attention_workspace(max(T, 1), max(B, 1), max(hq, 1), max(hkv, 1), d)
        return L.sdx_tree_attention_paged_whole(
            fake, 1, T, B, fake, hq, hkv, d, fake, fake, 8, 16, fake, mb, fake, fake, 1, scale, fake,
            need if nbytes is None else nbytes, out, None, None)

    assert call(T=0) == OK
    for bad in (dict(T=-1), dict(B=0), dict(hq=3), dict(scale=0.0), dict(out=None), dict(out=off)):
        assert call(**bad) == EINVAL, bad
    assert call(d=96) == EUNSUP and call(mb=1 << 28) == EUNSUP and call(nbytes=64) == EWS


def test_free_pages_of_many_pages_and_entries():
    """The tables are gone through once for every 2^18 pages: large pools behind large tables are refused,
    each of them by itself is not."""
    from specdec import _lib
    L = _lib.lib()
    fake = ctypes.c_void_p(4096)

    def call(B, mb, nb, nbytes=16):                    # (a workspace that is too small: nothing is launched)
        return L.sdx_free_pages(fake, B, mb, fake, 16, nb, fake, fake, fake, nbytes, None, None)

    assert call(1 << 15, 1 << 16, 1 << 23) == EWS and call(1 << 15, 1 << 16, (1 << 23) + 1) == EUNSUP
    assert call(1 << 8, 1 << 16, 1 << 30) == EWS and call((1 << 8) + 1, 1 << 16, 1 << 30) == EUNSUP
    assert L.sdx_free_pages_workspace(1 << 8, 1 << 16, 1 << 30) > 0
    assert L.sdx_free_pages_workspace((1 << 8) + 1, 1 << 16, 1 << 30) == 0
