"""CPU checks of arguments of the page operators that lie over one another: the C entry points
return their status before anything is launched (the pointers are never dereferenced)."""
import ctypes

OK, EINVAL = 0, -1


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
