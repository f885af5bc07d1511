"""Sizes that the paged cache's C entry points refuse (no device needed)."""
import ctypes as C

from test_paged_refusals import attend, desc, lib  # noqa: F401


def test_more_sequences_than_the_search_counts(lib):  # noqa: F811
    """The search for a token's sequence counts in 32 bits and looks up to 32 steps ahead."""
    d = desc()
    rows = (4096, 128, 64, 4096, 128, 64, 0, 4096, 1, 1)
    for n in (2**31 - 1, 2**30 + 1):
        assert lib.adaptq_paged_append(C.addressof(d), *rows, 4096, 0, 4096, n, 1, None, None) == -1
        assert "too many sequences" in lib.adaptq_last_error().decode()
        assert lib.adaptq_paged_read(C.addressof(d), *rows, 4096, 4096, n, 1, None) == -1
        assert "too many sequences" in lib.adaptq_last_error().decode()
        assert attend(lib, d, n_seqs=n) == -1 and "too many sequences" in lib.adaptq_last_error().decode()
