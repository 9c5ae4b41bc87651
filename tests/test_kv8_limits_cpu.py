"""Sizes whose numbers of pages would pass 32 bits are refused (nothing is launched)."""
from test_kv8_cpu import buf, cache_of  # noqa: F401  (a fixture)

from cats_b200 import _lib


def test_tables_beyond_32_bits_are_refused(buf):  # noqa: F811
    L, big = _lib.lib(), 1 << 40
    for n_seqs, max_pages, status in ((1024, 1 << 21, -9), (1024, 1 << 27, -9), (17, (1 << 27) - 1, -9)):
        c = cache_of(buf, n_seqs=n_seqs, max_pages=max_pages)
        assert L.cats_kv8_grow(c, None, 1, None) == status
        assert L.cats_kv8_reorder(c, buf, buf, big, None) == status
