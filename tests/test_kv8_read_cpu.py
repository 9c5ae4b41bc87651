"""``KVCache8.read`` is host code over the cache's tensors: sequences whose pages are not all there are refused
before a page number becomes an index.  Runs on CPU tensors; nothing is launched."""
import pytest
import torch

from cats_b200 import kv8


def cache(lens, table, pages=6, page=16):
    c = kv8.KVCache8.__new__(kv8.KVCache8)
    c.codes = torch.zeros((1, pages, 2, 1, page, 32), dtype=torch.uint8)
    for p in range(pages):
        c.codes[0, p] = 0x38 + p                           # 1.0 and the codes above it
    c.scales = torch.ones((1, pages, 2, 1))
    c.lens, c.table = torch.tensor(lens, dtype=torch.int32), torch.tensor(table, dtype=torch.int32)
    c.n_layers, c.n_pages, c.n_seqs, c.max_pages = 1, pages, len(lens), c.table.shape[1]
    c.n_kv_heads, c.page, c.head_dim, c.max_len = 1, page, 32, c.table.shape[1] * page
    return c


def test_rows_of_a_sequence():
    c = cache([20, 0], [[2, 0, -1], [-1, -1, -1]])
    k, v = c.read(0, 0)
    assert k.shape == v.shape == (1, 20, 32)
    assert (k[0, :16] == 1.25).all() and (k[0, 16:] == 1.0).all() and torch.equal(k, v)
    assert c.read(0, 1)[0].shape == (1, 0, 32)


@pytest.mark.parametrize("lens,table", [([20], [[2, -1, -1]]), ([33], [[2, 0, 6]]), ([5], [[-7, 0, 0]]),
                                        ([20], [[2, 1 << 30, 0]])])
def test_missing_and_bad_pages_are_refused(lens, table):
    with pytest.raises(RuntimeError, match="page"):
        cache(lens, table).read(0, 0)


@pytest.mark.parametrize("n", [-1, 49, 1 << 30])
def test_lengths_that_the_table_cannot_hold_are_refused(n):
    with pytest.raises(RuntimeError, match="long"):
        cache([n], [[2, 0, 1]]).read(0, 0)


def test_out_of_range():
    for call in (lambda c: c.read(1, 0), lambda c: c.read(0, 1), lambda c: c.read(0, -1)):
        with pytest.raises(RuntimeError, match="range"):
            call(cache([5], [[0, 1, 2]]))
