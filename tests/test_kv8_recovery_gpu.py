"""The paged 8-bit cache after a step that could not have what it asked for: what was cached stays as
it was, and once there is room again the cache works on."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as K
from test_kv8_gpu import cu_of, filled, np64, same_state

pytestmark = pytest.mark.gpu


def rows_of(c):
    """Every sequence's keys and values in every layer, and the scales of all pages."""
    return [[c.read(layer, b) for b in range(c.n_seqs)] for layer in range(c.n_layers)], c.scales.clone()


def same_rows(a, b, seqs):
    return all(torch.equal(x, y) for la, lb in zip(a[0], b[0]) for s in seqs for x, y in zip(la[s], lb[s]))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 16, 2, 13]])
def test_append_after_a_refused_grow_leaves_the_cached_rows(counts, dt, cuda_device):
    """Sequences 1 and 3 do not get their pages.  Their tokens are left out of every layer, the others'
    are not, and the same tokens go in once pages are free again."""
    uniform = len(set(counts)) == 1
    lens = [16, 32, 7, 48]
    lens = lens if uniform else [9, 32, 7, 48]
    c = filled(cuda_device, lens, 16, 1, 32, layers=2, spare=1 if uniform else 0)
    o = K.Cache.of(c)
    granted = o.grow(counts)
    assert granted == [True, False, True, False]
    before = rows_of(c)
    cu = None if uniform else cu_of(counts, cuda_device)
    c.grow(counts[0]) if uniform else c.grow(cu=cu)
    n = sum(counts)
    g = torch.Generator().manual_seed(1)
    qkv = [(torch.randn((n, 3 * 32), generator=g) * 50).to(dt).to(cuda_device) for _ in range(2)]
    kept = [k if ok else 0 for k, ok in zip(counts, granted)]
    at = np.concatenate([np.arange(k) + a if ok else np.arange(0) for k, a, ok in
                         zip(counts, np.concatenate(([0], np.cumsum(counts))), granted)]).astype(int)
    for layer in range(2):
        c.append(layer, qkv[layer], 1, cu=cu)
        o.append(layer, np64(qkv[layer]).reshape(n, 3, 32)[at], kept, 1)
    assert same_rows(before, rows_of(c), (1, 3))
    same_state(c, o)
    with pytest.raises(RuntimeError, match="no free page") as e:
        c.check()
    assert "had not lengthened" in str(e.value)
    # room again: sequence 2 goes, the refused ones get their pages and their tokens
    c.status.zero_()
    c.free([0, 2])
    o.reorder([-1, 1, -1, 3])
    again = [0, counts[1], 0, counts[3]]
    at = np.concatenate([np.arange(counts[b]) + sum(counts[:b]) for b in (1, 3)]).astype(int)
    c.grow(cu=cu_of(again, cuda_device))
    assert o.grow(again) == [False, True, False, True]
    for layer in range(2):
        c.append(layer, qkv[layer][torch.from_numpy(at).to(cuda_device)], 1, cu=cu_of(again, cuda_device))
        o.append(layer, np64(qkv[layer]).reshape(n, 3, 32)[at], again, 1)
    same_state(c, o)
    c.check()


def test_a_full_table_row_is_not_overwritten(cuda_device):
    c = filled(cuda_device, [64, 5], 16, 1, 32, max_pages=4)
    before = rows_of(c)
    for _ in range(2):                                     # refused again
        c.grow(1)
        c.append(0, torch.randn((2, 96), device=cuda_device), 1)
    assert same_rows(before, rows_of(c), (0,)) and c.lens.tolist() == [64, 7]
    with pytest.raises(RuntimeError, match="longer"):
        c.check()


def test_a_refusal_follows_the_sequence(cuda_device):
    """Sequences that continue a refused one are refused too, until they grow; ``reset`` forgets it."""
    c = filled(cuda_device, [16, 3, 0], 16, 1, 32, spare=0)
    c.grow(cu=cu_of([1, 1, 0], cuda_device))
    assert c.lens.tolist() == [16, 4, 0]
    c.reorder(torch.tensor([1, 0, -1], dtype=torch.int32, device=cuda_device))
    before = rows_of(c)
    c.append(0, torch.randn((3, 96), device=cuda_device), 1)
    assert same_rows(before, rows_of(c), (1,)) and not same_rows(before, rows_of(c), (0,))
    c.reset()
    c.check()
    c.grow(2)
    c.append(0, torch.randn((6, 96), device=cuda_device), 1)
    assert all(c.read(0, b)[0].abs().sum() > 0 for b in range(2)) and c.lens.tolist() == [2, 2, 0]


def test_a_thousand_sequences_of_which_some_grow(cuda_device):
    lens = [16 if i % 3 else 5 for i in range(1000)]
    c = filled(cuda_device, lens, 16, 1, 32, spare=100, poison=False)
    o = K.Cache.of(c)
    granted = np.array(o.grow([1] * 1000))
    assert 0 < granted.sum() < 1000
    c.grow(1)
    x = torch.randn((1000, 96), device=cuda_device)
    c.append(0, x, 1)
    o.append(0, np64(x).reshape(1000, 3, 32)[granted], granted.astype(int), 1)
    assert np.array_equal(c.lens.cpu().numpy(), o.lens)
    assert np.array_equal(np64(c.codes.view(torch.uint8).cpu().view(torch.float8_e4m3fn).float()), o.values)


# ---- the decoder after a search that ran out of pages
def test_a_search_that_ran_out_of_pages_does_not_spoil_the_next(cuda_device):
    from cats_b200 import decoder as D
    from test_decoder_paged8_gpu import SMALL, small_model

    dec = D.CatsDecoder(small_model(cuda_device), 4, 200, mlp="dense", cache="paged8", page=16, n_pages=10)
    ids = torch.randint(0, SMALL["vocab_size"], (2, 30), device=cuda_device)
    want = dec.beam_search(ids, 2, 3)
    with pytest.raises(RuntimeError, match="no free page"):
        dec.beam_search(ids, 2, 60)
    got = dec.beam_search(ids, 2, 3)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    one = torch.cat((ids, ids))
    dec.prefill(one)
    dec.decode(2)                                          # 32 tokens each: eight pages


def test_reset_forgets_what_was_recorded(cuda_device):
    c = filled(cuda_device, [20, 7], 16, 1, 32)
    c.reorder(torch.tensor([7, -5], dtype=torch.int32, device=cuda_device))
    with pytest.raises(RuntimeError, match="parent"):
        c.check()
    c.reset()
    c.check()
    assert c.lens.tolist() == [0, 0] and int(c.refs.sum()) == 0 and int((c.table >= 0).sum()) == 0


# ---- a parent whose last page is missing
def test_a_missing_page_is_not_handed_on_as_another(cuda_device):
    """Sequence 1 lacks its last page (an earlier reorder found none free).  Who continues it lacks the
    page too; it gets no page with somebody else's rows."""
    c = filled(cuda_device, [20, 37, 5, 16], 16, 1, 32, layers=2, spare=4)
    lost = int(c.table[1, 2])
    c.table[1, 2] = -1
    c.refs[lost] = 0
    o = K.Cache.of(c)
    o.reorder([1, 0, 1, 1])
    c.reorder(torch.tensor([1, 0, 1, 1], dtype=torch.int32, device=cuda_device))
    same_state(c, o, layers=False)
    assert c.lens.tolist() == [37, 20, 37, 37]
    assert c.table[:, 2].tolist() == [-1, -1, -1, -1]
    assert torch.equal(c.table[[0, 2, 3], :2], c.table[:1, :2].expand(3, 2)) and c.table[0, :2].min() >= 0
    held = torch.zeros_like(c.refs)
    t = c.table[c.table >= 0].long()
    held.index_add_(0, t, torch.ones_like(t, dtype=torch.int32))
    assert torch.equal(held, c.refs)
    k, v = c.read(0, 1)
    ko, vo = o.rows(0, 1, 20)
    assert np.array_equal(np64(k), ko) and np.array_equal(np64(v), vo)
    with pytest.raises(RuntimeError, match="page id"):
        c.check()


# ---- a capture that fails
def test_a_step_that_fails_while_it_is_captured_leaves_the_cache(cuda_device):
    """The warm-up of a capture runs over a cache of its own; the decoder's comes back even if a step raises."""
    from cats_b200 import decoder as D
    from test_decoder_paged8_gpu import SMALL, small_model

    dec = D.CatsDecoder(small_model(cuda_device), 2, 200, mlp="dense", cache="paged8", page=16)
    ids = torch.randint(0, SMALL["vocab_size"], (2, 30), device=cuda_device)
    kv = dec.kv
    dec.prefill(ids)
    tok, pos = dec.tok.clone(), dec.pos.clone()

    def step(_):
        dec.pos.add_(1)
        raise MemoryError("nothing left")

    with pytest.raises(MemoryError):
        dec._capture([dec.max_len], 30, step)
    assert dec.kv is kv and not dec.graphs
    assert torch.equal(dec.tok, tok) and torch.equal(dec.pos, pos)
    dec.decode(3)
    assert kv.lens.tolist() == [33, 33]
