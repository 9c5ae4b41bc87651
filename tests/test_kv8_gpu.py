"""Paged 8-bit key/value cache and beam selection on the GPU against oracle/kv8_oracle.py (64 bits).

Codes, exponents, tables, counts, tokens and rows are compared for equality.  Tolerances of computed
numbers, per output o = sum p v:
* rounding of the result to its type: eps / 2 * |o|;
* each p enters the product with V rounded to half precision (2^-11; split in two halves, 2^-22, for
  fp32) and is an exponential of a score that is off by at most (hd + 4) 2^-24 S, S the largest sum of
  |q k| (fp32 products and sums, the scale, the subtraction of the maximum); exponential and running
  sums 2^-22 and n 2^-23 for n keys; the same once more for the divisor: all relative to sum p |v|;
* a p below half precision's normal range is off by 2^-25 (2^-46 when split, bounded by the same):
  n 2^-25 max |v|.
"""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as K

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def np64(t):
    return t.detach().double().cpu().numpy()


def filled(dev, lens, page=16, nkv=2, hd=64, layers=1, spare=6, seed=0, max_pages=None, poison=True):
    """A cache whose sequences lie scattered over the pool, with random contents; rows that no sequence
    holds are NaN codes."""
    from cats_b200.kv8 import KVCache8

    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + spare
    max_pages = max_pages or max(held) + 3
    at, k = torch.randperm(pages, generator=g).tolist(), 0
    c = KVCache8(layers, pages, len(lens), max_pages * page, nkv, hd, page, dev)
    codes = torch.full((layers, pages, 2, nkv, page, hd), 127 if poison else 0, dtype=torch.uint8)
    exps = torch.randint(-3, 4, (layers, pages, 2, nkv), generator=g)
    for b, n in enumerate(lens):
        for j in range(held[b]):
            rows = min(page, n - j * page)
            v = torch.randn((layers, 2, nkv, rows, hd), generator=g) * 60
            codes[:, at[k], :, :, :rows] = v.to(torch.float8_e4m3fn).view(torch.uint8)
            c.table[b, j] = at[k]
            c.refs[at[k]] = 1
            k += 1
    c.codes.view(torch.uint8).copy_(codes)
    c.scales.copy_(torch.exp2(exps.float()))
    c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    return c


def same_state(c, o, layers=True):
    assert np.array_equal(c.table.cpu().numpy(), o.table)
    assert np.array_equal(c.lens.cpu().numpy(), o.lens)
    assert np.array_equal(c.refs.cpu().numpy(), o.refs)
    if layers:                                          # the rows that sequences hold
        for layer in range(c.n_layers):
            for b in range(c.n_seqs):
                k, v = c.read(layer, b)
                ko, vo = o.rows(layer, b, int(o.lens[b]))
                assert np.array_equal(np64(k), ko, equal_nan=True) and np.array_equal(np64(v), vo, equal_nan=True), (layer, b)


def tables(n, hd, dt, dev):
    a = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    return [torch.cat((f(a), f(a)), -1).to(dt).to(dev) for f in (torch.cos, torch.sin)]


def cu_of(counts, dev):
    return torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device=dev)


# ---- attend ---------------------------------------------------------------------------------------------
def attend_and_compare(c, counts, group, dt, seed=1, scale=None, strided=False, uniform=False, q=None):
    dev, n, nh, hd = c.device, int(sum(counts)), c.n_kv_heads * group, c.head_dim
    g = torch.Generator().manual_seed(seed)
    if q is None:
        q = torch.randn((n, nh + (3 if strided else 0), hd), generator=g).to(dt).to(dev)
    if strided:
        q = q[:, :nh]
    out = c.attend(0, q, cu=None if uniform else cu_of(counts, dev), scale=scale)
    want, m = K.Cache.of(c).attend(0, np64(q), counts, scale)
    eps = torch.finfo(dt).eps
    rel = (2.0 ** -21 if dt == torch.float32 else 2.0 ** -11) + 2 * ((hd + 4) * 2.0 ** -24 * m["s"] + 2.0 ** -22 + m["n"] * 2.0 ** -23)
    tol = eps / 2 * np.abs(want) + rel * m["pv"] + m["n"] * 2.0 ** -25 * m["v"] + 1e-30
    if dt == torch.float16:
        tol = tol + 2.0 ** -25                          # results below half precision's normal range
    got = np64(out)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    worst = float(np.max(np.where(nan, 0, np.abs(got - want) / tol)))
    assert worst <= 1, worst
    c.check()
    return out


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("page,nkv,group,hd", [(16, 2, 1, 64), (64, 3, 4, 128), (32, 1, 7, 96), (128, 2, 8, 32),
                                               (64, 1, 16, 128), (16, 2, 20, 32)])
def test_one_token_each(page, nkv, group, hd, dt, cuda_device):
    c = filled(cuda_device, [1, 2, 15, 16, 17, 63, 64, 65, 130, 300], page, nkv, hd)
    attend_and_compare(c, [1] * 10, group, TYPES[dt], uniform=True)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lens,counts", [([40, 7, 0, 129], [3, 7, 0, 1]), ([1], [1]), ([200], [200]), ([33, 500], [33, 61]),
                                         ([0, 0, 5], [0, 0, 2]), ([70, 70, 70], [5, 5, 5])])
def test_several_tokens_are_causal(lens, counts, dt, cuda_device):
    c = filled(cuda_device, lens, 32, 2, 64)
    attend_and_compare(c, counts, 3, TYPES[dt], strided=True)


@pytest.mark.parametrize("dt", list(TYPES))
def test_long_sequences_are_split_and_joined(dt, cuda_device):
    c = filled(cuda_device, [5000, 31, 1], 64, 1, 128)
    attend_and_compare(c, [1, 1, 1], 4, TYPES[dt], uniform=True)
    attend_and_compare(c, [9, 30, 1], 4, TYPES[dt], seed=2)


@pytest.mark.parametrize("n", [200, 700])
def test_many_short_sequences(n, cuda_device):
    c = filled(cuda_device, [1 + 37 * i % 97 for i in range(n)], 16, 2, 32, spare=1)
    attend_and_compare(c, [1] * n, 2, torch.float16, uniform=True)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("hd,page,group", [(32, 16, 3), (96, 32, 6), (64, 128, 1), (128, 16, 2)])
def test_many_sequences_with_several_tokens(hd, page, group, dt, cuda_device):
    lens = [5 + 53 * i % 211 for i in range(40)]
    c = filled(cuda_device, lens, page, 1, hd)
    attend_and_compare(c, [min(n, 1 + 29 * i % 37) for i, n in enumerate(lens)], group, TYPES[dt])


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("hd,counts", [(128, [130, 40, 1]), (64, [64, 300, 7]), (32, [40, 33, 9]), (96, [2, 2, 1])])
def test_long_sequences_with_many_tokens(hd, counts, dt, cuda_device):
    """Several tiles of rows, split over CTAs and joined."""
    c = filled(cuda_device, [3000, 411, 9], 64, 2, hd)
    attend_and_compare(c, counts, 2, TYPES[dt])


def test_a_padded_call_leaves_the_rows_behind(cuda_device):
    for dt in TYPES.values():
        for counts in ([1, 0, 1], [20, 3, 1]):
            c = filled(cuda_device, [40, 33, 7], 16, 2, 64)
            n = sum(counts)
            cu, cos = cu_of(counts, cuda_device), tables(c.max_len, 64, dt, cuda_device)
            qkv = torch.randn((n + 5, 8 * 64), device=cuda_device).to(dt)
            q = torch.full((n + 5, 4, 64), 7.0, device=cuda_device, dtype=dt)
            out = torch.full_like(q, 9.0)
            c.append(0, qkv, 4, *cos, cu=cu, q_out=q)
            c.attend(0, q, cu=cu, out=out)
            assert (q[n:] == 7).all() and (out[n:] == 9).all() and (out[:n] != 9).any()
            c.check()


def test_scores_of_any_size(cuda_device):
    """Peaked and flat softmax, large and tiny scales of pages, queries beyond half precision's range."""
    c = filled(cuda_device, [150, 90], 16, 2, 64)
    attend_and_compare(c, [2, 1], 2, torch.bfloat16, scale=3.0)
    attend_and_compare(c, [2, 1], 2, torch.float32, scale=0.0)
    attend_and_compare(c, [2, 1], 2, torch.float32, scale=-0.2)
    g = torch.Generator().manual_seed(5)
    q = (torch.randn((3, 4, 64), generator=g) * torch.tensor([1e-6, 1.0, 3e5])[:, None, None]).to(cuda_device)
    attend_and_compare(c, [2, 1], 2, torch.float32, q=q, scale=1e-4)
    attend_and_compare(c, [2, 1], 2, torch.bfloat16, q=q.bfloat16(), scale=1e-4)
    c.scales[0, :, 1] *= torch.exp2(torch.randint(-12, 13, c.scales[0, :, 1].shape, generator=g).float()).to(cuda_device)
    attend_and_compare(c, [2, 1], 2, torch.float32)
    c.scales[0, :, 1] *= 2.0 ** 20
    attend_and_compare(c, [2, 1], 2, torch.float32)


@pytest.mark.parametrize("dt,heads", [("f32", 4), ("f16", 2), ("bf16", 4), ("bf16", 2)])
def test_what_lies_behind_a_token_does_not_reach_it(dt, heads, cuda_device):
    """NaN values (and keys) of the later tokens of the same call: the earlier rows stay what they are."""
    for where in (0, 1):
        for counts in ([20, 33], [20, 3]):                                     # many rows per key head, few
            c = filled(cuda_device, [50, 60 + counts[1]], 32, 2, 64)
            q = torch.ones((sum(counts), heads, 64), device=cuda_device, dtype=TYPES[dt])
            clean = c.attend(0, q, cu=cu_of(counts, cuda_device))
            page = int(c.table[0, 45 // 32])
            c.codes.view(torch.uint8)[0, page, where, 1, 45 % 32, 7] = 127     # position 45, key head 1
            got = c.attend(0, q, cu=cu_of(counts, cuda_device))
            first = 45 - 30                                                    # the row at position 45
            hit = torch.zeros_like(got, dtype=torch.bool)
            if where == 0:
                hit[first:20, heads // 2:] = True                              # its score is NaN: the whole row
            else:
                hit[first:20, heads // 2:, 7] = True
            assert torch.equal(got.isnan(), hit)
            assert torch.equal(got[~hit], clean[~hit])


def test_one_new_token_behind_stale_nan_rows(cuda_device):
    """Rows of a sequence's last page behind its length hold NaN codes (see ``filled``): two tokens of
    eight rows, in the tile with the end of the sequence."""
    for dt in TYPES.values():
        c = filled(cuda_device, [33, 47, 5], 64, 1, 64)
        attend_and_compare(c, [2, 2, 2], 4, dt)
        attend_and_compare(c, [3, 1, 4], 2, dt)


def test_empty_sequences_give_zeros_and_bad_ids_are_reported(cuda_device):
    c = filled(cuda_device, [0, 40], 16, 1, 32)
    out = c.attend(0, torch.randn(2, 2, 32, device=cuda_device))
    assert out[0].abs().max() == 0 and out[1].isfinite().all()
    c.check()
    for bad in (-1, 12, 1 << 30):
        d = filled(cuda_device, [40, 40], 16, 1, 32)
        assert d.n_pages == 12
        q = torch.randn(2, 2, 32, device=cuda_device)
        clean = d.attend(0, q)
        d.table[1, 1] = bad
        got = d.attend(0, q)
        assert torch.equal(got[0], clean[0]) and got.isfinite().all()
        with pytest.raises(RuntimeError, match="page id"):
            d.check()
        o = K.Cache.of(d)                                # positions 16 .. 31 left out
        o.table[1, 1], x = 0, np64(q)
        k, v = (np.concatenate([a[:, :16], a[:, 32:]], 1) for a in o.rows(0, 1, 40))
        s = k[0] @ x[1].T * 32 ** -0.5
        p = np.exp(s - s.max(0))
        assert np.allclose(np64(got[1]), (p / p.sum(0)).T @ v[0], rtol=1e-5, atol=1e-5 * np.abs(v).max())


def test_lengths_that_the_table_cannot_hold_are_reported(cuda_device):
    for n in (-3, 10 ** 9):
        c = filled(cuda_device, [20, 40], 16, 1, 32)
        q = torch.randn(2, 1, 32, device=cuda_device)
        clean = c.attend(0, q)
        c.lens[0] = n
        got = c.attend(0, q)
        assert torch.equal(got[1], clean[1])
        with pytest.raises(RuntimeError):
            c.check()


def test_offsets_beyond_32_bits(cuda_device):
    """A pool of 5 GB: the last pages of the last layer."""
    from cats_b200.kv8 import KVCache8

    c = KVCache8(2, 20000, 1, 256, 8, 128, 64, cuda_device)
    c.table[0, :4] = torch.tensor([19999, 19998, 3, 19997], dtype=torch.int32)
    c.lens[0] = 200
    for p in (19999, 19998, 3, 19997):
        c.refs[p] = 1
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn((200, 24 * 128), generator=g).to(cuda_device).half()
    q = c.append(1, qkv, 8)
    out = c.attend(1, q, cu=cu_of([200], cuda_device))
    small = filled(cuda_device, [200], 64, 8, 128)
    small.append(0, qkv, 8)
    assert torch.equal(out, small.attend(0, q, cu=cu_of([200], cuda_device)))
    for a, b in zip(c.read(1, 0), small.read(0, 0)):
        assert torch.equal(a, b)
    assert int(c.codes.view(torch.uint8)[0].max()) == 0 and c.codes.view(torch.uint8)[1, 4].max() == 0
    c.check()


# ---- append ---------------------------------------------------------------------------------------------
def append_and_compare(c, counts, group, dt, seed=1, rope=True, uniform=False, strided=False, size=1.0, qkv=None):
    dev, n, nh, nkv, hd = c.device, int(sum(counts)), c.n_kv_heads * group, c.n_kv_heads, c.head_dim
    g = torch.Generator().manual_seed(seed)
    width = (nh + 2 * nkv) * hd
    if qkv is None:
        qkv = (torch.randn((n, width + (16 if strided else 0)), generator=g) * size).to(dt).to(dev)[:, :width]
    cos, sin = tables(c.max_len + 5, hd, dt, dev) if rope else (None, None)
    # the oracle's rotation in fp32 steps, as documented, so that the codes have to be equal
    o = K.Cache.of(c)
    x = qkv.float().view(n, -1, hd).cpu()
    if rope:
        pos = np.concatenate([np.arange(l - k, l) for l, k in zip(c.lens.tolist(), counts)]).astype(np.int64)
        cf, sf = cos.float().cpu()[pos][:, None], sin.float().cpu()[pos][:, None]
        qk = x[:, :nh + nkv]
        x = torch.cat((qk * cf + torch.cat((-qk[..., hd // 2:], qk[..., :hd // 2]), -1) * sf, x[:, nh + nkv:]), 1)
    want = o.append(0, x.double().numpy(), counts, nh)
    q = c.append(0, qkv, nh, cos, sin, cu=None if uniform else cu_of(counts, dev))
    assert np.array_equal(np64(q), np64(torch.from_numpy(want).float().to(dt)), equal_nan=True)
    c.check()
    assert np.array_equal(np64(c.codes.view(torch.uint8).cpu().view(torch.float8_e4m3fn).float()), o.values, equal_nan=True)
    used = c.refs.cpu().numpy() > 0
    assert np.array_equal(np.log2(c.scales.cpu().numpy())[:, used], o.exps[:, used])


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("page,nkv,group,hd", [(16, 2, 1, 64), (64, 3, 4, 128), (32, 1, 7, 96), (128, 2, 2, 32), (128, 1, 1, 128)])
def test_append_one_token_each(page, nkv, group, hd, dt, cuda_device):
    c = filled(cuda_device, [1, 2, 15, 16, 17, 63, 64, 65, 130], page, nkv, hd)
    append_and_compare(c, [1] * 9, group, TYPES[dt], uniform=True, size=20.0)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("lens,counts", [([40, 7, 0, 129], [3, 7, 0, 1]), ([200], [200]), ([33, 500, 64], [33, 61, 64]),
                                         ([0, 0, 5], [0, 0, 2]), ([70, 70, 70], [66, 66, 66])])
def test_append_several_tokens(lens, counts, dt, cuda_device):
    for page in (16, 64):
        c = filled(cuda_device, lens, page, 2, 96)
        append_and_compare(c, counts, 2, TYPES[dt], strided=True, size=3.0)
    c = filled(cuda_device, lens, 32, 1, 64)
    append_and_compare(c, counts, 1, TYPES[dt], rope=False)


def test_a_larger_row_rescales_the_page(cuda_device):
    """Exponents that grow by little and by a lot (older codes become subnormal and vanish), zeros,
    values that are exactly 448 times a power of two, the ends of the exponents' range."""
    c = filled(cuda_device, [10, 20, 33, 12, 5, 7], 16, 1, 32)
    c.scales.fill_(1.0)
    qkv = torch.randn((6, 3 * 32), device=cuda_device)
    for i, m in enumerate((447.9, 448.0, 448.1, 1e5, 1e9, 0.0)):
        qkv[i] *= 0 if m == 0 else m / qkv[i, 32:].abs().max()
        qkv[i, 40], qkv[i, 70] = m, -m
    append_and_compare(c, [1] * 6, 1, torch.float32, rope=False, uniform=True, qkv=qkv)
    c = filled(cuda_device, [1, 1, 1, 1], 16, 1, 32)
    qkv = torch.randn((4, 96), device=cuda_device) * torch.tensor([1e-30, 1e-9, 1e18, 1e30], device=cuda_device)[:, None]
    append_and_compare(c, [1] * 4, 1, torch.float32, rope=False, uniform=True, qkv=qkv)


def test_what_is_not_finite_is_stored_as_nan_and_sets_no_scale(cuda_device):
    c = filled(cuda_device, [3, 20], 16, 1, 32)
    qkv = torch.randn((2, 96), device=cuda_device)
    qkv[0, 33], qkv[0, 65], qkv[1, 64], qkv[1, 50] = float("inf"), float("-inf"), float("nan"), float("nan")
    append_and_compare(c, [1, 1], 1, torch.float32, rope=False, uniform=True, qkv=qkv)
    k, v = c.read(0, 0)
    assert k[0, 2, 1].isnan() and v[0, 2, 1].isnan() and k.isnan().sum() == 1 and v.isnan().sum() == 1


def test_append_writes_nothing_else(cuda_device):
    c = filled(cuda_device, [40, 7], 16, 2, 64, layers=3)
    before, scales = c.codes.view(torch.uint8).clone(), c.scales.clone()
    c.append(1, torch.randn((4, 6 * 64), device=cuda_device), 2, cu=cu_of([3, 1], cuda_device))
    touched = {(int(c.table[0, 2]), r) for r in (5, 6, 7)} | {(int(c.table[1, 0]), 6)}
    after = c.codes.view(torch.uint8)
    assert torch.equal(after[0], before[0]) and torch.equal(after[2], before[2])
    assert torch.equal(c.scales[::2], scales[::2])
    pages = {p for p, _ in touched}
    for p in range(c.n_pages):
        if p not in pages:
            assert torch.equal(after[1, p], before[1, p]) and torch.equal(c.scales[1, p], scales[1, p])
    assert torch.equal(after[1, int(c.table[1, 0]), :, :, 7:], before[1, int(c.table[1, 0]), :, :, 7:])


def test_append_never_writes_a_shared_or_bad_page(cuda_device):
    for change in ("shared", "bad", "long"):
        c = filled(cuda_device, [40, 7], 16, 1, 32)
        if change == "shared":
            c.refs[c.table[0, 2].long()] = 2
        elif change == "bad":
            c.table[0, 2] = c.n_pages
        else:
            c.lens[0] = c.max_len + 1
        before = c.codes.view(torch.uint8).clone()
        c.append(0, torch.randn((2, 96), device=cuda_device), 1)
        mine = int(c.table[1, 0])
        same = [p for p in range(c.n_pages) if p != mine]
        assert torch.equal(c.codes.view(torch.uint8)[:, same], before[:, same])
        assert not torch.equal(c.codes.view(torch.uint8)[:, mine], before[:, mine])
        with pytest.raises(RuntimeError, match="page id" if change != "long" else "longer"):
            c.check()


def test_cu_that_does_not_fit_is_reported_and_reads_nothing(cuda_device):
    c = filled(cuda_device, [40, 30], 16, 1, 32)
    before = c.codes.view(torch.uint8).clone()
    c.append(0, torch.randn((2, 96), device=cuda_device), 1,
             cu=torch.tensor([0, 20, 30], dtype=torch.int32, device=cuda_device))
    assert torch.equal(c.codes.view(torch.uint8), before)
    with pytest.raises(RuntimeError, match="cu does not fit"):
        c.check()


# ---- pages ----------------------------------------------------------------------------------------------
def test_grow_takes_the_lowest_free_pages_in_order(cuda_device):
    for counts in ([1, 1, 1, 1], [0, 16, 5, 40], [17, 0, 0, 0]):
        c = filled(cuda_device, [16, 7, 0, 33], 16, 1, 32, spare=12)
        o = K.Cache.of(c)
        o.grow(counts)
        if len(set(counts)) == 1:
            c.grow(counts[0])
        else:
            c.grow(cu=cu_of(counts, cuda_device))
        same_state(c, o, layers=False)
        c.check()


def test_grow_of_many_sequences_over_a_large_pool(cuda_device):
    from cats_b200.kv8 import KVCache8

    c = KVCache8(1, 30000, 1024, 640, 1, 32, 16, cuda_device)
    held = torch.randperm(30000, generator=torch.Generator().manual_seed(1))[:20000].to(cuda_device)
    c.refs[held] = 1
    o = K.Cache.of(c)
    counts = np.random.default_rng(2).integers(0, 250, 1024)
    o.grow(counts)
    c.grow(cu=cu_of(counts, cuda_device))
    same_state(c, o, layers=False)


def test_grow_without_pages_or_room_leaves_the_sequence(cuda_device):
    c = filled(cuda_device, [16, 16, 15, 16], 16, 1, 32, spare=1)
    o = K.Cache.of(c)
    assert o.grow([1, 1, 1, 1]) == [True, False, True, False]
    c.grow(1)
    same_state(c, o, layers=False)
    with pytest.raises(RuntimeError, match="no free page"):
        c.check()
    c = filled(cuda_device, [60, 5], 16, 1, 32, max_pages=4)
    c.grow(5)
    assert c.lens.tolist() == [60, 10]
    with pytest.raises(RuntimeError, match="longer"):
        c.check()


@pytest.mark.parametrize("page,hd,nkv", [(16, 32, 1), (64, 128, 3), (32, 96, 2)])
def test_reorder_shares_full_pages_and_copies_the_last(page, hd, nkv, cuda_device):
    lens = [page * 2 + 5, page * 3, 3, 0, page - 1, page * 4 + 1]
    for parents in ([0, 1, 2, 3, 4, 5], [0, 0, 0, 0, 0, 0], [5, 4, 3, 2, 1, 0], [1, 1, 2, 2, 5, 5], [-1, 0, -1, 0, 5, -1],
                    [-1] * 6, [3, 3, 0, 0, 5, 5]):
        c = filled(cuda_device, lens, page, nkv, hd, layers=2, spare=8)
        o = K.Cache.of(c)
        o.reorder(parents)
        c.reorder(torch.tensor(parents, dtype=torch.int32, device=cuda_device))
        same_state(c, o)
        c.check()


def test_reorder_again_and_again(cuda_device):
    """Shared pages with several holders, freed and taken again: 25 steps of growth and reordering."""
    r = np.random.default_rng(3)
    c = filled(cuda_device, [20, 0, 33, 5, 64], 16, 1, 32, spare=60, max_pages=12)
    o = K.Cache.of(c)
    for step in range(25):
        counts = r.integers(0, 9, 5) * (o.lens < 150)
        o.grow(counts)
        c.grow(cu=cu_of(counts, cuda_device))
        n = int(counts.sum())
        if n:
            qkv = torch.from_numpy(r.standard_normal((n, 96)).astype(np.float32)).to(cuda_device)
            o.append(0, np64(qkv).reshape(n, 3, 32), counts, 1)
            c.append(0, qkv, 1, cu=cu_of(counts, cuda_device))
        parents = r.integers(-1, 5, 5) if step % 3 else np.arange(5)
        o.reorder(parents)
        c.reorder(torch.tensor(parents, dtype=torch.int32, device=cuda_device))
        if step % 6 == 5:
            assert int(c.compact()) == o.compact()
        same_state(c, o)
        c.check()


def test_reorder_without_a_free_page(cuda_device):
    c = filled(cuda_device, [20, 20, 5], 16, 1, 32, spare=0)
    o = K.Cache.of(c)
    c.reorder(torch.tensor([0, 1, 1], dtype=torch.int32, device=cuda_device))     # frees a page, takes it
    o.reorder([0, 1, 1])
    same_state(c, o)
    c.check()
    c.reorder(torch.tensor([0, 0, 1], dtype=torch.int32, device=cuda_device))
    o.reorder([0, 0, 1])
    same_state(c, o)
    c = filled(cuda_device, [20, 17, 16], 16, 1, 32, spare=0)
    c.reorder(torch.tensor([0, 1, 1], dtype=torch.int32, device=cuda_device))
    c.reorder(torch.tensor([0, 1, 0], dtype=torch.int32, device=cuda_device))
    c.check()
    c.refs[c.refs == 0] = 1                                                      # nothing is free any more
    c.reorder(torch.tensor([0, 0, 0], dtype=torch.int32, device=cuda_device))
    assert c.lens.tolist() == [20, 20, 20] and (c.table[1:, 1] >= 0).sum() == 2
    c.reorder(torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device))


def test_bad_parents_are_reported(cuda_device):
    c = filled(cuda_device, [20, 7], 16, 1, 32)
    c.reorder(torch.tensor([7, -5], dtype=torch.int32, device=cuda_device))
    assert c.lens.tolist() == [0, 0] and int(c.refs.sum()) == 0
    with pytest.raises(RuntimeError, match="parent"):
        c.check()


def test_reorder_of_many_sequences(cuda_device):
    r = np.random.default_rng(4)
    lens = r.integers(0, 90, 1000)
    c = filled(cuda_device, lens.tolist(), 16, 1, 32, spare=1200)
    o = K.Cache.of(c)
    parents = r.integers(-1, 1000, 1000)
    o.reorder(parents)
    c.reorder(torch.tensor(parents, dtype=torch.int32, device=cuda_device))
    same_state(c, o, layers=False)
    ids = torch.from_numpy(o.table[o.table >= 0])
    got = c.codes.view(torch.uint8).cpu()[0, ids].view(torch.float8_e4m3fn).float().numpy()
    want = o.values[0, ids]
    held = ~np.isnan(want)
    assert np.array_equal(got[held], want[held])


def test_fork_and_free(cuda_device):
    c = filled(cuda_device, [20, 0, 7], 16, 1, 32)
    o = K.Cache.of(c)
    c.fork([0], [1])
    o.reorder([0, 0, 2])
    same_state(c, o)
    c.free([0, 2, 2])
    o.reorder([-1, 1, -1])
    same_state(c, o)
    for bad in (lambda: c.fork([0, 0], [1, 1]), lambda: c.fork([0], [3]), lambda: c.fork([3], [0]), lambda: c.fork([-1], [0]),
                lambda: c.free([3]), lambda: c.free([-1]), lambda: c.fork([0], [])):
        with pytest.raises(RuntimeError):
            bad()
    same_state(c, o)


@pytest.mark.parametrize("pages,live", [(1, 1), (1, 0), (40, 13), (40, 40), (20000, 9000)])
def test_compact(pages, live, cuda_device):
    from cats_b200.kv8 import KVCache8

    seqs, width = 8, max(1, -(-live // 8))
    c = KVCache8(2, pages, seqs, width * 16, 1, 32, 16, cuda_device)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(live))[:live]
    c.codes.view(torch.uint8).random_(0, 127)
    c.scales.copy_(torch.exp2(torch.randint(-20, 20, c.scales.shape).float()))
    flat = torch.full((seqs * width,), -1, dtype=torch.int32)
    flat[:live] = ids.int()
    c.table.copy_(flat.view(seqs, width))
    c.lens.copy_((c.table >= 0).sum(1) * 16)
    c.refs[ids.to(cuda_device)] = torch.randint(1, 5, (live,), dtype=torch.int32).to(cuda_device)
    o = K.Cache.of(c)
    assert int(c.compact()) == o.compact() == live
    same_state(c, o, layers=False)
    got = c.codes.view(torch.uint8).cpu().view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(got[:, :live], o.values[:, :live])
    assert np.array_equal(np.log2(c.scales.cpu().numpy())[:, :live], o.exps[:, :live])


# ---- selection ------------------------------------------------------------------------------------------
def select_and_compare(x, scores, k, done=None, eos=-1):
    from cats_b200 import ops

    got = ops.beam_select(x, scores, k, done=done, eos=eos)
    want = K.beam_select(np64(x), np64(scores), k, None if done is None else done.cpu().numpy(), eos)
    assert np.array_equal(got[1].cpu().numpy(), want[1]) and np.array_equal(got[2].cpu().numpy(), want[2])
    assert np.array_equal(got[3].cpu().numpy().astype(bool), want[3])
    # log-sum-exp: exponentials 2^-21, fp32 sums of at most 2^13 values 2^-11 at the very worst (they
    # are positive and of like size: 2^-20 is measured far above what occurs), the score's own rounding
    a, b = np64(got[0]), want[0]
    fin = np.isfinite(b)
    assert np.array_equal(fin, np.isfinite(a)) and np.array_equal(a[~fin], b[~fin])
    assert np.all(np.abs(a[fin] - b[fin]) <= 2.0 ** -24 * np.abs(b[fin]) + 2.0 ** -18)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n,beams,vocab,k", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 4), (1, 4, 32000, 4), (3, 2, 4097, 9), (2, 32, 515, 32),
                                             (5, 1, 8191, 32), (1, 8, 50257, 8), (40, 3, 2048, 3), (1, 2, 129283, 17)])
def test_select(n, beams, vocab, k, dt, cuda_device):
    g = torch.Generator().manual_seed(vocab + k)
    x = (torch.randn((n, beams, vocab), generator=g) * 3).to(TYPES[dt]).to(cuda_device)
    scores = (-10 * torch.rand((n, beams), generator=g)).to(cuda_device)
    select_and_compare(x, scores, k)
    done = (torch.rand((n, beams), generator=g) < 0.4).to(cuda_device)
    select_and_compare(x, scores, k, done, eos=vocab // 2)


def test_select_ties_go_to_the_lowest_beam_and_token(cuda_device):
    dev = cuda_device
    for dt in TYPES.values():
        flat = torch.zeros((2, 3, 9000), device=dev, dtype=dt)
        select_and_compare(flat, torch.zeros((2, 3), device=dev), 20)
        few = (torch.randint(0, 3, (2, 3, 9000), generator=torch.Generator().manual_seed(0))).to(dt).to(dev)
        few[:, 1] = few[:, 0]
        few[:, 2] = few[:, 0]
        select_and_compare(few, torch.full((2, 3), -1.5, device=dev), 32)
        select_and_compare(few, torch.tensor([[-1.5, -1.5, -1.0]] * 2, device=dev), 7)
        signs = torch.zeros((1, 2, 300), device=dev, dtype=dt)
        signs[0, 0, ::2] = -0.0
        select_and_compare(signs, torch.zeros((1, 2), device=dev), 12)


def test_select_of_rising_falling_and_masked_rows(cuda_device):
    dev = cuda_device
    up = torch.arange(60000, device=dev, dtype=torch.float32) * 1e-4
    x = torch.stack((up, up.flip(0), torch.where(up < 5.99, -float("inf"), up), up - 3)).view(1, 4, -1)
    for k in (1, 4, 32):
        select_and_compare(x, torch.tensor([[-1.0, -1.25, -3.0, -float("inf")]], device=dev), k)
    y = torch.full((1, 3, 700), -float("inf"), device=dev)
    y[0, 1, 13] = 2.0
    select_and_compare(y, torch.zeros((1, 3), device=dev), 6)
    select_and_compare(y, torch.zeros((1, 3), device=dev), 6, torch.tensor([[True, False, True]], device=dev), eos=3)
    low = torch.full((1, 2, 700), torch.finfo(torch.float32).min, device=dev)
    low[0, 1, ::5] = torch.randn(140, device=dev)
    select_and_compare(low, torch.zeros((1, 2), device=dev), 8)


def test_select_leaves_out_beams_that_are_not_finite(cuda_device):
    x = torch.randn((1, 5, 3000), device=cuda_device)
    x[0, 0, 2999] = float("nan")
    x[0, 1, 17] = float("inf")
    scores = torch.tensor([[0.0, 0.0, -float("inf"), float("nan"), -4.0]], device=cuda_device)
    select_and_compare(x, scores, 10)
    select_and_compare(x[:, :4], scores[:, :4].contiguous(), 10)                 # nothing usable at all


def test_select_of_strided_rows(cuda_device):
    x = torch.randn((3, 2, 1003), device=cuda_device).half()
    s = torch.randn((3, 2), device=cuda_device)
    for y in (x[:, :, :1000], x[:, :, 1:], x[:, :, 3:504]):
        select_and_compare(y, s, 5)
    select_and_compare(x[:, :1, 2:], s[:, :1].contiguous(), 5)


def test_front_end_refusals(cuda_device):
    from cats_b200 import ops
    from cats_b200.kv8 import KVCache8

    dev = cuda_device
    c = filled(dev, [20, 7], 16, 2, 64)
    r = lambda *s, dt=torch.float16, d=dev: torch.zeros(s, dtype=dt, device=d)  # noqa: E731
    cos = r(c.max_len, 64)
    for call in (lambda: c.append(0, r(2, 6 * 64).cpu(), 2), lambda: c.append(0, r(3, 6 * 64), 2), lambda: c.append(0, r(2, 5 * 64), 2),
                 lambda: c.append(0, r(2, 7 * 64), 3), lambda: c.append(1, r(2, 6 * 64), 2), lambda: c.append(0, r(2, 6 * 64, dt=torch.float64), 2),
                 lambda: c.append(0, r(6 * 64, 2).t(), 2), lambda: c.append(0, r(2, 6 * 64), 2, cos, None),
                 lambda: c.append(0, r(2, 6 * 64), 2, cos[:-1], cos[:-1]), lambda: c.append(0, r(2, 6 * 64), 2, cos.float(), cos.float()),
                 lambda: c.append(0, r(2, 6 * 64), 2, cu=torch.zeros(3, dtype=torch.int64, device=dev)),
                 lambda: c.append(0, r(2, 6 * 64), 2, cu=torch.zeros(2, dtype=torch.int32, device=dev)),
                 lambda: c.append(0, r(2, 6 * 64), 2, q_out=r(2, 2, 32)), lambda: c.append(0, r(2, 6 * 64 + 4)[:, 4:], 2),
                 lambda: c.attend(0, r(2, 3, 64)), lambda: c.attend(0, r(2, 2, 32)), lambda: c.attend(0, r(2, 2, 64).cpu()),
                 lambda: c.attend(0, r(2, 64, 2).transpose(1, 2)), lambda: c.attend(2, r(2, 2, 64)), lambda: c.attend(0, r(3, 2, 64)),
                 lambda: c.attend(0, r(2, 2, 64), out=r(2, 2, 64, dt=torch.float32)), lambda: c.attend(0, r(2, 2, 64), scale=float("nan")),
                 lambda: c.grow(0), lambda: c.grow(-1), lambda: c.reorder(torch.zeros(2, dtype=torch.int64, device=dev)),
                 lambda: c.reorder(torch.zeros(3, dtype=torch.int32, device=dev)), lambda: c.read(0, 2), lambda: c.read(1, 0),
                 lambda: KVCache8(1, 4, 1, 64, 1, 80, device=dev), lambda: KVCache8(1, 4, 1, 64, 1, 64, page=20, device=dev),
                 lambda: KVCache8(1, 4, 1025, 64, 1, 64, device=dev), lambda: KVCache8(0, 4, 1, 64, 1, 64, device=dev),
                 lambda: ops.beam_select(r(1, 2, 8), r(1, 2), 2), lambda: ops.beam_select(r(1, 2, 8), r(1, 3, dt=torch.float32), 2),
                 lambda: ops.beam_select(r(1, 33, 8), r(1, 33, dt=torch.float32), 2), lambda: ops.beam_select(r(1, 2, 8), r(1, 2, dt=torch.float32), 17),
                 lambda: ops.beam_select(r(1, 2, 8), r(1, 2, dt=torch.float32), 0), lambda: ops.beam_select(r(2, 8), r(1, 2, dt=torch.float32), 2),
                 lambda: ops.beam_select(r(1, 8, 2).transpose(1, 2), r(1, 2, dt=torch.float32), 2),
                 lambda: ops.beam_select(r(4, 2, 8)[::2, :1].expand(2, 2, 8), r(2, 2, dt=torch.float32), 2),
                 lambda: ops.beam_select(r(1, 2, 8), r(1, 2, dt=torch.float32), 2, done=r(1, 2, dt=torch.bool)),
                 lambda: ops.beam_select(r(1, 2, 8), r(1, 2, dt=torch.float32), 2, done=r(1, 2), eos=1)):
        with pytest.raises(RuntimeError):
            call()
    c.check()
    assert c.append(0, r(0, 6 * 64), 2, cu=cu_of([0, 0], dev)).shape == (0, 2, 64)
    assert c.attend(0, r(0, 2, 64), cu=cu_of([0, 0], dev)).shape == (0, 2, 64)


# ---- together -------------------------------------------------------------------------------------------
def beam_steps(dev, graph, seed=0):
    """Six steps of a beam search over two prompts, one layer: grow, append, attend, select, reorder."""
    from cats_b200 import ops

    beams, vocab = 3, 700
    c = filled(dev, [37, 37, 37, 5, 5, 5], 16, 1, 32, spare=30, seed=seed)
    g = torch.Generator().manual_seed(seed)
    w_in = torch.randn((vocab, 4 * 32), generator=g).to(dev)
    w_out = torch.randn((64, vocab), generator=g).to(dev)
    cos, sin = tables(c.max_len, 32, torch.float32, dev)
    tok = torch.arange(6, device=dev)
    scores = -torch.rand((2, beams), generator=g).to(dev)
    done = torch.zeros((2, beams), dtype=torch.bool, device=dev)
    log = []

    def step():
        c.grow(1)
        q = c.append(0, w_in[tok], 2, cos, sin)
        o = c.attend(0, q)
        s, rows, t, d = ops.beam_select((o.view(6, 64) @ w_out).view(2, beams, vocab), scores, beams, done=done, eos=3)
        c.reorder(rows.view(-1))
        scores.copy_(s)
        done.copy_(d)
        tok.copy_(t.view(-1))

    if graph:
        keep = [t.clone() for t in (c.codes.view(torch.uint8), c.scales, c.table, c.lens, c.refs, tok, scores, done)]
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream(dev).wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step()
        for t, k in zip((c.codes.view(torch.uint8), c.scales, c.table, c.lens, c.refs, tok, scores, done), keep):
            t.copy_(k)
    for _ in range(6):
        gr.replay() if graph else step()
        log.append((tok.clone(), scores.clone(), done.clone(), c.table.clone(), c.lens.clone(), c.refs.clone()))
    c.check()
    return log


def test_a_captured_step_replays_to_the_same_search(cuda_device):
    for a, b in zip(beam_steps(cuda_device, False), beam_steps(cuda_device, True)):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_two_searches_at_once_on_two_streams(cuda_device):
    """Different caches on different streams share nothing: eager and captured, interleaved."""
    dev = cuda_device
    want = [beam_steps(dev, False, s) for s in (1, 2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream(dev))
    got = []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            got.append(beam_steps(dev, False, i + 1))
    torch.cuda.synchronize(dev)
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert all(torch.equal(u, v) for u, v in zip(x, y))


def test_work_handed_to_another_stream(cuda_device):
    """Work handed over by an event to another stream, on scratch that the cache keeps."""
    c, d = (filled(cuda_device, [700, 31, 90], 64, 2, 128, seed=3) for _ in range(2))
    q = torch.randn((3, 8, 128), device=cuda_device).half()
    many = torch.randn((60, 8, 128), device=cuda_device).half()
    cu = cu_of([25, 5, 30], cuda_device)
    want = [c.attend(0, q), c.attend(0, many, cu=cu)]
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        got = [d.attend(0, q), d.attend(0, many, cu=cu)]
        d.reorder(torch.tensor([1, 1, 0], dtype=torch.int32).to(cuda_device))
        d.compact()
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert d.lens.tolist() == [31, 31, 700]
    d.check()


def test_results_do_not_depend_on_the_run(cuda_device):
    c = filled(cuda_device, [5000, 31, 700], 64, 2, 128)
    q = torch.randn((3, 8, 128), device=cuda_device).half()
    first = c.attend(0, q)
    x = torch.randn((4, 4, 32000), device=cuda_device)
    s = torch.randn((4, 4), device=cuda_device)
    from cats_b200 import ops
    best = ops.beam_select(x, s, 4)
    for _ in range(5):
        assert torch.equal(c.attend(0, q), first)
        assert all(torch.equal(a, b) for a, b in zip(ops.beam_select(x, s, 4), best))
