"""Attention over the paged 8-bit cache where the work is dealt out in equal shares (more (sequence, head,
tile)s than CTAs): segments that are split between CTAs, CTAs that have the end of one segment and the
beginning of another, every tile size of every kernel."""
import pytest
import torch

from test_kv8_gpu import TYPES, attend_and_compare, filled

pytestmark = pytest.mark.gpu


def segments(c, counts, group, rows):
    """(head, tile)s of the call."""
    return sum(-(-n * group // rows) for n in counts) * c.n_kv_heads


def compare(c, counts, group, rows, dt, **more):
    sms = torch.cuda.get_device_properties(c.device).multi_processor_count
    assert segments(c, counts, group, rows) > sms          # not by segments
    mean = -(-sum(counts) // c.n_seqs) * group
    assert {8: mean <= 8, 16: 8 < mean, 32: 16 < mean <= 32, 128: mean > 32}[rows]
    attend_and_compare(c, counts, group, dt, **more)
    c.check()


# uneven lengths: from less than a unit to many, borders of shares anywhere
def uneven(n, least, most):
    return [least + (most - least) * (i * i * 37 % 101) // 100 for i in range(n)]


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n,nkv,page,hd,most", [(24, 8, 16, 32, 3000), (40, 4, 64, 64, 1500), (9, 24, 32, 96, 1300), (160, 1, 128, 128, 900)])
def test_tiles_of_8_rows(n, nkv, page, hd, most, dt, cuda_device):
    c = filled(cuda_device, uneven(n, 200, most), page, nkv, hd)
    compare(c, [1] * n, 4, 8, TYPES[dt], uniform=True)
    compare(c, [1 + i % 3 for i in range(n)], 2, 8, TYPES[dt], seed=2)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("n,nkv,page,hd", [(24, 8, 16, 32), (40, 4, 64, 128)])
def test_tiles_of_16_rows(n, nkv, page, hd, dt, cuda_device):
    c = filled(cuda_device, uneven(n, 100, 1500), page, nkv, hd)
    compare(c, [3] * n, 5, 16, TYPES[dt], uniform=True)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("n,nkv,page,hd", [(24, 8, 16, 32), (40, 4, 64, 64), (20, 8, 32, 96), (22, 8, 128, 128)])
def test_tiles_of_32_rows(n, nkv, page, hd, dt, cuda_device):
    c = filled(cuda_device, uneven(n, 100, 1200), page, nkv, hd)
    compare(c, [8] * n, 3, 32, TYPES[dt], uniform=True)
    compare(c, [4 + 7 * i % 9 for i in range(n)], 3, 32, TYPES[dt], seed=2)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("n,nkv,page,hd,group,t", [(24, 8, 16, 64, 4, 10), (10, 4, 64, 128, 8, 64), (3, 8, 128, 64, 8, 120),
                                                   (40, 4, 32, 128, 6, 7)])
def test_tiles_of_128_rows(n, nkv, page, hd, group, t, dt, cuda_device):
    """The tensor-memory kernel: also as the second segment of a CTA, and with several tiles of rows."""
    c = filled(cuda_device, uneven(n, 130, 900), page, nkv, hd)
    counts = [t] * n
    compare(c, counts, group, 128, TYPES[dt], uniform=True)
    compare(c, [t // 2 + 1 + 37 * i % (t + 1) for i in range(n)], group, 128, TYPES[dt], seed=2)


def test_nan_values_of_one_segment_stay_out_of_the_next(cuda_device):
    """A CTA that has several segments: NaN values of the first reach none of the others."""
    for group, t in ((4, 1), (3, 8), (4, 20)):
        n = 30
        c = filled(cuda_device, uneven(n, 150, 700), 16, 6, 64)
        q = torch.randn((n * t, 6 * group, 64), device=cuda_device).half()
        clean = c.attend(0, q)
        for b in range(0, n, 3):
            c.codes.view(torch.uint8)[0, c.table[b, 0].long(), 1, :, 3, 9] = 127
        got = c.attend(0, q).view(n, t, 6 * group, 64)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0::3, :, :, 9] = True
        assert torch.equal(got.isnan(), hit)
        assert torch.equal(got[~hit], clean.view_as(got)[~hit])
        c.check()
