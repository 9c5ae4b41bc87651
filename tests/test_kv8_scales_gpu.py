"""Attention over pages whose scales lie far apart: a page with one very large channel must not cost the
other channels, or the other pages' rows, their precision.

Tolerance of an output o = sum p v, channel by channel: as in test_kv8_gpu, but for what half precision
loses of a small weight.  Weights are held relative to a reference that is at most the row's largest
score, and at most 2^4 above or below the scale of what they multiply; one below half precision's normal
range is off by at most 2^-25 of that: 2^-21 * max p * sum |v| over the channel's values.  (fp32: weights in
two halves, the second one's subnormals 2^-25 too.)"""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as K
from test_kv8_gpu import TYPES, cu_of, filled, np64

pytestmark = pytest.mark.gpu


def compare(c, counts, group, dt, seed=1, spread=400):
    n, nh, hd = sum(counts), c.n_kv_heads * group, c.head_dim
    q = torch.randn((n, nh, hd), generator=torch.Generator().manual_seed(seed)).to(dt).to(c.device)
    scale = hd ** -0.5 / spread                            # (codes of some 60: 400 makes the scores of like size)
    got = np64(c.attend(0, q, cu=cu_of(counts, c.device), scale=scale))
    c.check()
    o = K.Cache.of(c)
    want, m = o.attend(0, np64(q), counts, scale)
    small, t, qn = np.zeros_like(want), 0, np64(q)
    for b, k in enumerate(counts):
        for i in range(k):
            key, val = o.rows(0, b, int(o.lens[b]) - k + i + 1)
            for h in range(nh):
                x = key[h // group] @ qn[t, h] * scale
                small[t, h] = np.abs(val[h // group]).sum(0) / np.exp(x - x.max()).sum()
            t += 1
    rel = (2.0 ** -21 if dt == torch.float32 else 2.0 ** -11) + 2 * ((hd + 4) * 2.0 ** -24 * m["s"] + 2.0 ** -22 + m["n"] * 2.0 ** -23)
    tol = torch.finfo(dt).eps / 2 * np.abs(want) + rel * m["pv"] + 2.0 ** -21 * small + 1e-30
    if dt == torch.float16:
        tol = tol + 2.0 ** -25
    worst = float(np.max(np.abs(got - want) / tol))
    assert worst <= 1, worst


def outliers(c, b, at, shift, low=0):
    """Pages ``at`` of sequence b: values 2^shift times as large in one channel, zero in the others.  All
    scales of values 2^low times what they were (fp16 results have to hold the large ones)."""
    c.scales[:, :, 1] *= 2.0 ** low
    for j in at:
        page = int(c.table[b, j])
        codes = c.codes.view(torch.uint8)[:, page, 1]
        keep = codes[..., 5].clone()
        codes.zero_()
        codes[..., 5] = keep
        c.scales[:, page, 1] *= 2.0 ** shift


@pytest.mark.parametrize("dt,shift", [("f16", 6), ("f16", 14), ("f16", 18), ("bf16", 14), ("bf16", 22), ("bf16", 40), ("f32", 18), ("f32", 30),
                                      ("f32", 50)])
@pytest.mark.parametrize("page,nkv,group,hd,counts", [(16, 2, 2, 64, [1, 1, 1]), (64, 1, 4, 128, [1, 1, 1]), (32, 2, 3, 96, [4, 5, 3]),
                                                      (16, 1, 5, 64, [5, 5, 5]), (16, 1, 4, 64, [20, 33, 9]), (64, 2, 2, 128, [40, 30, 60]),
                                                      (16, 1, 2, 32, [30, 40, 9])])
def test_one_page_far_above_the_others(page, nkv, group, hd, counts, dt, shift, cuda_device):
    for at in ([0], [1], [1, 3]):
        c = filled(cuda_device, [300, 2700 if max(counts) < 9 else 700, 70], page, nkv, hd, poison=False)
        low = -14 if dt == "f16" else 0
        for b in range(3):
            pages = -(-int(c.lens[b]) // page)
            outliers(c, b, [j for j in at if j < pages], shift, low if b == 0 else 0)
        compare(c, counts, group, TYPES[dt])
        compare(c, counts, group, TYPES[dt], spread=20)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("hd,counts", [(64, [1, 1]), (96, [7, 8]), (128, [40, 50])])
def test_every_page_at_another_scale(hd, counts, dt, cuda_device):
    """Scales over the whole range that the cache can store, page by page, in no order."""
    c = filled(cuda_device, [400, 190], 16, 2, hd, poison=False)
    g = torch.Generator().manual_seed(3)
    for width in (8, 20, 40):
        c.scales[:, :, 1] = torch.exp2(torch.randint(-width // 2, width // 2 + 1, c.scales[:, :, 1].shape, generator=g).float()).to(c.device)
        compare(c, counts, 2, TYPES[dt])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1], [9, 8], [40, 30]])
def test_the_ends_of_the_range_of_scales(counts, dt, cuda_device):
    """Pages at 2^60 beside pages at 2^-24, with and without rows that are one position alone."""
    for at in ([0], [2], [1, 5]):
        c = filled(cuda_device, [400, 190], 16, 1, 64, poison=False)
        c.scales[:, :, 1] = 2.0 ** -24
        for b in range(2):
            outliers(c, b, at, 84)
        compare(c, counts, 2, TYPES[dt])
        compare(c, counts, 2, TYPES[dt], spread=1)
