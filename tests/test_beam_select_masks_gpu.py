"""Beam selection over logits that carry finite masks or lie far from zero, against
oracle/kv8_oracle.py (64 bits).  Rows, tokens and ended beams equal; scores within the tolerance that
``select_and_compare`` derives."""
import pytest
import torch

from test_kv8_gpu import TYPES, select_and_compare

pytestmark = pytest.mark.gpu


def masked(dt, vocab, kept, mask, dev, seed=0):
    """Four beams of ``vocab`` logits at ``mask`` but for those of ``kept``, which are of usual size."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((1, 4, vocab), float(mask))
    x[:, :, kept] = torch.randn((1, 4, len(kept)), generator=g) * 3
    return x.to(dt).to(dev), (-torch.rand((1, 4), generator=g)).to(dev)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("mask", [-88.0, -89.0, -100.0, -1e4, -65504.0, -1e9])
def test_finite_masks_leave_the_beam_in(mask, dt, cuda_device):
    """Most of a row masked by a finite number: short rows, rows of several tiles, rows whose first
    tiles are masked as a whole, rows that are masked as a whole."""
    if dt == "f16" and abs(mask) > 65504:
        pytest.skip("not a number of the type")
    for vocab, kept in ((700, [5, 333]), (40000, [3, 39990]), (150000, list(range(149000, 149040))), (5000, list(range(0, 5000, 7)))):
        x, s = masked(TYPES[dt], vocab, kept, mask, cuda_device)
        select_and_compare(x, s, 2)
        select_and_compare(x, s, 7)
    x, s = masked(TYPES[dt], 9000, [], mask, cuda_device)
    select_and_compare(x, s, 5)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("size", [7e5, 3e6, 1e10, 3e12, 1e20, 1e30])
def test_logits_far_from_zero(size, dt, cuda_device):
    """Masks that a threshold near zero does not catch, and rows that lie far from zero as a whole."""
    for sign in (1, -1):
        for vocab, kept in ((700, [5, 333]), (40000, [3, 39990]), (5000, list(range(0, 5000, 7)))):
            if sign < 0:                                   # masked by a large negative number
                x, s = masked(TYPES[dt], vocab, kept, -size, cuda_device)
                select_and_compare(x, s, 2)
                select_and_compare(x, s, 6)
            g = torch.Generator().manual_seed(vocab)       # all of the row there
            x = torch.full((1, 3, vocab), sign * size)
            x[0, 1] *= 1 - 0.5 * torch.rand(vocab, generator=g)
            x[0, 2, ::3] *= 0.75
            select_and_compare(x.to(TYPES[dt]).to(cuda_device), (-torch.rand((1, 3), generator=g)).to(cuda_device), 6)


def test_rows_across_the_border_of_the_two_exponentials(cuda_device):
    """Maxima that rise from tile to tile through 2^20 / log2(e) = 726817, up and down, half a unit a tile."""
    n = 60000
    ramp = 726817 + (torch.arange(n) // 4096 - 7).float() * 0.5
    x = torch.stack((ramp, ramp.flip(0), -ramp, -ramp.flip(0)))[None]
    for at in (0, 5000, 59000):
        y = x.clone()
        y[:, :, at] = y.amax(-1) + 0.25
        select_and_compare(y.to(cuda_device), torch.tensor([[-1.0, -1.25, -1.5, -1.75]], device=cuda_device), 5)


def test_sums_of_very_many_values(cuda_device):
    """Thirty-two rows of 16.8 M equal logits with a few larger ones, one to a thread and part: a thread adds
    thousands of values, always with the same rounding.  Of a sum of positive numbers: exponentials 2^-21, 48
    roundings in fp32 (32 tiles and the 16 values of one) 2^-18.4, fp64 above that, the part's sum as fp32 2^-24."""
    from cats_b200 import ops

    parts, tiles = 6, 683
    vocab = 4096 * parts * tiles
    low = (-0.5 - torch.arange(32) * 0.17).half()          # of each beam
    x = low.to(cuda_device).view(1, 32, 1).expand(1, 32, vocab).contiguous()
    first = (torch.arange(parts)[:, None] * (4096 * tiles) + torch.arange(256) * 8).view(-1)
    x[:, :, first.to(cuda_device)] = 0
    x[:, :, 0] = 1
    lse = torch.log(torch.e + (len(first) - 1) + (vocab - len(first)) * torch.exp(low.double()))
    scores = (lse - 1).float().view(1, 32)                 # every beam's best comes out near zero
    got = ops.beam_select(x, scores.to(cuda_device), 32)
    rows = got[1].view(-1).long().cpu()
    want = (scores.double().view(-1) + 1 - lse)[rows]
    assert sorted(rows.tolist()) == list(range(32)) and int(got[2].abs().max()) == 0
    assert float((got[0].double().view(-1).cpu() - want).abs().max()) <= 2.0 ** -18 + 2.0 ** -21 + 2.0 ** -23
