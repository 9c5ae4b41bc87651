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
