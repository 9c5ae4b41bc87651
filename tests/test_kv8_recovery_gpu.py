"""The paged 8-bit cache after a step that could not have what it asked for: what was cached stays as
it was, and once there is room again the cache works on."""
import pytest
import torch

from test_kv8_gpu import filled

pytestmark = pytest.mark.gpu


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
