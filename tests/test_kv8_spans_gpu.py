"""Spans of new tokens (``cu``) that do not fit: what does not fit is left out and recorded, whatever the numbers are."""
import pytest
import torch

from test_kv8_gpu import TYPES, cu_of, filled

pytestmark = pytest.mark.gpu

NUMBERS = [-2 ** 31, -5, 0, 1, 3, 2 ** 30, 2 ** 31 - 1]


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("heads", [2, 20, 100])
def test_attend_leaves_out_a_call_whose_spans_are_not_in_order(heads, n, cuda_device):
    c = filled(cuda_device, [20 + i for i in range(n)], 16, 1, 64)
    q = torch.randn((2 * n, heads, 64), device=cuda_device).half()
    for cu in ([0, 2, 1] + [4] * (n - 2), [0, 2 * n] * n, [-2 ** 31, 2 ** 31 - 1] * n, [5, 3, 2, 1] + [0] * n):
        out = torch.full_like(q, 7.0)
        c.attend(0, q, cu=ints(cu[:n + 1], c.device), out=out)
        assert (out == 7).all()
        with pytest.raises(RuntimeError, match="cu does not fit"):
            c.check()
        c.status.zero_()


def test_spans_that_are_too_many_to_count(cuda_device):
    """1024 sequences of which every other one claims all of the tokens: their units pass 32 bits."""
    from cats_b200.kv8 import KVCache8

    c = KVCache8(1, 4, 1024, 32768, 2, 64, 64, cuda_device)
    c.table.fill_(1)
    c.lens.fill_(32768)
    c.refs.fill_(1)
    q = torch.zeros((40000, 64, 64), dtype=torch.float16, device=cuda_device)
    out = torch.full_like(q, 7.0)
    c.attend(0, q, cu=ints([0, 40000] * 512 + [0], cuda_device), out=out)
    assert (out == 7).all()
    with pytest.raises(RuntimeError, match="cu does not fit"):
        c.check()


@pytest.mark.parametrize("dt", list(TYPES))
def test_a_span_beyond_the_tokens_is_left_out(dt, cuda_device):
    c = filled(cuda_device, [40, 30, 50], 16, 1, 64)
    q = torch.randn((4, 2, 64), device=cuda_device).to(TYPES[dt])
    want = c.attend(0, q, cu=cu_of([2, 0, 2], c.device))
    out = torch.full_like(q, 7.0)
    c.attend(0, q, cu=ints([0, 2, 2, 9], c.device), out=out)
    assert torch.equal(out[:2], want[:2]) and (out[2:] == 0).all()
    with pytest.raises(RuntimeError, match="cu does not fit"):
        c.check()


@pytest.mark.parametrize("page", [16, 64])
def test_append_and_grow_with_any_numbers(page, cuda_device):
    """Nothing is written that is not a row of the sequence whose span it is, and nothing read out of range."""
    g = torch.Generator().manual_seed(0)
    n = 70
    c = filled(cuda_device, [60] * n, page, 1, 32, spare=2)
    # every page but those of the last rows stays what it is: a span that fits has at most 20 tokens here
    first = sorted({int(p) for p in c.table[:, :40 // page].reshape(-1).tolist()})
    before = c.codes.view(torch.uint8)[:, first].clone()
    qkv = torch.randn((20, 3 * 32), generator=g).to(cuda_device)
    for trial in range(60):
        cu = [NUMBERS[int(i)] for i in torch.randint(0, len(NUMBERS), (n + 1,), generator=g)]
        if trial % 3 == 0:
            cu = sorted(cu)
        c.append(0, qkv, 1, cu=ints(cu, cuda_device))
        lens = c.lens.clone()
        c.grow(cu=ints(cu, cuda_device))
        assert int(c.lens.max()) <= c.max_len and int(c.lens.min()) >= 60
        c.lens.copy_(lens)
        c._state.zero_()
    assert torch.equal(c.codes.view(torch.uint8)[:, first], before)
