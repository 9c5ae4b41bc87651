"""The paged 8-bit cache at the ends of what a call may be: as many sequences as it takes, calls with more tokens than
their sequence holds, results written over the queries, calls of which most sequences have no part."""
import pytest
import torch

from test_kv8_gpu import TYPES, append_and_compare, attend_and_compare, cu_of, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [32, 33, 511, 512, 513, 1023, 1024])
def test_any_number_of_sequences(n, cuda_device):
    lens = [(37 * i) % 83 + (300 if i == n - 1 else 0) for i in range(n)]
    c = filled(cuda_device, lens, 16, 1, 32, spare=1)
    attend_and_compare(c, [min(1, k) for k in lens], 2, torch.float16)
    attend_and_compare(c, [min(3 if i % 5 else 9, k) for i, k in enumerate(lens)], 2, torch.bfloat16, seed=2)
    append_and_compare(c, [min(2, k) for k in lens], 2, torch.float32)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("hd,group,counts", [(64, 2, [3, 1, 8]), (64, 8, [4, 2, 9]), (128, 4, [20, 9, 30]), (32, 4, [9, 5, 20])])
def test_tokens_before_a_sequence_begins(hd, group, counts, dt, cuda_device):
    """More new tokens than the sequence has: those before its first position see nothing and give zeros."""
    c = filled(cuda_device, [2, 40, 7], 16, 2, hd)
    out = attend_and_compare(c, counts, group, TYPES[dt])
    assert out[:counts[0] - 2].abs().max() == 0 and out[counts[0] - 2:counts[0]].abs().max() > 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [9, 3, 40, 1], [70, 30, 90, 20]])
def test_results_over_the_queries(counts, dt, cuda_device):
    c = filled(cuda_device, [3000, 500, 90, 33], 64, 2, 128)
    q = torch.randn((sum(counts), 8, 128), device=cuda_device).to(TYPES[dt])
    cu = cu_of(counts, cuda_device)
    want = c.attend(0, q, cu=cu)
    assert c.attend(0, q, cu=cu, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("n,tokens", [(64, 100), (300, 40)])
def test_one_long_call_among_idle_sequences(n, tokens, dt, cuda_device):
    """Kernels are chosen by the mean number of rows; the tokens of one sequence are right with each."""
    lens = [20 + i % 60 for i in range(n)]
    lens[n // 2] = 700
    c = filled(cuda_device, lens, 16, 1, 64, spare=1)
    counts = [0] * n
    counts[n // 2] = tokens
    attend_and_compare(c, counts, 4, TYPES[dt])
    counts[3] = counts[n - 1] = 1
    attend_and_compare(c, counts, 4, TYPES[dt], seed=2)


def test_the_same_call_gives_the_same_bits(cuda_device):
    """Every kernel, split segments and not: the order of the joins does not depend on the run."""
    g = torch.Generator().manual_seed(0)
    for lens, counts, nkv, group, hd in (([640], [1], 32, 1, 128), ([512 + 130 * i for i in range(8)], [1] * 8, 8, 4, 128),
                                         ([1000 + 2900 * i for i in range(10)], [1] * 10, 8, 8, 128), ([2000, 6000], [200, 256], 8, 4, 128),
                                         ([900, 3000, 40], [5, 6, 7], 4, 4, 64), ([900, 3000, 40], [3, 4, 2], 4, 4, 96)):
        c = filled(cuda_device, lens, 64, nkv, hd)
        for dt in TYPES.values():
            q = torch.randn((sum(counts), nkv * group, hd), generator=g).to(dt).to(cuda_device)
            cu = cu_of(counts, cuda_device)
            first = c.attend(0, q, cu=cu)
            assert all(torch.equal(c.attend(0, q, cu=cu), first) for _ in range(20))
        c.check()
