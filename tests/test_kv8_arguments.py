"""Arguments of another kind than the calls take are refused like all others (nothing is launched)."""
import pytest
import torch

from cats_b200 import kv8


def cache():
    """A cache's sizes on CPU tensors: enough for the checks, which come before any launch."""
    c = kv8.KVCache8.__new__(kv8.KVCache8)
    c.device, c.n_seqs, c.n_layers, c.n_kv_heads, c.head_dim, c.max_len = torch.device("cpu"), 2, 1, 1, 32, 64
    return c


@pytest.mark.parametrize("call", [
    lambda c: c.append(0, torch.tensor(1.0), 1), lambda c: c.attend(0, torch.tensor(1.0)), lambda c: c.append(0, [[1.0]], 1),
    lambda c: c.attend(0, None), lambda c: c.append(0, torch.zeros(2, 96), 1, q_out=[0.0] * 64),
    lambda c: c.attend(0, torch.zeros(2, 1, 32), out=[0.0] * 64), lambda c: c.attend(0, torch.zeros(2)), lambda c: c.append(0, torch.zeros(2), 1)])
def test_other_things_than_rows(call):
    with pytest.raises(RuntimeError, match="kv8"):
        call(cache())


@pytest.mark.gpu
def test_ended_beams_that_are_no_tensor(cuda_device):
    from cats_b200 import ops

    with pytest.raises(RuntimeError, match="done"):
        ops.beam_select(torch.zeros((1, 2, 8), device=cuda_device), torch.zeros((1, 2), device=cuda_device), 2, done=[False, True], eos=1)
