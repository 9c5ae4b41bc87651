"""Selections of different sizes from several threads at once: each needs its own amount of shared memory
above 48 KB, and a launch must not lose it to another thread's."""
import threading

import pytest
import torch

from cats_b200 import _lib

pytestmark = pytest.mark.gpu


def test_selections_of_two_sizes_from_several_threads(cuda_device):
    """The C entry point in a loop on each thread (the interpreter's lock is free during a call)."""
    L, dev, jobs = _lib.lib(), cuda_device, []
    g = torch.Generator().manual_seed(0)
    for parts in (6, 5, 6, 5):                             # 64 KB and 56 KB in the joining kernel
        vocab = 4096 * parts
        x = torch.randn((1, 32, vocab), generator=g).half().to(dev)
        s = torch.randn((1, 32), generator=g).to(dev)
        outs = [torch.zeros(32, dtype=dt, device=dev) for dt in (torch.float32, torch.int32, torch.int64, torch.uint8)]
        nbytes = int(L.cats_beam_select_bytes(1, 32, vocab, 32))
        ws, st = torch.empty(nbytes, dtype=torch.uint8, device=dev), torch.cuda.Stream(dev)
        args = (x.data_ptr(), vocab, s.data_ptr(), None, 1, 32, vocab, 32, -1, _lib.F16, *(t.data_ptr() for t in outs), ws.data_ptr(),
                nbytes, st.cuda_stream)
        jobs.append((args, outs, st, (x, s, ws)))
    torch.cuda.synchronize(dev)
    bad, start = [], threading.Barrier(len(jobs))

    def work(args, st):
        torch.cuda.set_device(dev)
        start.wait()
        for i in range(20000):
            status = L.cats_beam_select(*args)
            if status:
                bad.append((status, L.cats_last_cuda_error().decode()))
                return
            if i % 200 == 199:
                st.synchronize()

    threads = [threading.Thread(target=work, args=(a, st)) for a, _, st, _ in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize(dev)
    assert not bad, bad
    for args, outs, st, _ in jobs:
        last = [t.clone() for t in outs]
        with torch.cuda.stream(st):
            assert L.cats_beam_select(*args) == 0
        st.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(last, outs)) and int(outs[1].max()) < 32
