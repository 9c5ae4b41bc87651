"""Searches over different caches that run at the same time, on different streams: they share nothing."""
import pytest
import torch

from test_kv8_gpu import filled, tables

pytestmark = pytest.mark.gpu


class Search:
    """A beam search of two prompts over one layer; ``step`` is grow, append, attend, select, reorder.
    Sequences long enough for their segments to be split between CTAs and joined."""

    def __init__(self, dev, seed):
        beams, vocab = 3, 9000
        self.c = filled(dev, [1500, 1500, 1500, 2600, 2600, 2600], 16, 2, 64, spare=60, seed=seed)
        g = torch.Generator().manual_seed(seed)
        self.w_in, self.w_out = (torch.randn(s, generator=g).to(dev) for s in ((vocab, 8 * 64), (4 * 64, vocab)))
        self.cos, self.sin = tables(self.c.max_len, 64, torch.float32, dev)
        self.tok = torch.arange(6, device=dev)
        self.scores = -torch.rand((2, beams), generator=g).to(dev)
        self.done = torch.zeros((2, beams), dtype=torch.bool, device=dev)
        self.shape = (2, beams, vocab)
        self.log = []

    def state(self):
        c = self.c
        return [c.codes.view(torch.uint8), c.scales, c.table, c.lens, c.refs, self.tok, self.scores, self.done]

    def step(self):
        from cats_b200 import ops

        self.c.grow(1)
        q = self.c.append(0, self.w_in[self.tok], 4, self.cos, self.sin)
        o = self.c.attend(0, q)
        s, rows, t, d = ops.beam_select((o.view(6, 256) @ self.w_out).view(self.shape), self.scores, 3, done=self.done, eos=3)
        self.c.reorder(rows.view(-1))
        for to, what in ((self.scores, s), (self.done, d), (self.tok, t.view(-1))):
            to.copy_(what)

    def capture(self):
        keep = [t.clone() for t in self.state()]
        self.step()
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.step()
        for t, k in zip(self.state(), keep):
            t.copy_(k)
        torch.cuda.synchronize()

    def record(self):
        self.log.append([t.clone() for t in self.state()])


def alone(dev, seed, steps):
    s = Search(dev, seed)
    for _ in range(steps):
        s.step()
        s.record()
    s.c.check()
    return s.log


@pytest.mark.parametrize("captured", [(False, False), (True, False), (True, True)])
def test_two_searches_at_the_same_time(captured, cuda_device):
    dev, steps = cuda_device, 12
    want = [alone(dev, s, steps) for s in (1, 2)]
    searches = [Search(dev, s) for s in (1, 2)]
    for s, as_graph in zip(searches, captured):
        if as_graph:
            s.capture()
    streams = [torch.cuda.Stream(dev) for _ in searches]
    torch.cuda.synchronize(dev)
    for st in streams:                                     # both queues fill before either starts
        with torch.cuda.stream(st):
            torch.cuda._sleep(20_000_000)
    for _ in range(steps):                                 # no wait of the host in here
        for s, st, as_graph in zip(searches, streams, captured):
            with torch.cuda.stream(st):
                s.graph.replay() if as_graph else s.step()
                s.record()
    torch.cuda.synchronize(dev)
    for s, w in zip(searches, want):
        s.c.check()
        for got, ref in zip(s.log, w):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
