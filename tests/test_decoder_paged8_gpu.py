"""The decode loop over the paged 8-bit cache, and beam search, on the GPU.

The reference for a step is the static-cache decoder whose cache is filled with the very values that
the 8-bit cache stands for, so that what is compared is attention and bookkeeping, not the loss of
eight bits.  (It keeps the current token's own keys and values unrounded: a share of 1 / positions of
the weights that is off by at most 2^-4, far below the bound.)"""
import numpy as np
import pytest
import torch

from oracle import cats_oracle as O

pytestmark = pytest.mark.gpu

SMALL = dict(hidden_size=512, intermediate_size=1408, num_attention_heads=4, vocab_size=1500, head_dim=128)


def to_np(t):
    return t.detach().float().cpu().numpy()


def small_model(dev, dtype=torch.float32, kv=2, layers=2):
    from cats_b200 import decoder as D

    return D.build_random_model("mistral", dtype, dev, layers=layers, seed=3, num_key_value_heads=kv, **SMALL)


@pytest.mark.parametrize("dtype,kv,page", [(torch.float32, 2, 16), (torch.float16, 1, 64), (torch.bfloat16, 4, 32)])
def test_steps_over_the_paged_cache_follow_the_static_cache(dtype, kv, page, cuda_device):
    from cats_b200 import decoder as D

    model = small_model(cuda_device, dtype, kv)
    ids = torch.randint(0, SMALL["vocab_size"], (3, 40), device=cuda_device)
    ref = D.CatsDecoder(model, 3, 200, mlp="dense")
    dec = D.CatsDecoder(model, 3, 200, mlp="dense", cache="paged8", page=page)
    l0, l1 = ref.prefill(ids), dec.prefill(ids)
    assert torch.equal(l0, l1)                             # the prompt's own attention is the same
    for step in range(30):                                 # crosses pages
        n = 40 + step
        for l in range(2):
            for b in range(3):
                k, v = dec.kv.read(l, b)
                assert k.shape[1] == n
                ref.kc[l][b, :, :n], ref.vc[l][b, :, :n] = k.to(dtype), v.to(dtype)
        ref.tok.copy_(dec.tok)
        ref._step(D.BUCKET)
        dec._step(D.BUCKET)
        assert O.rel_l2(to_np(dec.logits), to_np(ref.logits)) <= 3e-2, step
    dec.kv.check()
    assert dec.kv.lens.tolist() == [70] * 3


def test_the_cats_mlp_runs_with_the_paged_cache_eager_and_captured(cuda_device):
    from cats_b200 import decoder as D

    model = small_model(cuda_device, torch.float16)
    thr = D.calibrate(model, 0.5, n_prompts=2, prompt_len=64)
    ids = torch.randint(0, SMALL["vocab_size"], (1, 250), device=cuda_device)
    runs = []
    for use_graph in (False, True):
        dec = D.CatsDecoder(model, 1, 300, mlp="cats", thresholds=thr, cache="paged8")
        dec.prefill(ids)
        toks, tps, logs = dec.decode(12, use_graph=use_graph, keep_logits=True)
        runs.append((toks, torch.stack(logs)))
        assert tps > 0 and dec.kv.lens.tolist() == [262]
        dec.kv.check()
        if use_graph:
            assert len(dec.graphs) == 1                    # one graph for all positions
    assert O.rel_l2(to_np(runs[1][1][:4]), to_np(runs[0][1][:4])) <= 2e-2
    assert torch.equal(runs[0][0][:, :2], runs[1][0][:, :2])


def forced_score(model, ids, tokens):
    """Summed log-probability of ``tokens`` (n) after the prompt ``ids`` (1, T), one sequence alone."""
    from cats_b200 import decoder as D

    dec = D.CatsDecoder(model, 1, 200, mlp="dense", cache="paged8", page=16)
    logits, total = dec.prefill(ids), 0.0
    for t in tokens.tolist():
        total += float(torch.log_softmax(logits[0].double(), -1)[t])
        dec.tok.fill_(t)
        dec._forward(dec.max_len)
        logits = dec.logits
    return total


def test_beam_search_scores_are_those_of_its_sequences(cuda_device):
    """fp32: the scores of the returned sequences equal those of each sequence decoded alone (noise of
    fp32 products in another batch, and now and then a key one code off: below 1e-2 in the sum)."""
    from cats_b200 import decoder as D

    model = small_model(cuda_device)
    ids = torch.randint(0, SMALL["vocab_size"], (2, 21), device=cuda_device)
    found = []
    for use_graph in (False, True):
        dec = D.CatsDecoder(model, 6, 200, mlp="dense", cache="paged8", page=16)
        tokens, scores = dec.beam_search(ids, 3, 14, length_penalty=0.0, use_graph=use_graph)
        dec.kv.check()
        assert tokens.shape == (2, 3, 14) and scores.shape == (2, 3)
        assert (scores[:, :-1] >= scores[:, 1:]).all()
        assert len({tuple(t) for t in tokens.view(6, 14).tolist()}) == 6 or not torch.equal(ids[0], ids[1])
        found.append((tokens, scores))
        # every page is held by somebody, and shared pages are counted
        held = torch.zeros_like(dec.kv.refs)
        t = dec.kv.table[dec.kv.table >= 0].long()
        held.index_add_(0, t, torch.ones_like(t, dtype=torch.int32))
        assert torch.equal(held, dec.kv.refs)
        assert int((dec.kv.refs > 0).sum()) < int((dec.kv.table >= 0).sum())
    assert torch.allclose(found[0][1], found[1][1], atol=1e-2)
    tokens, scores = found[0]
    for p in range(2):
        assert len({tuple(t) for t in tokens[p].tolist()}) == 3
        for b in range(3):
            assert abs(forced_score(model, ids[p:p + 1], tokens[p, b]) - float(scores[p, b])) <= 1e-2


def test_one_beam_is_greedy_decoding(cuda_device):
    from cats_b200 import decoder as D

    model = small_model(cuda_device)
    ids = torch.randint(0, SMALL["vocab_size"], (2, 17), device=cuda_device)
    dec = D.CatsDecoder(model, 2, 100, mlp="dense", cache="paged8")
    tokens, _ = dec.beam_search(ids, 1, 9, use_graph=False)
    dec.prefill(ids)
    greedy, _, _ = dec.decode(8, use_graph=False)
    assert torch.equal(tokens[:, 0], greedy)


def test_beams_that_end_keep_their_score(cuda_device):
    from cats_b200 import decoder as D

    model = small_model(cuda_device)
    ids = torch.randint(0, SMALL["vocab_size"], (1, 12), device=cuda_device)
    dec = D.CatsDecoder(model, 4, 100, mlp="dense", cache="paged8")
    free, _ = dec.beam_search(ids, 4, 8)
    eos = int(free[0, 0, 2])                               # what the best beam says third
    tokens, scores = dec.beam_search(ids, 4, 8, eos=eos, length_penalty=0.0)
    for b in range(4):
        t = tokens[0, b].tolist()
        if eos in t:
            n = t.index(eos) + 1
            assert set(t[n:]) <= {eos}
            alone = forced_score(model, ids, tokens[0, b, :n])
        else:
            alone = forced_score(model, ids, tokens[0, b])
        assert abs(alone - float(scores[0, b])) <= 1e-2
    assert any(eos in t for t in tokens[0].tolist())
    half, _ = dec.beam_search(ids, 4, 8, eos=eos, length_penalty=1.0)
    assert half.shape == (1, 4, 8)


def test_refusals(cuda_device):
    from cats_b200 import decoder as D

    model = small_model(cuda_device)
    ids = torch.randint(0, SMALL["vocab_size"], (2, 12), device=cuda_device)
    static = D.CatsDecoder(model, 4, 100, mlp="dense")
    paged = D.CatsDecoder(model, 4, 100, mlp="dense", cache="paged8")
    for call in (lambda: static.beam_search(ids, 2, 4), lambda: paged.beam_search(ids, 3, 4), lambda: paged.beam_search(ids, 2, 0),
                 lambda: paged.beam_search(ids, 2, 1000), lambda: D.CatsDecoder(model, 1, 100, cache="8bit"),
                 lambda: paged.beam_search(ids, 2, 4, eos=SMALL["vocab_size"])):
        with pytest.raises(RuntimeError):
            call()
    assert np.isfinite(to_np(paged.beam_search(ids, 2, 1)[1])).all()
