"""Paged 8-bit cache and beam selection without a GPU: refusals of the C ABI and of the Python front
end, and the oracle's own arithmetic.  Nothing is launched."""
import ctypes

import numpy as np
import pytest
import torch

from cats_b200 import _lib, kv8, ops
from oracle import kv8_oracle as K


@pytest.fixture(scope="module")
def buf():
    raw = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(raw) + 15) // 16 * 16
    yield p
    del raw


def cache_of(p, **over):
    f = dict(codes=p, scales=p, table=p, lens=p, refs=p, status=p, n_layers=2, n_pages=8, n_seqs=4, max_pages=4,
             n_kv_heads=2, page=16, head_dim=64)
    f.update(over)
    return ctypes.byref(_lib.Kv8(*[f[n] for n, _ in _lib.Kv8._fields_]))


@pytest.mark.parametrize("over,status", [
    (dict(codes=None), -4), (dict(scales=None), -4), (dict(table=None), -4), (dict(lens=None), -4),
    (dict(refs=None), -4), (dict(status=None), -4), (dict(page=48), -9), (dict(page=8), -9),
    (dict(head_dim=80), -9), (dict(head_dim=256), -9), (dict(n_seqs=0), -9), (dict(n_seqs=1025), -9),
    (dict(n_pages=0), -9), (dict(max_pages=0), -9), (dict(n_layers=0), -9), (dict(n_kv_heads=0), -9),
    (dict(max_pages=1 << 28), -9)])
def test_bad_caches_are_refused_by_every_entry_point(over, status, buf):
    L, c, big = _lib.lib(), cache_of(buf, **over), 1 << 30
    assert L.cats_kv8_grow(c, None, 1, None) == status
    assert L.cats_kv8_append(c, 0, buf, 512, None, 4, None, None, 0, buf, 4, 1, None) == status
    assert L.cats_kv8_attend(c, 0, buf, 256, None, 4, 4, 0.1, buf, buf, big, 1, None) == status
    assert L.cats_kv8_reorder(c, buf, buf, big, None) == status
    assert L.cats_kv8_compact(c, buf, buf, big, None) == status
    assert L.cats_kv8_grow(None, None, 1, None) == -4


def test_misaligned_codes(buf):
    assert _lib.lib().cats_kv8_grow(cache_of(buf, codes=buf + 8), None, 1, None) == -3


def test_bad_steps_are_refused(buf):
    L, c, big = _lib.lib(), cache_of(buf), 1 << 30
    ap = lambda layer=0, qkv=buf, ld=512, n=4, cos=None, sin=None, rope=0, q=buf, nh=4, dt=1: L.cats_kv8_append(  # noqa: E731
        c, layer, qkv, ld, None, n, cos, sin, rope, q, nh, dt, None)
    assert L.cats_kv8_grow(c, None, 0, None) == -9
    assert ap(dt=7) == -1
    assert ap(layer=2) == -9 and ap(layer=-1) == -9
    assert ap(qkv=None) == -4 and ap(cos=buf) == -4 and ap(sin=buf) == -4
    assert ap(cos=buf, sin=buf, rope=63) == -9                 # the cache takes 64 positions
    assert ap(ld=511) == -9 and ap(n=3) == -9 and ap(n=0) == -9 and ap(nh=3) == -9 and ap(nh=0) == -9
    assert ap(qkv=buf + 8) == -3 and ap(ld=514) == -3 and ap(q=buf + 8) == -3
    assert ap(cos=buf + 2, sin=buf, rope=64) == -3
    at = lambda layer=0, q=buf, ld=256, n=4, nh=4, scale=0.1, out=buf, ws=buf, nb=big, dt=1: L.cats_kv8_attend(  # noqa: E731
        c, layer, q, ld, None, n, nh, scale, out, ws, nb, dt, None)
    assert at(dt=3) == -1 and at(layer=5) == -9 and at(nh=5) == -9 and at(n=5) == -9 and at(ld=255) == -9
    assert at(q=None) == -4 and at(out=None) == -4 and at(ws=None) == -4
    assert at(q=buf + 4) == -3 and at(out=buf + 4) == -3 and at(ld=260) == -3
    assert at(scale=float("nan")) == -9 and at(scale=float("inf")) == -9
    assert at(nb=0) == -5
    assert L.cats_kv8_reorder(c, None, buf, big, None) == -4
    assert L.cats_kv8_reorder(c, buf, buf, 8, None) == -5
    assert L.cats_kv8_compact(c, None, buf, big, None) == -4
    assert L.cats_kv8_compact(c, buf, buf, 8, None) == -5


def test_bad_selections_are_refused(buf):
    L, big = _lib.lib(), 1 << 30
    sel = lambda x=buf, ld=100, sc=buf, done=None, n=2, beams=3, vocab=100, k=4, eos=-1, dt=1, nb=big: L.cats_beam_select(  # noqa: E731
        x, ld, sc, done, n, beams, vocab, k, eos, dt, buf, buf, buf, buf, buf, nb, None)
    assert sel(dt=5) == -1
    assert sel(n=0) == -9 and sel(beams=0) == -9 and sel(beams=33) == -9 and sel(k=0) == -9 and sel(k=33) == -9
    assert sel(vocab=1, k=4) == -9 and sel(ld=99) == -9
    assert sel(done=buf, eos=-1) == -9 and sel(done=buf, eos=100) == -9
    assert sel(x=None) == -4 and sel(sc=None) == -4
    assert sel(x=buf + 1) == -3 and sel(nb=16) == -5
    assert sel(n=65536, beams=1) == -9 and sel(vocab=(1 << 30) + 1, ld=1 << 31) == -9


def test_python_front_end_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv8.KVCache8(1, 4, 2, 64, 2, 64, device="cpu")
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        kv8.KVCache8.from_tensors(z(1, 4, 2, 2, 16, 64, dt=torch.uint8), z(1, 4, 2, 2, dt=torch.float32), z(2, 4), z(2), z(4))
    with pytest.raises(RuntimeError, match="codes"):
        kv8.KVCache8.from_tensors(z(1, 4, 2, 2, 16, 64), z(1, 4, 2, 2, dt=torch.float32), z(2, 4), z(2), z(4))


def test_the_decoders_paged_cache_needs_a_gpu():
    from transformers import MistralConfig, MistralForCausalLM

    from cats_b200 import decoder as D

    cfg = MistralConfig(hidden_size=64, intermediate_size=96, num_hidden_layers=1, num_attention_heads=2,
                        num_key_value_heads=1, vocab_size=64, max_position_embeddings=64)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.CatsDecoder(MistralForCausalLM(cfg), 1, 64, mlp="dense", cache="paged8")


def test_the_oracles_e4m3_is_the_format():
    """Every finite code is a fixed point, and values between two neighbours go to the nearer one,
    halves to the even code: torch's conversion says the same."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    fin = codes[torch.isfinite(codes)].double().numpy()
    assert np.array_equal(K.e4m3(fin), fin)
    pos = np.unique(np.abs(fin))
    mid = (pos[1:] + pos[:-1]) / 2
    x = np.concatenate([mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9), -mid])
    near = np.minimum(np.abs(x[:, None] - pos), np.abs(x[:, None] + pos)).min(1)
    got = K.e4m3(x)
    assert np.allclose(np.abs(got - x), near, rtol=0, atol=0)
    exact_halves = np.concatenate([mid, -mid])
    assert np.array_equal(K.e4m3(exact_halves), torch.from_numpy(exact_halves).to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(K.e4m3(np.inf)) and K.e4m3(1e9) == 448.0
    assert K.exponent(448.0) == 0 and K.exponent(448.0001) == 1 and K.exponent(0) == -24 and K.exponent(1e30) == 60


def test_the_oracles_bookkeeping_keeps_counts_and_tables_consistent():
    r = np.random.default_rng(0)
    c = K.Cache(np.zeros((1, 24, 2, 1, 16, 32)), np.zeros((1, 24, 2, 1)), -np.ones((5, 8)), np.zeros(5), np.zeros(24))
    for step in range(30):
        c.grow(r.integers(0, 12, 5) * (c.lens < 90))
        c.reorder(r.integers(-1, 5, 5))
        if step % 7 == 6:
            n = c.compact()
            assert (c.refs[:n] > 0).all() and (c.refs[n:] == 0).all()
        held = np.zeros(24, int)
        for b in range(5):
            for j in range(8):
                if j < -(-c.lens[b] // 16):
                    if c.table[b, j] >= 0:
                        held[c.table[b, j]] += 1
                else:
                    assert c.table[b, j] == -1
        assert np.array_equal(held, c.refs)
