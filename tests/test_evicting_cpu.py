"""The evicting KV cache's and the sampling's oracle against hand-made values, and the refusals of their
entry points that need no GPU (nothing is launched: every call is refused by its arguments)."""
import ctypes

import numpy as np
import pytest

from oracle import kve

FAKE = 0x10000          # an aligned address that no refused call touches


def cache(pkg, **over):
    c = dict(keys=FAKE, values=FAKE, weights=FAKE, positions=FAKE, block_table=FAKE, turns=FAKE, num_sequences=2,
             max_pages=8, page_size=16, num_pages=16, num_kv_heads=2, head_dim=128, dtype=0, rotary_dim=128,
             interleaved=0)
    c.update(over)
    return pkg._lib.KVECache(**c)


BAD = [dict(head_dim=96), dict(head_dim=0), dict(page_size=24), dict(page_size=8), dict(page_size=65536),
       dict(num_sequences=0), dict(max_pages=0), dict(num_kv_heads=0), dict(num_kv_heads=65536), dict(num_pages=0),
       dict(rotary_dim=24), dict(rotary_dim=144), dict(rotary_dim=-16), dict(turns=None), dict(keys=FAKE + 4),
       dict(values=FAKE + 8), dict(dtype=3), dict(dtype=4), dict(dtype=-1), dict(max_pages=1 << 27),
       dict(max_pages=(0x7ff00000 >> 4) + 1)]


@pytest.mark.parametrize("over", BAD, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_bad_cache_is_refused(pkg, over):
    L, c = pkg.lib(), cache(pkg, **over)
    ref = ctypes.addressof(c)
    assert L.ojasx_kve_append_device(ref, None, 0, 0, 0, None, FAKE, 256, 128, FAKE, 256, 128, None, 2, FAKE, None,
                                     None, None) == -3
    assert L.ojasx_kve_decode_workspace(ref, 4, 0, 1) == -3
    assert L.ojasx_kve_decode_device(ref, FAKE, 4, FAKE, 0, -1.0, 1, FAKE, FAKE, 1 << 40, None) == -3
    assert L.ojasx_kve_evict_workspace(ref, 8, 0) == -3
    assert L.ojasx_kve_evict_device(ref, FAKE, 8, 0, 0, 0, FAKE, 1 << 40, None) == -3
    assert L.ojasx_get_last_error()


def test_the_most_slots_are_taken(pkg):
    """Kernels step past a sequence's end by some thousands of slots, in 32 bits."""
    L, c = pkg.lib(), cache(pkg, max_pages=0x7ff00000 >> 4, num_sequences=1)
    assert L.ojasx_kve_decode_workspace(ctypes.addressof(c), 4, 0, 0) > 0
    assert L.ojasx_kve_evict_workspace(ctypes.addressof(c), 8, 0) > 0


def test_null_buffers_are_refused(pkg):
    L = pkg.lib()
    for name in ("keys", "values", "weights", "positions", "block_table"):
        ref = cache(pkg, **{name: None})
        assert L.ojasx_kve_decode_workspace(ctypes.addressof(ref), 4, 0, 1) == -1
        assert L.ojasx_kve_evict_workspace(ctypes.addressof(ref), 4, 0) == -1
    assert L.ojasx_kve_decode_workspace(None, 4, 0, 1) == -1 and L.ojasx_kve_evict_workspace(None, 4, 0) == -1


def test_bad_calls_are_refused(pkg):
    L, c = pkg.lib(), cache(pkg)
    ref = ctypes.addressof(c)

    def append(n=2, cu=None, k=FAKE, v=FAKE, q=None, heads=0, qo=None, ts=256, hs=128, start=FAKE):
        return L.ojasx_kve_append_device(ref, q, ts, hs, heads, qo, k, ts, hs, v, ts, hs, None, n, start, None, cu, None)

    assert append(n=3) == -3 and append(n=-1, cu=FAKE) == -3 and append(n=(1 << 25) + 1, cu=FAKE) == -3
    assert append(k=None) == -1 and append(v=None) == -1 and append(start=None) == -1
    assert append(heads=4) == -1 and append(heads=4, q=FAKE) == -1 and append(heads=-1) == -3
    assert append(ts=257) == -3 and append(hs=130) == -3 and append(k=FAKE + 8) == -3 and append(ts=-256) == -3
    assert append(heads=4, q=FAKE, qo=FAKE + 2) == -3
    assert append(n=0, cu=FAKE) == 0                                  # nothing to do

    need = L.ojasx_kve_decode_workspace(ref, 4, 0, 1)
    assert need > L.ojasx_kve_decode_workspace(ref, 4, 0, 0) > 0      # without weights no scores are kept
    assert need > L.ojasx_kve_decode_workspace(ref, 4, 20, 1) > 0     # and shorter sequences keep fewer

    def decode(heads=4, q=FAKE, held=FAKE, most=0, scale=-1.0, out=FAKE, ws=FAKE, n=need):
        return L.ojasx_kve_decode_device(ref, q, heads, held, most, scale, 1, out, ws, n, None)

    assert decode(heads=3) == -3 and decode(heads=0) == -3 and decode(heads=258) == -3 and decode(most=-1) == -3
    assert decode(q=None) == -1 and decode(held=None) == -1 and decode(out=None) == -1
    assert decode(q=FAKE + 8) == -3 and decode(out=FAKE + 4) == -3
    assert decode(n=need - 1) == -3 and decode(ws=None) == -3 and decode(ws=FAKE + 4) == -3
    for s in (float("nan"), float("inf"), 3e38):
        assert decode(scale=s) == -3 and b"scale" in L.ojasx_get_last_error()

    need = L.ojasx_kve_evict_workspace(ref, 8, 0)

    def evict(budget=8, sink=2, recent=2, most=0, held=FAKE, ws=FAKE, n=need):
        return L.ojasx_kve_evict_device(ref, held, budget, sink, recent, most, ws, n, None)

    assert evict(budget=0) == -3 and evict(sink=-1) == -3 and evict(recent=-1) == -3 and evict(most=-1) == -3
    assert evict(sink=5, recent=4) == -3 and evict(sink=2**31 - 1, recent=2**31 - 1) == -3 and evict(held=None) == -1
    assert evict(ws=None) == -3 and evict(n=need - 1) == -3 and evict(ws=FAKE + 4) == -3
    # no sequence can hold more than the budget: nothing to do
    assert evict(budget=128) == 0 and evict(budget=100, most=100) == 0


def test_calls_past_a_launch_are_refused(pkg):
    L = pkg.lib()
    big = cache(pkg, num_sequences=1 << 20, num_kv_heads=64)
    assert L.ojasx_kve_decode_workspace(ctypes.addressof(big), 64, 0, 1) == -3
    assert L.ojasx_kve_evict_workspace(ctypes.addressof(big), 8, 0) == -3


def test_workspace_counts_past_32_bits(pkg):
    """Scores of many long sequences: bytes past 2^32."""
    L = pkg.lib()
    big = cache(pkg, num_sequences=64, max_pages=1 << 16, num_pages=1 << 20, num_kv_heads=8)
    assert L.ojasx_kve_decode_workspace(ctypes.addressof(big), 32, 0, 1) > 64 * 32 * (1 << 20) * 4 > 1 << 32


def test_python_refusals(pkg):
    import torch
    from importlib import import_module
    lc, dec = import_module(pkg.__name__ + ".long_context"), import_module(pkg.__name__ + ".decoder")
    for kw in (dict(head_dim=96), dict(page_size=20), dict(page_size=8), dict(num_sequences=0), dict(max_pages=0),
               dict(num_pages=0), dict(rotary_dim=24), dict(rotary_dim=256), dict(rope_theta=None, rotary_dim=64),
               dict(rope_theta=0.0), dict(rope_theta=float("nan")), dict(inv_freq=torch.ones(63))):
        with pytest.raises(ValueError):
            # as far as a GPU is needed for nothing
            lc.PagedEvictingKVCache(2, **kw)
    for dtype in (torch.float64, torch.int8):
        with pytest.raises(TypeError):
            lc.PagedEvictingKVCache(2, dtype=dtype)
    with pytest.raises(RuntimeError):
        lc.PagedEvictingKVCache(2, device="cpu")
    with pytest.raises(RuntimeError):
        dec.sample_tokens(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError):
        dec.sample_tokens(torch.zeros(8), torch.zeros(1))


def test_bad_sampling_is_refused(pkg):
    L = pkg.lib()
    S = pkg._lib.Sampling
    need = L.ojasx_sample_workspace(2, 100)
    assert need > 0 and L.ojasx_sample_workspace(0, 100) == 0
    for rows, vocab in ((-1, 100), (2, 0), (2, -5), (2, (1 << 22) + 1), (0x7fffffff, 100000), (1 << 22, 100)):
        assert L.ojasx_sample_workspace(rows, vocab) == -3

    def call(logits=FAKE, dtype=0, rows=2, vocab=100, stride=100, u=FAKE, tokens=FAKE, ws=FAKE, n=need, s=None, **kw):
        s = S(**{**dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0), **kw})
        return L.ojasx_sample_device(logits, dtype, rows, vocab, stride, u, ctypes.addressof(s), tokens, ws, n, None)

    assert call(dtype=3) == -3 and call(dtype=4) == -3 and call(rows=-1) == -3 and call(vocab=0) == -3
    assert call(logits=None) == -1 and call(u=None) == -1 and call(tokens=None) == -1
    assert call(stride=-1) == -3 and call(logits=FAKE + 2) == -3 and call(logits=FAKE + 1, dtype=1) == -3
    assert call(ws=None) == -3 and call(ws=FAKE + 8) == -3 and call(n=need - 1) == -3
    nan, inf = float("nan"), float("inf")
    for kw in (dict(temperature=-1.0), dict(temperature=nan), dict(temperature=inf), dict(temperature=1e300),
               dict(top_p=-0.1), dict(top_p=nan), dict(min_p=-0.1), dict(min_p=nan), dict(min_p=1.5)):
        assert call(**kw) == -3 and b"sampling" in L.ojasx_get_last_error()
    assert L.ojasx_sample_device(FAKE, 0, 2, 100, 100, FAKE, None, FAKE, FAKE, need, None) == -1
    assert call(rows=0, logits=None, ws=None, n=0) == 0


def test_oracle_eviction():
    w = np.array([5, 1, 3, 3, 0, 9, 2, 3], np.float32)
    pos = np.arange(8)
    assert kve.kept(w, pos, 4, 0, 0) == ([0, 2, 3, 5], [1], [5])                # of three threes the first two
    assert kve.kept(w, pos, 4, 0, 1) == ([0, 2, 5, 7], [1, 3], [5, 7])          # the newest stays
    assert kve.kept(w, pos, 4, 2, 0) == ([0, 1, 2, 5], [3], [5])                # the first two stay
    assert kve.kept(w, pos[::-1].copy(), 3, 1, 0)[0] == [0, 5, 7]               # positions, not slots
    w[5] = np.nan
    assert kve.kept(w, pos, 4, 0, 0)[0] == [0, 2, 3, 7]
    assert kve.kept(w, pos, 8, 0, 0)[1:] == ([], [])
    assert kve.kept(w, pos, 3, 0, 0, there=np.array([0, 1, 1, 1, 1, 1, 1, 1], bool))[0] == [2, 3, 7]


def test_oracle_draws():
    x = np.log(np.array([1.0, 4.0, 2.0, 1.0]))
    assert [kve.draw(x, u) for u in (0.0, 0.124, 0.126, 0.62, 0.63, 0.87, 0.88, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [kve.draw(x, u, k=2) for u in (0.0, 0.66, 0.67)] == [1, 1, 2]
    assert [kve.draw(x, u, k=3) for u in (0.0, 0.14, 0.15)] == [0, 0, 1]        # of two equal ones the first
    assert [kve.draw(x, u, p=0.5) for u in (0.0, 0.99)] == [1, 1]               # reached, not passed
    assert [kve.draw(x, u, p=0.51) for u in (0.0, 0.99)] == [1, 2]
    assert [kve.draw(x, u, m=0.3) for u in (0.0, 0.99)] == [1, 2]
    assert kve.draw(x, 0.99, T=0) == 1 and kve.draw([1.0, np.nan], 0.5) == -1 and kve.draw([-np.inf] * 3, 0.5) == -1
    assert kve.draw([0.0, np.inf], 0.5) == -1 and kve.draw([0.0, -np.inf], 0.999) == 0


def test_bad_sampled_generation_is_refused(pkg):
    import torch
    dec = pkg.decoder
    call = pkg._lib.lib().ojasx_decoder_generate_sampled
    u, toks = (ctypes.c_float * 2)(0.1, 0.2), (ctypes.c_int * 2)()
    assert call(None, 0, 2, 0, u, 1.0, 0, 1.0, 0.0, toks, None) == -1
    assert call(FAKE, 0, 2, 0, None, 1.0, 0, 1.0, 0.0, toks, None) == -1
    assert call(FAKE, 0, 2, 0, u, 1.0, 0, 1.0, 0.0, None, None) == -1
    d = object.__new__(dec.LUTDecoder)
    d.cfg, d._h = dec.DecoderConfig(), None
    with pytest.raises(ValueError, match="uniform"):
        d.generate(0, 2, temperature=0.5)
    with pytest.raises(ValueError, match="uniform"):
        d.generate(0, 2, uniform=torch.zeros(3))
