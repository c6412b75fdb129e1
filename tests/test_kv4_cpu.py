"""The 4-bit KV cache's oracle against hand-made values, and the refusals of its entry points
that need no GPU (nothing is launched: every call is refused by its arguments)."""
import ctypes

import numpy as np
import pytest

from oracle import kv4

FAKE = 0x10000          # an aligned address that no refused call touches


def cache(pkg, **over):
    c = dict(k_codes=FAKE, v_codes=FAKE, k_steps=FAKE, v_steps=FAKE, block_table=FAKE, turns=FAKE,
             num_sequences=2, max_pages=8, sink_pages=1, page_size=16, num_pages=16, num_kv_heads=2,
             head_dim=128, group_size=32, rotary_dim=128, interleaved=0)
    c.update(over)
    return pkg._lib.KV4Cache(**c)


BAD = [dict(head_dim=96), dict(head_dim=64, group_size=128), dict(group_size=16), dict(page_size=24),
       dict(page_size=8), dict(page_size=65536), dict(num_sequences=0), dict(max_pages=1),
       dict(sink_pages=-1), dict(num_kv_heads=0), dict(num_pages=0), dict(rotary_dim=24),
       dict(rotary_dim=144), dict(turns=None), dict(k_codes=FAKE + 4)]


@pytest.mark.parametrize("over", BAD, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_bad_cache_is_refused(pkg, over):
    L, c = pkg.lib(), cache(pkg, **over)
    ref = ctypes.addressof(c)
    assert L.ojasx_kv4_append_device(ref, None, 0, 0, 0, None, FAKE, 256, 128, None, FAKE, 256, 128, 2, 0,
                                     FAKE, None, None) == -3
    assert L.ojasx_kv4_read_device(ref, FAKE, None, None, 2, FAKE, FAKE, 0, None) == -3
    assert L.ojasx_kv4_decode_workspace(ref, 4, 0) == -3
    assert L.ojasx_kv4_decode_device(ref, FAKE, 4, 0, FAKE, 0, -1.0, FAKE, FAKE, 1 << 30, None) == -3
    assert L.ojasx_get_last_error()


def test_null_buffers_are_refused(pkg):
    L = pkg.lib()
    for name in ("k_codes", "v_codes", "k_steps", "v_steps", "block_table"):
        c = cache(pkg, **{name: None})
        assert L.ojasx_kv4_decode_workspace(ctypes.addressof(c), 4, 0) == -1
    assert L.ojasx_kv4_decode_workspace(None, 4, 0) == -1


def test_bad_calls_are_refused(pkg):
    L, c = pkg.lib(), cache(pkg)
    ref = ctypes.addressof(c)

    def append(n=2, dtype=0, cu=None, k=FAKE, v=FAKE, q=None, heads=0, qo=None, ko=None, ts=256, hs=128,
               start=FAKE):
        return L.ojasx_kv4_append_device(ref, q, ts, hs, heads, qo, k, ts, hs, ko, v, ts, hs, n, dtype, start,
                                         cu, None)

    assert append(n=3) == -3 and append(n=-1, cu=FAKE) == -3          # one token a sequence without cu
    assert append(dtype=3) == -3 and append(dtype=4) == -3
    assert append(k=None) == -1 and append(v=None) == -1 and append(start=None) == -1
    assert append(heads=4) == -1 and append(heads=4, q=FAKE) == -1 and append(heads=-1) == -3
    assert append(ts=257) == -3 and append(hs=130) == -3 and append(k=FAKE + 8) == -3
    assert append(ko=FAKE + 2) == -3 and append(ts=-256) == -3
    assert append(n=0, cu=FAKE) == 0                                  # nothing to do
    assert L.ojasx_kv4_read_device(ref, FAKE, None, None, 3, FAKE, FAKE, 0, None) == -3
    assert L.ojasx_kv4_read_device(ref, FAKE, FAKE, None, 0, FAKE, FAKE, 0, None) == 0
    assert L.ojasx_kv4_read_device(ref, None, FAKE, None, 3, FAKE, FAKE, 0, None) == -1
    assert L.ojasx_kv4_read_device(ref, FAKE, FAKE, None, 3, FAKE, FAKE, 3, None) == -3
    need = L.ojasx_kv4_decode_workspace(ref, 4, 0)
    decode = lambda heads=4, dtype=0, q=FAKE, ws=FAKE, n=need: L.ojasx_kv4_decode_device(  # noqa: E731
        ref, q, heads, dtype, FAKE, 0, -1.0, FAKE, ws, n, None)
    assert decode(heads=3) == -3 and decode(heads=0) == -3 and decode(dtype=3) == -3 and decode(q=None) == -1
    assert decode(n=need - 1) == -3 and decode(ws=None) == -3 and decode(ws=FAKE + 4) == -3


def test_workspace_covers_the_runs(pkg):
    """(runs + sequences) x query heads x (head_dim + 2) floats; no more runs than tiles."""
    L = pkg.lib()
    big = cache(pkg, num_sequences=1, max_pages=2048, num_pages=2048)
    row = 4 * 130 * 4
    need = [L.ojasx_kv4_decode_workspace(ctypes.addressof(big), 4, m) for m in (0, 64, 65, 1 << 30)]
    assert all(n > 0 and n % row == 0 for n in need)
    assert need[1] == 2 * row and need[2] == 3 * row and need[0] == need[3]


def test_python_refusals(pkg):
    from importlib import import_module
    lc = import_module(pkg.__name__ + ".long_context")
    for kw in (dict(head_dim=96), dict(group_size=48), dict(head_dim=64, group_size=128), dict(page_size=20),
               dict(page_size=8), dict(num_sequences=0), dict(max_resident_pages=2, sink_pages=2),
               dict(num_pages=0), dict(rotary_dim=24), dict(rotary_dim=256), dict(rope_theta=None, rotary_dim=64)):
        with pytest.raises(ValueError):
            lc.PagedInt4KVCache(2, **kw)
    with pytest.raises(RuntimeError):
        lc.PagedInt4KVCache(2, device="cpu")


def test_oracle_held_values():
    x = np.zeros((4, 32), np.float32)
    x[0] = np.arange(32) % 16 - 3            # lo -3, s 1: exact
    x[1] = 7.25                              # a constant group: lo alone
    x[2, 5] = np.inf
    x[3, :16] = np.arange(16) + 0.5          # lo 0, s fp16(15.5 / 15)
    h = kv4.held(x, 32)
    assert np.array_equal(h[0], x[0]) and np.array_equal(h[1], x[1]) and np.isnan(h[2]).all()
    s = float(np.float16(np.float32(15.5 / 15)))
    assert np.array_equal(h[3, :16], s * np.clip(np.rint(x[3, :16].astype(np.float64) / s), 0, 15))
    r = np.random.default_rng(0).normal(size=(50, 64)).astype(np.float32)
    # half a step, and what fp16 rounds off lo and s
    span = r.max() - r.min()
    assert np.abs(kv4.held(r, 32) - r).max() <= span / 30 * (1 + 2 ** -10) + np.abs(r).max() * 2 ** -10


def test_oracle_residents_and_rotation():
    assert list(kv4.resident(5, 2, 3, 1)) == [0, 1, 2, 3, 4]
    assert list(kv4.resident(7, 2, 3, 1)) == [0, 1, 4, 5, 6]      # page 1 (tokens 2, 3) is gone
    x = np.random.default_rng(1).normal(size=(3, 2, 16))
    f = kv4.inv_freq(16, 1e4)
    for inter in (False, True):
        y = kv4.rotate(x, [0, 1, 1000], f, inter)
        assert np.array_equal(y[0], x[0])
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-13)
    assert not np.allclose(kv4.rotate(x, [1] * 3, f), kv4.rotate(x, [1] * 3, f, True))


def test_prompt_attention_refusals(pkg):
    L = pkg.lib()

    def call(q=FAKE, k=FAKE, v=FAKE, ts=512, hs=128, dtype=0, nq=4, nk=4, H=4, Hkv=2, D=128, cu=FAKE, ck=FAKE,
             B=1, scale=0.1, out=FAKE):
        return L.ojasx_prompt_attention_device(q, ts, hs, k, ts, hs, v, ts, hs, dtype, nq, nk, H, Hkv, D, cu, ck,
                                               B, 1, scale, 0, out, None, None)

    assert call(dtype=3) == -3 and call(nq=-1) == -3 and call(nk=-1) == -3 and call(H=3) == -3
    assert call(Hkv=0) == -3 and call(D=0) == -3 and call(D=12) == -3 and call(D=264) == -3 and call(B=0) == -3
    assert call(scale=0.0) == -3 and call(scale=-1.0) == -3 and call(scale=float("inf")) == -3
    assert call(scale=float("nan")) == -3 and call(ts=514) == -3 and call(hs=-128) == -3
    assert call(q=FAKE + 8) == -3 and call(k=FAKE + 4) == -3 and call(out=FAKE + 2) == -3
    assert call(q=None) == -1 and call(k=None) == -1 and call(cu=None) == -1 and call(ck=None) == -1
    assert call(out=None) == -1 and call(nq=0, q=None) == 0
    assert L.ojasx_get_last_error()


def test_launches_past_the_grid_are_refused(pkg):
    """More tokens than a grid of fewer than 2^32 threads, or than row numbers of 32 bits, take."""
    L, c = pkg.lib(), cache(pkg)
    ref = ctypes.addressof(c)
    for n in ((1 << 25) + 1, 0x7fffffff):
        assert L.ojasx_kv4_append_device(ref, None, 0, 0, 0, None, FAKE, 256, 128, None, FAKE, 256, 128, n, 0,
                                         FAKE, FAKE, None) == -3
        assert L.ojasx_kv4_read_device(ref, FAKE, FAKE, None, n, FAKE, FAKE, 0, None) == -3
    prompt = lambda nq, nk, H, B: L.ojasx_prompt_attention_device(  # noqa: E731
        FAKE, 64, 8, FAKE, 64, 8, FAKE, 64, 8, 0, nq, nk, H, H, 8, FAKE, FAKE, B, 1, 0.5, 0, FAKE, None, None)
    assert prompt(0x7fffffff, 1, 1, 1) == -3 and prompt(1, 0x7fffffff, 1, 1) == -3
    assert prompt(1 << 26, 1, 64, 1) == -3          # 2^19 blocks of rows by 64 heads: 2^25 workgroups
    assert prompt(1, 1, 8, 1 << 22) == -3           # every sequence has a workgroup for each head


ROWS = [  # shape, strides: torch calls all of them contiguous, or takes them for rows of 16 bytes
    ((1, 4, 64), (259, 64, 1)), ((7, 1, 64), (64, 1, 1)), ((1, 1, 64), (3, 5, 1)), ((1, 4, 64), (0, 64, 1)),
    ((5, 1, 64), (72, 3, 1)), ((1, 3, 64), (1, 72, 1)), ((4, 2, 64), (128, 64, 1)), ((4, 2, 64), (200, 64, 1)),
    ((4, 2, 64), (259, 64, 1)), ((4, 2, 64), (128, 1, 2)), ((4, 2, 64), (0, 0, 1)), ((0, 2, 64), (259, 64, 1)),
    ((2, 0, 64), (259, 1, 1)),
]


@pytest.mark.parametrize("shape,strides", ROWS, ids=str)
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("es", [2, 4])
def test_aligned_rows_of_any_strides(pkg, shape, strides, offset, es):
    """Rows for a kernel: 16-byte aligned, strides of dimensions of one entry too, the same values."""
    import torch
    from importlib import import_module
    lc = import_module(pkg.__name__ + ".long_context")
    dtype = torch.float32 if es == 4 else torch.bfloat16
    base = torch.arange(2048 + offset).to(dtype)
    t = base.as_strided(shape, strides, offset)
    rows, at, ts, hs = lc._aligned_rows(t, es)
    assert torch.equal(rows, t) and at == rows.data_ptr()
    assert at % 16 == 0 and ts * es % 16 == 0 and hs * es % 16 == 0
    if t.numel():
        assert torch.equal(rows.as_strided(shape, (ts, hs, 1), rows.storage_offset()), t)


def test_scales_that_are_not_finite_are_refused(pkg):
    """NaN is no request for the default, and a scale whose product with log2(e) overflows fp32 makes
    every score an infinity or a NaN."""
    L, c = pkg.lib(), cache(pkg)
    ref = ctypes.addressof(c)
    need = L.ojasx_kv4_decode_workspace(ref, 4, 0)
    for s in (float("nan"), float("inf"), 3e38):
        assert L.ojasx_kv4_decode_device(ref, FAKE, 4, 0, FAKE, 0, s, FAKE, FAKE, need, None) == -3
        assert b"scale" in L.ojasx_get_last_error()
        assert L.ojasx_prompt_attention_device(FAKE, 512, 128, FAKE, 512, 128, FAKE, 512, 128, 0, 4, 4, 4, 4, 128, FAKE,
                                               FAKE, 1, 1, s, 0, FAKE, None, None) == -3
        assert b"scale" in L.ojasx_get_last_error()


def test_frequencies_that_are_not_finite_are_refused(pkg):
    """They would rotate every key into NaN, which the cache then holds."""
    import torch
    from importlib import import_module
    lc = import_module(pkg.__name__ + ".long_context")
    for kw in (dict(rope_theta=0.0), dict(rope_theta=-1e4), dict(rope_theta=float("nan")), dict(rope_theta=float("inf")),
               dict(inv_freq=torch.full((64,), float("nan"))), dict(inv_freq=[float("inf")] + [0.0] * 63),
               dict(inv_freq=torch.ones(63))):
        with pytest.raises(ValueError):
            lc.PagedInt4KVCache(2, **kw)


def test_no_kv_heads_are_refused(pkg):
    """0 kv heads are not the default."""
    from importlib import import_module
    lc = import_module(pkg.__name__ + ".long_context")
    with pytest.raises(ValueError):
        lc.PackedPromptAttention(4, 0, 64)
    assert lc.PackedPromptAttention(4, None, 64).num_kv_heads == 4
