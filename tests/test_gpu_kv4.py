"""PagedInt4KVCache on the GPU: rotation, encoding, reading back and decode attention against
the fp64 oracle (oracle/kv4.py), at lengths, pages, masks and layouts where they can go wrong."""
import math

import numpy as np
import pytest

from oracle import kv4

pytestmark = pytest.mark.gpu

THETA = 1e6


@pytest.fixture(scope="module")
def lc(pkg):
    from importlib import import_module
    return import_module(pkg.__name__ + ".long_context")


def i32(dev, values):
    import torch
    return torch.tensor(list(values), dtype=torch.int32, device=dev)


def cum(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(int).tolist()


def rand(dev, dtype, *shape, seed):
    import torch
    r = np.random.default_rng(seed)
    x = r.normal(size=shape) * (0.5 + r.random(shape[-1])) + (r.random(shape[-1]) < 0.1) * r.normal(size=shape[-1])
    return torch.from_numpy(x.astype(np.float32)).to(dev).to(getattr(torch, dtype))


def f64(t):
    return t.detach().double().cpu().numpy()


def eps_half(dtype):
    import torch
    return torch.finfo(getattr(torch, dtype)).eps / 2


def positions(starts, lengths):
    return np.concatenate([np.arange(s, s + n) for s, n in zip(starts, lengths)] or [[]]).astype(int)


def want_kv(k, v, pos, D, group, rot=None, theta=THETA, interleaved=False):
    freq = kv4.inv_freq(D if rot is None else rot, theta)
    kr = kv4.rotate(f64(k), pos, freq, interleaved)
    return kr, kv4.held(kr.astype(np.float32), group), kv4.held(f64(v).astype(np.float32), group)


SHAPES = [  # D, group, dtype, page, kv heads, query heads, rotary, interleaved
    (128, 32, "bfloat16", 16, 8, 32, 128, False),
    (128, 32, "float32", 32, 1, 3, 128, False),
    (128, 64, "float16", 16, 3, 3, 64, False),
    (128, 128, "bfloat16", 64, 2, 10, 128, True),
    (64, 32, "float32", 16, 5, 5, 32, True),
    (64, 64, "bfloat16", 128, 4, 4, 64, False),
    (256, 32, "float16", 16, 1, 16, 256, False),
    (256, 64, "float32", 16, 2, 2, 16, False),
    (256, 128, "bfloat16", 32, 2, 6, 48, True),
]


@pytest.mark.parametrize("D,group,dtype,page,Hkv,Hq,rot,inter", SHAPES)
def test_append_and_read(lc, dev, D, group, dtype, page, Hkv, Hq, rot, inter):
    """The held values are the format's own, bit for bit (fp64 rotation and encoding; the sum
    lo + s code rounds once in fp32); the rotated queries and keys are theirs rounded to fp32
    and to the type: two half steps."""
    import torch
    lengths, starts = [37, 0, 1, 90, 16], [0, 5, 70001, 15, 64]
    B, N = len(lengths), sum(lengths)
    c = lc.PagedInt4KVCache(Hkv, D, num_sequences=B, page_size=page, max_resident_pages=8192 // page * 16,
                            group_size=group, rope_theta=THETA, rotary_dim=rot, interleaved=inter, device=dev)
    k, v, q = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((Hkv, 1), (Hkv, 2), (Hq, 3)))
    start, cu = i32(dev, starts), i32(dev, cum(lengths))
    qr, kr = c.append(k, v, start, cu, query=q, return_key=True)
    pos = positions(starts, lengths)
    kf, hk, hv = want_kv(k, v, pos, D, group, rot, interleaved=inter)
    rk, rv = c.read(start, cu, N)
    assert np.array_equal(f64(rk), hk.astype(np.float32).astype(np.float64))
    assert np.array_equal(f64(rv), hv.astype(np.float32).astype(np.float64))
    qf = kv4.rotate(f64(q), pos, kv4.inv_freq(rot, THETA), inter)
    e = 2 * eps_half(dtype)
    assert qr.dtype == q.dtype and (np.abs(f64(qr) - qf) <= e * np.abs(qf) + 1e-7 * (dtype == "float16")).all()
    assert kr.dtype == k.dtype and (np.abs(f64(kr) - kf) <= e * np.abs(kf) + 1e-7 * (dtype == "float16")).all()
    # in the cache's other types: the same values rounded
    for t in ("bfloat16", "float16"):
        bk, bv = c.read(start, cu, N, dtype=getattr(torch, t))
        assert torch.equal(bk, rk.to(bk.dtype)) and torch.equal(bv, rv.to(bv.dtype))


def test_single_tokens_without_lengths(lc, dev):
    """One token a sequence: the same as with cu_seqlens, at a batch on each side of the launch's split."""
    import torch
    for B in (1, 3, 300):
        c = [lc.PagedInt4KVCache(2, 64, num_sequences=B, max_resident_pages=8, device=dev) for _ in range(2)]
        k, v, q = (rand(dev, "bfloat16", B, h, 64, seed=h) for h in (2, 2, 6))
        start = i32(dev, [7 * b % 100 for b in range(B)])
        a = c[0].append(k, v, start, query=q)[0]
        b = c[1].append(k, v, start, i32(dev, range(B + 1)), query=q)[0]
        assert torch.equal(a, b)
        for x, y in zip(c[0].read(start), c[1].read(start, i32(dev, range(B + 1)), B)):
            assert torch.equal(x, y) and x.abs().sum() > 0


def test_no_rotation_and_given_frequencies(lc, dev):
    import torch
    k, v = rand(dev, "float32", 20, 2, 128, seed=4), rand(dev, "float32", 20, 2, 128, seed=5)
    s, cu = i32(dev, [1000]), i32(dev, [0, 20])
    plain = lc.PagedInt4KVCache(2, rope_theta=None, device=dev)
    q, kr = plain.append(k, v, s, cu, query=k, return_key=True)
    assert torch.equal(q, k) and torch.equal(kr, k)
    assert np.array_equal(f64(plain.read(s, cu, 20)[0]),
                          kv4.held(f64(k).astype(np.float32), 32).astype(np.float32).astype(np.float64))
    freq = kv4.inv_freq(128, 5e5) * 0.25
    c = lc.PagedInt4KVCache(2, inv_freq=torch.from_numpy(freq), device=dev)
    _, kr = c.append(k, v, s, cu, return_key=True)
    want = kv4.rotate(f64(k), np.arange(1000, 1020), freq)
    assert (np.abs(f64(kr) - want) <= 2 ** -23 * np.abs(want)).all()


def test_hard_values(lc, dev):
    """Ties, constant groups, values fp16 cannot hold, infinities and NaN: as the format says."""
    import torch
    x = np.zeros((12, 1, 64), np.float32)
    x[0, 0] = np.arange(64) % 16                       # exact
    x[1, 0] = np.tile(np.r_[0, 15, np.arange(14) + 0.5], 4)   # ties: to even
    x[2, 0] = -3.140625
    x[3, 0, 7] = np.nan
    x[4, 0, 40] = -np.inf
    x[5, 0] = np.linspace(-2e5, 3e5, 64)               # lo saturates
    x[6, 0] = np.linspace(0, 3e38, 64)                 # s too
    x[7, 0] = np.linspace(-1e-7, 1e-7, 64)             # subnormal steps
    x[8, 0] = np.linspace(1, 1 + 1e-6, 64)
    x[9, 0] = np.r_[np.full(32, -65504.0), np.linspace(100, 101, 32)]
    x[10, 0] = np.tile(np.r_[0, 7.5, np.arange(14) * 0.5 + 0.25], 4)  # step 0.5, ties
    x[11, 0] = np.tile([-1e-30, 1.0], 32)
    v = torch.from_numpy(x).to(dev)
    c = lc.PagedInt4KVCache(1, 64, rope_theta=None, device=dev)
    s, cu = i32(dev, [0]), i32(dev, [0, 12])
    c.append(v, v, s, cu)
    for got in c.read(s, cu, 12):
        assert np.array_equal(f64(got), kv4.held(x, 32).astype(np.float32).astype(np.float64), equal_nan=True)


def test_ring_of_pages(lc, dev):
    """Appends past the page limit: the sink pages stay, the rest are the newest; evicted tokens read
    as 0, also those that one call evicts again."""
    import torch
    P, pages, sink = 16, 5, 2
    c = lc.PagedInt4KVCache(2, 64, num_sequences=2, page_size=P, max_resident_pages=pages, sink_pages=sink,
                            group_size=64, rope_theta=THETA, device=dev)
    for calls in ([40, 30, 1, 1, 9, 50], [300], [80, 1], [16] * 9):
        N = sum(calls)
        k, v = rand(dev, "float32", N, 2, 64, seed=N), rand(dev, "float32", N, 2, 64, seed=N + 1)
        at = 0
        for n in calls:                        # sequence 1 gets the tokens, sequence 0 none
            c.append(k[at:at + n], v[at:at + n], i32(dev, [0, at]), i32(dev, [0, 0, n]))
            at += n
        zero, cu, seen = i32(dev, [0, 0]), i32(dev, [0, 0, N]), i32(dev, [0, N])
        rk, rv = c.read(zero, cu, N, seen=seen)
        _, hk, hv = want_kv(k, v, np.arange(N), 64, 64)
        gone = np.ones(N, bool)
        gone[kv4.resident(N, P, pages, sink)] = False
        hk[gone], hv[gone] = 0, 0
        assert np.array_equal(f64(rk), hk.astype(np.float32)) and np.array_equal(f64(rv), hv.astype(np.float32))
        q = rand(dev, "float32", 2, 4, 64, seed=7)
        out = f64(c.decode(q, seen))
        assert (out[0] == 0).all()
        for h in range(4):
            w, _ = kv4.attention(f64(q)[1, h:h + 1], hk[~gone, h // 2], hv[~gone, h // 2], 1 / 8)
            assert np.abs(out[1, h] - w[0]).max() <= 2e-6 * np.abs(hv).max(), (calls, h)


def test_rows_of_no_sequence(lc, dev):
    """Rows before the first and behind the last sequence: nothing is written, the results are 0."""
    import torch
    c = lc.PagedInt4KVCache(1, 64, num_sequences=2, max_resident_pages=8, device=dev)
    k, v, q = (rand(dev, "float16", 20, 1, 64, seed=s) for s in (1, 2, 3))
    k[:3], k[12:], v[:3], v[12:], q[:3], q[12:] = (float("nan"),) * 6
    s, cu = i32(dev, [0, 0]), i32(dev, [3, 8, 12])
    before = [t.clone() for t in (c.k_codes, c.v_codes, c.k_steps, c.v_steps)]
    qr, kr = c.append(k, v, s, cu, query=q, return_key=True)
    rk, rv = c.read(s, cu, 20)
    for t in (qr, kr, rk, rv):
        t = f64(t)
        assert (t[:3] == 0).all() and (t[12:] == 0).all() and np.isfinite(t).all() and (t[3:12] != 0).any()
    c.append(k, v, s, i32(dev, [0, 0, 0]))             # all rows of no sequence
    c2 = lc.PagedInt4KVCache(1, 64, num_sequences=2, max_resident_pages=8, device=dev)
    c2.append(k[3:12], v[3:12], s, i32(dev, [0, 5, 9]))
    for a, b, z in zip((c.k_codes, c.v_codes, c.k_steps, c.v_steps),
                       (c2.k_codes, c2.v_codes, c2.k_steps, c2.v_steps), before):
        assert torch.equal(a, b) and not torch.equal(a, z)


def test_block_table_of_the_caller(lc, dev):
    """Shuffled pages, a shared prefix, and entries that map no page."""
    import torch
    c = lc.PagedInt4KVCache(2, 128, num_sequences=2, page_size=16, max_resident_pages=4, sink_pages=1,
                            num_pages=9, device=dev)
    k, v = rand(dev, "bfloat16", 60, 2, 128, seed=1), rand(dev, "bfloat16", 60, 2, 128, seed=2)
    s = i32(dev, [0, 0])
    q = rand(dev, "float32", 2, 2, 128, seed=3)
    c.append(k, v, s, i32(dev, [0, 60, 60]))           # no page is mapped yet
    assert not c.k_codes.any() and not c.v_steps.any()
    assert not c.decode(q, i32(dev, [60, 0])).any()
    c.block_table.copy_(i32(dev, [7, 2, 8, 0, 7, -1, 99, 5]).view(2, 4))
    c.append(k, v, s, i32(dev, [0, 60, 60]))
    # sequence 1 reads sequence 0's first page, has none for its next two and writes the last
    c.append(k[48:60], v[48:60], i32(dev, [60, 48]), i32(dev, [0, 0, 12]))
    _, hk, hv = want_kv(k, v, np.arange(60), 128, 32)
    rk, rv = c.read(s, i32(dev, [0, 60, 60]), 60)
    assert np.array_equal(f64(rk), hk.astype(np.float32)) and np.array_equal(f64(rv), hv.astype(np.float32))
    out = f64(c.decode(q, i32(dev, [60, 60])))
    there = np.r_[0:16, 48:60]
    for h in range(2):
        for b, rows in ((0, np.arange(60)), (1, there)):
            w, _ = kv4.attention(f64(q)[b, h:h + 1], hk[rows, h], hv[rows, h], 128 ** -0.5)
            assert np.abs(out[b, h] - w[0]).max() <= 2e-6 * np.abs(hv).max(), (b, h)


def test_strided_and_unaligned_inputs(lc, dev):
    """Views of one packed projection, transposed heads, odd offsets: the same as contiguous copies."""
    import torch
    n, Hkv, Hq, D = 21, 2, 4, 64
    s, cu = i32(dev, [3]), i32(dev, [0, n])
    qkv = rand(dev, "bfloat16", n, (Hq + 2 * Hkv) * D, seed=5).view(n, Hq + 2 * Hkv, D)
    wide = rand(dev, "bfloat16", n, Hkv, D + 8, seed=6)
    odd = rand(dev, "bfloat16", 1, n * Hkv * D + 1, seed=7)[0, 1:].view(n, Hkv, D)
    turned = rand(dev, "bfloat16", Hkv, n, D, seed=8).transpose(0, 1)
    columns = rand(dev, "bfloat16", n, D, Hkv, seed=9).transpose(1, 2)
    repeated = rand(dev, "bfloat16", n, 1, D, seed=10).expand(n, Hkv, D)
    for k, v, q in ((qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], qkv[:, :Hq]), (wide[..., :D], wide[..., 1:D + 1], qkv[:, 1:3]),
                    (odd, turned, odd), (turned, columns, columns), (columns, odd, repeated), (repeated, repeated, qkv[:, ::2])):
        got, want = (lc.PagedInt4KVCache(Hkv, D, device=dev) for _ in range(2))
        a = got.append(k, v, s, cu, query=q, return_key=True)
        b = want.append(k.contiguous().clone(), v.contiguous().clone(), s, cu, query=q.contiguous().clone(), return_key=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(got.k_codes, want.k_codes) and torch.equal(got.v_codes, want.v_codes)
        assert torch.equal(got.k_steps, want.k_steps) and torch.equal(got.v_steps, want.v_steps)


# decode: lengths around a block, a tile, a workgroup's tiles and its splits
DECODE = [  # D, group, dtype, page, kv heads, share, lengths, pages
    (128, 32, "float32", 16, 8, 4, [2048], 2048),
    (128, 32, "bfloat16", 16, 2, 4, [0, 1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000], 128),
    (128, 32, "float16", 32, 1, 5, [300, 33], 64),
    (128, 64, "bfloat16", 64, 2, 8, [5000, 3, 777], 128),
    (128, 128, "float32", 16, 2, 17, [129, 640], 64),
    (128, 128, "float16", 16, 4, 1, [1500], 128),
    (64, 32, "float32", 16, 3, 2, [1, 100, 2000], 128),
    (64, 64, "float16", 16, 2, 16, [4097, 0], 512),
    (64, 64, "bfloat16", 128, 1, 3, [130], 4),
    (256, 32, "float32", 16, 1, 2, [77, 1025], 128),
    (256, 64, "bfloat16", 16, 2, 5, [513], 64),
    (256, 128, "float16", 256, 2, 9, [900, 12], 8),
]


def decode_case(lc, dev, D, group, dtype, page, Hkv, share, lengths, pages, seed=11):
    B, N, Hq = len(lengths), sum(lengths), Hkv * share
    c = lc.PagedInt4KVCache(Hkv, D, num_sequences=B, page_size=page, max_resident_pages=pages, sink_pages=1,
                            group_size=group, device=dev)
    k, v = rand(dev, dtype, N, Hkv, D, seed=seed), rand(dev, dtype, N, Hkv, D, seed=seed + 1)
    q = rand(dev, dtype, B, Hq, D, seed=seed + 2)
    if N:
        c.append(k, v, i32(dev, [0] * B), i32(dev, cum(lengths)))
    _, hk, hv = want_kv(k, v, positions([0] * B, lengths), D, group)
    return c, q, hk, hv


def check_decode(out, q, hk, hv, lengths, share, dtype, scale, group):
    """Bound: a score is a sum of D + 2 D / group products and step products in fp32; its
    rounding is a random walk, held to 16 half steps of sum |q| (|lo| + 15 s) <= 3 sum |q| |k|max
    scale.  It enters the weights twice (numerator and denominator).  A weight is rounded to fp16
    for bf16 outputs, 2^-12, and in two pieces else, 2^-22.  The output rounds once."""
    at = 0
    for b, n in enumerate(lengths):
        for h in range(q.shape[1]):
            o = f64(out)[b, h]
            if n == 0:
                assert (o == 0).all()
                continue
            K, V = hk[at:at + n, h // share], hv[at:at + n, h // share]
            x = f64(q)[b, h]
            want, _ = kv4.attention(x[None], K, V, scale)
            score = 16 * 2 ** -24 * 3 * (np.abs(x) * np.abs(K).max(0)).sum() * scale
            tol = np.abs(V).max() * (2 * score + (2 ** -12 if dtype == "bfloat16" else 2 ** -22))
            tol = tol + eps_half(dtype) * np.abs(want[0]) + 1e-7 * (dtype == "float16")
            assert (np.abs(o - want[0]) <= tol).all(), (b, h, np.abs(o - want[0]).max())
        at += n


@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"d{c[0]}g{c[1]}{c[2]}x{c[5]}")
def test_decode(lc, dev, case):
    D, group, dtype, page, Hkv, share, lengths, pages = case
    c, q, hk, hv = decode_case(lc, dev, *case)
    seen = i32(dev, lengths)
    for kw, scale in ((dict(), D ** -0.5), (dict(max_seen=max(lengths)), D ** -0.5), (dict(scale_factor=0.05), 0.05),
                      (dict(max_seen=1), D ** -0.5)):
        out = c.decode(q, seen, **kw)
        assert out.dtype == q.dtype and out.shape == q.shape
        check_decode(out, q, hk, hv, lengths, share, dtype, scale, group)


def test_decode_leaves_out_what_is_not_held(lc, dev):
    """Slots past a sequence's end hold NaN and infinite tokens from an earlier use: they reach nothing."""
    import torch
    c = lc.PagedInt4KVCache(2, 128, num_sequences=2, max_resident_pages=64, device=dev)
    bad = torch.full((1024, 2, 128), float("nan"), device=dev)
    bad[::3] = float("inf")
    bad[1::3] = 6e4
    s, cu = i32(dev, [0, 0]), i32(dev, [0, 512, 1024])
    c.append(bad, bad, s, cu)
    k, v = rand(dev, "float32", 150, 2, 128, seed=1), rand(dev, "float32", 150, 2, 128, seed=2)
    lengths = [101, 49]
    c.append(k, v, s, i32(dev, [0, 101, 150]))
    q = rand(dev, "float32", 2, 8, 128, seed=3)
    _, hk, hv = want_kv(k, v, positions([0, 0], lengths), 128, 32)
    check_decode(c.decode(q, i32(dev, lengths)), q, hk, hv, lengths, 4, "float32", 128 ** -0.5, 32)
    # a NaN among the held tokens does reach the heads that read it
    k[5, 1, 3] = float("nan")
    c.append(k, v, s, i32(dev, [0, 101, 150]))
    out = f64(c.decode(q, i32(dev, lengths)))
    assert np.isnan(out[0, 4:]).all() and np.isfinite(out[0, :4]).all() and np.isfinite(out[1]).all()


def test_decode_large_and_small_values(lc, dev):
    """Scores far apart, queries near the types' ends, steps from 1e-6 to 1e3: the scalings hold."""
    import torch
    n = 200
    for qs, ks, vs in ((1e4, 1e-3, 1e3), (1e-6, 30.0, 1e-5), (3e-3, 1e3, 1.0), (1e30, 1e-30, 1e-2)):
        c = lc.PagedInt4KVCache(1, 64, rope_theta=None, device=dev)
        k, v = rand(dev, "float32", n, 1, 64, seed=1) * ks, rand(dev, "float32", n, 1, 64, seed=2) * vs
        v[::7] *= 1e-3
        q = rand(dev, "float32", 1, 2, 64, seed=3) * qs
        c.append(k, v, i32(dev, [0]), i32(dev, [0, n]))
        hk, hv = kv4.held(f64(k).astype(np.float32), 32), kv4.held(f64(v).astype(np.float32), 32)
        check_decode(c.decode(q, i32(dev, [n])), q, hk, hv, [n], 2, "float32", 1 / 8, 32)


def test_decode_constant_groups(lc, dev):
    """Groups of one value that fp16 rounds up or down: their step is 0 (or the smallest there is), never
    negative, and the weights' scaling holds beside them."""
    import torch
    n = 500
    for seed in range(3):
        g = np.random.default_rng(seed)
        x = [np.repeat(g.normal(size=(n, 1, 4, 1)), 32, -1).reshape(n, 1, 128).astype(np.float32) for _ in range(2)]
        x[1][::9, 0, 5] += 1e-3
        c = lc.PagedInt4KVCache(1, 128, rope_theta=None, device=dev)
        k, v = (torch.from_numpy(a).to(dev) for a in x)
        q = rand(dev, "float32", 1, 4, 128, seed=3)
        c.append(k, v, i32(dev, [0]), i32(dev, [0, n]))
        assert (c.k_steps.view(-1, 2)[:, 0] >= 0).all() and (c.v_steps.view(-1, 2)[:, 0] >= 0).all()
        hk, hv = kv4.held(x[0], 32), kv4.held(x[1], 32)
        for ms in (0, 64):
            check_decode(c.decode(q, i32(dev, [n]), max_seen=ms), q, hk, hv, [n], 4, "float32", 128 ** -0.5, 32)


def test_captured_steps(lc, dev):
    """A captured decode step replays as the sequences grow: rotation, append and attention follow the
    lengths that the graph advances itself; every replay equals the eager step."""
    import torch
    B, Hkv, Hq, D = 3, 2, 8, 128
    g, e = (lc.PagedInt4KVCache(Hkv, D, num_sequences=B, max_resident_pages=6, sink_pages=1, device=dev) for _ in range(2))
    starts = [0, 30, 94]
    k0, v0 = rand(dev, "bfloat16", sum(starts), Hkv, D, seed=1), rand(dev, "bfloat16", sum(starts), Hkv, D, seed=2)
    for c in (g, e):
        c.append(k0, v0, i32(dev, [0] * B), i32(dev, cum(starts)))
    q, k, v = (torch.empty(B, h, D, dtype=torch.bfloat16, device=dev) for h in (Hq, Hkv, Hkv))
    start = i32(dev, starts)
    seen = start + 1

    def step(c, start, seen):
        qr, _ = c.append(k, v, start, query=q)
        return c.decode(qr, seen)

    q.normal_(), k.normal_(), v.normal_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(g, start, seen)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(g, start, seen)
        start.add_(1)
        seen.add_(1)
    for i in range(40):
        for t, s in ((q, 1), (k, 2), (v, 3)):
            t.copy_(rand(dev, "bfloat16", *t.shape, seed=100 * i + s))
        graph.replay()
        torch.cuda.synchronize()
        at = i32(dev, [x + i for x in starts])
        assert torch.equal(out, step(e, at, at + 1)), i
        assert out.abs().sum() > 0


def test_streams_and_repeat(lc, dev):
    """Calls on another stream follow that stream, and the same call gives the same bits."""
    import torch
    c, q, hk, hv = decode_case(lc, dev, *DECODE[3])
    lengths = DECODE[3][6]
    seen = i32(dev, lengths)
    first = c.decode(q, seen)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        outs = [c.decode(q, seen) for _ in range(5)]
    s.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    out = torch.full_like(first, 9.0)
    assert c.decode(q, seen, out=out) is out and torch.equal(out, first)


def test_refusals(lc, dev):
    import torch
    c = lc.PagedInt4KVCache(2, 64, num_sequences=3, max_resident_pages=4, device=dev)
    k = torch.zeros(3, 2, 64, device=dev)
    s = i32(dev, [0, 0, 0])
    bad = [
        (RuntimeError, lambda: c.append(k.cpu(), k, s)),
        (ValueError, lambda: c.append(k, k.half(), s)),
        (TypeError, lambda: c.append(k.double(), k.double(), s)),
        (ValueError, lambda: c.append(k[:2], k[:2], s)),
        (ValueError, lambda: c.append(k, k[:2], s)),
        (ValueError, lambda: c.append(k[:, :1], k, s)),
        (ValueError, lambda: c.append(k[..., :32], k[..., :32], s)),
        (ValueError, lambda: c.append(k, k, s.long())),
        (ValueError, lambda: c.append(k, k, s[:2])),
        (ValueError, lambda: c.append(k, k, s.cpu())),
        (ValueError, lambda: c.append(k, k, s, s)),
        (ValueError, lambda: c.append(k, k, s, query=k[:2])),
        (ValueError, lambda: c.append(k, k, s, query=k.half())),
        (RuntimeError, lambda: c.append(k.clone().requires_grad_(), k, s)),
        (ValueError, lambda: c.read(s, i32(dev, [0, 1, 2, 3]))),
        (ValueError, lambda: c.read(s, num_tokens=2)),
        (TypeError, lambda: c.read(s, dtype=torch.float64)),
        (ValueError, lambda: c.decode(k[:2], s)),
        (ValueError, lambda: c.decode(torch.zeros(3, 3, 64, device=dev), s)),
        (ValueError, lambda: c.decode(k, s, max_seen=-1)),
        (ValueError, lambda: c.decode(k, s, out=torch.zeros(3, 2, 64, device=dev, dtype=torch.half))),
        (RuntimeError, lambda: c.decode(k.clone().requires_grad_(), s)),
        (TypeError, lambda: c.decode(k.double(), s)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    with torch.no_grad():
        c.append(k.clone().requires_grad_(), k, s)
    assert c.append(k[:0], k[:0], s, i32(dev, [0] * 4)) == (None, None)


def test_offsets_past_32_bits(lc, dev):
    """A pool of more than 2^32 bytes of codes: pages at its far end."""
    import torch
    pages = (1 << 32) // (2 * 16 * 128) + 64            # 2 heads, 16 slots, 128 bytes a row (head_dim 256)
    c = lc.PagedInt4KVCache(2, 256, num_sequences=1, max_resident_pages=8, sink_pages=1, num_pages=pages,
                            group_size=128, device=dev)
    assert c.k_codes.numel() > 1 << 32
    c.block_table.copy_(torch.arange(pages - 8, pages, dtype=torch.int32, device=dev).view(1, 8))
    k, v = rand(dev, "bfloat16", 100, 2, 256, seed=1), rand(dev, "bfloat16", 100, 2, 256, seed=2)
    s, cu = i32(dev, [0]), i32(dev, [0, 100])
    c.append(k, v, s, cu)
    _, hk, hv = want_kv(k, v, np.arange(100), 256, 128)
    rk, rv = c.read(s, cu, 100)
    assert np.array_equal(f64(rk), hk.astype(np.float32)) and np.array_equal(f64(rv), hv.astype(np.float32))
    q = rand(dev, "bfloat16", 1, 4, 256, seed=3)
    check_decode(c.decode(q, i32(dev, [100])), q, hk, hv, [100], 2, "bfloat16", 1 / 16, 128)


def test_block_table_is_filled_in_not_replaced(lc, dev):
    import torch
    c = lc.PagedInt4KVCache(1, 64, max_resident_pages=4, group_size=64, num_pages=4, device=dev)
    with pytest.raises(AttributeError):
        c.block_table = torch.zeros(1, 4, dtype=torch.int32, device=dev)


def test_decode_into_the_query(lc, dev):
    """out may be the query: a long sequence, cut into runs, and short ones, written whole."""
    import torch
    g = torch.Generator(device=dev).manual_seed(3)
    c = lc.PagedInt4KVCache(2, 128, num_sequences=3, max_resident_pages=64, device=dev)
    n = [1000, 3, 0]
    cu = i32(dev, [0, 1000, 1003, 1003])
    k, v = (torch.randn(1003, 2, 128, generator=g, device=dev) for _ in range(2))
    c.append(k, v, i32(dev, [0, 0, 0]), cu)
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.randn(3, 16, 128, generator=g, device=dev).to(dtype)
        want = c.decode(q, i32(dev, n))
        assert c.decode(q, i32(dev, n), out=q) is q and torch.equal(q, want)


FEW = [  # as DECODE: no more heads per kv head than a quarter of the columns
    (128, 32, "float32", 16, 3, 1, [0, 1, 3, 4, 5, 11, 12, 13, 16, 17, 63, 64, 65, 700], 64),
    (128, 64, "bfloat16", 32, 2, 2, [1, 4, 6, 900, 0, 31], 64),
    (128, 128, "float16", 16, 1, 3, [1030, 7], 128),
    (64, 32, "bfloat16", 16, 2, 1, [2, 500, 66], 64),
    (64, 64, "float32", 64, 2, 4, [1, 8, 129, 0], 16),
    (64, 64, "bfloat16", 16, 16, 1, [1300, 5, 9, 14], 128),
    (256, 64, "bfloat16", 16, 2, 1, [10, 333], 64),
    (256, 128, "float32", 16, 1, 2, [3, 260], 64),
]


@pytest.mark.parametrize("case", FEW, ids=lambda c: f"d{c[0]}g{c[1]}{c[2]}x{c[5]}")
def test_decode_few_heads(lc, dev, case):
    D, group, dtype, page, Hkv, share, lengths, pages = case
    c, q, hk, hv = decode_case(lc, dev, *case)
    seen = i32(dev, lengths)
    for kw in (dict(), dict(max_seen=max(lengths))):
        check_decode(c.decode(q, seen, **kw), q, hk, hv, lengths, share, dtype, D ** -0.5, group)


@pytest.mark.parametrize("B,N,dtype", [(3, 1500, "bfloat16"), (70, 2500, "float16"), (130, 5000, "float32")])
def test_append_many_tokens(lc, dev, B, N, dtype):
    """Tokens that share their waves' work over fewer of them, and one wave for a whole token; more
    sequences than lanes."""
    r = np.random.default_rng(B)
    cuts = np.sort(r.integers(0, N + 1, B - 1)).tolist()
    cu = [0] + cuts + [N]
    lengths = np.diff(cu).tolist()
    starts = r.integers(0, 100, B).tolist()
    pages = (max(lengths) + 100) // 16 + 1
    c = lc.PagedInt4KVCache(2, 128, num_sequences=B, max_resident_pages=pages, sink_pages=1, rope_theta=THETA,
                            device=dev)
    k, v, q = (rand(dev, dtype, N, h, 128, seed=s) for h, s in ((2, 1), (2, 2), (12, 3)))
    qr, _ = c.append(k, v, i32(dev, starts), i32(dev, cu), query=q)
    pos = positions(starts, lengths)
    _, hk, hv = want_kv(k, v, pos, 128, 32)
    rk, rv = c.read(i32(dev, starts), i32(dev, cu), N)
    assert np.array_equal(f64(rk), hk.astype(np.float32).astype(np.float64))
    assert np.array_equal(f64(rv), hv.astype(np.float32).astype(np.float64))
    qf = kv4.rotate(f64(q), pos, kv4.inv_freq(128, THETA))
    assert (np.abs(f64(qr) - qf) <= 2 * eps_half(dtype) * np.abs(qf) + 1e-7 * (dtype == "float16")).all()


@pytest.mark.parametrize("share", [1, 5])
def test_decode_many_sequences(lc, dev, share):
    """More sequences than lanes, some without tokens, runs that begin in any of them."""
    lengths = np.random.default_rng(share).integers(-20, 200, 150).clip(0).tolist()
    lengths[149] = 1000
    c, q, hk, hv = decode_case(lc, dev, 64, 32, "float32", 16, 2, share, lengths, 64)
    seen = i32(dev, lengths)
    for kw in (dict(), dict(max_seen=40)):
        check_decode(c.decode(q, seen, **kw), q, hk, hv, lengths, share, "float32", 0.125, 32)
