"""PackedPromptAttention on the GPU against the fp64 oracle (oracle/kv4.py): lengths around its
tiles, grouped heads, head dims, masks that leave rows empty, rows of no sequence, hidden
infinities, layouts, captured calls; and the serving path that it begins: prompts, their cache,
decode steps."""
import math

import numpy as np
import pytest

from oracle import kv4
from test_gpu_kv4 import cum, eps_half, f64, i32, positions, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc(pkg):
    from importlib import import_module
    return import_module(pkg.__name__ + ".long_context")


def check(out, q, k, v, cq, ck, causal, scale, dtype, lse=None):
    """Bound: a score is an fp32 sum of D exact products, its rounding a random walk held to 16 half
    steps of sum |q k| scale and 2 of the score in log2; it moves the weights twice (numerator and
    sum).  A weight is rounded to the inputs' type (none for fp32; the hardware's exp2 is within two
    fp32 half steps); the output rounds once."""
    import torch
    q, k, v, o = f64(q), f64(k), f64(v), f64(out)
    share = q.shape[1] // k.shape[1]
    half = eps_half(dtype)
    for b in range(len(cq) - 1):
        n, t = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        for h in range(q.shape[1]):
            K, V = k[ck[b]:ck[b + 1], h // share], v[ck[b]:ck[b + 1], h // share]
            x = q[cq[b]:cq[b + 1], h]
            hidden = np.arange(n) + t - n + 1 if causal else np.full(n, t)
            want, wl = kv4.attention(x, K, V, scale, hidden)
            got = o[cq[b]:cq[b + 1], h]
            if t == 0:
                assert (got == 0).all(), (b, h)
                continue
            absw, _ = kv4.attention(x, K, np.abs(V), scale, hidden)          # sum of weights times |v|
            score = 2 ** -24 * (16 * scale * (np.abs(x) @ np.abs(K).max(0)) + 2 * 1.45 * np.abs(scale * (x @ K.T)).max(1))
            rel = 2 * score + (half if dtype != "float32" else 0) + 2 ** -22
            tol = rel[:, None] * absw + half * np.abs(want) + 1e-7 * (dtype == "float16")
            bad = np.abs(got - want) > tol
            assert not bad.any(), (b, h, np.argwhere(bad)[:3], np.abs(got - want).max())
            if lse is not None:
                gl = f64(lse)[cq[b]:cq[b + 1], h]
                empty = ~np.isfinite(wl)
                assert (gl[empty] == -np.inf).all()
                assert (np.abs(gl[~empty] - wl[~empty]) <= score[~empty] + 2 ** -22 * (1 + np.abs(wl[~empty]))).all()


LENGTHS = [0, 1, 2, 31, 33, 64, 65, 0, 127, 129, 200]
SHAPES = [  # Hq, Hkv, D, dtype
    (4, 4, 128, "bfloat16"), (8, 2, 128, "float16"), (5, 1, 128, "bfloat16"), (16, 2, 64, "bfloat16"),
    (6, 3, 64, "float16"), (8, 1, 256, "bfloat16"), (3, 3, 256, "float16"), (2, 1, 8, "bfloat16"),
    (4, 2, 40, "float16"), (12, 4, 80, "bfloat16"), (4, 1, 136, "bfloat16"), (1, 1, 104, "float16"),
    (4, 1, 128, "float32"), (8, 8, 64, "float32"), (6, 2, 256, "float32"), (2, 2, 72, "float32"),
    (16, 1, 24, "float32"), (32, 2, 128, "bfloat16"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", SHAPES)
def test_packed_prompts(lc, dev, Hq, Hkv, D, dtype, causal):
    N = sum(LENGTHS)
    q, k, v = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
    cu = cum(LENGTHS)
    a = lc.PackedPromptAttention(Hq, Hkv, D, causal=causal)
    out, lse = a(q, k, v, i32(dev, cu), return_lse=True)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == q.shape[:2]
    check(out, q, k, v, cu, cu, causal, D ** -0.5, dtype, lse)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_one_long_prompt(lc, dev, dtype):
    """A prompt of many tiles and row blocks, with a scale of its own and scores far apart."""
    n, D = 1111, 128
    q, k, v = (rand(dev, dtype, n, h, D, seed=s) for h, s in ((4, 1), (1, 2), (1, 3)))
    for scale in (0.02, 1.0):
        a = lc.PackedPromptAttention(4, 1, D, scale=scale)
        out, lse = a(q, k, v, i32(dev, [0, n]), return_lse=True)
        check(out, q, k, v, [0, n], [0, n], True, scale, dtype, lse)


@pytest.mark.parametrize("dtype,D", [("bfloat16", 128), ("float32", 64), ("float16", 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_their_own_lengths(lc, dev, dtype, D, causal):
    """More keys than queries (a context before the prompt's rows), fewer (the first rows see none),
    none at all, and queries none."""
    nq, nk = [10, 70, 5, 40, 0, 3], [100, 70, 300, 7, 20, 0]
    q, k, v = rand(dev, dtype, sum(nq), 4, D, seed=1), rand(dev, dtype, sum(nk), 2, D, seed=2), \
        rand(dev, dtype, sum(nk), 2, D, seed=3)
    a = lc.PackedPromptAttention(4, 2, D, causal=causal)
    out, lse = a(q, k, v, i32(dev, cum(nq)), i32(dev, cum(nk)), return_lse=True)
    check(out, q, k, v, cum(nq), cum(nk), causal, D ** -0.5, dtype, lse)
    if causal:
        assert (f64(out)[85:85 + 33] == 0).all() and (f64(lse)[85:85 + 33] == -np.inf).all()
    assert (f64(out)[-3:] == 0).all()
    none = a(q, k[:0], v[:0], i32(dev, cum(nq)), i32(dev, [0] * 7))
    assert not none.any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_of_no_sequence(lc, dev, dtype):
    """Rows before the first and behind the last sequence: 0 in a new result, as they were in a given
    one; what they hold reaches nothing."""
    import torch
    q, k, v = (rand(dev, dtype, 300, h, 64, seed=s) for h, s in ((4, 1), (2, 2), (2, 3)))
    for t in (q, k, v):
        t[:77], t[250:] = float("nan"), float("inf")
    cu = [77, 140, 140, 250]
    a = lc.PackedPromptAttention(4, 2, 64)
    out, lse = a(q, k, v, i32(dev, cu), return_lse=True)
    check(out, q, k, v, cu, cu, True, 0.125, dtype, lse)
    assert not out[:77].any() and not out[250:].any()
    assert (lse[:77] == -math.inf).all() and (lse[250:] == -math.inf).all()
    mine = torch.full_like(out, 5.0)
    got, l2 = a(q, k, v, i32(dev, cu), out=mine, return_lse=True)
    assert got is mine and (mine[:77] == 5).all() and (mine[250:] == 5).all()
    assert torch.equal(mine[77:250], out[77:250]) and torch.equal(l2, lse)
    for empty in ([0, 0], [300, 300, 300], [120, 120]):
        assert not a(q, k, v, i32(dev, empty)).any()


def test_bounds_that_are_none(lc, dev):
    """Bounds past the rows, negative or descending: no access outside the tensors, rows of proper
    sequences as ever."""
    import torch
    q, k, v = (rand(dev, "bfloat16", 100, 1, 64, seed=s) for s in (1, 2, 3))
    a = lc.PackedPromptAttention(1, 1, 64)
    whole = a(q, k, v, i32(dev, [0, 100]))
    assert torch.equal(a(q, k, v, i32(dev, [-50, 1000])), whole)
    for cu in ([0, 90, 30, 100], [100, 0], [2 ** 31 - 1, -2 ** 31], [50, 2 ** 31 - 1, 60]):
        assert torch.isfinite(a(q, k, v, i32(dev, cu))).all()
        assert torch.isfinite(a(q, k, v, i32(dev, [0] + [100] * (len(cu) - 1)), i32(dev, cu))).all()


@pytest.mark.parametrize("dtype,D", [("bfloat16", 128), ("float16", 64), ("float32", 128), ("bfloat16", 256)])
def test_hidden_keys_reach_nothing(lc, dev, dtype, D):
    """Infinities and NaN in keys and values that a row does not see: in the same tile, behind the
    sequence's end, in the next sequence.  A row that sees one has what its dot products give."""
    import torch
    lengths = [90, 45, 70]
    N, cu = sum(lengths), cum(lengths)
    q, k, v = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((4, 1), (2, 2), (2, 3)))
    a = lc.PackedPromptAttention(4, 2, D)
    clean, lse = a(q, k, v, i32(dev, cu), return_lse=True)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(k.dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[40], v2[40], v2[cu[1]], v2[cu[3] - 1, 0, 3] = bad, bad, bad, bad
        out, l2 = a(q, k2, v2, i32(dev, cu), return_lse=True)
        check(out[:40], q[:40], k[:40], v[:40], [0, 40], [0, 40], True, D ** -0.5, dtype, l2[:40])
        check(out[cu[2]:N - 1], q[cu[2]:N - 1], k[cu[2]:N - 1], v[cu[2]:N - 1], [0, N - 1 - cu[2]],
              [0, N - 1 - cu[2]], True, D ** -0.5, dtype, l2[cu[2]:N - 1])
        if not math.isfinite(bad):
            assert not torch.isfinite(out[cu[1]:cu[2]]).any()                # all of sequence 1 sees it
            last = out[N - 1]
            assert not torch.isfinite(last[:2, 3]).any() and torch.isfinite(last[2:]).all()
            assert torch.isfinite(last[:2, :3]).all() and torch.isfinite(last[:2, 4:]).all()
    q2 = q.clone()
    q2[50, 1] = float("nan")                                                 # one query row
    out = a(q2, k, v, i32(dev, cu))
    assert torch.isnan(out[50, 1]).all()
    ok = torch.ones(N, 4, dtype=torch.bool, device=dev)
    ok[50, 1] = False
    assert torch.isfinite(out[ok]).all()
    want = out.clone()
    want[50, 1] = clean[50, 1]
    check(want, q, k, v, cu, cu, True, D ** -0.5, dtype)


def test_strided_and_unaligned_inputs(lc, dev):
    import torch
    n, Hq, Hkv, D = 150, 4, 2, 64
    cu = i32(dev, [0, 60, n])
    a = lc.PackedPromptAttention(Hq, Hkv, D)
    qkv = rand(dev, "bfloat16", n, (Hq + 2 * Hkv) * D, seed=5).view(n, Hq + 2 * Hkv, D)
    wide = rand(dev, "bfloat16", n, Hkv, D + 8, seed=6)
    odd = rand(dev, "bfloat16", 1, n * Hkv * D + 1, seed=7)[0, 1:].view(n, Hkv, D)
    heads = rand(dev, "bfloat16", Hq, n, D, seed=8).transpose(0, 1)
    columns = rand(dev, "bfloat16", n, D, Hkv, seed=9).transpose(1, 2)
    one = rand(dev, "bfloat16", n, 1, D, seed=10).expand(n, Hkv, D)
    back = rand(dev, "bfloat16", 2 * n, Hkv, D, seed=11)[::2]
    for q, k, v in ((qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]), (heads, wide[..., :D], wide[..., 3:D + 3]),
                    (heads, odd, columns), (qkv[:, ::2], one, back), (qkv[:, 2:6], columns, odd)):
        out = a(q, k, v, cu)
        assert torch.equal(out, a(q.contiguous().clone(), k.contiguous().clone(), v.contiguous().clone(), cu))


def test_offsets_past_32_bits(lc, dev):
    """Rows more than 2^32 bytes apart."""
    import torch
    n, D = 130, 64
    stride = (1 << 33) // (2 * n) // 8 * 8 + 64
    buf = torch.empty(n * stride + 1024, dtype=torch.bfloat16, device=dev)
    q, k, v = (rand(dev, "bfloat16", n, h, D, seed=s) for h, s in ((2, 1), (1, 2), (1, 3)))
    qs, ks, vs = (torch.as_strided(buf, (n, h, D), (stride, D, 1), at) for h, at in ((2, 0), (1, 256), (1, 512)))
    for a, b in ((qs, q), (ks, k), (vs, v)):
        a.copy_(b)
    att = lc.PackedPromptAttention(2, 1, D)
    cu = i32(dev, [0, 1, n])
    assert torch.equal(att(qs, ks, vs, cu), att(q, k, v, cu))


def test_many_sequences(lc, dev):
    """More sequences than lanes; a batch of single tokens returns its values."""
    import torch
    r = np.random.default_rng(4)
    lengths = r.integers(0, 9, 500).tolist()
    N, cu = sum(lengths), cum(lengths)
    q, k, v = (rand(dev, "bfloat16", N, h, 64, seed=s) for h, s in ((2, 1), (1, 2), (1, 3)))
    check(lc.PackedPromptAttention(2, 1, 64)(q, k, v, i32(dev, cu)), q, k, v, cu, cu, True, 0.125, "bfloat16")
    ones = lc.PackedPromptAttention(2, 1, 64)(q, k, v, i32(dev, range(N + 1)))
    assert torch.equal(ones, v.expand(N, 2, 64))


def test_captured_and_streams(lc, dev):
    """A captured call follows the lengths and inputs of each replay; other streams give the same bits."""
    import torch
    N = 260
    a = lc.PackedPromptAttention(8, 2, 128)
    q, k, v = (rand(dev, "bfloat16", N, h, 128, seed=s) for h, s in ((8, 1), (2, 2), (2, 3)))
    cu = i32(dev, [0, 100, 260])
    first = a(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [a(q, k, v, cu) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = a(q, k, v, cu, return_lse=True)
    for i, bounds in enumerate(([0, 100, 260], [0, 0, 260], [10, 33, 200], [0, 259, 260])):
        cu.copy_(i32(dev, bounds))
        q.copy_(rand(dev, "bfloat16", N, 8, 128, seed=50 + i))
        g.replay()
        torch.cuda.synchronize()
        e, el = a(q, k, v, cu, return_lse=True)
        assert torch.equal(out, e) and torch.equal(lse, el), i
        check(out, q, k, v, bounds, bounds, True, 128 ** -0.5, "bfloat16", lse)


def test_refusals(lc, dev):
    import torch
    for kw in (dict(num_heads=3, num_kv_heads=2), dict(num_heads=2, head_dim=260), dict(num_heads=2, head_dim=12),
               dict(num_heads=0), dict(num_heads=2, scale=0.0), dict(num_heads=2, scale=float("nan")),
               dict(num_heads=2, scale=-1.0)):
        with pytest.raises(ValueError):
            lc.PackedPromptAttention(**kw)
    a = lc.PackedPromptAttention(4, 2, 64)
    q, k = torch.zeros(10, 4, 64, device=dev), torch.zeros(10, 2, 64, device=dev)
    cu = i32(dev, [0, 10])
    for kind, call in [
            (RuntimeError, lambda: a(q.cpu(), k, k, cu)), (ValueError, lambda: a(q.half(), k, k, cu)),
            (TypeError, lambda: a(q.double(), k.double(), k.double(), cu)), (ValueError, lambda: a(k, k, k, cu)),
            (ValueError, lambda: a(q, q, k, cu)), (ValueError, lambda: a(q, k[:9], k, cu)),
            (ValueError, lambda: a(q, k[:9], k[:9], cu)), (ValueError, lambda: a(q, k, k, cu.long())),
            (ValueError, lambda: a(q, k, k, cu.cpu())), (ValueError, lambda: a(q, k, k, cu[:1])),
            (ValueError, lambda: a(q, k, k, cu, i32(dev, [0, 5, 10]))), (ValueError, lambda: a(q, k, k, cu[None])),
            (ValueError, lambda: a(q, k, k, cu, out=q.half())), (ValueError, lambda: a(q, k, k, cu, out=q[:9])),
            (ValueError, lambda: a(q, k, k, cu, out=torch.zeros(4, 10, 64, device=dev).transpose(0, 1))),
            (RuntimeError, lambda: a(q.clone().requires_grad_(), k, k, cu))]:
        with pytest.raises(kind):
            call()
    assert a(q[:0], k[:0], k[:0], i32(dev, [0, 0])).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_serving_path(lc, dev, dtype):
    """Prompts and decode steps of one layer as a server runs them: rotate and append, attend over the
    prompt's own keys, then steps over the cache; two of the prompts arrive while the others decode.
    The prompts' rows equal attention over the rotated inputs, the steps' rows attention over what
    the cache holds."""
    import torch
    B, Hq, Hkv, D, group = 4, 8, 2, 128, 32
    cache = lc.PagedInt4KVCache(Hkv, D, num_sequences=B, max_resident_pages=24, sink_pages=1, group_size=group, device=dev)
    att = lc.PackedPromptAttention(Hq, Hkv, D)
    seen = np.zeros(B, int)
    hist = [[np.zeros((0, Hkv, D))] * 2 for _ in range(B)]

    def feed(lengths, seed):
        N = sum(lengths)
        q, k, v = (rand(dev, dtype, N, h, D, seed=seed + s) for h, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
        qr, kr = cache.append(k, v, i32(dev, seen), i32(dev, cum(lengths)), query=q, return_key=True)
        kf, hk, hv = kv4.rotate(f64(k), positions(seen, lengths), kv4.inv_freq(D, 1e6)), None, None
        hk, hv = kv4.held(kf.astype(np.float32), group), kv4.held(f64(v).astype(np.float32), group)
        for b, (lo, hi) in enumerate(zip(cum(lengths), cum(lengths)[1:])):
            hist[b] = [np.concatenate([hist[b][0], hk[lo:hi]]), np.concatenate([hist[b][1], hv[lo:hi]])]
            seen[b] += hi - lo
        return qr, kr, v

    for first in ([37, 0, 300, 0], [0, 64, 0, 129]):
        q, k, v = feed(first, 10 + first[0])
        out = att(q, k, v, i32(dev, cum(first)))
        check(out, q, k, v, cum(first), cum(first), True, D ** -0.5, dtype)
        for step in range(3):
            alive = (seen > 0).astype(int).tolist()
            qs, _, _ = feed(alive, 100 + step)
            query = torch.zeros(B, Hq, D, dtype=q.dtype, device=dev)
            query[torch.tensor(np.nonzero(alive)[0], device=dev)] = qs
            got = f64(cache.decode(query, i32(dev, seen)))
            for b in range(B):
                if not seen[b]:
                    assert (got[b] == 0).all()
                    continue
                keep = kv4.resident(seen[b], 16, 24, 1)
                for h in range(Hq):
                    want, _ = kv4.attention(f64(query)[b, h:h + 1], hist[b][0][keep, h // 4], hist[b][1][keep, h // 4], D ** -0.5)
                    V = np.abs(hist[b][1][keep, h // 4]).max()
                    tol = V * (2 ** -12 + 1e-5 if dtype == "bfloat16" else 1e-5) + eps_half(dtype) * np.abs(want[0])
                    assert (np.abs(got[b, h] - want[0]) <= tol).all(), (b, h)


@pytest.mark.parametrize("name", ["float32", "bfloat16"])
def test_out_is_the_query(lc, dev, name):
    import torch
    dtype = getattr(torch, name)
    g = torch.Generator(device=dev).manual_seed(4)
    cu = torch.tensor([0, 70, 70, 301], dtype=torch.int32, device=dev)
    q, k, v = (torch.randn(301, h, 64, generator=g, device=dev).to(dtype) for h in (4, 2, 2))
    a = lc.PackedPromptAttention(4, 2, 64)
    want = a(q, k, v, cu)
    assert a(q, k, v, cu, out=q) is q and torch.equal(q, want)


MANY = LENGTHS + [300, 1, 95, 260, 0, 32, 128, 17, 250, 3, 63, 190, 64, 1, 97, 33, 5]


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [
    (32, 32, 64, "float16"), (32, 8, 128, "bfloat16"), (16, 16, 128, "float16"), (32, 16, 96, "bfloat16"),
    (16, 8, 256, "bfloat16")])
def test_more_workgroups_than_are_resident(lc, dev, Hq, Hkv, D, dtype):
    """Grids past the rule that splits a tile's keys over two waves: more workgroups (of up to four
    heads and 128 rows by head) than the 768, 512 or 256 that it has by head dim.  Infinities and
    NaN in the second half of the longest prompt's keys reach no row before them."""
    N, cu = sum(MANY), cum(MANY)
    share = Hq // Hkv
    heads = min(share & -share, 4)
    assert (N * heads // 128 + len(MANY) + 2) * (Hq // heads) > (768 if D <= 64 else 512 if D <= 128 else 256)
    q, k, v = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
    a = lc.PackedPromptAttention(Hq, Hkv, D)
    out, lse = a(q, k, v, i32(dev, cu), return_lse=True)
    check(out, q, k, v, cu, cu, True, D ** -0.5, dtype, lse)
    b = MANY.index(300)
    lo, mid = cu[b], cu[b] + 150
    k[mid:lo + 300:2] = float("inf")
    k[mid + 1:lo + 300:2] = float("nan")
    v[mid:lo + 300] = float("-inf")
    out = a(q, k, v, i32(dev, cu))
    check(out[lo:mid], q[lo:mid], k[lo:mid], v[lo:mid], [0, 150], [0, 150], True, D ** -0.5, dtype)
    assert out[mid:lo + 300].isnan().all()
