"""PackedPromptAttention on the GPU at the ends of its range: scores of -inf, past what fp32 tells
apart, weights below fp16's steps, infinities and NaN that many rows see; prompts over keys read back
from the 4-bit cache.  The oracle is oracle/kv4.py in fp64."""
import math

import numpy as np
import pytest

from oracle import kv4
from test_gpu_kv4 import cum, eps_half, f64, i32, positions, rand, want_kv
from test_gpu_prompt import check

pytestmark = pytest.mark.gpu

TYPES = ["bfloat16", "float16", "float32"]


@pytest.fixture(scope="module")
def lc(pkg):
    from importlib import import_module
    return import_module(pkg.__name__ + ".long_context")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_scores_of_minus_infinity(lc, dev, dtype, causal):
    """A row whose keys all score -inf has no softmax: NaN, as the definition gives, with a
    log-sum-exp of -inf.  Only a row that sees no key is 0."""
    import torch
    N, D = 150, 64
    q, k, v = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((4, 1), (2, 2), (2, 3)))
    k[..., 5] = k[..., 5].abs() + 0.5
    bad = torch.zeros(N, 4, dtype=torch.bool, device=dev)
    bad[::31, 0] = bad[149, 3] = True
    q2 = q.clone()
    q2[..., 5][bad] = -float("inf")
    a = lc.PackedPromptAttention(4, 2, D, causal=causal)
    out, lse = a(q2, k, v, i32(dev, [0, N]), return_lse=True)
    assert torch.isnan(out[bad]).all() and (lse[bad] == -math.inf).all()
    out[bad], lse[bad] = (x[bad] for x in a(q, k, v, i32(dev, [0, N]), return_lse=True))
    check(out, q, k, v, [0, N], [0, N], causal, D ** -0.5, dtype, lse)
    # queries before the first key see none: 0, whatever they hold
    few = a(q2, k[:7], v[:7], i32(dev, [0, N]), i32(dev, [0, 7]))
    if causal:
        assert not few[:N - 7].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_small_weights(lc, dev, dtype, D):
    """One key that takes nearly all the weight and 60000 that have about 2^-25 of it each: their sum
    is a share of 2^-9, held as exactly as any other."""
    import torch
    n, scale = 60000, 1.0
    k = torch.zeros(n, 1, D, device=dev)
    k[7, 0, 0] = 25.4 / 1.4427                             # log2 distance 25.4 to the others
    k = k.to(getattr(torch, dtype))
    v = torch.ones(n, 1, D, device=dev).to(k.dtype)
    v[7] = 0
    q = torch.zeros(3, 2, D, device=dev).to(k.dtype)
    q[..., 0] = 1
    a = lc.PackedPromptAttention(2, 1, D, causal=False, scale=scale)
    got = f64(a(q, k, v, i32(dev, [0, 3]), i32(dev, [0, n])))
    far = math.exp(-float(k[7, 0, 0]))
    want = (n - 1) * far / (1 + (n - 1) * far)
    # equal weights, so their roundings to the inputs' type are all alike: half a step of that type,
    # of weights and sum; the fp32 sums of 60000 equal terms in blocks of 32, held to 2^-12
    tol = want * (2 * eps_half(dtype) + 2 ** -12)
    if dtype == "float16":
        # weights of 2^-25.4 times 2^7 are among fp16's subnormals, 2^-24 apart: each is off by half of
        # that, 2^-32 of the row's largest, all alike
        tol += n * 2 ** -32
    assert (np.abs(got - want) <= tol + 1e-7 * (dtype == "float16")).all(), (got.ravel()[:4], want)


@pytest.mark.parametrize("dtype,D", [(t, D) for t in TYPES for D in (64, 128, 256)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (16, 16)])
def test_infinities_that_many_rows_see(lc, dev, dtype, D, bad, Hq, Hkv):
    """One value, one key entry that later rows see and earlier rows do not, in prompts of several
    tiles and blocks: the value reaches its own dimension of the rows that see it, as itself; the
    key's rows are what their dot products give; all else is as ever."""
    import torch
    lengths = [450, 70, 333]
    N, cu = sum(lengths), cum(lengths)
    q, k, v = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
    share = Hq // Hkv
    a = lc.PackedPromptAttention(Hq, Hkv, D)
    v2, k2 = v.clone(), k.clone()
    v2[140, 0, 3] = v2[cu[1] + 69, 1, 5] = bad             # a value of sequence 0, the last of sequence 1
    k2[cu[2] + 100, 1, 2] = bad                            # a key of sequence 2
    out, lse = a(q, k2, v2, i32(dev, cu), return_lse=True)
    got = f64(out)
    seen = np.zeros(got.shape, bool)
    seen[140:450, :share, 3] = seen[cu[1] + 69, share:2 * share, 5] = True
    if math.isnan(bad):
        assert np.isnan(got[seen]).all()
    else:
        assert (got[seen] == bad).all()
    # of the key's rows those whose score is +inf or NaN are NaN; a score of -inf weighs nothing
    rows = slice(cu[2] + 100, N)
    score = f64(q)[rows, share:2 * share, 2] * bad
    lost = ~(score == -math.inf)
    assert np.isnan(got[rows, share:2 * share][lost]).all()
    seen[rows, share:2 * share] |= lost[..., None]
    for b in range(3):
        s = slice(cu[b], cu[b + 1])
        n = lengths[b]
        for h in range(Hq):
            kh, vh = f64(k2)[s, h // share], f64(v2)[s, h // share]
            # the oracle's sums have no infinite or NaN terms: a key that scores -inf is left out by
            # rows of its own, values at `seen` are not compared
            vh = np.where(np.isfinite(vh), vh, 0)
            clean, _ = kv4.attention(f64(q)[s, h], f64(k)[s, h // share], vh, D ** -0.5, np.arange(n) + 1)
            if b == 2 and h // share == 1:
                x = f64(q)[s, h]
                for i in range(100, n):
                    if not lost[i - 100, h - share]:
                        keep = np.r_[0:100, 101:i + 1]
                        clean[i] = kv4.attention(x[i:i + 1], kh[keep], vh[keep], D ** -0.5)[0][0]
            absw = np.abs(vh).max()
            score_err = 2 ** -24 * (16 * D ** -0.5 * np.abs(f64(q)[s, h]).max(0) @ np.abs(f64(k)[s, h // share]).max(0) + 30)
            tol = absw * (2 * score_err + (eps_half(dtype) if dtype != "float32" else 0) + 2 ** -22)
            tol = tol + eps_half(dtype) * np.abs(clean) + 1e-7 * (dtype == "float16")
            ok = (np.abs(got[s, h] - clean) <= tol) | seen[s, h]
            assert ok.all(), (b, h, np.argwhere(~ok)[:3])


@pytest.mark.parametrize("dtype", TYPES)
def test_huge_finite_values(lc, dev, dtype):
    """Values at the type's largest (past bfloat16's range for float32): finite weights of them are
    finite, hidden ones reach nothing."""
    import torch
    n, D = 200, 128
    most = torch.finfo(getattr(torch, dtype)).max
    q, k, v = (rand(dev, dtype, n, h, D, seed=s) for h, s in ((2, 1), (1, 2), (1, 3)))
    k.zero_()                                              # weights of 1: the sums stay in range
    v[150, 0] = most
    v[90, 0, :7] = -most
    out = f64(lc.PackedPromptAttention(2, 1, D)(q, k, v, i32(dev, [0, n])))
    for h in range(2):
        want, _ = kv4.attention(f64(q)[:, h], f64(k)[:, 0], f64(v)[:, 0], D ** -0.5, np.arange(n) + 1)
        absw, _ = kv4.attention(f64(q)[:, h], f64(k)[:, 0], np.abs(f64(v)[:, 0]), D ** -0.5, np.arange(n) + 1)
        score = 2 ** -24 * (16 * D ** -0.5 * np.abs(f64(q)[:, h]).max(0) @ np.abs(f64(k)[:, 0]).max(0) + 30)
        # the sums of equal weights run key by key over up to 95 keys where a tile has hidden values:
        # as many half steps of fp32, at worst, and 33 for the rest
        tol = absw * (2 * score + (eps_half(dtype) if dtype != "float32" else 0) + 2 ** -17) + eps_half(dtype) * np.abs(want)
        assert (np.abs(out[:, h] - want) <= tol + 1e-7 * (dtype == "float16")).all()


def test_a_nan_does_not_stall_a_batch(lc, dev):
    """One NaN among the values that almost all rows see costs a second pass, not a walk over every
    key: a call of 4096 tokens takes less than six times as long with it."""
    import torch
    n, D = 4096, 128
    q, k, v = (rand(dev, "bfloat16", n, h, D, seed=s) for h, s in ((32, 1), (8, 2), (8, 3)))
    a = lc.PackedPromptAttention(32, 8, D)
    cu = i32(dev, [0, n])

    def took(v):
        a(q, k, v, cu)
        best = math.inf
        for _ in range(5):
            t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            t[0].record()
            a(q, k, v, cu)
            t[1].record()
            torch.cuda.synchronize()
            best = min(best, t[0].elapsed_time(t[1]))
        return best

    v2 = v.clone()
    v2[100, :, 3] = float("nan")
    assert took(v2) < 6 * took(v)


@pytest.mark.parametrize("dtype,Hq,Hkv,n", [("bfloat16", 4, 2, 400), ("bfloat16", 32, 32, 900), ("float32", 4, 1, 300),
                                            ("bfloat16", 32, 8, 3000), ("float16", 48, 48, 2500)])
def test_out_is_the_query_with_a_nan(lc, dev, dtype, Hq, Hkv, n):
    """A second pass reads the queries again: rows already written into them take no part."""
    import torch
    q, k, v = (rand(dev, dtype, n, h, 64, seed=s) for h, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
    v[n // 2, 0, 3] = float("nan")
    k[n // 3, Hkv - 1, 3] = float("inf")
    cu = i32(dev, [0, 3, 3, n - 50, n])
    a = lc.PackedPromptAttention(Hq, Hkv, 64)
    want, lse = a(q, k, v, cu, return_lse=True)
    got, l2 = a(q, k, v, cu, out=q, return_lse=True)
    assert got is q and torch.equal(q.isnan(), want.isnan()) and torch.equal(q.nan_to_num(7), want.nan_to_num(7))
    assert torch.equal(l2.nan_to_num(7), lse.nan_to_num(7)) and want.isnan().any()


@pytest.mark.parametrize("dtype,size", [("bfloat16", 3e3), ("bfloat16", 3e4), ("bfloat16", 1e8), ("bfloat16", 1e15),
                                        ("float16", 3e3), ("float16", 6e3), ("float32", 3e4), ("float32", 1e8),
                                        ("float32", 1e15)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_far_apart(lc, dev, dtype, size, D):
    """Scores of 2^23 to 2^100 and as far apart: all weight on the largest, which fp32 still tells from
    the next (rows where it does not are left out: a few)."""
    import torch
    n, scale = 200, D ** -0.5
    q, k, v = (rand(dev, dtype, n, h, D, seed=s) for h, s in ((2, 1), (1, 2), (1, 3)))
    q, k = ((x * size).to(x.dtype) for x in (q, k))
    out, lse = lc.PackedPromptAttention(2, 1, D)(q, k, v, i32(dev, [0, n]), return_lse=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    qf, kf, vf, o = f64(q), f64(k)[:, 0], f64(v)[:, 0], f64(out)
    taken = 0
    for h in range(2):
        for i in range(n):
            s = kf[:i + 1] @ qf[i, h] * scale
            top = np.argsort(s)[::-1]
            err = 16 * 2 ** -24 * scale * (np.abs(kf[:i + 1]).max(0) * np.abs(qf[i, h])).sum()
            assert abs(f64(lse)[i, h] - s.max()) <= 2 * err + 1
            if i and s[top[0]] - s[top[1]] < 2 * err + 40:
                continue
            taken += 1
            want = vf[top[0]]
            assert (np.abs(o[i, h] - want) <= (eps_half(dtype) + 2 ** -21) * np.abs(want) + 1e-7 * (dtype == "float16")).all()
    assert taken > n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(5, 5, 128), (3, 1, 64), (20, 4, 64), (7, 7, 256)])
def test_single_rows_over_long_keys(lc, dev, dtype, Hq, Hkv, D):
    """One to 33 rows of each sequence over some hundred keys, head counts that leave waves of a
    workgroup without rows: these add nothing, and a NaN in the last row's query stays in it."""
    nq, nk = [1, 1, 0, 33, 2], [700, 1, 30, 400, 65]
    q, k, v = rand(dev, dtype, sum(nq), Hq, D, seed=1), rand(dev, dtype, sum(nk), Hkv, D, seed=2), \
        rand(dev, dtype, sum(nk), Hkv, D, seed=3)
    a = lc.PackedPromptAttention(Hq, Hkv, D)
    out, lse = a(q, k, v, i32(dev, cum(nq)), i32(dev, cum(nk)), return_lse=True)
    check(out, q, k, v, cum(nq), cum(nk), True, D ** -0.5, dtype, lse)
    q[-1, 0, 0] = float("nan")
    got = a(q, k, v, i32(dev, cum(nq)), i32(dev, cum(nk)))
    assert got[-1, 0].isnan().all() and got.isnan().sum() == D
    got[-1, 0] = out[-1, 0]
    q[-1, 0, 0] = 0
    check(got[:-1], q[:-1], k[:-65], v[:-65], cum(nq[:-1]), cum(nk[:-1]), True, D ** -0.5, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_over_the_cache(lc, dev, dtype):
    """A prompt that arrives in parts: each part's rows over all the sequence's keys so far, read back
    from the 4-bit cache, through cu_seqlens_kv."""
    import torch
    Hq, Hkv, D, group = 4, 2, 128, 32
    cache = lc.PagedInt4KVCache(Hkv, D, num_sequences=2, max_resident_pages=32, group_size=group, device=dev)
    a = lc.PackedPromptAttention(Hq, Hkv, D)
    seen, dt = np.zeros(2, int), getattr(torch, dtype)
    hist = [[np.zeros((0, Hkv, D))] * 2 for _ in range(2)]
    for part, lengths in enumerate(([100, 7], [65, 0], [1, 200], [130, 33])):
        N = sum(lengths)
        q, k, v = (rand(dev, dtype, N, h, D, seed=10 * part + s) for h, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
        qr, _ = cache.append(k, v, i32(dev, seen), i32(dev, cum(lengths)), query=q)
        _, hk, hv = want_kv(k, v, positions(seen, lengths), D, group)
        for b, (lo, hi) in enumerate(zip(cum(lengths), cum(lengths)[1:])):
            hist[b] = [np.concatenate([hist[b][0], hk[lo:hi]]), np.concatenate([hist[b][1], hv[lo:hi]])]
            seen[b] += hi - lo
        ck = cum(seen)
        rk, rv = cache.read(i32(dev, [0, 0]), i32(dev, ck), ck[-1], dtype=dt)
        for got, i in ((rk, 0), (rv, 1)):
            want = torch.from_numpy(np.concatenate([hist[0][i], hist[1][i]]).astype(np.float32)).to(dt)
            assert torch.equal(got.cpu(), want)
        out = a(qr, rk, rv, i32(dev, cum(lengths)), i32(dev, ck))
        check(out, qr, rk, rv, cum(lengths), ck, True, D ** -0.5, dtype)


@pytest.mark.parametrize("dtype,H,D", [("bfloat16", 80, 64), ("float16", 64, 128), ("bfloat16", 64, 128), ("float16", 32, 256),
                                       ("float16", 80, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_infinities_in_large_grids(lc, dev, dtype, H, D, causal):
    """As test_infinities_that_many_rows_see, past the rule that splits a tile's keys over two waves: each
    wave has rows of its own, and those without a NaN are written before the second pass."""
    import torch
    lengths = [450, 70, 333]
    N, cu = sum(lengths), cum(lengths)
    assert (N // 128 + 5) * H > (768 if D <= 64 else 512 if D <= 128 else 256)
    q, k, v = (rand(dev, dtype, N, H, D, seed=s) for s in (1, 2, 3))
    a = lc.PackedPromptAttention(H, H, D, causal=causal)
    v2 = v.clone()
    inf = float("inf")
    v2[140, 0, 3], v2[200, 0, 4], v2[300, 0, 4], v2[cu[1] + 69, 1, 5], v2[310, H - 1, 6] = inf, -inf, inf, -inf, float("nan")
    out, lse = a(q, k, v2, i32(dev, cu), return_lse=True)
    got, l2 = f64(out), f64(lse)
    for b in range(3):
        s, n = slice(cu[b], cu[b + 1]), lengths[b]
        for h in (0, 1, 2, H - 1):
            x, K, V = f64(q)[s, h], f64(k)[s, h], f64(v2)[s, h]
            sc = x @ K.T * D ** -0.5
            if causal:
                sc = np.where(np.tri(n, dtype=bool), sc, -np.inf)
            w = np.exp(sc - sc.max(1, keepdims=True))
            total = w.sum(1, keepdims=True)
            seen = np.tri(n) if causal else np.ones((n, n))
            up, down, nan = (seen @ m for m in (V == inf, V == -inf, np.isnan(V)))
            F = np.where(np.isfinite(V), V, 0)
            want = (w @ F) / total
            score = 2 ** -24 * (16 * D ** -0.5 * np.abs(x).max(0) @ np.abs(K).max(0) + 30)
            tol = (w @ np.abs(F)) / total * (2 * score + eps_half(dtype) + 2 ** -21) + eps_half(dtype) * np.abs(want) + 1e-7
            ok = np.abs(got[s, h] - want) <= tol
            g = got[s, h]
            both = (up > 0) & (down > 0) | (nan > 0)
            ok = np.where(both, np.isnan(g), np.where(up > 0, g == inf, np.where(down > 0, g == -inf, ok)))
            assert ok.all(), (b, h, np.argwhere(~ok)[:3])
            want_l = (sc.max(1, keepdims=True) + np.log(total))[:, 0]
            assert (np.abs(l2[s, h] - want_l) <= score + 2 ** -21 * (1 + np.abs(want_l))).all()
