"""PagedInt4KVCache.decode and append on the GPU at the ends of their ranges: queries of zeros,
scores past what fp32 tells apart or holds, single tokens of large batches, rows whose layout torch
calls contiguous.  The oracle is oracle/kv4.py in fp64."""
import numpy as np
import pytest

from oracle import kv4
from test_gpu_kv4 import check_decode, cum, decode_case, eps_half, f64, i32, positions, rand, want_kv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc(pkg):
    from importlib import import_module
    return import_module(pkg.__name__ + ".long_context")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("share", [1, 4])
def test_decode_query_of_zeros(lc, dev, dtype, share):
    """A head of zeros weighs all tokens alike, at every scale: the mean of the held values, also
    where the last tile is not full.  The other heads beside it keep their results."""
    lengths = [1, 37, 64, 100, 500, 0]
    c, q, hk, hv = decode_case(lc, dev, 128, 32, dtype, 16, 2, share, lengths, 64)
    q[:, 0] = 0
    q[3] = 0
    for scale in (-1.0, 4e-8, 1e-30, 1e-45):
        out = c.decode(q, i32(dev, lengths), scale)
        check_decode(out, q, hk, hv, lengths, share, dtype, 128 ** -0.5 if scale < 0 else scale, 32)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("share", [1, 4])
def test_decode_scores_of_minus_infinity(lc, dev, dtype, share):
    """A head whose held tokens all score -inf has no softmax: NaN, as the definition gives.  A
    sequence without tokens, or with unmapped pages alone, stays 0."""
    import torch
    lengths = [1, 70, 300, 0, 20]
    N, D = sum(lengths), 64
    c = lc.PagedInt4KVCache(2, D, num_sequences=5, max_resident_pages=32, rope_theta=None, device=dev, num_pages=160)
    c.block_table.copy_(torch.arange(160, dtype=torch.int32, device=dev).view(5, 32))
    k = torch.ones(N, 2, D, device=dev)
    k[..., 0] = 2                                          # lo 1, step 1 / 15, code 15: both terms of one sign
    k = k.to(getattr(torch, dtype))
    v = rand(dev, dtype, N, 2, D, seed=1)
    c.append(k, v, i32(dev, [0] * 5), i32(dev, cum(lengths)))
    c.block_table[4] = -1
    q = rand(dev, dtype, 5, 2 * share, D, seed=2)
    q[:, 0, 0] = -float("inf")
    out = c.decode(q, i32(dev, lengths))
    assert torch.isnan(out[:3, 0]).all()
    assert torch.isfinite(out[:, 1:]).all() and not out[3:].any()
    hk, hv = kv4.held(f64(k).astype(np.float32), 32), kv4.held(f64(v).astype(np.float32), 32)
    q[:, 0], out[:3, 0] = 0, 0
    hv0 = hv.copy()
    if share == 1:
        hv0[:, 0] = 0                                      # head 0 is the one left out
        check_decode(out[:3], q[:3], hk, hv0, lengths[:3], share, dtype, 0.125, 32)


@pytest.mark.parametrize("share", [1, 4])
def test_decode_some_scores_past_fp32(lc, dev, share):
    """Tokens whose score is below every fp32 value have no weight beside tokens that have one,
    whichever wave or run they lie in."""
    import torch
    for first in (1, 64, 130, 1000):
        n, D = first + 137, 64
        c = lc.PagedInt4KVCache(1, D, max_resident_pages=128, rope_theta=None, device=dev)
        k = torch.zeros(n, 1, D, device=dev)
        k[:first] = 6e4
        v = rand(dev, "float32", n, 1, D, seed=first)
        c.append(k, v, i32(dev, [0]), i32(dev, [0, n]))
        q = torch.full((1, share, D), -3e38, device=dev)
        hv = kv4.held(f64(v).astype(np.float32), 32)[first:, 0]
        # weights are equal: sums of 137 values in fp32, a pairwise order's error held to 16 half steps
        got = f64(c.decode(q, i32(dev, [n])))[0]
        assert (np.abs(got - hv.mean(0)) <= 16 * 2 ** -24 * np.abs(hv).max()).all(), first


@pytest.mark.parametrize("dtype,size", [("bfloat16", 1e2), ("bfloat16", 3e4), ("bfloat16", 1e8), ("bfloat16", 1e15),
                                        ("float16", 1e3), ("float16", 6e3), ("float32", 3e4), ("float32", 1e8),
                                        ("float32", 1e15)])
@pytest.mark.parametrize("share", [1, 4])
def test_decode_scores_far_apart(lc, dev, dtype, size, share):
    """Scores of 2^17 to 2^60 and as far apart: all weight on the largest, which fp32 still tells
    from the next (a head where it does not, by the scores' error in fp32, is only finite)."""
    import torch
    n, D, scale = 333, 128, 128 ** -0.5
    c = lc.PagedInt4KVCache(1, D, max_resident_pages=64, rope_theta=None, device=dev)
    k, v = rand(dev, dtype, n, 1, D, seed=1) * 5e3, rand(dev, dtype, n, 1, D, seed=2)
    q = (rand(dev, dtype, 1, share, D, seed=3) * size).to(getattr(torch, dtype))
    c.append(k, v, i32(dev, [0]), i32(dev, [0, n]))
    hk, hv = kv4.held(f64(k).astype(np.float32), 32)[:, 0], kv4.held(f64(v).astype(np.float32), 32)[:, 0]
    got = f64(c.decode(q, i32(dev, [n])))[0]
    taken = 0
    for h in range(share):
        x = f64(q)[0, h]
        s = hk @ x * scale
        top = np.argsort(s)[::-1]
        err = 16 * 2 ** -24 * 3 * (np.abs(x) * np.abs(hk).max(0)).sum() * scale      # as check_decode
        assert np.abs(s).max() * 1.4427 > 2 ** 17 and np.isfinite(got[h]).all()
        if s[top[0]] - s[top[1]] <= 2 * err + 40:
            continue
        taken += 1
        want = hv[top[0]]
        # one weight: fp16 of 2^-12 (bf16 outputs), two pieces else; the output rounds once
        tol = np.abs(hv).max() * (2 ** -12 if dtype == "bfloat16" else 2 ** -21) + eps_half(dtype) * np.abs(want)
        assert (np.abs(got[h] - want) <= tol + 1e-7 * (dtype == "float16")).all(), (h, got[h][:4], want[:4])
    assert 4 * taken >= 3 * share


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_append_of_one_row_of_a_wider_projection(lc, dev, dtype):
    """One token, or one kv head, of a tensor whose other strides are not 16-byte: as contiguous copies."""
    import torch
    wide = rand(dev, dtype, 7, 259, seed=1)
    token = wide[:, :256].view(7, 4, 64)[3:4]
    head = rand(dev, dtype, 5, 64, 1, seed=2).transpose(1, 2)
    for t, heads in ((token, 4), (head, 1)):
        n = len(t)
        got, want = (lc.PagedInt4KVCache(heads, 64, device=dev) for _ in range(2))
        s, cu = i32(dev, [3]), i32(dev, [0, n])
        a = got.append(t, t, s, cu, query=t, return_key=True)
        p = torch.empty(t.shape, dtype=t.dtype, device=dev).copy_(t)
        b = want.append(p, p, s, cu, query=p, return_key=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(got.k_codes, want.k_codes)
        at = lc.PackedPromptAttention(heads, heads, 64)
        assert torch.equal(at(t, t, t, cu), at(p, p, p, cu))


def test_forward_tangents_are_refused(lc, dev):
    """A dual tensor's tangent would be lost without a word: refused, also under no_grad, which keeps
    forward mode on."""
    import torch
    import torch.autograd.forward_ad as fw
    c = lc.PagedInt4KVCache(2, 64, num_sequences=3, max_resident_pages=4, device=dev)
    a = lc.PackedPromptAttention(2, 2, 64)
    k, s, cu = torch.randn(3, 2, 64, device=dev), i32(dev, [0, 0, 0]), i32(dev, [0, 3])
    with fw.dual_level():
        d = fw.make_dual(k, torch.ones_like(k))
        calls = [lambda x: c.append(x, k, s), lambda x: c.append(k, x, s), lambda x: c.append(k, k, s, query=x),
                 lambda x: c.decode(x, s + 1), lambda x: a(x, k, k, cu), lambda x: a(k, x, k, cu), lambda x: a(k, k, x, cu)]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(d)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(d)
            call(k), call(fw.unpack_dual(d).primal)
            with torch.inference_mode():
                call(k)


def test_counts_past_an_int_are_refused(lc, dev):
    """Rows of stride 0 can be more than 2^32: their count must not lose its high bits on the way."""
    import torch
    c = lc.PagedInt4KVCache(1, 64, max_resident_pages=4, rope_theta=None, device=dev)
    a = lc.PackedPromptAttention(1, 1, 64)
    row = torch.ones(1, 1, 64, device=dev)
    many = row.expand(2 ** 32 + 3, 1, 64)
    cu = i32(dev, [0, 3])
    for call in (lambda: c.append(many, many, i32(dev, [0]), cu), lambda: a(row, many, many, i32(dev, [0, 1]), cu)):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    assert not c.k_steps.any()


def test_single_tokens_of_a_large_batch(lc, dev):
    """Append and read of one token a sequence with one wave for a whole token (more than 4096 waves)."""
    import torch
    B = 5000
    c = [lc.PagedInt4KVCache(2, 64, num_sequences=B, max_resident_pages=7, device=dev) for _ in range(2)]
    k, v, q = (rand(dev, "bfloat16", B, h, 64, seed=s) for s, h in enumerate((2, 2, 6)))
    starts = [7 * b % 100 for b in range(B)]
    start = i32(dev, starts)
    a = c[0].append(k, v, start, query=q)[0]
    b = c[1].append(k, v, start, i32(dev, range(B + 1)), query=q)[0]
    assert torch.equal(a, b)
    _, hk, hv = want_kv(k, v, np.array(starts), 64, 32)
    for x, y, want in zip(c[0].read(start), c[1].read(start, i32(dev, range(B + 1)), B), (hk, hv)):
        assert torch.equal(x, y) and np.array_equal(f64(x), want.astype(np.float32).astype(np.float64))
    qf = kv4.rotate(f64(q), starts, kv4.inv_freq(64, 1e6))
    assert (np.abs(f64(a) - qf) <= 2 * eps_half("bfloat16") * np.abs(qf)).all()


@pytest.mark.parametrize("name", ["k_codes", "v_codes", "k_steps", "v_steps", "block_table"])
def test_buffers_are_filled_in_not_replaced(lc, dev, name):
    """The kernels hold the buffers' addresses: a tensor put in a buffer's place would be ignored, and
    the memory that they go on writing freed."""
    c = lc.PagedInt4KVCache(1, 64, max_resident_pages=4, device=dev)
    t = getattr(c, name)
    with pytest.raises(AttributeError):
        setattr(c, name, t.clone())
    assert getattr(c, name) is t


def test_two_streams_at_once(lc, dev):
    """Decodes of one cache and prompts on two streams at the same time, one prompt with a NaN that
    takes its second pass: each has its own workspace, the results are the calls' own."""
    import torch
    c, q, hk, hv = decode_case(lc, dev, 128, 32, "bfloat16", 16, 2, 4, [900, 3, 2000, 77], 128)
    seen, n = i32(dev, [900, 3, 2000, 77]), 700
    pq, pk, pv = (rand(dev, "bfloat16", n, h, 128, seed=s) for h, s in ((8, 1), (2, 2), (2, 3)))
    pn = pv.clone()
    pn[100, 0, 3] = float("nan")
    a, cu = lc.PackedPromptAttention(8, 2, 128), i32(dev, [0, 300, n])
    qs = [q, q * 0.5]
    want = [(c.decode(x, seen), a(pq, pk, v, cu)) for x, v in zip(qs, (pv, pn))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((c.decode(qs[i], seen), a(pq, pk, (pv, pn)[i], cu)))
    torch.cuda.synchronize()
    for i in range(2):
        for d, p in got[i]:
            assert torch.equal(d, want[i][0]) and torch.equal(p.nan_to_num(7), want[i][1].nan_to_num(7))
