"""PagedEvictingKVCache on the GPU against the fp64 oracle (oracle/kve.py, oracle/kv4.py): append with
rotation, decode attention with counted weights and eviction, at lengths, pages, masks and layouts
where they can go wrong."""
import math

import numpy as np
import pytest

from oracle import kv4, kve

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


def half_step(dtype):
    import torch
    return torch.finfo(getattr(torch, dtype)).eps / 2


def shuffled(c, seed):
    """Every sequence's pages at random places of the pool."""
    import torch
    r = np.random.default_rng(seed)
    p = r.permutation(c.num_pages)[:c.num_sequences * c.max_pages].astype(np.int32)
    c.block_table.copy_(torch.from_numpy(p.reshape(c.num_sequences, c.max_pages)))
    return c


def place(c, b, t):
    """(pages, slots) of slots t of sequence b."""
    table = c.block_table[b].cpu().numpy()
    return table[np.asarray(t) // c.page_size], np.asarray(t) % c.page_size


SHAPES = [  # D, dtype, page, kv heads, query heads, rotary, interleaved
    (128, "bfloat16", 16, 8, 32, 128, False),
    (128, "float32", 32, 1, 3, 128, False),
    (128, "float16", 16, 3, 3, 64, False),
    (128, "bfloat16", 64, 2, 10, 128, True),
    (64, "float32", 16, 5, 5, 32, True),
    (64, "bfloat16", 128, 4, 4, 64, False),
    (256, "float16", 16, 1, 16, 256, False),
    (256, "float32", 16, 2, 2, 16, False),
    (256, "bfloat16", 32, 2, 6, 48, True),
]


@pytest.mark.parametrize("D,dtype,page,Hkv,Hq,rot,inter", SHAPES)
def test_append(lc, dev, D, dtype, page, Hkv, Hq, rot, inter):
    """Keys and queries are the rotation's fp64 values rounded to fp32 and to the type: two half steps.
    Values are copied; slots that nothing is written to stay as they are."""
    import torch
    lengths, starts, at = [37, 0, 1, 90, 16], [0, 5, 75, 15, 64], [0, 7, 1 << 20, 70001, 64]
    B, N = len(lengths), sum(lengths) + 3        # the last three rows belong to no sequence
    c = shuffled(lc.PagedEvictingKVCache(Hkv, D, num_sequences=B, page_size=page, max_pages=-(-128 // page),
                                         num_pages=B * -(-128 // page) + 2, rope_theta=THETA, rotary_dim=rot,
                                         interleaved=inter, dtype=getattr(torch, dtype), device=dev), 1)
    assert c.keys.dtype == getattr(torch, dtype) and c.capacity == max(128, page)
    c.keys.fill_(7.0), c.values.fill_(8.0), c.weights.fill_(9.0), c.positions.fill_(-3)
    k, v, q = (rand(dev, dtype, N, h, D, seed=s) for h, s in ((Hkv, 1), (Hkv, 2), (Hq, 3)))
    v[5, 0, 3], v[6, 0, 4] = math.nan, -math.inf
    w = torch.rand(N, Hkv, device=dev)
    kept = [t.clone() for t in (k, v, q, w)]
    qr = c.append(k, v, i32(dev, starts), i32(dev, cum(lengths)), position=i32(dev, at), query=q, weight=w)
    assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in zip((k, v, q, w), kept))
    freq, e = kv4.inv_freq(rot, THETA), 2 * half_step(dtype)
    tiny = 1e-7 * (dtype == "float16")
    seen = np.zeros((c.num_pages, page), bool)
    for b, (first, n) in enumerate(zip(cum(lengths), lengths)):
        pos, rows = at[b] + np.arange(n), slice(first, first + n)
        pages, slots = place(c, b, starts[b] + np.arange(n))
        seen[pages, slots] = True
        want = kv4.rotate(f64(k[rows]), pos, freq, inter)
        got = f64(c.keys)[pages, :, slots]
        assert (np.abs(got - want) <= e * np.abs(want) + tiny).all()
        want = kv4.rotate(f64(q[rows]), pos, freq, inter)
        assert (np.abs(f64(qr[rows]) - want) <= e * np.abs(want) + tiny).all()
        assert np.array_equal(f64(c.values)[pages, :, slots], f64(v[rows]), equal_nan=True)
        assert np.array_equal(f64(c.weights)[pages, :, slots], f64(w[rows]))
        assert (c.positions.cpu().numpy()[pages, :, slots] == pos[:, None]).all()
    assert not qr[sum(lengths):].any()
    rest = ~seen
    for t, was in ((c.keys, 7), (c.values, 8), (c.weights, 9), (c.positions, -3)):
        x = t.float().cpu().numpy()
        assert (np.moveaxis(x, 1, 2)[rest] == was).all()


def test_append_single_tokens(lc, dev):
    """One token a sequence: the same as with cu_seqlens, at a batch on each side of the launch's split."""
    import torch
    for B in (1, 3, 300):
        c = [lc.PagedEvictingKVCache(2, 64, num_sequences=B, max_pages=8, device=dev) for _ in range(2)]
        k, v, q = (rand(dev, "bfloat16", B, h, 64, seed=h) for h in (2, 2, 6))
        start = i32(dev, [7 * b % 100 for b in range(B)])
        a = c[0].append(k, v, start, query=q)
        b = c[1].append(k, v, start, i32(dev, range(B + 1)), query=q)
        assert torch.equal(a, b) and torch.equal(c[0].keys, c[1].keys) and torch.equal(c[0].values, c[1].values)
        assert torch.equal(c[0].positions, c[1].positions) and c[0].keys.any() and not c[0].weights.any()


def test_append_past_the_pages(lc, dev):
    """Slots past the sequence's pages, below 0 and of pages that are not there are not written; their
    queries are rotated all the same."""
    import torch
    c = lc.PagedEvictingKVCache(1, 64, num_sequences=3, page_size=16, max_pages=2, num_pages=6, dtype=torch.float32,
                                device=dev)
    c.block_table.copy_(torch.tensor([[0, 1], [2, -1], [99, 3]], dtype=torch.int32))
    k, v = rand(dev, "float32", 60, 1, 64, seed=1), rand(dev, "float32", 60, 1, 64, seed=2)
    q = c.append(k, v, i32(dev, [20, 10, -5]), i32(dev, [0, 20, 40, 60]), position=i32(dev, [0, 0, 0]), query=k)
    pos = np.tile(np.arange(20), 3)
    want = kv4.rotate(f64(k), pos, kv4.inv_freq(64, 1e6))
    assert (np.abs(f64(q) - want) <= 2 * 2.0 ** -24 * np.abs(want) + 1e-12).all()
    written = {(1, s) for s in range(4, 16)} | {(2, s) for s in range(10, 16)}
    there = c.values[:, 0].abs().sum(-1).cpu().numpy() > 0
    assert {(p, s) for p, s in zip(*there.nonzero())} == written


def test_append_of_any_strides(lc, dev):
    import torch
    c = [lc.PagedEvictingKVCache(2, 128, num_sequences=1, max_pages=4, dtype=torch.float32, device=dev) for _ in range(2)]
    fused = rand(dev, "float32", 40, 8, 128, seed=1)           # 4 query heads, 2 kv heads of keys and values
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    s, cu = i32(dev, [3]), i32(dev, [0, 40])
    a = c[0].append(k, v, s, cu, query=q)
    b = c[1].append(k.contiguous(), v.contiguous(), s, cu, query=q.contiguous())
    assert torch.equal(a, b) and torch.equal(c[0].keys, c[1].keys) and torch.equal(c[0].values, c[1].values)
    odd = torch.zeros(128, 2, 41, device=dev).permute(2, 1, 0)[1:]     # the dimensions far apart, off by 4 bytes
    odd.copy_(k)
    c[0].append(odd, v.transpose(0, 1).contiguous().transpose(0, 1), s, cu)
    assert torch.equal(c[0].keys, c[1].keys) and torch.equal(c[0].values, c[1].values)


# ---- decode --------------------------------------------------------------------------------

def filled(lc, dev, D, dtype, page, Hkv, lengths, seed=0, pages=None, poison=True):
    """A cache whose sequences hold the lengths, at random pages, with NaN wherever no token is."""
    import torch
    B = len(lengths)
    most = pages or max(1, -(-max(lengths) // page))
    c = shuffled(lc.PagedEvictingKVCache(Hkv, D, num_sequences=B, page_size=page, max_pages=most, num_pages=B * most + 3,
                                         dtype=getattr(torch, dtype), device=dev), seed)
    k, v = rand(dev, dtype, c.num_pages * page, Hkv, D, seed=seed + 1), rand(dev, dtype, c.num_pages * page, Hkv, D, seed=seed + 2)
    c.keys.copy_(k.view(c.num_pages, page, Hkv, D).transpose(1, 2))
    c.values.copy_(v.view(c.num_pages, page, Hkv, D).transpose(1, 2))
    c.weights.copy_(torch.rand(c.weights.shape, generator=torch.Generator().manual_seed(seed)))
    c.positions.copy_(torch.arange(c.positions.numel()).view(c.positions.shape) % 100003)
    if poison:
        there = torch.zeros(c.num_pages, page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            p, s = place(c, b, np.arange(n))
            there[torch.from_numpy(p).long(), torch.from_numpy(s).long()] = True
        gone = (~there).to(dev)[:, None].expand(c.num_pages, Hkv, page)
        for t in (c.keys, c.values, c.weights):
            t[gone] = math.nan
    return c


def check_decode(c, q, lengths, out, before, dtype, scale=None, counted=True):
    """Out and weights within what the arithmetic rounds.

    A score's products are exact and its sums fp32: off by (D + 3) 2^-24 of the largest score's terms,
    and 2^-23 of its size for the scaling; a softmax weight by the relative double of that, 2^-22 of
    exp2 and of the maximum's factors, and 1024 2^-24 of the sums (a wave's way through a chunk and the
    chunks of a sequence are each shorter than that here).  16-bit types round the weights of the value
    product by half a step, and the output by another one."""
    D, Hkv, Hq = c.head_dim, c.num_kv_heads, q.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    K, V, Q, O, W = f64(c.keys), f64(c.values), f64(q), f64(out), f64(c.weights)
    u = half_step(dtype)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not O[b].any()
            continue
        pages, slots = place(c, b, np.arange(n))
        for h in range(Hkv):
            k, v = K[pages, h, slots], V[pages, h, slots]
            got, slack = np.zeros(n), np.zeros(n)
            for j in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                want, w, size, terms = kve.attend(Q[b, j], k, v, scale)
                e = 2 * ((D + 3) * 2.0 ** -24 * terms + 2.0 ** -23 * terms) + 2.0 ** -22 + 1024 * 2.0 ** -24
                tol = u * np.abs(want) + (e + (2 * u if dtype != "float32" else 0)) * size
                if dtype == "float16":
                    tol += 2.0 ** -24
                assert (np.abs(O[b, j] - want) <= tol).all(), (b, j, np.abs(O[b, j] - want).max())
                got += w
                slack += 2 * e * w
            if counted:
                want = before[pages, h, slots] + got
                assert (np.abs(W[pages, h, slots] - want) <= slack + 2.0 ** -23 * np.abs(want)).all(), (b, h)
    if not counted:
        assert np.array_equal(W, before, equal_nan=True)


DECODES = [  # D, dtype, page, kv heads, query heads, lengths
    (128, "bfloat16", 16, 8, 32, [1, 31, 32, 33, 0, 500, 129]),
    (128, "bfloat16", 32, 1, 5, [700, 2, 64]),
    (128, "float16", 16, 4, 4, [15, 16, 17, 300]),
    (128, "float32", 16, 2, 8, [1, 15, 16, 17, 0, 300, 63, 64, 65]),
    (128, "float32", 64, 1, 1, [1000]),
    (64, "float16", 16, 16, 16, [40, 257, 3]),
    (64, "bfloat16", 128, 2, 32, [127, 128, 129, 5]),        # 16 query heads of a kv head: a whole product
    (64, "float32", 16, 3, 51, [90, 1]),                      # 17: one more
    (256, "bfloat16", 16, 1, 33, [200, 0, 47]),               # 33: two passes
    (256, "float32", 16, 2, 40, [70, 33]),                    # 20, in passes of 16
    (256, "float16", 32, 2, 4, [260]),
    (128, "bfloat16", 16, 1, 128, [75, 130]),                 # the most query heads of a kv head
    (64, "float32", 16, 1, 128, [35]),
    (128, "float16", 16, 2, 46, [99, 32]),
    # every build's most shared memory: scores of more tokens than it holds
    (256, "bfloat16", 16, 1, 32, [600, 33]),
    (256, "float32", 16, 2, 32, [900, 770, 12]),
    (256, "float16", 16, 2, 8, [3500]),
    (128, "float32", 16, 1, 32, [500, 390]),
    (128, "bfloat16", 16, 2, 64, [388, 800]),
    (64, "float32", 16, 2, 64, [388, 400]),
    (64, "float16", 16, 2, 32, [449, 900, 448]),
]


@pytest.mark.parametrize("D,dtype,page,Hkv,Hq,lengths", DECODES)
def test_decode(lc, dev, D, dtype, page, Hkv, Hq, lengths):
    import torch
    c = filled(lc, dev, D, dtype, page, Hkv, lengths, seed=D + Hq)
    q = rand(dev, dtype, len(lengths), Hq, D, seed=9)
    held, before = i32(dev, lengths), f64(c.weights)
    out = c.decode(q, held)
    check_decode(c, q, lengths, out, before, dtype)
    # again: the weights go on; with a bound; without weights
    mid = f64(c.weights)
    again = c.decode(q, held, max_held=max(lengths))
    check_decode(c, q, lengths, again, mid, dtype)
    mid = f64(c.weights)
    other = c.decode(q, held, 0.3, count=False, out=q.clone())
    check_decode(c, q, lengths, other, mid, dtype, scale=0.3, counted=False)
    assert torch.isfinite(out).all() and out.dtype == q.dtype
    # into the query itself
    x = q.clone()
    assert c.decode(x, held, 0.3, count=False, out=x) is x and torch.equal(x, other)


def cycled(lengths, n):
    return (lengths * n)[:n]


@pytest.mark.parametrize("dtype,Hq,lengths", [
    # 32 query heads a kv head: scores of 384 tokens lie in LDS, chunks have 512
    ("bfloat16", 64, cycled([590, 600, 540, 600, 500, 0, 600, 385, 384, 600], 130)),
    # 16: scores of 448 tokens, chunks of 800
    ("float32", 32, cycled([900, 900, 790, 769, 830, 900, 768, 900, 900, 1], 260)),
    # sequences cut into chunks of 512, more than LDS has room for
    ("float16", 64, cycled([590, 1000, 540, 600, 500, 0, 600, 385, 384, 600], 130)),
    # a kv head for each query head: all of the longest
    ("float16", 2, cycled([70, 31, 0, 128, 129, 1], 513)),
])
def test_decode_of_whole_sequences(lc, dev, dtype, Hq, lengths):
    """A batch whose sequences are a workgroup's each, with their scores in LDS and past it, some cut in two."""
    c = filled(lc, dev, 64, dtype, 16, 2, lengths, seed=31)
    q = rand(dev, dtype, len(lengths), Hq, 64, seed=32)
    before = f64(c.weights)
    check_decode(c, q, lengths, c.decode(q, i32(dev, lengths)), before, dtype)


def test_decode_one_long_sequence(lc, dev):
    """More tiles than a launch has chunks for at their least size, with a strided query."""
    import torch
    n = 70001
    c = filled(lc, dev, 64, "bfloat16", 64, 2, [n], seed=5)
    q = rand(dev, "bfloat16", 1, 8, 128, seed=6)[..., 1:65]
    before = f64(c.weights)
    check_decode(c, q, [n], c.decode(q, i32(dev, [n])), before, "bfloat16")


def test_decode_many_sequences(lc, dev):
    """More sequences than chunks, of no, one and some tokens: a prefix over several blocks of threads."""
    r = np.random.default_rng(3)
    lengths = r.integers(0, 40, size=3001).tolist()
    c = filled(lc, dev, 64, "float32", 16, 1, lengths, seed=7)
    q = rand(dev, "float32", len(lengths), 2, 64, seed=8)
    before = f64(c.weights)
    check_decode(c, q, lengths, c.decode(q, i32(dev, lengths)), before, "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_decode_bound_and_lengths_out_of_range(lc, dev, dtype):
    """Lengths past the bound or the pages are cut to it, below 0 they are 0."""
    import torch
    c = filled(lc, dev, 64, dtype, 16, 2, [96, 96, 96, 96], seed=1)
    q = rand(dev, dtype, 4, 4, 64, seed=2)
    before = f64(c.weights)
    out = c.decode(q, i32(dev, [2**31 - 1, 97, -1, -2**31]))
    check_decode(c, q, [96, 96, 0, 0], out, before, dtype)
    before = f64(c.weights)
    out = c.decode(q, i32(dev, [2**31 - 1, 50, 51, 3]), max_held=50)
    check_decode(c, q, [50, 50, 50, 3], out, before, dtype)
    out = c.decode(q, i32(dev, [96] * 4), max_held=2**31 - 1, count=False)
    assert torch.equal(out, c.decode(q, i32(dev, [96] * 4), count=False))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_decode_pages_that_are_not_there(lc, dev, dtype):
    """Their tokens are not attended and get no weight; a sequence of such pages alone is one without
    tokens."""
    import torch
    c = filled(lc, dev, 128, dtype, 16, 2, [80, 80, 80], seed=4, poison=False)
    c.block_table[0, 1], c.block_table[0, 4], c.block_table[1] = -1, c.num_pages, -7
    q = rand(dev, dtype, 3, 6, 128, seed=5)
    before, table = f64(c.weights), c.block_table.clone()
    out = c.decode(q, i32(dev, [80, 80, 80]))
    assert not out[1].any()
    # the same with the tokens of the pages that are there alone
    ref = c.keys.clone(), c.weights.clone()
    want = lc.PagedEvictingKVCache(2, 128, num_sequences=3, max_pages=5, num_pages=c.num_pages, dtype=c.dtype, device=dev)
    want.keys.copy_(c.keys), want.values.copy_(c.values), want.weights.copy_(torch.from_numpy(before))
    want.block_table.copy_(table)
    want.block_table[0, :3] = table[0, [0, 2, 3]]
    check_decode(want, q, [48, 0, 80], out, before, dtype, counted=False)
    o2 = want.decode(q, i32(dev, [48, 0, 80]))
    check_decode(want, q, [48, 0, 80], o2, before, dtype)
    assert torch.allclose(want.weights, c.weights, rtol=1e-4, atol=1e-6) and torch.equal(ref[0], c.keys)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_decode_extreme_scores(lc, dev, dtype):
    """Scores of -inf alone: no softmax, NaN.  Some of -inf: no weight.  From 2^24 on: the largest one's
    value.  A NaN key or an infinite value that a head sees shows in it alone."""
    import torch
    n, D = 70, 64
    big = 60000.0 if dtype == "float16" else 1e6
    c = lc.PagedEvictingKVCache(2, D, num_sequences=1, max_pages=8, rope_theta=None, dtype=getattr(torch, dtype), device=dev)
    v = rand(dev, dtype, 128, 2, D, seed=3).view(8, 16, 2, D).transpose(1, 2)
    c.values.copy_(v)
    q = torch.ones(1, 4, D, dtype=c.dtype, device=dev)
    held = i32(dev, [n])
    flat = lambda: c.values.transpose(1, 2).reshape(128, 2, D).double()  # noqa: E731
    # kv head 0 scores -inf everywhere, head 1 on all but two tokens
    c.keys.zero_()
    c.keys[:, 0, :, 0] = -math.inf
    c.keys[:, 1, :, 0] = -math.inf
    c.keys[1, 1, 5, 0], c.keys[4, 1, 3, 0] = 0.0, 0.0
    out = c.decode(q, held)
    assert torch.isnan(out[0, :2]).all()
    want = (flat()[21, 1] + flat()[67, 1]) / 2
    assert torch.allclose(out[0, 2].double(), want, rtol=2 * half_step(dtype), atol=2 * half_step(dtype) * 4)
    w = c.weights.transpose(1, 2).reshape(128, 2)
    assert torch.isnan(w[:n, 0]).all() and not w[n:].any()
    assert w[21, 1] == 1.0 and w[67, 1] == 1.0 and w[:n, 1].sum() == 2.0      # two query heads of one half each
    # huge scores
    c.weights.zero_(), c.keys.zero_()
    c.keys[:, :, :, 0] = big
    c.keys[2, :, 7, 1] = big / 2
    out = c.decode(q * (1.0 if dtype == "float16" else 300.0), held, 100.0)
    want = flat()[39]
    assert torch.allclose(out[0].double(), want.repeat_interleave(2, 0), rtol=half_step(dtype), atol=1e-6)
    # an infinite value with a weight is infinite, and in its dimension and head alone
    c.weights.zero_(), c.keys.zero_()
    c.values[1, 0, 2, 9] = math.inf
    out = c.decode(q, held)
    bad = torch.isinf(out)
    assert bad[0, :2, 9].all() and bad.sum() == 2 and torch.isfinite(out[~bad]).all()
    # a NaN key
    c.keys[3, 1, 1, 4] = math.nan
    out = c.decode(q, held)
    assert torch.isnan(out[0, 2:]).all() and not torch.isnan(out[0, :2]).any()


@pytest.mark.parametrize("D,Hq", [(64, 1), (64, 20), (128, 4), (256, 1), (256, 17)])
@pytest.mark.parametrize("dtype,p", [("bfloat16", 0.5 + 0.99 * 2.0 ** -9), ("float16", 0.5 + 0.99 * 2.0 ** -12),
                                     ("bfloat16", 0.3 + 2.0 ** -12), ("float16", 0.7), ("float32", 0.7)])
@pytest.mark.parametrize("n", [40, 300])
def test_decode_weights_that_the_type_cannot_hold(lc, dev, D, Hq, dtype, p, n):
    """Half the tokens of weight 1 and half of p, a number in the middle between two of the type, with values
    that cancel: what remains shows how weights are rounded.

    Of the scores one product is exact and its scaling off by 2^-23 of |ln p| < 2; exp2 and the maximum's factor
    2^-22; sums of n terms, two products each, 2 n 2^-24 and 8 2^-24 for joins and the division; the weights'
    two numbers 2^-14 (bfloat16) or 2^-20."""
    import torch
    page = 32
    c = lc.PagedEvictingKVCache(1, D, num_sequences=1, page_size=page, max_pages=-(-n // page), rope_theta=None,
                                dtype=getattr(torch, dtype), device=dev)
    scale = float(np.float32(-math.log(p)))
    r = rand(dev, dtype, D, seed=61)
    c.keys[:, 0, 1::2, 0] = -1.0
    c.values[:, 0, ::2] = r
    c.values[:, 0, 1::2] = (-r.double() / p).to(c.dtype)
    q = torch.zeros(1, Hq, D, dtype=c.dtype, device=dev)
    q[..., 0] = 1.0
    out = f64(c.decode(q, i32(dev, [n]), scale))
    k, v = (f64(t).transpose(0, 2, 1, 3).reshape(-1, D)[:n] for t in (c.keys, c.values))
    want, _, size, _ = kve.attend(f64(q)[0, 0], k, v, scale)
    own = {"bfloat16": 2.0 ** -14, "float16": 2.0 ** -20, "float32": 0.0}[dtype]
    tol = half_step(dtype) * np.abs(want) + (2.0 ** -22 + 2.0 ** -22 + (2 * n + 8) * 2.0 ** -24 + own) * size
    tol += 2.0 ** -25 * (dtype == "float16")
    assert (np.abs(out[0] - want) <= tol).all(), np.abs((out[0] - want) / size).max()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_decode_infinite_values_of_small_weights(lc, dev, dtype):
    """An infinite value shows as such, however small its weight is beside the largest one, and a token whose
    weight is 1 alone is its value bit for bit."""
    import torch
    D = 64
    c = lc.PagedEvictingKVCache(1, D, num_sequences=1, page_size=16, max_pages=4, rope_theta=None,
                                dtype=getattr(torch, dtype), device=dev)
    v = rand(dev, dtype, 4, 1, 16, D, seed=62)
    q = torch.zeros(1, 3, D, dtype=c.dtype, device=dev)
    q[..., 0] = 1.0
    for at, bits in ((3, 0.0), (17, 1.0), (40, 11.5), (9, 15.0), (50, 20.25), (33, 28.0), (2, 36.5), (1, 37.9)):
        for sign in (1, -1):
            c.values.copy_(v)
            c.keys.zero_()
            c.keys[at // 16, 0, at % 16, 0] = -bits
            c.values[at // 16, 0, at % 16, 5] = sign * math.inf
            out = c.decode(q, i32(dev, [50 + 14 * (at >= 50)]), math.log(2.0), count=False)
            assert (out[..., 5] == sign * math.inf).all() and torch.isfinite(out).sum() == 3 * (D - 1), bits
    c.values.copy_(v), c.keys.zero_()
    assert torch.equal(c.decode(q, i32(dev, [1])), v[0, 0, :1].expand(3, D)[None])
    c.keys[1, 0, 4, 0] = 1.0                          # the others' weights are 0 in fp32
    assert torch.equal(c.decode(q, i32(dev, [60]), 1000.0), v[1, 0, 4:5].expand(3, D)[None])


def test_decode_small_weights_keep_their_share(lc, dev):
    """One token of weight 1 and 100000 of 2^-24 each: together they are as much as 0.6 % of it, in fp16
    as well, whose smallest number is 2^-24."""
    import torch
    n, D = 100001, 64
    for dtype in ("float16", "bfloat16", "float32"):
        c = lc.PagedEvictingKVCache(1, D, num_sequences=1, page_size=1024, max_pages=98, rope_theta=None,
                                    dtype=getattr(torch, dtype), device=dev)
        c.values.fill_(1.0)
        c.values[0, 0, 0] = 0.0
        c.keys[0, 0, 0, 0] = 1.0
        q = torch.zeros(1, 1, D, dtype=c.dtype, device=dev)
        q[0, 0, 0] = 1.0
        out = c.decode(q, i32(dev, [n]), 24 * math.log(2.0), count=False)
        w = 100000 * 2.0 ** -24
        want = w / (1 + w)
        assert (out.double() - want).abs().max() <= want * (half_step(dtype) + 2.0 ** -10), dtype


# ---- evict ---------------------------------------------------------------------------------

def check_evict(c, held, budget, sink, recent, **kw):
    """The whole pool as the definition leaves it, bit for bit."""
    import torch
    was = {n: getattr(c, n).clone().cpu() for n in ("keys", "values", "weights", "positions")}
    want = {n: t.clone() for n, t in was.items()}
    h = i32(c.device, held)
    assert c.evict(h, budget, sink_tokens=sink, recent_tokens=recent, **kw) is None
    assert h.tolist() == list(held)
    table = c.block_table.cpu().numpy()
    for b, n in enumerate(held):
        n = min(max(n, 0), kw.get("max_held") or c.capacity, c.capacity)
        if n <= budget:
            continue
        pages, slots = place(c, b, np.arange(n))
        there = (pages >= 0) & (pages < c.num_pages)
        safe = np.where(there, pages, 0)
        for g in range(c.num_kv_heads):
            w, p = was["weights"].numpy()[safe, g, slots], was["positions"].numpy()[safe, g, slots]
            _, places, moved = kve.kept(w, p, budget, sink, recent, there)
            for to, of in zip(places, moved):
                if there[to] and there[of]:
                    for name in want:
                        want[name][pages[to], g, slots[to]] = was[name][pages[of], g, slots[of]]
    for name, t in want.items():
        got = getattr(c, name).cpu()
        assert torch.equal(got.view(torch.int16 if t.element_size() == 2 else torch.int32),
                           t.view(torch.int16 if t.element_size() == 2 else torch.int32)), name
    assert np.array_equal(table, c.block_table.cpu().numpy())


EVICTS = [  # D, dtype, page, kv heads, held, budget, sink, recent
    (128, "bfloat16", 16, 8, [33, 40, 32, 5, 0, 64], 32, 4, 8),
    (64, "float16", 32, 3, [100, 101, 99], 99, 0, 0),
    (256, "float32", 16, 2, [70, 300], 17, 2, 15),
    (64, "bfloat16", 16, 1, [2, 500, 1], 1, 0, 0),
    (64, "bfloat16", 16, 1, [400], 5, 0, 1),
    (128, "float32", 128, 2, [1500, 900], 700, 4, 100),        # moves of a launch of their own
    (64, "float16", 64, 2, [5000], 300, 0, 300),
    (256, "bfloat16", 16, 1, [2048], 2040, 4, 64),
]


@pytest.mark.parametrize("D,dtype,page,Hkv,held,budget,sink,recent", EVICTS)
def test_evict(lc, dev, D, dtype, page, Hkv, held, budget, sink, recent):
    import torch
    c = filled(lc, dev, D, dtype, page, Hkv, held, seed=budget, poison=False)
    for b, n in enumerate(held):                     # positions in order of the slots, from 3 b on
        p, s = place(c, b, np.arange(n))
        c.positions[torch.from_numpy(p).long().to(dev), :, torch.from_numpy(s).long().to(dev)] = \
            (torch.arange(n, device=dev) + 3 * b).to(torch.int32)[:, None]
    check_evict(c, held, budget, sink, recent)
    # again on what is left: positions and slots in different orders now
    left = [min(n, budget) for n in held]
    check_evict(c, left, max(1, budget // 2), sink // 2, recent // 2)
    # with a bound below the lengths
    check_evict(c, left, max(1, budget // 4), 0, 0, max_held=max(2, budget // 3))


@pytest.mark.parametrize("held,budget", [([1024, 1000, 7], 400), ([1025, 1000, 512], 400), ([1024, 1023], 1020),
                                         ([1025, 1024], 1020), ([4096, 4097], 4000), ([4097], 1000)])
def test_evict_at_the_sizes_that_change_the_launch(lc, dev, held, budget):
    c = filled(lc, dev, 128, "bfloat16", 16, 2, held, seed=41, poison=False)
    check_evict(c, held, budget, 4, 64, max_held=max(held))
    check_evict(c, [min(n, budget) for n in held], budget - 3, 4, 64)


@pytest.mark.parametrize("B,held,budget", [(86, [1024, 1000, 7], 400), (86, [1025, 1000, 512], 400), (86, [1024, 1023], 1020),
                                           (86, [1025, 1024], 1020), (85, [1500, 1490], 1480), (86, [4100, 20, 4096], 4000)])
def test_evict_of_many_sequences(lc, dev, B, held, budget):
    """More (sequence, kv head) pairs than the card has CUs, and 255 of them."""
    held = cycled(held, B)
    c = filled(lc, dev, 64, "float16", 32, 3, held, seed=42, poison=False)
    check_evict(c, held, budget, 4, 64, max_held=max(held))


def test_evict_ties_and_odd_weights(lc, dev):
    """Equal weights (the lowest slots stay), zeros of both signs, negative ones, infinities and NaN."""
    import torch
    c = filled(lc, dev, 64, "bfloat16", 16, 4, [200, 130, 64], seed=11, poison=False)
    odd = torch.tensor([0.0, -0.0, 1.0, 1.0, -1.0, math.inf, -math.inf, math.nan, -math.nan, 1e-45, 3e38, 1.0])
    pick = torch.randint(0, 12, c.weights.shape, generator=torch.Generator().manual_seed(1))
    for budget in (100, 63, 7, 1):
        c.weights.copy_(odd[pick])
        check_evict(c, [200, 130, 64], budget, 0, 0)
    c.weights.fill_(0.25)
    check_evict(c, [200, 130, 64], 50, 0, 0)
    c.positions.zero_()                              # every token protected: the lowest slots
    check_evict(c, [200, 130, 64], 50, 1, 0)
    c.positions.fill_(2**31 - 1)
    check_evict(c, [200, 130, 64], 50, 1, 49)
    c.positions.fill_(-2**31)
    check_evict(c, [200, 130, 64], 50, 0, 50)


def test_evict_pages_that_are_not_there(lc, dev):
    c = filled(lc, dev, 64, "float32", 16, 2, [96, 96], seed=12, poison=False)
    c.block_table[0, 1], c.block_table[0, 4] = -1, c.num_pages
    c.block_table[1] = -1
    for budget in (80, 50, 20):
        check_evict(c, [96, 96], budget, 0, 3)


def test_evict_loses_what_goes_to_a_page_that_is_not_there(lc, dev):
    """As documented: of the tokens behind the budget those whose place is such a page's are gone, the others
    move."""
    import torch
    c = filled(lc, dev, 64, "float32", 16, 1, [64], seed=15, poison=False)
    c.block_table[0, 1] = -1
    c.weights.fill_(1.0)
    p, s = (torch.from_numpy(x).long() for x in place(c, 0, np.arange(64)))
    c.weights[p[40:], 0, s[40:]] = 2.0                # 24 behind the budget: 8 and then 16 of slots 8 to 31
    c.weights[p[:8], 0, s[:8]] = 3.0
    was = c.values[p[40:], 0, s[40:]].clone(), c.values.clone()
    check_evict(c, [64], 32, 0, 0)
    assert torch.equal(c.values[p[8:16], 0, s[8:16]], was[0][:8])
    was[1][p[8:16], 0, s[8:16]] = was[0][:8]
    assert torch.equal(c.values, was[1])


@pytest.mark.parametrize("n,budget", [(33000, 32900), (40001, 8192)])
def test_evict_long(lc, dev, n, budget):
    """More tokens than the ranks' place in LDS."""
    c = filled(lc, dev, 64, "bfloat16", 64, 1, [n, n // 2], seed=13, poison=False)
    check_evict(c, [n, n // 2], budget, 4, 1000)


def roomy(lc, dev, dtype, Hkv, held, capacity, seed):
    """Sequences with pages for what they hold alone, in a table of `capacity` slots each; positions from a
    place of each sequence's own on, in order."""
    import torch
    page, B = 64, len(held)
    pages = [-(-n // page) for n in held]
    c = lc.PagedEvictingKVCache(Hkv, 64, num_sequences=B, page_size=page, max_pages=capacity // page, num_pages=sum(pages),
                                dtype=getattr(torch, dtype), device=dev)
    order, first = np.random.default_rng(seed).permutation(sum(pages)).astype(np.int32), cum(pages)
    for b in range(B):
        c.block_table[b, :pages[b]] = torch.from_numpy(order[first[b]:first[b + 1]]).to(dev)
    for t, s in ((c.keys, 1), (c.values, 2)):
        t.copy_(rand(dev, dtype, t.shape[0], Hkv, page, 64, seed=seed + s))
    c.weights.copy_(torch.rand(c.weights.shape, generator=torch.Generator().manual_seed(seed)))
    for b, n in enumerate(held):
        p, s = place(c, b, np.arange(n))
        c.positions[torch.from_numpy(p).long().to(dev), :, torch.from_numpy(s).long().to(dev)] = \
            (torch.arange(n, device=dev) + 5 * b).to(torch.int32)[:, None]
    return c


@pytest.mark.parametrize("dtype,Hkv,Hq", [("bfloat16", 2, 8), ("float32", 1, 3), ("float16", 3, 102)])
def test_decode_short_sequences_of_a_large_pool(lc, dev, dtype, Hkv, Hq):
    """Without a bound, sequences of some tokens in a table of 40960 slots each."""
    held = [700, 0, 1, 64, 65, 129, 2500]
    c = roomy(lc, dev, dtype, Hkv, held, 40960, seed=52)
    q = rand(dev, dtype, len(held), Hq, 64, seed=53)
    before = f64(c.weights)
    check_decode(c, q, held, c.decode(q, i32(dev, held)), before, dtype)


@pytest.mark.parametrize("held,Hkv", [([40001, 3000, 4096, 4097, 900, 0], 2), ([2064, 33, 1], 1),
                                      (cycled([900, 4096, 201, 4097, 20, 1025, 1024], 86), 3)])
@pytest.mark.parametrize("budget,recent", [(200, 64), (800, 128), (2900, 0)])     # moves in place, by a launch of their own
@pytest.mark.parametrize("max_held", [0, 40001, 32768])     # the last: all ranks in LDS, as many as there can be
def test_evict_short_sequences_of_a_large_pool(lc, dev, held, Hkv, budget, recent, max_held):
    """A bound past the ranks' place in LDS, sequences that hold few tokens: the newest and the first stay,
    of the others those of largest weight."""
    c = roomy(lc, dev, "bfloat16", Hkv, held, 40960, seed=51)
    check_evict(c, held, budget, 4, recent, **(dict(max_held=max_held) if max_held else {}))


def test_evict_lengths_out_of_range(lc, dev):
    c = filled(lc, dev, 64, "bfloat16", 16, 2, [96, 96, 96], seed=14, poison=False)
    check_evict(c, [2**31 - 1, -4, 97], 40, 4, 4)
    check_evict(c, [96, 96, 96], 96, 0, 0)           # nothing to do
    check_evict(c, [96, 96, 96], 2**31 - 1, 0, 0)


# ---- as they are used ----------------------------------------------------------------------

def test_steps_in_bounded_memory(lc, dev, pkg):
    """A generation past the cache's size: append, decode, draw and evict, captured once and replayed,
    gives what the eager calls give and what the oracle says of every step's attention and eviction."""
    import torch
    from importlib import import_module
    sample = import_module(pkg.__name__ + ".decoder").sample_tokens
    B, Hkv, Hq, D, budget, room, V = 3, 2, 8, 64, 48, 56, 500
    g = torch.Generator(device=dev).manual_seed(2)
    emb = torch.randn(V, (Hq + 2 * Hkv) * D, generator=g, device=dev)
    head = torch.randn(Hq * D, V, generator=g, device=dev) * 0.2
    us = torch.rand(40, B, generator=g, device=dev)

    def start():
        c = lc.PagedEvictingKVCache(Hkv, D, num_sequences=B, max_pages=-(-room // 16), dtype=torch.float32, device=dev)
        pk, pv = (torch.randn(B * 30, Hkv, D, generator=torch.Generator(device=dev).manual_seed(s), device=dev) for s in (5, 6))
        c.append(pk, pv, i32(dev, [0] * B), i32(dev, [0, 30, 60, 90]))
        return dict(c=c, held=i32(dev, [30, 30, 30]), pos=i32(dev, [30, 30, 30]), token=i32(dev, [1, 2, 3]),
                    u=torch.zeros(B, device=dev), out=torch.zeros(B, Hq, D, device=dev))

    def step(s):
        x = emb[s["token"].long()].view(B, Hq + 2 * Hkv, D)
        q = s["c"].append(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], s["held"], position=s["pos"], query=x[:, :Hq])
        s["held"].add_(1), s["pos"].add_(1)
        s["c"].decode(q, s["held"], max_held=room, out=s["out"])
        s["c"].evict(s["held"], budget, sink_tokens=2, recent_tokens=8, max_held=room)
        s["held"].clamp_(max=budget)
        sample(s["out"].view(B, -1) @ head, s["u"], temperature=0.8, top_p=0.9, out=s["token"])

    eager, tokens = start(), []
    for t in range(40):
        eager["u"].copy_(us[t])
        step(eager)
        tokens.append(eager["token"].tolist())
    assert eager["pos"].tolist() == [70] * B and eager["held"].tolist() == [budget] * B
    assert len({tuple(x) for x in tokens}) > 5
    warm = start()
    step(warm)
    s = start()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(s)
    fresh = start()
    for name in ("held", "pos", "token"):
        s[name].copy_(fresh[name])
    for name in ("keys", "values", "weights", "positions"):
        getattr(s["c"], name).copy_(getattr(fresh["c"], name))
    for t in range(40):
        s["u"].copy_(us[t])
        graph.replay()
        torch.cuda.synchronize()
        torch.randn(1000, device=dev).sort()          # other work between the replays
        assert s["token"].tolist() == tokens[t], t
    assert torch.equal(s["c"].keys, eager["c"].keys) and torch.equal(s["c"].weights, eager["c"].weights)
    assert torch.equal(s["c"].positions, eager["c"].positions) and torch.equal(s["out"], eager["out"])


def test_on_other_streams(lc, dev):
    """Two caches' calls on two streams at once, each with a workspace of its own."""
    import torch
    cs = [filled(lc, dev, 128, "bfloat16", 16, 4, [600, 500], seed=20 + i) for i in range(2)]
    q = rand(dev, "bfloat16", 2, 16, 128, seed=1)
    held = i32(dev, [600, 500])
    want = [c.decode(q, held, count=False) for c in cs]
    before = [f64(c.weights) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    outs = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                outs[i] = c.decode(q, held)
    torch.cuda.synchronize()
    for c, a, b, w in zip(cs, outs, want, before):
        assert torch.equal(a, b)
        one = f64(c.weights)
        pages, slots = place(c, 0, np.arange(600))
        grown = one[pages, :, slots] - w[pages, :, slots]
        assert np.allclose(grown.sum(0), 5 * 4, rtol=1e-3)      # five steps, four query heads a kv head


def test_weights_with_a_gradient_are_refused(lc, dev):
    """As keys, values and queries with one are: what the cache holds has none."""
    import torch
    from torch.autograd import forward_ad
    c = lc.PagedEvictingKVCache(2, 64, num_sequences=2, max_pages=4, dtype=torch.bfloat16, device=dev)
    k, one = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=dev), i32(dev, [1, 1])
    w = torch.ones(2, 2, device=dev)
    with pytest.raises(RuntimeError, match="no gradient"):
        c.append(k, k, one, weight=w.clone().requires_grad_())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        c.append(k, k, one, weight=forward_ad.make_dual(w, w))
    assert not c.weights.any()
    with torch.no_grad():
        c.append(k, k, one, weight=w.clone().requires_grad_())
    assert c.weights.sum() == 4


def test_refusals(lc, dev):
    import torch
    c = lc.PagedEvictingKVCache(2, 64, num_sequences=2, max_pages=4, dtype=torch.float32, device=dev)
    k, q, one = torch.zeros(2, 2, 64, device=dev), torch.zeros(2, 4, 64, device=dev), i32(dev, [1, 1])
    for bad in (lambda: c.append(k[:1], k[:1], one), lambda: c.append(k, k, one.long()), lambda: c.append(k, k, one[:1]),
                lambda: c.append(k, k, one, i32(dev, [0, 1])), lambda: c.append(k, k[:, :1], one),
                lambda: c.append(k.bfloat16(), k.bfloat16(), one), lambda: c.append(k, k, one, position=one.float()),
                lambda: c.append(k, k, one, weight=torch.zeros(2, 3, device=dev)),
                lambda: c.append(k, k, one, weight=torch.zeros(2, 2)), lambda: c.append(k, k, one.cpu()),
                lambda: c.append(k, k, one, query=q[:, :, :32]), lambda: c.decode(q[:, :3], one),
                lambda: c.decode(q[:1], one), lambda: c.decode(q[:, :0], one), lambda: c.decode(q, one[:1]),
                lambda: c.decode(q.half(), one), lambda: c.decode(q, one, max_held=-1),
                lambda: c.decode(q, one, out=q.half()), lambda: c.decode(q, one, out=q[:, ::2].expand(2, 2, 64)),
                lambda: c.evict(one, 0), lambda: c.evict(one, 3), lambda: c.evict(one, 8, sink_tokens=5, recent_tokens=4),
                lambda: c.evict(one, 8, sink_tokens=-1), lambda: c.evict(one, 8, recent_tokens=-1),
                lambda: c.evict(one, 8, max_held=-1), lambda: c.evict(one[:1], 8), lambda: c.evict(one, 2**31)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.decode(q, one, math.nan), lambda: c.decode(q, one, math.inf)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError):
        c.append(k.clone().requires_grad_(), k, one)
    with pytest.raises(RuntimeError):
        c.decode(q.clone().requires_grad_(), one)
    with pytest.raises(AttributeError):
        c.keys = k
    assert not c.keys.any() and not c.positions.any()
    # empty calls
    assert c.append(k[:0], k[:0], one, i32(dev, [0, 0, 0]), query=q[:0]).shape == (0, 4, 64)
    assert not c.decode(q, i32(dev, [0, 0])).any()
