"""decoder.sample_tokens on the GPU: the token is the fp64 oracle's own (oracle/kve.py), at cuts, ties,
masks and sizes where it can go wrong."""
import math

import numpy as np
import pytest

from oracle import kve

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sample(pkg):
    from importlib import import_module
    return import_module(pkg.__name__ + ".decoder").sample_tokens


def logits(rows, vocab, dtype, seed, spread=2.0, peaks=12):
    import torch
    r = np.random.default_rng(seed)
    x = r.normal(size=(rows, vocab)) * spread
    for b in range(rows):
        x[b, r.integers(0, vocab, size=peaks)] += 4 + 3 * r.normal(size=peaks)
    return torch.from_numpy(x.astype(np.float32)).to(getattr(torch, dtype))


def check(sample, dev, x, u, T=1.0, k=0, p=1.0, m=0.0):
    """Settings: numbers, or lists of one for each row."""
    import torch
    rows = x.shape[0]

    def given(v, dtype):
        return torch.tensor(v, dtype=dtype, device=dev) if isinstance(v, list) else v

    got = sample(x.to(dev), torch.tensor(u, dtype=torch.float32, device=dev), temperature=given(T, torch.float32),
                 top_k=given(k, torch.int32), top_p=given(p, torch.float32), min_p=given(m, torch.float32))
    assert got.dtype == torch.int32 and tuple(got.shape) == (rows,)
    f = lambda v: np.asarray(v, np.float32).astype(np.float64) if isinstance(v, list) else np.full(rows, v)  # noqa: E731
    xs, uf = x.double().cpu().numpy(), np.asarray(u, np.float32).astype(np.float64)
    want = [kve.draw(xs[b], uf[b], a, int(kk), pp, mm) for b, (a, kk, pp, mm) in
            enumerate(zip(f(T), k if isinstance(k, list) else [k] * rows, f(p), f(m)))]
    assert got.tolist() == want
    return want


def grid(n):
    """n numbers over [0, 1), both ends among them."""
    return [min(i / (n - 1), 1 - 2.0 ** -24) for i in range(n)]


SETTINGS = [dict(), dict(T=0.3), dict(T=1.7), dict(k=1), dict(k=50), dict(k=5000), dict(p=0.9), dict(p=0.5, T=0.7),
            dict(p=0.999), dict(m=0.05), dict(m=0.5, T=1.3), dict(k=40, p=0.8), dict(k=1000, p=0.95, m=0.01, T=0.8),
            dict(k=3, m=0.9), dict(T=0.0), dict(T=0.0, k=5, p=0.5), dict(T=0.05, k=50, p=0.9), dict(T=1e-4),
            dict(T=25.0, p=0.6), dict(T=25.0, k=20000), dict(T=1e6, p=0.3, k=9000), dict(p=0.0), dict(m=1.0),
            dict(p=1e-9), dict(p=1 - 1e-12), dict(k=2**31 - 1, p=2.0)]


@pytest.mark.parametrize("s", SETTINGS, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()) or "plain")
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_settings(sample, dev, s, dtype):
    """A vocabulary of several slices with an odd end; bfloat16 has many equal logits."""
    check(sample, dev, logits(24, 30011, dtype, seed=1), grid(24), **s)


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 255, 1000, 8191, 8192, 8193, 16384, 151936, 262144])
def test_vocabularies(sample, dev, vocab):
    x = logits(5, vocab, "float32", seed=vocab)
    for s in (dict(), dict(k=20, p=0.9), dict(p=0.95, T=1.2), dict(T=0.0), dict(m=0.1)):
        check(sample, dev, x, grid(5), **s)


def test_largest_vocabulary(sample, dev):
    x = logits(2, 1 << 22, "bfloat16", seed=5)
    for s in (dict(), dict(p=0.9), dict(k=100000, p=0.99)):
        check(sample, dev, x, [0.31, 0.83], **s)


def test_settings_of_each_row(sample, dev):
    r = np.random.default_rng(4)
    rows = 200
    check(sample, dev, logits(rows, 9001, "bfloat16", seed=6), r.random(rows).tolist(),
          T=[float(r.choice([0.0, 0.2, 0.7, 1.0, 1.5, 30.0])) for _ in range(rows)],
          k=[int(r.choice([0, -5, 1, 2, 40, 700, 9000, 9001, 10000])) for _ in range(rows)],
          p=[float(r.choice([1.0, 0.9, 0.5, 0.05, 0.0, -1.0, 1.5])) for _ in range(rows)],
          m=[float(r.choice([0.0, 0.02, 0.3, 1.0, 1.5, -0.5])) for _ in range(rows)])


def test_equal_logits(sample, dev):
    """Cuts within equal logits keep the first ones of the vocabulary, over slices too."""
    import torch
    V = 20000
    flat = torch.zeros(16, V)
    u = grid(16)
    for s in (dict(), dict(k=1), dict(k=8192), dict(k=8193), dict(k=12345), dict(p=0.25), dict(p=0.5), dict(p=0.75),
              dict(k=16000, p=0.5), dict(m=1.0), dict(T=0.0), dict(T=3.0, k=100, p=0.5), dict(p=0.99999)):
        want = check(sample, dev, flat, u, **s)
        n = s.get("k") or V
        assert max(want) < (n if "p" not in s else math.ceil(n * s["p"]))
    two = torch.where(torch.arange(V) % 3 == 0, 0.5, -0.25).repeat(16, 1)
    for s in (dict(k=100), dict(k=6667), dict(k=6668), dict(k=15000), dict(p=0.3), dict(p=0.8), dict(k=9000, p=0.9)):
        check(sample, dev, two, u, **s)
        check(sample, dev, -two * 1e-3 + 1e4, u, **s)
        check(sample, dev, two.bfloat16(), u, T=0.4, **s)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_tokens_next_to_those_not_drawn(sample, dev, dtype):
    """Tokens 36.4 temperatures below the largest, e about 2^-52.5, in a slice whose own largest is below the
    row's: none is drawn, and a top-k cut among them keeps all that can be."""
    import torch
    x = torch.full((12, 24576), -60000.0)
    x[:, 0] = 0.0
    for b, top in enumerate((-1.0, -0.125, -3.0, -20.0) * 3):
        x[b, 8192 + b] = top
        x[b, 8300:8310] = -25.5
        x[b, 16384 + b:16390] = -25.5                 # a slice of nothing else
    x = x.to(getattr(torch, dtype))
    for k in (1, 2, 3, 5, 11, 12, 13, 18, 30):
        for s in (dict(), dict(p=0.5), dict(p=0.999999), dict(m=1e-12), dict(p=0.9, m=0.01)):
            got = check(sample, dev, x, grid(12), T=0.7, k=k, **s)
            assert all(t in (0, 8192 + b) for b, t in enumerate(got))
    for s in (dict(), dict(p=0.5), dict(p=1 - 1e-7)):
        check(sample, dev, x, grid(12), T=0.7, **s)


def test_masked_logits(sample, dev):
    """Logits of -inf are never drawn, the type's lowest value only where nothing else is."""
    import torch
    for low in (-math.inf, torch.finfo(torch.float32).min):
        x = logits(12, 20001, "float32", seed=7)
        x[:, 3:19000] = low
        x[1, :] = low
        x[1, [77, 15000]] = torch.tensor([1.0, 2.0])
        x[2, :8192] = low                             # whole slices of it
        x[3, 8192:] = low
        x[4, :20000] = low
        for s in (dict(), dict(p=0.9), dict(k=30), dict(k=5000, p=0.99), dict(m=0.1), dict(T=0.0), dict(T=1e-3, p=0.5)):
            got = check(sample, dev, x, grid(12), **s)
            assert all(x[b, t] > -1e30 for b, t in enumerate(got))
    x = torch.full((2, 9000), torch.finfo(torch.float32).min)
    for s in (dict(), dict(k=100), dict(p=0.5), dict(T=0.0)):
        check(sample, dev, x, [0.0, 0.9999], **s)


def test_rows_without_a_distribution(sample, dev):
    import torch
    x = logits(8, 10000, "bfloat16", seed=8)
    x[0] = -math.inf
    x[1, 9999] = math.nan
    x[2, 0] = math.inf
    x[3, 4000] = -math.nan
    for s in (dict(), dict(k=20), dict(p=0.9), dict(m=0.2), dict(T=0.0)):
        got = check(sample, dev, x, grid(8), **s)
        assert got[:4] == [-1] * 4 and min(got[4:]) >= 0
    T = [1.0, 1.0, 1.0, 1.0, -1.0, math.nan, math.inf, 1.0]
    got = sample(x.to(dev), torch.tensor(grid(8), device=dev), temperature=torch.tensor(T, device=dev), top_p=0.9)
    assert got.tolist()[:7] == [-1] * 7 and got[7] >= 0


def test_settings_that_are_nan(sample, dev):
    """A NaN among a row's settings gives -1, not the row without that cut or with its largest token alone;
    infinities count as the nearest setting in range."""
    import torch
    x, u = logits(8, 10000, "bfloat16", seed=14).to(dev), torch.tensor(grid(8), device=dev)
    nan, inf = math.nan, math.inf
    p, m = [nan, 0.9, 0.9, inf, -inf, 0.9, nan, 0.9], [0.0, nan, 0.0, 0.0, 0.0, inf, nan, -inf]
    for T in (1.0, 0.0):
        for k in (0, 30):
            got = sample(x, u, temperature=T, top_k=k, top_p=torch.tensor(p, device=dev),
                         min_p=torch.tensor(m, device=dev)).tolist()
            want = [kve.draw(x[b].double().cpu().numpy(), float(u[b]), T, k, min(max(p[b], 0.0), 1.0), min(max(m[b], 0.0), 1.0))
                    for b in range(8)]
            assert got == [-1, -1, want[2], want[3], want[4], want[5], -1, want[7]]


def test_extreme_values(sample, dev):
    """Logits at the ends of the type, tiny and huge temperatures, a cut at a value next to 0."""
    import torch
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[big, -big, 0.0, big, 1e-45, -1e-45, -0.0, 0.0, 1e38, -1e38]] * 6)
    u = grid(6)
    for s in (dict(), dict(k=2), dict(k=5), dict(p=0.5), dict(m=0.5), dict(T=1e38), dict(T=1e38, k=5), dict(T=1e-38, k=2),
              dict(T=3e38, p=0.7), dict(T=1e-45), dict(T=1e38, m=0.1), dict(T=1e38, k=7, p=0.9)):
        check(sample, dev, x, u, **s)
    near = torch.tensor([[0.0, -0.0, 1e-45, 0.0, -0.0, -1e-45, 2e-45, -1e-3, 1e-3, -0.0]] * 6)
    for k in range(1, 10):
        check(sample, dev, near, u, k=k)
        check(sample, dev, near, u, k=k, p=0.6, T=0.5)
    check(sample, dev, near, u, m=0.9999)
    for v in (0.0, 1e4, -1e4, 60000.0):
        check(sample, dev, torch.full((3, 9000), v, dtype=torch.float16), [0.0, 0.4, 0.99], k=8500, p=0.7)


def test_random_numbers_out_of_range(sample, dev):
    import torch
    x = torch.full((5, 9000), -math.inf)
    x[:, 10:8990] = 0.0
    u = torch.tensor([1.0, 7.0, -1.0, math.nan, math.inf], device=dev)
    for kw in (dict(), dict(top_k=100), dict(top_p=0.5)):
        got = sample(x.to(dev), u, **kw).tolist()
        last = {0: 8989, 100: 109}.get(kw.get("top_k", 0)) if "top_p" not in kw else 4499
        assert got == [last, last, 10, 10, last], kw


def test_many_tokens_of_one_bin(sample, dev):
    """More candidates of a cut than the list in LDS takes, over a wide range of keys."""
    r = np.random.default_rng(9)
    import torch
    x = torch.from_numpy((r.random((6, 60000)) * 0.1).astype(np.float32))
    x[3:] -= 0.05                                     # both signs
    for s in (dict(k=20000), dict(p=0.4), dict(k=50000, p=0.7), dict(m=0.95), dict(k=30000, m=0.93, p=0.99)):
        check(sample, dev, x, grid(6), **s)


@pytest.mark.parametrize("dtype,V,g", [("bfloat16", 151936, -20.75), ("float16", 151936, -20.75), ("float32", 151936, -20.7),
                                       ("float32", 151936, -19.9), ("bfloat16", 1 << 22, -18.0), ("float32", 1 << 22, -17.3)])
def test_top_p_among_many_small_equal_logits(sample, dev, dtype, V, g):
    """One peak and small e = exp(g) everywhere else: top-p between the sums after the j-th of them and the
    next one keeps j + 1.  Half an e from either border: 4.8e-10 of all or more, 7.1e-9 with 2^22 logits, where
    sums may be off by 8e-11 and 1.9e-9."""
    import torch
    x = torch.full((6, V), g).to(getattr(torch, dtype))
    x[:, 0] = 0.0
    e = math.exp(float(x[0, 1]))
    u = torch.ones(1, device=dev)                     # counts as the last number: the last kept token
    for j in (0, 9, 1000, V // 3, V // 2 + 1, V - 3):
        p = (1 + (j + 0.5) * e) / (1 + (V - 1) * e)
        assert sample(x[:1].to(dev), u, top_p=p).tolist() == [j + 1], j
        # top-k takes from the same tokens: their sum is the whole of top-p
        k = V - V // 10
        if j < k - 2:
            p = (1 + (j + 0.5) * e) / (1 + (k - 1) * e)
            assert sample(x[:1].to(dev), u, top_k=k, top_p=p).tolist() == [j + 1], j


ONE_BIN = [  # dtype, vocabulary, temperature, two logits of one bin
    ("bfloat16", 151936, 7.89, -164.0, -165.0),
    ("float16", 151936, 7.89, -164.0, -165.0),
    ("float32", 151936, 7.84, -164.1, -164.7),
    ("float32", 151936, 0.858, -18.1, -18.15),
    ("bfloat16", 1 << 22, 7.75, -139.0, -140.0),
]


@pytest.mark.parametrize("dtype,V,T,a,b", ONE_BIN)
def test_top_p_behind_many_small_equal_logits(sample, dev, dtype, V, T, a, b):
    """The cut lies among the smaller of two values of one bin, behind the sum of all of the larger: half a share
    from either border, as above."""
    import torch
    n, m = V * 2 // 3, V // 4
    x = torch.full((1, V), -60000.0)
    x[:, 0], x[:, 1:1 + n], x[:, 1 + n:1 + n + m] = 0.0, a, b
    x = x.to(getattr(torch, dtype))
    ea, eb = (math.exp(float(x[0, i]) / T) for i in (1, 1 + n))
    for j in (0, 5, m // 2, m - 2):
        p = (1 + n * ea + (j + 0.5) * eb) / (1 + n * ea + m * eb)
        assert sample(x.to(dev), torch.ones(1, device=dev), temperature=T, top_p=p).tolist() == [1 + n + j], j


@pytest.mark.parametrize("dtype,V,T,a,b", ONE_BIN)
def test_draws_among_many_small_equal_logits(sample, dev, dtype, V, T, a, b):
    """Two values of one bin, the cut within the smaller: numbers in the middle of a token's share draw that
    token, in early and late slices.  Half a share is 3.2e-10 of all or more (2^22 logits: 7e-9)."""
    import torch
    n, m, k = V * 2 // 3, V // 4, V * 2 // 3 + V // 8
    x = torch.full((8, V), -60000.0)
    x[:, :n], x[:, n:n + m], x[:, n + m] = a, b, 0.0
    x = x.to(getattr(torch, dtype))
    ea, eb = (math.exp(float(x[0, i]) / T) for i in (0, n))
    at = [0, 1, 8191, 8192, n // 2, n - 1, n, n + V // 8 - 2]          # the peak is one of the k
    total = 1 + n * ea + (k - 1 - n) * eb
    u = [(min(i, n) * ea + max(i - n, 0) * eb + 0.5 * (ea if i < n else eb)) / total for i in at]
    assert check(sample, dev, x, u, T=T, k=k) == at


def test_strides_and_rows(sample, dev):
    import torch
    base = logits(6, 5003, "bfloat16", seed=10).to(dev)
    u = torch.tensor(grid(6), device=dev)
    want = sample(base, u, top_p=0.9)
    wide = torch.empty(6, 9001, dtype=base.dtype, device=dev)
    wide[:, 7:5010] = base
    assert torch.equal(sample(wide[:, 7:5010], u, top_p=0.9), want)          # rows 2-byte aligned
    assert torch.equal(sample(base.t().contiguous().t(), u, top_p=0.9), want)
    one = base[2:3].expand(6, -1)                     # a row for all
    assert torch.equal(sample(one, u, top_p=0.9), sample(one.contiguous(), u, top_p=0.9))
    out = torch.empty(6, dtype=torch.int32, device=dev)
    assert sample(base, u, top_p=0.9, out=out) is out and torch.equal(out, want)
    # a row alone is what it is among others
    for b in range(6):
        assert sample(base[b:b + 1], u[b:b + 1], top_p=0.9).item() == want[b]
    assert sample(base[:0], u[:0]).shape == (0,)


def test_many_rows(sample, dev):
    """More rows than a grid's second dimension would take."""
    import torch
    x = logits(70000, 40, "float32", seed=11, peaks=2)
    r = np.random.default_rng(12)
    u = r.random(70000).astype(np.float32)
    got = sample(x.to(dev), torch.from_numpy(u).to(dev), top_k=10, top_p=0.9).tolist()
    xs = x.double().numpy()
    for b in range(0, 70000, 701):
        assert got[b] == kve.draw(xs[b], float(u[b]), 1.0, 10, 0.9)
    assert min(got) >= 0 and max(got) < 40


def test_frequencies(sample, dev):
    """Over an even grid of random numbers every token comes as often as its probability, to one."""
    import torch
    p = np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    n = 4096
    x = torch.from_numpy(np.log(p).astype(np.float32)).repeat(n, 1)
    u = (torch.arange(n) + 0.5) / n
    got = np.bincount(sample(x.to(dev), u.to(dev)).cpu().numpy(), minlength=5)
    assert (np.abs(got - p * n) <= 1).all()


def test_captured_and_on_a_stream(sample, dev):
    import torch
    x, u = logits(9, 20000, "bfloat16", seed=13).to(dev), torch.rand(9, device=dev)
    T, out = torch.full((9,), 0.7, device=dev), torch.empty(9, dtype=torch.int32, device=dev)
    sample(x, u, temperature=T, top_k=50, top_p=0.9, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample(x, u, temperature=T, top_k=50, top_p=0.9, out=out)
    for i in range(4):
        u.copy_(torch.rand(9, device=dev))
        T.fill_(0.3 + 0.4 * i)
        x.copy_(logits(9, 20000, "bfloat16", seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, sample(x, u, temperature=T, top_k=50, top_p=0.9))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = sample(x, u, temperature=T, top_k=50, top_p=0.9)
    s.synchronize()
    assert torch.equal(a, got)


def test_refusals(sample, dev):
    import torch
    x, u = torch.zeros(2, 50, device=dev), torch.zeros(2, device=dev)
    for bad in (lambda: sample(x[0], u[:1]), lambda: sample(x, u[:1]), lambda: sample(x, u.double()),
                lambda: sample(x, u.cpu()), lambda: sample(x[:, :0], u), lambda: sample(x, u, temperature=-1.0),
                lambda: sample(x, u, temperature=math.nan), lambda: sample(x, u, temperature=math.inf),
                lambda: sample(x, u, top_p=-0.1), lambda: sample(x, u, top_p=math.nan), lambda: sample(x, u, min_p=1.1),
                lambda: sample(x, u, min_p=math.nan), lambda: sample(x, u, temperature=u.double()),
                lambda: sample(x, u, top_k=u), lambda: sample(x, u, top_p=u[:1]), lambda: sample(x, u, out=u),
                lambda: sample(x, u, out=torch.zeros(2, dtype=torch.int64, device=dev))):
        with pytest.raises(ValueError):
            bad()
    for bad in (x.double(), x.long()):
        with pytest.raises(TypeError):
            sample(bad, u)
    with pytest.raises(RuntimeError):
        sample(x.cpu(), u.cpu())


@pytest.mark.parametrize("T", [5e-324, 1e-310, 1e-300, 1e-90, 1e-60])
def test_temperatures_below_any_fp32(sample, dev, T):
    """Only tokens that equal the largest logit are drawn, however near the others are."""
    import torch
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[0.0, 3.0, -1.0, 3.0, big, big], [1e-45, 0.0, -0.0, 1e-45, -1e-45, 1e-45], [-big, big, 1.0, big, -1.0, 5.0]] * 2)
    for s in (dict(), dict(k=1), dict(k=2), dict(k=4, p=0.9), dict(p=0.3), dict(m=0.5), dict(m=1.0, p=0.6)):
        check(sample, dev, x, grid(6), T=T, **s)
