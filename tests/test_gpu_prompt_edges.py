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


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
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
    assert (np.abs(got - want) <= tol + 1e-7 * (dtype == "float16")).all(), (got.ravel()[:4], want)
