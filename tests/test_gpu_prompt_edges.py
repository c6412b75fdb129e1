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
