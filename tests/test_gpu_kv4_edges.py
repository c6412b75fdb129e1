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
