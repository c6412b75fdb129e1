"""The 4-bit KV cache, its rotation and the attentions around it, in fp64 numpy from
their definitions (include/ojasx_lut_c_api.h, "4-bit paged KV cache")."""
import numpy as np


def inv_freq(rot, theta):
    return theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


def rotate(x, pos, freq, interleaved=False):
    """x [n, heads, D] rotated by positions pos [n]; fp64, not rounded."""
    x = np.asarray(x, np.float64).copy()
    rot = 2 * len(freq)
    ang = np.asarray(pos, np.float64)[:, None] * freq
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    xa, xb = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x


def held(x, group):
    """The fp64 values that the format holds for fp32 x [..., D]: lo + s code."""
    x = np.asarray(x, np.float32)
    y = x.astype(np.float64).reshape(*x.shape[:-1], -1, group)
    bad = ~np.isfinite(y).all(-1, keepdims=True)
    y = np.where(bad, 0.0, y)
    lo = np.clip(y.min(-1, keepdims=True), -65504, 65504).astype(np.float16).astype(np.float64)
    step = np.float32((y.max(-1, keepdims=True) - lo) / 15)
    s = np.clip(step, np.float32(0), np.float32(65504)).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(s > 0, np.clip(np.rint((y - lo) / s), 0, 15), 0)
    return np.where(bad, np.nan, lo + s * code).reshape(x.shape)


def resident(seen, page, pages, sink):
    """Positions that a sequence of ``seen`` tokens holds, ascending."""
    opened = -(-seen // page)
    j = np.arange(seen) // page
    return np.nonzero((j < sink) | (j >= opened - (pages - sink)))[0]


def attention(q, k, v, scale, first_hidden=None):
    """softmax(scale q k^T) v of q [m, D] over k, v [t, D] in fp64; row i sees the keys
    before first_hidden[i] (all without it); a row that sees none is 0.  Hidden keys
    take no part.  Returns (out, log-sum-exp)."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, lse = np.zeros((len(q), v.shape[1])), np.full(len(q), -np.inf)
    for i in range(len(q)):
        t = len(k) if first_hidden is None else int(np.clip(first_hidden[i], 0, len(k)))
        if t:
            s = k[:t] @ q[i] * scale
            m = s.max()
            w = np.exp(s - m)
            out[i] = w @ v[:t] / w.sum()
            lse[i] = m + np.log(w.sum())
    return out, lse
