"""Performance cases of the packed-prompt serving path: prompts of different lengths through
causal attention, their keys and values rotated and appended to a 4-bit paged cache, and the
decode steps over that cache.

``listed()`` holds the named cases, ``draw(rng)`` one more case of the same ranges.  A case's
``kind`` names the entry point:

* ``prompt``  ``long_context.PackedPromptAttention.forward``: attention of packed prompts;
* ``append``  ``long_context.PagedInt4KVCache.append`` of a decode step or of whole prompts, with
              the queries rotated in the same call, and ``read`` of the appended tokens;
* ``decode``  ``long_context.PagedInt4KVCache.decode``: one query token of every sequence over
              its resident tokens.

The 4-bit format: of every token, head and group of ``group`` dimensions the smallest value
lo in fp16, the step s = (largest - lo) / 15 rounded to fp32 and then to fp16, and
code = round((x - lo) / s) in 0 .. 15 for the value lo + s * code.  Keys are rotated by
their position first (angles in 64 bits), to fp32.
"""
import math
import random

import torch

own = False

SINK = 2                 # pages kept from the start of a sequence
THETA = 1e6              # base of the rotation's frequencies
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # three short prompts that arrive together: the smallest prefill call
        dict(name="prompt_3x50_bf16", kind="prompt", seqs=3, tokens=150, q_heads=32, kv_heads=8, D=128, dtype="bf16"),
        # a batch of eight prompts of different lengths, an ordinary prefill step
        dict(name="prompt_8seq_8k_bf16", kind="prompt", seqs=8, tokens=8192, q_heads=32, kv_heads=8, D=128,
             dtype="bf16"),
        # one long document
        dict(name="prompt_16k_bf16", kind="prompt", seqs=1, tokens=16384, q_heads=32, kv_heads=8, D=128, dtype="bf16"),
        # narrow heads, every query head with its own keys, odd lengths
        dict(name="prompt_5seq_d64_f16", kind="prompt", seqs=5, tokens=4999, q_heads=16, kv_heads=16, D=64,
             dtype="f16"),
        # the activations of this engine's fp32 linears
        dict(name="prompt_2seq_2k_f32", kind="prompt", seqs=2, tokens=2048, q_heads=32, kv_heads=8, D=128, dtype="f32"),
        # one decode step of one sequence: the smallest append
        dict(name="append_1tok_f32", kind="append", seqs=1, tokens=1, past=4095, step=True, q_heads=32, kv_heads=8,
             D=128, dtype="f32", group=32, page=16, pages=512),
        # one decode step of a serving batch
        dict(name="append_64seq_step_bf16", kind="append", seqs=64, tokens=64, past=3000, step=True, q_heads=32,
             kv_heads=8, D=128, dtype="bf16", group=32, page=16, pages=512),
        # the prompts of a prefill step
        dict(name="append_8seq_8k_bf16", kind="append", seqs=8, tokens=8192, past=0, step=False, q_heads=32,
             kv_heads=8, D=128, dtype="bf16", group=32, page=16, pages=512),
        # a decode step at the context where one sequence no longer fills the card by itself
        dict(name="decode_1x2048_f32", kind="decode", seqs=1, tokens=2048, q_heads=32, kv_heads=8, D=128, dtype="f32",
             group=32, page=16, pages=2048),
        # a serving batch of ragged lengths
        dict(name="decode_64seq_bf16", kind="decode", seqs=64, tokens=64 * 3000, q_heads=32, kv_heads=8, D=128,
             dtype="bf16", group=32, page=16, pages=1024),
        # one very long sequence
        dict(name="decode_1x131072_bf16", kind="decode", seqs=1, tokens=131072, q_heads=32, kv_heads=8, D=128,
             dtype="bf16", group=64, page=64, pages=2048),
        # narrow heads without sharing, past the page limit: the sliding window has dropped the middle
        dict(name="decode_16seq_d64_f16", kind="decode", seqs=16, tokens=16 * 2500 + 7, q_heads=16, kv_heads=16, D=64,
             dtype="f16", group=64, page=16, pages=130),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "append", "decode"])
    kvh = rng.choice([1, 2, 4, 8, 16])
    share = rng.choice([1, 2, 4, 4, 5, 8])
    qh = kvh * share
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "prompt":
        D = rng.choice([64, 80, 128, 128, 256])
        most = 16384 if dtype != "f32" else 4096
        tokens = _log(rng, 20, most)
        seqs = min(_log(rng, 1, 24), tokens)
        # as much work as a 16k prompt of 32 heads of 128 at most, sequences of one length taken
        while tokens * tokens / seqs * qh * D > (2.0 if dtype != "f32" else 0.1) * 16384 * 16384 * 32 * 64:
            tokens -= tokens // 4
        return dict(kind=kind, seqs=min(seqs, tokens), tokens=tokens, q_heads=qh, kv_heads=kvh, D=D, dtype=dtype)
    D = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (32, 32, 64, 128) if g <= D])
    page = rng.choice([16, 16, 32, 64])
    if kind == "append":
        step = rng.random() < 0.5
        seqs = _log(rng, 1, 64 if step else 8)
        tokens = seqs if step else max(seqs, _log(rng, 16, 6000 * 40 * 128 // (D * (qh + kvh))))
        tokens = min(tokens, 8192)
        past = rng.choice([0, _log(rng, 1, 5000)])
        return dict(kind=kind, seqs=seqs, tokens=tokens, past=past, step=step, q_heads=qh, kv_heads=kvh, D=D,
                    dtype=dtype, group=group, page=page, pages=16384 // page)
    seqs = _log(rng, 1, 64)
    tokens = seqs * _log(rng, 20, 60000)
    while tokens * kvh * D > 64 * 2400 * 8 * 128:
        tokens -= tokens // 4
    tokens = max(tokens, seqs)
    pages = max(4, (tokens // seqs * 2 if rng.random() < 0.7 else tokens // seqs) // page)
    return dict(kind=kind, seqs=seqs, tokens=tokens, q_heads=qh, kv_heads=kvh, D=D, dtype=dtype, group=group,
                page=page, pages=pages)


def _lengths(total, n):
    """``total`` tokens in ``n`` sequences of unlike lengths, one token each at least."""
    r = random.Random(total * 131 + n)
    w = [r.uniform(0.3, 1.7) for _ in range(n)]
    got = [1 + int((total - n) * x / sum(w)) for x in w]
    got[-1] += total - sum(got)
    return got


def _starts(case):
    """Tokens that each sequence of an append case holds before the call."""
    r = random.Random(case["past"] * 17 + case["seqs"])
    return [int(case["past"] * r.uniform(0.5, 1.0)) if case["seqs"] > 1 else case["past"] for _ in range(case["seqs"])]


def _resident(seen, page, pages):
    """Tokens of a sequence that its pages hold: the first SINK pages and the newest ones."""
    opened = -(-seen // page)
    return seen if opened <= pages else (pages - 1) * page + seen - (opened - 1) * page


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    D, Hq, Hkv = c["D"], c["q_heads"], c["kv_heads"]
    if c["kind"] == "prompt":
        pairs = sum(n * (n + 1) // 2 for n in _lengths(c["tokens"], c["seqs"]))
        return dict(bytes=e * c["tokens"] * D * (2 * Hq + 2 * Hkv), flops=4 * Hq * D * pairs)
    row = D // 2 + 4 * D // c["group"]                       # one token's K or V of one head
    if c["kind"] == "append":
        N = c["tokens"]
        return dict(bytes=e * N * D * (2 * Hq + 4 * Hkv) + 4 * N * Hkv * row, flops=6 * N * D * (Hq + 2 * Hkv))
    held = sum(_resident(n, c["page"], c["pages"]) for n in _lengths(c["tokens"], c["seqs"]))
    return dict(bytes=2 * held * Hkv * row + 2 * e * c["seqs"] * Hq * D, flops=4 * Hq * D * held)


def _cum(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _keys(g, n, heads, D):
    """Keys as projections give them: some channels larger than others and off centre."""
    gain = 0.6 + 0.8 * torch.rand(heads, D, generator=g, device="cuda")
    mean = 0.8 * _normal(g, heads, D) * (torch.rand(heads, D, generator=g, device="cuda") < 0.1)
    return _normal(g, n, heads, D) * gain + mean


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    N, D, Hq, Hkv, B = c["tokens"], c["D"], c["q_heads"], c["kv_heads"], c["seqs"]
    if c["kind"] == "prompt":
        lengths = _lengths(N, B)
        st = dict(case=c, lengths=lengths, cu=_int32(_cum(lengths)), q=_normal(g, N, Hq, D).to(dt),
                  k=_keys(g, N, Hkv, D).to(dt), v=_normal(g, N, Hkv, D).to(dt))
        if own:
            st["attention"] = _long_context().PackedPromptAttention(Hq, Hkv, D)
        return st
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    if c["kind"] == "append":
        lengths = [1] * B if c["step"] else _lengths(N, B)
        starts = _starts(c)
        st = dict(case=c, inv=inv, cu=_int32(_cum(lengths)), start=_int32(starts),
                  q=_normal(g, N, Hq, D).to(dt), k=_keys(g, N, Hkv, D).to(dt), v=_normal(g, N, Hkv, D).to(dt))
        if own:
            st["cache"] = _cache(c)
        else:
            rows = B * c["pages"] * c["page"]
            st["codes"] = torch.zeros(2, rows, Hkv, D // 2, dtype=torch.uint8, device="cuda")
            st["steps"] = torch.zeros(2, rows, Hkv, D // c["group"], 2, dtype=torch.float16, device="cuda")
        return st
    lengths = _lengths(N, B)
    k, v = _keys(g, N, Hkv, D).to(dt), _normal(g, N, Hkv, D).to(dt)
    st = dict(case=c, inv=inv, seen=_int32(lengths), q=_normal(g, B, Hq, D).to(dt))
    if own:
        st["cache"] = _cache(c)
        st["cache"].append(k, v, _int32([0] * B), _int32(_cum(lengths)))
    else:
        st.update(_filled(c, inv, lengths, k, v))
    return st


def run(state):
    c = state["case"]
    if own:
        if c["kind"] == "prompt":
            return state["attention"].forward(state["q"], state["k"], state["v"], state["cu"])
        if c["kind"] == "append":
            cu = None if c["step"] else state["cu"]
            q, _ = state["cache"].append(state["k"], state["v"], state["start"], cu, query=state["q"])
            k, v = state["cache"].read(state["start"], cu, c["tokens"], dtype=q.dtype)
            return q, k, v
        return state["cache"].decode(state["q"], state["seen"])
    if c["kind"] == "prompt":
        return _plain_prompt(state)
    return _plain_append(state) if c["kind"] == "append" else _plain_decode(state)


def _long_context():
    import importlib

    import __graft_entry__
    return importlib.import_module(__graft_entry__.load_package().__name__ + ".long_context")


def _cache(c):
    return _long_context().PagedInt4KVCache(c["kv_heads"], c["D"], num_sequences=c["seqs"], page_size=c["page"],
                                            max_resident_pages=c["pages"], sink_pages=SINK, group_size=c["group"],
                                            rope_theta=THETA, device="cuda")


# ---- the plain forms ----------------------------------------------------------------------

def _plain_prompt(st):
    c = st["case"]
    Hkv, D = c["kv_heads"], c["D"]
    R = c["q_heads"] // Hkv
    outs, at = [], 0
    for n in st["lengths"]:                                # every prompt by itself
        q = st["q"][at:at + n].float().view(n, Hkv, R, D).permute(1, 2, 0, 3).reshape(Hkv, R * n, D)
        k = st["k"][at:at + n].float().permute(1, 2, 0).contiguous()
        v = st["v"][at:at + n].float().transpose(0, 1).contiguous()
        s = torch.matmul(q, k).view(Hkv, R, n, n).mul_(1.0 / math.sqrt(D))
        i = torch.arange(n, device="cuda")
        s.masked_fill_(i[None, :] > i[:, None], -math.inf)
        s.sub_(s.amax(-1, keepdim=True)).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(Hkv, R * n, n), v).view(Hkv, R, n, D) / total
        outs.append(o.permute(2, 0, 1, 3).reshape(n, Hkv * R, D).to(st["q"].dtype))
        at += n
    return torch.cat(outs)


def _rotate(x, pos, inv):
    """fp32 of x [n, heads, D] rotated at positions pos [n], in 64 bits."""
    ang = pos.double()[:, None] * inv
    co, si = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat((a * co - b * si, b * co + a * si), dim=-1).float()


def _encode(x, group):
    """Codes (two to a byte) and (step, lo) of fp32 x [n, heads, D]."""
    x = x.double().unflatten(-1, (-1, group))
    lo = x.amin(-1).clamp(-65504, 65504).half()
    step = ((x.amax(-1) - lo.double()) / 15).float().clamp(max=65504).half()
    code = ((x - lo.double()[..., None]) / step.double()[..., None]).round().clamp(0, 15)
    code = torch.where(step[..., None] > 0, code, 0).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.stack((step, lo), dim=-1)


def _decode_values(codes, steps):
    """fp32 values of packed codes [..., D / 2] with (step, lo) [..., D / group, 2]."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).unflatten(-1, (steps.shape[-2], -1))
    s = steps.float()
    return (c.float() * s[..., :1] + s[..., 1:]).flatten(-2)


def _slots(pos, page, pages):
    """Place of a position within its sequence's pages: the first SINK pages stay, the others take turns."""
    j = pos // page
    j = torch.where(j < SINK, j, SINK + (j - SINK) % (pages - SINK))
    return j * page + pos % page


def _plain_append(st):
    c = st["case"]
    n = c["tokens"]
    cu, start = st["cu"].long(), st["start"].long()
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = start[seq] + row - cu[seq]
    q = _rotate(st["q"], pos, st["inv"]).to(st["q"].dtype)
    k = _rotate(st["k"], pos, st["inv"])
    at = seq * (c["pages"] * c["page"]) + _slots(pos, c["page"], c["pages"])
    out = []
    for i, x in enumerate((k, st["v"].float())):           # keys, then values
        codes, steps = _encode(x, c["group"])
        st["codes"][i, at], st["steps"][i, at] = codes, steps
        out.append(_decode_values(st["codes"][i, at], st["steps"][i, at]).to(st["q"].dtype))
    return q, out[0], out[1]


def _filled(c, inv, lengths, k, v):
    """The resident tokens of every sequence, encoded, padded to the longest: [B, heads, T, ...]."""
    B, T = c["seqs"], max(_resident(n, c["page"], c["pages"]) for n in lengths)
    Hkv, D, G = c["kv_heads"], c["D"], c["D"] // c["group"]
    codes = torch.zeros(2, B, Hkv, T, D // 2, dtype=torch.uint8, device="cuda")
    steps = torch.zeros(2, B, Hkv, T, G, 2, dtype=torch.float16, device="cuda")
    held = []
    for b, (n, at) in enumerate(zip(lengths, _cum(lengths))):
        m = _resident(n, c["page"], c["pages"])
        pos = torch.arange(n, device="cuda")
        if m < n:
            first = SINK * c["page"]
            pos = torch.cat((pos[:first], pos[n - (m - first):]))
        rows = at + pos
        for i, x in enumerate((_rotate(k[rows], pos, inv), v[rows].float())):
            a, s = _encode(x, c["group"])
            codes[i, b, :, :m], steps[i, b, :, :m] = a.transpose(0, 1), s.transpose(0, 1)
        held.append(m)
    return dict(codes=codes, steps=steps, held=_int32(held))


def _plain_decode(st):
    c = st["case"]
    B, Hq, Hkv, D = c["seqs"], c["q_heads"], c["kv_heads"], c["D"]
    k, v = _decode_values(st["codes"][0], st["steps"][0]), _decode_values(st["codes"][1], st["steps"][1])
    q = st["q"].float().view(B, Hkv, Hq // Hkv, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(D))
    hidden = torch.arange(k.shape[2], device="cuda")[None] >= st["held"][:, None]
    s.masked_fill_(hidden[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    return o.reshape(B, Hq, D).to(st["q"].dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------

def exact(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    N, D, Hq, Hkv, B = c["tokens"], c["D"], c["q_heads"], c["kv_heads"], c["seqs"]
    if c["kind"] == "prompt":
        q, k, v = _normal(g, N, Hq, D).to(dt).double(), _keys(g, N, Hkv, D).to(dt).double(), _normal(g, N, Hkv, D).to(dt).double()
        out, at = torch.empty_like(q), 0
        for n in _lengths(N, B):
            for h in range(Hq):
                kh, vh = k[at:at + n, h * Hkv // Hq], v[at:at + n, h * Hkv // Hq]
                for i in range(0, n, 2048):
                    m = min(i + 2048, n)
                    s = (q[at + i:at + m, h] @ kh[:m].t()) / math.sqrt(D)
                    w = torch.exp(s - s.max(dim=1, keepdim=True).values).tril(i)
                    out[at + i:at + m, h] = (w @ vh[:m]) / w.sum(dim=1, keepdim=True)
            at += n
        return out
    freq = torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"),
                     torch.arange(D // 2, dtype=torch.float64, device="cuda").mul(-2.0 / D))

    def turned(x, pos):
        h = D // 2
        z = torch.complex(x[..., :h].double(), x[..., h:].double())
        ang = torch.outer(pos.double(), freq)[:, None]
        z = z * torch.complex(torch.cos(ang), torch.sin(ang))
        return torch.cat((z.real, z.imag), dim=2)

    def held(x):
        """The value that the 4-bit format holds for fp32 x."""
        y = x.float().double().reshape(*x.shape[:-1], D // c["group"], c["group"])
        low = torch.clip(y.min(dim=-1, keepdim=True).values, -65504.0, 65504.0).to(torch.float16).double()
        unit = (y.max(dim=-1, keepdim=True).values - low).div(15.0).to(torch.float32).to(torch.float16).double()
        n = torch.where(unit > 0, torch.clip(torch.round((y - low) / unit), 0, 15), torch.zeros_like(y))
        return (low + unit * n).reshape(x.shape)

    if c["kind"] == "append":
        lengths = [1] * B if c["step"] else _lengths(N, B)
        pos = torch.cat([torch.arange(s, s + n, device="cuda") for s, n in zip(_starts(c), lengths)])
        q, k, v = _normal(g, N, Hq, D).to(dt), _keys(g, N, Hkv, D).to(dt), _normal(g, N, Hkv, D).to(dt)
        return turned(q, pos), held(turned(k, pos)), held(v)
    lengths = _lengths(N, B)
    k, v = _keys(g, N, Hkv, D).to(dt), _normal(g, N, Hkv, D).to(dt)
    q = _normal(g, B, Hq, D).to(dt).double()
    out, at = torch.empty_like(q), 0
    for b, n in enumerate(lengths):
        opened = (n + c["page"] - 1) // c["page"]
        page = torch.arange(n, device="cuda") // c["page"]
        pos = torch.nonzero((page < SINK) | (page >= opened - (c["pages"] - SINK))).flatten()
        kk, vv = held(turned(k[at:at + n][pos], pos)), held(v[at:at + n][pos])
        for h in range(Hq):
            w = torch.softmax((kk[:, h * Hkv // Hq] @ q[b, h]) / math.sqrt(D), dim=0)
            out[b, h] = w @ vv[:, h * Hkv // Hq]
        at += n
    return out
