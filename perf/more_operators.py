"""Performance cases of a serving batch's decode steps in bounded memory: a paged key-value cache
that counts the attention its tokens get and drops those that get least, and the draw of the
next token from the logits.

``listed()`` holds the named cases, ``draw(rng)`` one more case of the same ranges.  A case's
``kind`` names the entry point:

* ``append``  ``long_context.PagedEvictingKVCache.append`` of a decode step or of whole prompts, keys
              and the queries beside them rotated by their positions;
* ``decode``  ``long_context.PagedEvictingKVCache.decode``: one query token of every sequence over the
              tokens that it holds, the softmax's weights added to each token's count;
* ``evict``   ``long_context.PagedEvictingKVCache.evict`` behind the append that filled the cache up:
              of a chunk of new tokens (``chunk``), or of whole prompts;
* ``sample``  ``decoder.sample_tokens``: temperature, top-k, top-p and min-p, and one token of every
              row from a given random number.

The cache: token t of a sequence lies in slot t % page of page block_table[sequence, t // page], with
its key, value, weight (the softmax weights that it got, summed over the query heads of its kv head)
and position.  Eviction keeps ``budget`` tokens of each sequence and kv head: those at positions
below ``sink``, the ``recent`` newest positions, and of the others the ones of largest weight, ties to
the lowest slot.  A kept token from behind the budget takes the place of a dropped one before it,
the i-th of them the i-th place.
"""
import math
import random

import torch

own = False

THETA = 1e6              # base of the rotation's frequencies
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one decode step of a serving batch: the smallest append
        dict(name="append_64seq_step_bf16", kind="append", seqs=64, tokens=64, past=900, step=True, q_heads=32,
             kv_heads=8, D=128, dtype="bf16", page=16, pages=64),
        # the prompts of a prefill step
        dict(name="append_8seq_8k_bf16", kind="append", seqs=8, tokens=8192, past=0, step=False, q_heads=32,
             kv_heads=8, D=128, dtype="bf16", page=16, pages=128),
        # one sequence that does not fill the card, in the type of this engine's linears
        dict(name="decode_1x2048_f32", kind="decode", seqs=1, tokens=2048, q_heads=32, kv_heads=8, D=128, dtype="f32",
             page=16, pages=128),
        # a serving batch of ragged lengths
        dict(name="decode_64seq_bf16", kind="decode", seqs=64, tokens=64 * 3000, q_heads=32, kv_heads=8, D=128,
             dtype="bf16", page=16, pages=352),
        # one very long sequence
        dict(name="decode_1x131072_bf16", kind="decode", seqs=1, tokens=131072, q_heads=32, kv_heads=8, D=128,
             dtype="bf16", page=64, pages=2048),
        # narrow heads without sharing, odd lengths
        dict(name="decode_16seq_d64_f16", kind="decode", seqs=16, tokens=16 * 2500 + 7, q_heads=16, kv_heads=16, D=64,
             dtype="f16", page=16, pages=288),
        # one sequence at its budget, the smallest eviction: a step's chunk of tokens for as many old ones
        dict(name="evict_1seq_step_f32", kind="evict", seqs=1, budget=1000, chunk=8, sink=4, recent=64, q_heads=32,
             kv_heads=8, D=128, dtype="f32", page=16),
        # a serving batch at its budget, evicting every 16 tokens
        dict(name="evict_64seq_16new_bf16", kind="evict", seqs=64, budget=2048, chunk=16, sink=4, recent=256,
             q_heads=32, kv_heads=8, D=128, dtype="bf16", page=16),
        # prompts cut down to the budget that they are decoded with
        dict(name="evict_8seq_prompts_bf16", kind="evict", seqs=8, budget=1024, tokens=8 * 4096, sink=4, recent=128,
             q_heads=32, kv_heads=8, D=128, dtype="bf16", page=16),
        # a decode step of one sequence over this engine's vocabulary
        dict(name="sample_1x151936_f32", kind="sample", rows=1, vocab=151936, dtype="f32", T=0.7, k=50, p=0.9, m=0.0,
             mixed=False),
        # a serving batch whose requests ask for different settings
        dict(name="sample_64x151936_bf16", kind="sample", rows=64, vocab=151936, dtype="bf16", T=1.0, k=0, p=0.95,
             m=0.0, mixed=True),
        # a large batch without truncation
        dict(name="sample_256x32000_f16", kind="sample", rows=256, vocab=32000, dtype="f16", T=0.8, k=0, p=1.0, m=0.0,
             mixed=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "evict", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "sample":
        rows = _log(rng, 1, 256)
        vocab = _log(rng, 500, min(260000, 64 * 151936 // rows))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, T=round(rng.uniform(0.2, 1.6), 3),
                    k=rng.choice([0, 0, 1, _log(rng, 2, 400)]), p=rng.choice([1.0, 0.9, round(rng.uniform(0.05, 1.0), 3)]),
                    m=rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.0, 0.4), 3)]), mixed=rng.random() < 0.4)
    kvh = rng.choice([1, 2, 4, 8, 16])
    qh = kvh * rng.choice([1, 2, 4, 4, 5, 8])
    D = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64])
    shape = dict(kind=kind, q_heads=qh, kv_heads=kvh, D=D, dtype=dtype, page=page)
    if kind == "append":
        step = rng.random() < 0.5
        seqs = _log(rng, 1, 64 if step else 8)
        tokens = seqs if step else max(seqs, _log(rng, 16, 6000 * 40 * 128 // (D * (qh + kvh))))
        tokens = min(tokens, 8192)
        past = rng.choice([0, _log(rng, 1, 1000)])
        most = past + (1 if step else max(_lengths(tokens, seqs)))
        return dict(shape, seqs=seqs, tokens=tokens, past=past, step=step, pages=-(-most // page))
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        tokens = seqs * _log(rng, 20, 60000)
        while tokens * kvh * D * (2 if dtype == "f32" else 1) > 64 * 2500 * 8 * 128:
            tokens -= tokens // 4
        tokens = max(tokens, seqs)
        return dict(shape, seqs=seqs, tokens=tokens, pages=-(-max(_lengths(tokens, seqs)) // page))
    seqs = _log(rng, 1, 32)
    budget = _log(rng, 32, 4096)
    while seqs * budget * kvh * D > 64 * 1500 * 8 * 128:
        budget -= budget // 4
    sink = rng.choice([0, 4])
    if rng.random() < 0.5:
        return dict(shape, seqs=seqs, budget=budget, sink=sink, recent=rng.randint(0, (budget - sink) // 2),
                    chunk=_log(rng, 1, max(2, budget // 8)))
    longer = rng.uniform(1.0, 6.0)
    while seqs * budget * longer * (qh + 2 * kvh) * D > 32768 * 48 * 128:
        budget -= budget // 4
    return dict(shape, seqs=seqs, budget=budget, sink=sink, recent=rng.randint(0, (budget - sink) // 2),
                tokens=seqs * int(budget * longer) + rng.randint(0, 9))


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


def _held(case):
    """Tokens that each sequence of an evict case holds before the eviction."""
    if "chunk" in case:
        return [case["budget"] + case["chunk"]] * case["seqs"]
    return _lengths(case["tokens"], case["seqs"])


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "sample":
        # one exponential of every logit: about 20 operations
        return dict(bytes=c["rows"] * (c["vocab"] * e + 8), flops=20 * c["rows"] * c["vocab"])
    D, Hq, Hkv = c["D"], c["q_heads"], c["kv_heads"]

    def append(n, weights):
        return e * n * D * (2 * Hq + 4 * Hkv) + n * Hkv * (12 if weights else 8), 6 * n * D * (Hq + Hkv)

    if c["kind"] == "append":
        b, f = append(c["tokens"], False)
        return dict(bytes=b, flops=f)
    if c["kind"] == "decode":
        n = c["tokens"]
        return dict(bytes=n * Hkv * (2 * D * e + 8) + 2 * e * c["seqs"] * Hq * D, flops=4 * Hq * D * n)
    # each held token's weight and position is read; moves: of the kept ones, those behind the budget
    held = _held(c)
    if "chunk" in c:
        b, f = append(c["seqs"] * c["chunk"], True)
        moved = c["seqs"] * c["chunk"]
    else:
        b, f = append(c["tokens"], True)
        moved = sum(c["budget"] * (n - c["budget"]) // n for n in held if n > c["budget"])
    return dict(bytes=b + 8 * Hkv * sum(held) + 2 * Hkv * moved * (2 * D * e + 8), flops=f)


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


def _weights(g, *shape):
    """Attention weights summed over some steps: a few tokens have most of them."""
    return (2.0 * _normal(g, *shape) - 4.0).exp()


def _logits(case, g):
    """Logits as a language model gives them: a wide body and a few tokens that stand out."""
    B, V = case["rows"], case["vocab"]
    x = 2.0 * _normal(g, B, V) - 2.0
    top = torch.randint(0, V, (B, 12), generator=g, device="cuda")
    x.scatter_add_(1, top, 4.0 + 3.0 * _normal(g, B, 12))
    return x.to(DTYPES[case["dtype"]])


def _settings(case):
    """Temperature, top-k, top-p and min-p: one value for all rows, or a tensor of a value for each."""
    B = case["rows"]
    if not case["mixed"]:
        return case["T"], case["k"], case["p"], case["m"]
    r = random.Random(case["vocab"] * 7 + B)
    T = [r.choice([case["T"], 0.0, 0.3, 0.7, 1.0, 1.4]) for _ in range(B)]
    k = [r.choice([case["k"], 0, 1, 40, 200]) for _ in range(B)]
    p = [r.choice([case["p"], 1.0, 0.9, 0.5]) for _ in range(B)]
    m = [r.choice([case["m"], 0.0, 0.02, 0.1]) for _ in range(B)]
    return (torch.tensor(T, device="cuda"), _int32(k), torch.tensor(p, device="cuda"), torch.tensor(m, device="cuda"))


def _inputs(case, seed):
    """What the plain forms, the kernels and the definitions all begin with."""
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "sample":
        return dict(logits=_logits(c, g), uniform=torch.rand(c["rows"], generator=g, device="cuda"))
    dt = DTYPES[c["dtype"]]
    D, Hq, Hkv, B, P = c["D"], c["q_heads"], c["kv_heads"], c["seqs"], c["page"]
    pages = c["pages"] if "pages" in c else -(-max(_held(c)) // P)
    got = dict(table=torch.randperm(B * pages, generator=g, device="cuda").to(torch.int32).view(B, pages))
    pool = (B * pages, Hkv, P)
    if c["kind"] == "decode" or "chunk" in c:              # the tokens that are there already
        n = B * pages * P
        got["keys"] = _keys(g, n, Hkv, D).view(B * pages, P, Hkv, D).transpose(1, 2).to(dt).contiguous()
        got["values"] = _normal(g, *pool, D).to(dt)
        got["weights"] = _weights(g, *pool)
        first = torch.empty(B, pages, dtype=torch.int64, device="cuda").copy_(torch.arange(pages, device="cuda") * P)
        base = torch.empty(B * pages, dtype=torch.int64, device="cuda")
        base[got["table"].flatten().long()] = first.flatten()
        slot = base[:, None] + torch.arange(P, device="cuda")
        got["positions"] = slot[:, None].expand(pool).to(torch.int32).contiguous()
    else:
        got["keys"] = torch.zeros(*pool, D, dtype=dt, device="cuda")
        got["values"] = torch.zeros_like(got["keys"])
        got["weights"] = torch.zeros(pool, device="cuda")
        got["positions"] = torch.zeros(pool, dtype=torch.int32, device="cuda")
    if c["kind"] == "decode":
        got["held"] = _int32(_lengths(c["tokens"], B))
        got["q"] = _normal(g, B, Hq, D).to(dt)
        return got
    if c["kind"] == "append":
        lengths = [1] * B if c["step"] else _lengths(c["tokens"], B)
        start, at = _starts(c), [100 + 3 * n for n in _starts(c)]
    elif "chunk" in c:                                     # behind the budget, at positions far past it
        lengths, start, at = [c["chunk"]] * B, [c["budget"]] * B, [3 * c["budget"]] * B
    else:
        lengths, start, at = _held(c), [0] * B, [0] * B
    N = sum(lengths)
    got.update(lengths=lengths, cu=_int32(_cum(lengths)), start=_int32(start), position=_int32(at),
               q=_normal(g, N, Hq, D).to(dt), k=_keys(g, N, Hkv, D).to(dt), v=_normal(g, N, Hkv, D).to(dt))
    if c["kind"] == "evict":
        got["held"], got["w"] = _int32(_held(c)), _weights(g, N, Hkv)
    return got


def prepare(case, seed):
    c = case
    st = dict(_inputs(c, seed), case=c)
    if c["kind"] == "sample":
        st["settings"] = _settings(c)
    else:
        st["most"] = max(_held(c)) if c["kind"] == "evict" else 0
        if own:
            cache = _module("long_context").PagedEvictingKVCache(
                c["kv_heads"], c["D"], num_sequences=c["seqs"], page_size=c["page"], max_pages=st["table"].shape[1],
                num_pages=st["table"].numel(), rope_theta=THETA, dtype=DTYPES[c["dtype"]], device="cuda")
            cache.block_table.copy_(st.pop("table"))
            for name in ("keys", "values", "weights", "positions"):
                getattr(cache, name).copy_(st.pop(name))
            st["cache"] = cache
        else:
            st["inv"] = THETA ** (-torch.arange(0, c["D"], 2, dtype=torch.float64, device="cuda") / c["D"])
            st["index"] = _index(c, st["table"])
    return st


def run(state):
    c = state["case"]
    if c["kind"] == "sample":
        if not own:
            return _plain_sample(state)
        T, k, p, m = state["settings"]
        return _module("decoder").sample_tokens(state["logits"], state["uniform"], temperature=T, top_k=k, top_p=p, min_p=m)
    if c["kind"] == "decode":
        if not own:
            return _plain_decode(state), state["weights"]
        return state["cache"].decode(state["q"], state["held"]), state["cache"].weights
    pool = state["cache"] if own else None
    one = c.get("step", False)                             # a token of every sequence: no bounds needed
    if own:
        q = pool.append(state["k"], state["v"], state["start"], None if one else state["cu"],
                        position=state["position"], query=state["q"], weight=state.get("w"))
    else:
        q = _plain_append(state)
    if c["kind"] == "evict":
        if own:
            pool.evict(state["held"], c["budget"], sink_tokens=c["sink"], recent_tokens=c["recent"],
                       max_held=state["most"])
        else:
            _plain_evict(state)
        if "chunk" in c:                                   # the next chunk's positions
            state["position"].add_(c["chunk"])
    if own:
        return q, pool.keys, pool.values, pool.weights, pool.positions
    return q, state["keys"], state["values"], state["weights"], state["positions"]


def _module(name):
    import importlib

    import __graft_entry__
    return importlib.import_module(__graft_entry__.load_package().__name__ + "." + name)


# ---- the plain forms ----------------------------------------------------------------------

def _index(c, table):
    """Of each sequence, kv head and slot its row of the pool: [B, heads, slots]."""
    P, H = c["page"], c["kv_heads"]
    t = torch.arange(table.shape[1] * P, device="cuda")
    page = table.long()[:, t // P]
    return (page[:, None] * H + torch.arange(H, device="cuda")[None, :, None]) * P + t % P


def _rotate(x, pos, inv):
    """x [n, heads, D] rotated at positions pos [n], in 64 bits, in its own type."""
    ang = pos.double()[:, None] * inv
    co, si = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat((a * co - b * si, b * co + a * si), dim=-1).to(x.dtype)


def _plain_append(st):
    D = st["case"]["D"]
    n = st["k"].shape[0]
    cu, row = st["cu"].long(), torch.arange(n, device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    ahead = row - cu[seq]
    pos = st["position"].long()[seq] + ahead
    at = st["index"][seq, :, st["start"].long()[seq] + ahead]          # [n, heads]
    st["keys"].view(-1, D)[at] = _rotate(st["k"], pos, st["inv"])
    st["values"].view(-1, D)[at] = st["v"]
    st["weights"].view(-1)[at] = st["w"] if "w" in st else 0.0
    st["positions"].view(-1)[at] = pos.to(torch.int32)[:, None].expand_as(at)
    return _rotate(st["q"], pos, st["inv"])


def _plain_decode(st):
    c = st["case"]
    B, Hq, Hkv, D = c["seqs"], c["q_heads"], c["kv_heads"], c["D"]
    k, v = (st[name].view(-1, D)[st["index"]].float() for name in ("keys", "values"))
    q = st["q"].float().view(B, Hkv, Hq // Hkv, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(D))
    hidden = torch.arange(k.shape[2], device="cuda")[None] >= st["held"][:, None]
    s.masked_fill_(hidden[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s.div_(s.sum(-1, keepdim=True))
    w = st["weights"].view(-1)
    w[st["index"]] = w[st["index"]] + s.sum(2)
    return torch.matmul(s, v).reshape(B, Hq, D).to(st["q"].dtype)


def _plain_evict(st):
    c = st["case"]
    index, held, budget = st["index"], st["held"].long()[:, None, None], c["budget"]
    t = torch.arange(index.shape[2], device="cuda")
    there = (t < held).expand(index.shape)
    pos = st["positions"].view(-1)[index].long().masked_fill(~there, -1)
    rank = st["weights"].view(-1)[index].double()
    rank = rank.masked_fill((pos < c["sink"]) | (pos > pos.amax(-1, keepdim=True) - c["recent"]), math.inf)
    rank = rank.masked_fill(~there, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(there).scatter_(-1, order[..., :budget], True) & there
    full = held > budget
    to, of = index[full & ~keep & (t < budget)], index[full & keep & (t >= budget)]
    for name in ("keys", "values", "weights", "positions"):
        rows = st[name].view(-1, c["D"]) if st[name].dim() == 4 else st[name].view(-1)
        rows[to] = rows[of]


def _plain_sample(st):
    x = st["logits"].double()
    B, V = x.shape
    T, k, p, m = (torch.as_tensor(a, dtype=torch.float64, device="cuda").expand(B)[:, None] for a in st["settings"])
    greedy = T == 0.0
    e = ((x - x.amax(1, keepdim=True)) / T.masked_fill(greedy, 1.0)).exp()
    order = x.sort(dim=1, descending=True, stable=True).indices
    rank = torch.arange(V, device="cuda")
    s = e.gather(1, order)
    keep = (rank < k) | (k <= 0.0)
    s = s * keep
    before = torch.nn.functional.pad(s.cumsum(1), (1, 0))
    keep &= (before[:, :-1] < p * before[:, -1:]) | (p >= 1.0) | (rank == 0)
    keep &= (s >= m) & (~greedy | (rank == 0))
    w = e * torch.zeros_like(keep).scatter_(1, order, keep)
    total = w.cumsum(1)
    hit = total > st["uniform"].double()[:, None] * total[:, -1:]
    return hit.to(torch.int32).argmax(1).to(torch.int32)


# ---- the definitions in 64 bits -----------------------------------------------------------

def exact(case, seed):
    c = case
    x = _inputs(c, seed)
    if c["kind"] == "sample":
        return _exact_sample(c, x)
    D, Hq, Hkv, B, P = c["D"], c["q_heads"], c["kv_heads"], c["seqs"], c["page"]
    K, V, W, pos = x["keys"].double(), x["values"].double(), x["weights"].double(), x["positions"].clone()
    table = x["table"].long()

    def slots(b, t):
        return table[b, torch.div(t, P, rounding_mode="floor")], torch.remainder(t, P)

    if c["kind"] == "decode":
        out = torch.empty(B, Hq, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(x["held"].tolist()):
            page, slot = slots(b, torch.arange(n, device="cuda"))
            for h in range(Hkv):
                k, v, group = K[page, h, slot], V[page, h, slot], range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                for j in group:
                    w = torch.softmax(torch.mv(k, x["q"][b, j].double()) / math.sqrt(D), dim=0)
                    out[b, j] = torch.mv(v.t(), w)
                    W[page, h, slot] += w
        return out, W
    freq = torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"),
                     torch.arange(D // 2, dtype=torch.float64, device="cuda").mul(-2.0 / D))

    def turned(y, at):
        h = D // 2
        z = torch.complex(y[..., :h].double(), y[..., h:].double())
        ang = torch.outer(at.double(), freq)[:, None]
        z = z * torch.complex(torch.cos(ang), torch.sin(ang))
        return torch.cat((z.real, z.imag), dim=2)

    q = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    first, start, turn = 0, x["start"].tolist(), x["position"].tolist()
    for b, n in enumerate(x["lengths"]):
        rows = slice(first, first + n)
        t = torch.arange(n, device="cuda")
        page, slot = slots(b, start[b] + t)
        K[page, :, slot] = turned(x["k"][rows], turn[b] + t)
        V[page, :, slot] = x["v"][rows].double()
        W[page, :, slot] = x["w"][rows].double() if "w" in x else 0.0
        pos[page, :, slot] = (turn[b] + t).to(torch.int32)[:, None]
        q[rows] = turned(x["q"][rows], turn[b] + t)
        first += n
    if c["kind"] == "evict":
        for b, n in enumerate(x["held"].tolist()):
            if n <= c["budget"]:
                continue
            page, slot = slots(b, torch.arange(n, device="cuda"))
            for h in range(Hkv):
                at = pos[page, h, slot].cpu()
                w = W[page, h, slot].cpu()
                safe = (at < c["sink"]) | (at > int(at.max()) - c["recent"])
                first_of_all = sorted(range(n), key=lambda i, s=safe.tolist(), u=w.tolist(): (not s[i], 0.0 if s[i] else -u[i], i))
                kept = set(first_of_all[:c["budget"]])
                to = [i for i in range(c["budget"]) if i not in kept]
                of = sorted(i for i in kept if i >= c["budget"])
                to, of = torch.tensor(to, device="cuda", dtype=torch.int64), torch.tensor(of, device="cuda", dtype=torch.int64)
                for y in (K, V, W, pos):
                    y[page[to], h, slot[to]] = y[page[of], h, slot[of]]
    return q, K, V, W, pos


def _exact_sample(c, x):
    """Row by row: sorted by value and place, cut, and the running sum in the vocabulary's order."""
    settings = [a.double().tolist() if torch.is_tensor(a) else [float(a)] * c["rows"] for a in _settings(c)]
    got = []
    for b, (T, k, p, m) in enumerate(zip(*settings)):
        row = x["logits"][b].double().cpu()
        at = torch.argsort(-row, stable=True)
        if T == 0.0:
            got.append(int(at[0]))
            continue
        e = torch.exp((row[at] - row[at[0]]) / T)
        if k > 0:
            e = e[:int(k)]
        if p < 1.0:
            run_sum = torch.cumsum(e, 0)
            e = e[:max(1, int((run_sum < p * run_sum[-1]).sum()) + 1)]
        e = e[e >= m]
        at, back = torch.sort(at[:e.numel()])
        run_sum = torch.cumsum(e[back], 0)
        i = int(torch.searchsorted(run_sum, x["uniform"][b].double().cpu() * run_sum[-1], right=True))
        got.append(int(at[min(i, at.numel() - 1)]))
    return torch.tensor(got, dtype=torch.int32)
