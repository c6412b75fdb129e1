"""Paged KV storage on the GPU, on the kernels of csrc/kv_pages.hip and
csrc/lut_kv.hip.

* ``PagedCompressedKVCache`` mirrors ojasx_24x96/long_context.py:212-279: the
  int8 cache with per-token fp16 scales and sink + sliding-window eviction.
  Names, argument meaning, validation, the page list ``_pages`` of
  ``(qk, sk, qv, sv)`` and ``storage_bytes`` match the reference.  Each page
  gets tensors of its own length, so an evicted page keeps its values for a
  caller that still holds it, as the reference's popped page does; the memory
  of an evicted page nobody holds returns to torch's caching allocator and is
  reused by a later page without a device allocation.
* ``PagedCodeKVCache`` is the code-domain counterpart for decode: per token
  and kv head, 8-bit codes into a 256-centroid codebook (or the reference's
  scalar quantiser, ojasx_lut_kv_cache.cpp:16-65) and an fp32 scale, in the
  page layout [page][kv head][slot][group] that ``decode`` reads through a
  block table.  Tokens fill pages in order; opening a page beyond
  ``max_resident_pages`` evicts the oldest page after the ``sink_pages`` first
  ones (the reference's eviction rule, long_context.py:255-257).

* ``OnlineSoftmaxBlockAttention`` mirrors long_context.py:47-209: exact
  attention over streamed (K, V) tiles with fp64 online-softmax state, on the
  kernels of csrc/attn_stream.hip.  ``forward_stream`` takes any iterable of
  tiles (one device update per tile, tiles moved to the query's device as the
  reference moves them) or a ``PagedCompressedKVCache`` itself, whose int8
  pages are then read in place and dequantised in registers, all pages in
  one update.

* ``PagedInt4KVCache`` is the cache of a serving batch: the keys and values of
  several sequences in 4 bits, with the position rotation applied on the way
  in (csrc/kv4_append.hip, csrc/kv4_decode.hip).  The sequences' lengths are
  the caller's, in device memory, so its calls can be captured.
* ``PagedEvictingKVCache`` holds keys and values of a serving batch in their own
  type, counts the attention that each token gets and drops those that get
  least (csrc/kve_append.hip, csrc/kve_decode.hip, csrc/kve_evict.hip).
* ``PackedPromptAttention`` is the prefill beside them: attention of a batch of
  prompts of different lengths, packed row by row, causal, grouped heads
  (csrc/prompt_attn.hip).

Everything runs on the GPU; CPU queries raise.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Iterable, Iterator, List, Optional, Tuple

import numpy as np

from . import _lib


def _torch():
    import torch
    return torch


def _vp(t):
    return t.data_ptr()


def _stream():
    return _lib.raw_stream(_torch().cuda.current_device())


def _require_gpu(t, what):
    if not t.is_cuda:
        raise RuntimeError(f"{what}: the KV cache runs on the GPU only (got a {t.device} tensor)")


def _dtype_tag(dtype):
    torch = _torch()
    tags = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}
    if dtype not in tags:
        raise TypeError(f"unsupported KV dtype {dtype}: float32, bfloat16, float16 or float64")
    return tags[dtype]


def _quantize_into(t, q, s):
    """Quantise t [..., R, D] (contiguous over its last two dimensions, uniform
    stride over the leading ones) into q [..., >=R, D] int8 and s [..., >=R, 1]
    fp16 views with the same leading shape."""
    lead = int(np.prod(t.shape[:-2])) if t.dim() > 2 else 1
    rows, dim = t.shape[-2], t.shape[-1]
    if rows > 2**31 - 1 or dim > 2**31 - 1:
        raise ValueError("int8 quantisation: more than 2^31 - 1 rows or columns in one call")
    xs = t.stride(-3) if t.dim() > 2 else rows * dim
    qs = q.stride(-3) if q.dim() > 2 else 0
    ss = s.stride(-3) if s.dim() > 2 else 0
    rc = _lib.lib().ojasx_quantize_int8_device(_vp(t), lead, rows, dim, xs, _dtype_tag(t.dtype),
                                               _vp(q), qs, _vp(s), ss, _stream())
    _lib.check(rc, "ojasx_quantize_int8_device")


class PagedCompressedKVCache:
    """Bounded-memory int8 paged KV cache (long_context.py:212-279): K/V pages
    of ``page_size`` tokens quantised per token to int8 with an fp16 scale;
    beyond ``max_resident_pages`` pages the oldest page after the
    ``sink_pages`` first ones is evicted."""

    def __init__(self, page_size: int = 256, max_resident_pages: int = 64,
                 sink_pages: int = 2) -> None:
        if page_size <= 0 or max_resident_pages <= sink_pages:
            raise ValueError("Invalid page configuration for PagedCompressedKVCache")
        self.page_size = int(page_size)
        self.max_resident_pages = int(max_resident_pages)
        self.sink_pages = int(sink_pages)
        self.total_tokens_seen: int = 0
        self._pages: List[Tuple] = []
        self._layout = None              # (B, H, D, device) of the first append
        self._version = 0                # bumped by every append
        self._tiles = None               # (version, attention tile array, tokens, max page)

    @staticmethod
    def _quantize_int8(t):
        """long_context.py:234-240 on the GPU: t [..., D] float32/bfloat16/
        float16/float64 -> (q int8 [..., D], scale float16 [..., 1])."""
        torch = _torch()
        _require_gpu(t, "PagedCompressedKVCache._quantize_int8")
        t = t.contiguous()
        q = torch.empty(t.shape, dtype=torch.int8, device=t.device)
        s = torch.empty((*t.shape[:-1], 1), dtype=torch.float16, device=t.device)
        if t.numel():
            flat = t.reshape(1, -1, t.shape[-1])
            _quantize_into(flat, q.view(1, -1, t.shape[-1]), s.view(1, -1, 1))
        return q, s

    @staticmethod
    def _dequantize_int8(q, scale, dtype):
        """long_context.py:242-244 on the GPU: float(q) * float(scale) in
        float32, returned as ``dtype``."""
        torch = _torch()
        _require_gpu(q, "PagedCompressedKVCache._dequantize_int8")
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
        if q.numel():
            dim = q.shape[-1]
            qs, ss = _group_stride(q), _group_stride(scale)
            if q.dim() < 3 or qs is None or ss is None or q.stride(-1) != 1 or \
                    q.stride(-2) != dim or scale.stride(-2) != 1:
                q, scale = q.contiguous().view(1, -1, dim), scale.contiguous().view(1, -1, 1)
                qs = ss = 0
            groups, rows = q.numel() // (q.shape[-2] * dim), q.shape[-2]
            rc = _lib.lib().ojasx_dequantize_int8_device(
                _vp(q), _vp(scale), groups, rows, dim, qs, ss, _vp(out), _dtype_tag(dtype),
                _stream())
            _lib.check(rc, "ojasx_dequantize_int8_device")
        return out

    @staticmethod
    def _new_page(B, H, n, D, device):
        torch = _torch()
        qk = torch.empty(B, H, n, D, dtype=torch.int8, device=device)
        sk = torch.empty(B, H, n, 1, dtype=torch.float16, device=device)
        return qk, sk, torch.empty_like(qk), torch.empty_like(sk)

    def append(self, key, value) -> None:
        """Quantise and append a K/V chunk ``[B, H, S, D]`` into bounded pages
        (long_context.py:246-257)."""
        _require_gpu(key, "PagedCompressedKVCache.append")
        _require_gpu(value, "PagedCompressedKVCache.append")
        if key.dim() != 4 or key.shape != value.shape:
            raise ValueError("key and value must both be [B, H, S, D] of one shape")
        B, H, S, D = key.shape
        layout = (B, H, D, key.device)
        if self._layout is None:
            self._layout = layout
        elif layout != self._layout:
            raise ValueError(f"chunk layout {layout[:3]} differs from the cache's {self._layout[:3]}")
        self.total_tokens_seen += S
        self._version += 1
        key, value = key.contiguous(), value.contiguous()
        for start in range(0, S, self.page_size):
            n = min(start + self.page_size, S) - start
            if len(self._pages) == self.max_resident_pages:
                # Evicting before the append leaves the same pages as the
                # reference's append-then-pop(sink_pages); the popped page's
                # memory can then serve the new page when nobody holds it.
                self._pages.pop(self.sink_pages)
            qk, sk, qv, sv = self._new_page(B, H, n, D, key.device)
            _quantize_into(key[:, :, start:start + n], qk, sk)
            _quantize_into(value[:, :, start:start + n], qv, sv)
            self._pages.append((qk, sk, qv, sv))

    def iter_dequantized_pages(self, dtype=None) -> Iterator[Tuple]:
        """Lazily dequantise resident pages one by one (long_context.py:259-267)."""
        torch = _torch()
        dtype = torch.float32 if dtype is None else dtype
        for qk, sk, qv, sv in self._pages:
            yield (self._dequantize_int8(qk, sk, dtype), self._dequantize_int8(qv, sv, dtype))

    @property
    def resident_tokens(self) -> int:
        return sum(p[0].shape[2] for p in self._pages)

    @property
    def storage_bytes(self) -> int:
        total = 0
        for page in self._pages:
            for t in page:
                total += t.numel() * t.element_size()
        return total


@dataclass(frozen=True)
class BlockAttentionReport:
    """Telemetry of an online-softmax pass (long_context.py:36-44)."""

    query_tokens: int
    kv_tokens: int
    num_kv_blocks: int
    peak_tile_elements: int
    max_logsumexp: float


def _attn_tag(dtype):
    torch = _torch()
    return {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
            torch.float16: _lib.DTYPE_F16, torch.float64: _lib.DTYPE_F64}.get(dtype)


def _float_tile(k, v, keep):
    """AttnTile of float K/V blocks [B, H_kv, S, D] (k and v of one dtype,
    rows contiguous and aligned; otherwise contiguous copies, kept alive in
    ``keep`` until the update is enqueued)."""
    torch = _torch()
    if k.dtype != v.dtype or _attn_tag(k.dtype) is None:
        k, v = k.to(torch.float64), v.to(torch.float64)
    es = k.element_size()
    ak, av = min(16, 8 * es), min(16, 4 * es)

    def fits(t, a):
        return (t.stride(-1) == 1 and t.data_ptr() % a == 0 and
                all((st * es) % ak == 0 for st in t.stride()[:3]) and t.stride(2) >= t.shape[3])

    if not fits(k, ak) or not fits(v, av) or k.stride() != v.stride():
        k, v = k.contiguous(), v.contiguous()
    keep.extend((k, v))
    tile = _lib.AttnTile(k.data_ptr(), v.data_ptr(), None, None, k.shape[2],
                         k.stride(0), k.stride(1), k.stride(2), 0, 0, 0)
    return tile, _attn_tag(k.dtype)


class OnlineSoftmaxBlockAttention:
    """Exact attention of queries over streamed (K, V) tiles with fp64
    (m, l, acc) state (long_context.py:47-209): MHA, GQA and MQA, optional
    causal masking.  Constructor arguments, validation and the scale
    1/sqrt(head_dim) follow the reference; the arithmetic runs on the GPU
    (scores and state in fp64, tiles read in their own type)."""

    _STATE_BYTES = 256 << 20         # fp64 state of one pass of ``forward``

    def __init__(self, num_heads: int, num_kv_heads: Optional[int] = None, head_dim: int = 64,
                 *, q_block_size: int = 128, kv_block_size: int = 256,
                 causal: bool = True) -> None:
        if min(num_heads, head_dim, q_block_size, kv_block_size) <= 0:
            raise ValueError("Attention dimensions and block sizes must be positive")
        self.num_heads = int(num_heads)
        self.num_kv_heads = self.num_heads if num_kv_heads is None else int(num_kv_heads)
        if self.num_heads % self.num_kv_heads != 0:
            raise ValueError(f"num_heads ({self.num_heads}) must be divisible by num_kv_heads "
                             f"({self.num_kv_heads})")
        self.num_queries_per_kv = self.num_heads // self.num_kv_heads
        self.head_dim = int(head_dim)
        self.q_block_size = int(q_block_size)
        self.kv_block_size = int(kv_block_size)
        self.causal = bool(causal)
        self.scale = 1.0 / math.sqrt(self.head_dim)
        # the kernels take head dims in multiples of 8: others run zero-padded
        # to the next one (exact: the added products are fp64 zeros; the
        # scale stays 1/sqrt(head_dim)) and the output is cut back
        self._dpad = -(-self.head_dim // 8) * 8

    def _pad_d(self, t):
        extra = self._dpad - t.shape[-1]
        return t if extra == 0 else _torch().nn.functional.pad(t, (0, extra))

    def _expand_kv_heads(self, tensor):
        """[B, H_kv, S, D] -> [B, H_q, S, D], each kv head repeated for its
        query heads (a view)."""
        if self.num_queries_per_kv == 1:
            return tensor
        B, H_kv, S, D = tensor.shape
        return tensor.unsqueeze(2).expand(B, H_kv, self.num_queries_per_kv, S, D).reshape(
            B, self.num_heads, S, D)

    def _check_query(self, query):
        if query.dim() != 4:
            raise ValueError(f"Expected query [B, H, S_q, D], got {tuple(query.shape)}")
        B, H_q, S_q, D = query.shape
        if H_q != self.num_heads or D != self.head_dim:
            raise ValueError(f"Expected query heads={self.num_heads}, dim={self.head_dim}, "
                             f"got ({H_q}, {D})")
        _require_gpu(query, "OnlineSoftmaxBlockAttention")
        if _attn_tag(query.dtype) is None:
            raise TypeError(f"unsupported query dtype {query.dtype}: float32, bfloat16, "
                            "float16 or float64")

    def _init(self, query):
        torch = _torch()
        B, H_q, S_q, D = query.shape
        rows = B * H_q * S_q
        state = torch.empty(rows, 2 * D + 2, dtype=torch.float64, device=query.device)
        q = query.contiguous()
        rc = _lib.lib().ojasx_attention_stream_init_device(_vp(state), _vp(q), _attn_tag(q.dtype),
                                                          rows, D, _stream())
        _lib.check(rc, "ojasx_attention_stream_init_device")
        return state

    def _page_tiles(self, cache, query):
        """The cache's resident pages as int8 attention tiles, rebuilt only
        after an append: (tile array, resident tokens, longest page)."""
        if cache._tiles is not None and cache._tiles[0] == cache._version:
            return cache._tiles[1:]
        tiles = []
        for qk, sk, qv, sv in cache._pages:
            if qk.device != query.device:
                raise ValueError("the cache's pages live on another device than the query")
            self._check_block(qk, query.shape[0], "key")
            if qk.shape[2]:
                tiles.append(_lib.AttnTile(qk.data_ptr(), qv.data_ptr(), sk.data_ptr(),
                                           sv.data_ptr(), qk.shape[2], qk.stride(0), qk.stride(1),
                                           qk.stride(2), sk.stride(0), sk.stride(1), sk.stride(2)))
        arr = (_lib.AttnTile * len(tiles))(*tiles)
        cache._tiles = (cache._version, arr, sum(t.n_tokens for t in tiles),
                        max((t.n_tokens for t in tiles), default=0))
        return cache._tiles[1:]

    def _update(self, state, query, tiles, kv_tag, query_start_pos, kv_offset):
        B, H_q, S_q, D = query.shape
        arr = tiles if isinstance(tiles, ctypes.Array) else (_lib.AttnTile * len(tiles))(*tiles)
        rc = _lib.lib().ojasx_attention_stream_update_device(
            _vp(state), B, H_q, self.num_kv_heads, S_q, D, arr, len(tiles), kv_tag,
            int(self.causal), int(query_start_pos), int(kv_offset), float(self.scale), _stream())
        _lib.check(rc, "ojasx_attention_stream_update_device")

    def _finalize(self, state, query, lse=None):
        torch = _torch()
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        rc = _lib.lib().ojasx_attention_stream_finalize_device(
            _vp(state), state.shape[0], query.shape[3], _vp(out), _attn_tag(query.dtype),
            _vp(lse) if lse is not None else None, _stream())
        _lib.check(rc, "ojasx_attention_stream_finalize_device")
        return out

    def _check_block(self, t, B, name):
        if t.dim() != 4 or t.shape[0] != B or t.shape[1] != self.num_kv_heads or \
                t.shape[3] != self.head_dim:
            raise ValueError(f"Expected {name} block [B={B}, H_kv={self.num_kv_heads}, S, "
                             f"D={self.head_dim}], got {tuple(t.shape)}")

    def forward_stream(self, query, kv_stream, *, query_start_pos: int = 0):
        """Attention of ``query`` [B, H_q, S_q, D] over a stream of
        ``(K_block, V_block)`` tiles [B, H_kv, S_k, D] (long_context.py:92-176),
        or over every resident page of a ``PagedCompressedKVCache`` passed
        as the stream.  Returns ``(out, BlockAttentionReport)``; ``out`` has
        the query's dtype."""
        torch = _torch()
        self._check_query(query)
        B, H_q, S_q, D = query.shape
        qp = self._pad_d(query)
        state = self._init(qp)
        kv_offset = num_blocks = peak = 0
        if isinstance(kv_stream, PagedCompressedKVCache) and kv_stream._pages and \
                kv_stream._pages[0][0].shape[3] % 16 == 0:
            self._check_block(kv_stream._pages[0][0], B, "key")
            arr, kv_offset, max_n = self._page_tiles(kv_stream, query)
            num_blocks = len(arr)
            peak = B * H_q * S_q * max_n
            self._update(state, qp, arr, _lib.DTYPE_INT8, query_start_pos, 0)
        else:
            if isinstance(kv_stream, PagedCompressedKVCache):
                kv_stream = kv_stream.iter_dequantized_pages()   # head_dim not a multiple of 16

            for k_blk, v_blk in kv_stream:
                k_blk = k_blk.to(device=query.device)
                v_blk = v_blk.to(device=query.device)
                self._check_block(k_blk, B, "key")
                self._check_block(v_blk, B, "value")
                if k_blk.shape[2] != v_blk.shape[2]:
                    raise ValueError("key and value blocks differ in length")
                S_k = k_blk.shape[2]
                if S_k == 0:
                    continue
                keep = []
                tile, tag = _float_tile(self._pad_d(k_blk), self._pad_d(v_blk), keep)
                self._update(state, qp, [tile], tag, query_start_pos, kv_offset)
                num_blocks += 1
                peak = max(peak, B * H_q * S_q * S_k)
                kv_offset += S_k
        lse = torch.empty(state.shape[0], dtype=torch.float64, device=query.device)
        out = self._finalize(state, qp, lse)
        if qp is not query:
            out = out[..., :D].contiguous()
        # the rows' log-sum-exps copied out and reduced on the host: one
        # synchronising copy, no reduction kernel
        max_lse = float(lse.cpu().max()) if kv_offset > 0 else 0.0
        return out, BlockAttentionReport(query_tokens=S_q, kv_tokens=kv_offset,
                                         num_kv_blocks=num_blocks, peak_tile_elements=peak,
                                         max_logsumexp=max_lse)

    def forward(self, query, key, value, *, query_start_pos: int = 0):
        """Tiled exact attention of ``query`` over ``key`` / ``value``
        [B, H_kv, S_k, D] (long_context.py:178-209): query blocks of
        q_block_size over the kv blocks of kv_block_size their causal horizon
        reaches, many query blocks and all their kv blocks in one update."""
        torch = _torch()
        self._check_query(query)
        B, H_q, S_q, D = query.shape
        key = key.to(device=query.device)
        value = value.to(device=query.device)
        self._check_block(key, B, "key")
        self._check_block(value, B, "value")
        key, value, qp = self._pad_d(key), self._pad_d(value), self._pad_d(query)
        S_k = key.shape[2]
        # whole query blocks per pass: as many as keep the fp64 state (query,
        # sums, maximum and weight of every row) within _STATE_BYTES and the rows
        # of a kv head within what an update takes (65535 blocks of 8)
        per_query = 8 * B * H_q * (2 * self._dpad + 2)
        step = min(self._STATE_BYTES // per_query, 8 * 65535 // self.num_queries_per_kv)
        step = max(1, step // self.q_block_size) * self.q_block_size
        outs = []
        for q_start in range(0, S_q, step):
            q_stop = min(q_start + step, S_q)
            q_chunk = qp[:, :, q_start:q_stop, :]
            eff_k = min(S_k, query_start_pos + q_stop) if self.causal else S_k
            state = self._init(q_chunk)
            keep, tiles, tag = [], [], None
            for k_start in range(0, max(eff_k, 0), self.kv_block_size):
                k_stop = min(k_start + self.kv_block_size, eff_k)
                tile, tag = _float_tile(key[:, :, k_start:k_stop, :],
                                        value[:, :, k_start:k_stop, :], keep)
                tiles.append(tile)
            if tiles:
                self._update(state, q_chunk, tiles, tag, query_start_pos + q_start, 0)
            outs.append(self._finalize(state, q_chunk))
        out = outs[0] if len(outs) == 1 else torch.cat(outs, dim=2)
        return out if qp is query else out[..., :D].contiguous()

    __call__ = forward


def _group_stride(t):
    """Element stride between consecutive [rows, last] matrices of t when its
    leading dimensions collapse into one, else None."""
    if t.dim() < 3:
        return 0
    gs = t.stride(-3)
    expect = gs * t.shape[-3]
    for i in range(t.dim() - 4, -1, -1):
        if t.shape[i] > 1 and t.stride(i) != expect:
            return None
        expect *= t.shape[i]
    return gs


class PageTable:
    """Host bookkeeping of a token-filled paged cache with sink + sliding
    eviction: logical pages in order (``pages``, physical ids), tokens in the
    last page (``tail``) and the free physical pages.  ``plan(n)`` places n
    new tokens and returns each token's slot (page * page_size + offset), -1
    for a token whose page is evicted again within the same call."""

    def __init__(self, page_size: int, max_pages: int, sink_pages: int) -> None:
        if page_size <= 0 or max_pages <= sink_pages or sink_pages < 0:
            raise ValueError("Invalid page configuration for PagedCodeKVCache")
        self.page_size = page_size
        self.max_pages = max_pages
        self.sink_pages = sink_pages
        self.pages: List[int] = []
        self.opened = 0                  # pages opened so far: changes whenever ``pages`` does
        self.ids = np.zeros(max_pages, np.int32)   # ``pages`` as an array
        self._gen: List[int] = []
        self._next_gen = 0
        self.tail = 0
        self._free = list(range(max_pages - 1, -1, -1))

    @property
    def seq_len(self) -> int:
        return (len(self.pages) - 1) * self.page_size + self.tail if self.pages else 0

    def _open_page(self) -> None:
        if len(self.pages) == self.max_pages:
            self._free.append(self.pages.pop(self.sink_pages))
            self._gen.pop(self.sink_pages)
            self.ids[self.sink_pages:-1] = self.ids[self.sink_pages + 1:]
        self.pages.append(self._free.pop())
        self.ids[len(self.pages) - 1] = self.pages[-1]
        self.opened += 1
        self._gen.append(self._next_gen)
        self._next_gen += 1
        self.tail = 0

    def plan(self, n: int) -> np.ndarray:
        P = self.page_size
        if n == 1:                       # a decode step: no page evicted within the call
            if not self.pages or self.tail == P:
                self._open_page()
            self.tail += 1
            return np.array([self.pages[-1] * P + self.tail - 1], np.int32)
        slots = np.empty(n, np.int32)
        gens = np.empty(n, np.int64)
        t = 0
        while t < n:
            if not self.pages or self.tail == P:
                self._open_page()
            m = min(P - self.tail, n - t)
            slots[t:t + m] = self.pages[-1] * P + self.tail + np.arange(m, dtype=np.int32)
            gens[t:t + m] = self._gen[-1]
            self.tail += m
            t += m
        slots[~np.isin(gens, np.asarray(self._gen, np.int64))] = -1
        return slots


class PagedCodeKVCache:
    """Code-domain paged KV cache of one attention layer on the GPU.

    ``append(k, v)`` encodes ``[S, num_kv_heads, head_dim]`` fp32 tokens in one
    launch: per token and head the scale s = max(1e-8, max|k|)/127
    (ojasx_lut_kv_cache.cpp:29-34) and per group of ``block_dim`` coordinates
    the nearest of the 256 centroids of ``k_codebook``/``v_codebook``
    ([num_kv_heads, 256, block_dim] or one [256, block_dim] for all heads),
    or, with no codebooks, the reference's scalar quantiser.  ``decode(q)``
    runs the paged code-domain attention of ``[num_q_heads, head_dim]``
    queries over the resident tokens.
    """

    def __init__(self, num_kv_heads: int, head_dim: int = 128, block_dim: int = 16,
                 page_size: int = 16, max_resident_pages: int = 2048, sink_pages: int = 2,
                 k_codebook=None, v_codebook=None, device="cuda") -> None:
        torch = _torch()
        if head_dim <= 0 or block_dim <= 0 or head_dim % block_dim:
            raise ValueError("head_dim must be a positive multiple of block_dim")
        if head_dim // block_dim > 32 or block_dim > 32:
            raise ValueError("the decode kernels take head_dim / block_dim <= 32, block_dim <= 32")
        if (k_codebook is None) != (v_codebook is None):
            raise ValueError("give both codebooks or neither")
        self.table = PageTable(page_size, max_resident_pages, sink_pages)
        self.num_kv_heads, self.head_dim, self.block_dim = num_kv_heads, head_dim, block_dim
        self.page_size, self.max_resident_pages, self.sink_pages = (
            page_size, max_resident_pages, sink_pages)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedCodeKVCache runs on the GPU only")
        G = head_dim // block_dim
        self.total_tokens_seen = 0
        self.scalar_codes = k_codebook is None
        if self.scalar_codes:
            # The reference's implicit codebook C[c] = (c - 128) e_0.
            cb = torch.zeros(num_kv_heads, 256, block_dim, dtype=torch.float32)
            cb[:, :, 0] = torch.arange(256, dtype=torch.float32) - 128
            self.k_codebook = cb.to(self.device)
            self.v_codebook = self.k_codebook
        else:
            self.k_codebook = self._codebook(k_codebook)
            self.v_codebook = self._codebook(v_codebook)
        shape = (max_resident_pages, num_kv_heads, page_size)
        self.k_codes = torch.zeros(*shape, G, dtype=torch.uint8, device=self.device)
        self.v_codes = torch.zeros_like(self.k_codes)
        self.k_scales = torch.zeros(shape, dtype=torch.float32, device=self.device)
        self.v_scales = torch.zeros_like(self.k_scales)
        self._bt = torch.zeros(max_resident_pages, dtype=torch.int32, device=self.device)
        self._bt_opened = 0              # table.opened when _bt was written

    def _codebook(self, cb):
        torch = _torch()
        cb = torch.as_tensor(cb, dtype=torch.float32)
        if cb.dim() == 2:
            cb = cb.unsqueeze(0).expand(self.num_kv_heads, -1, -1)
        if tuple(cb.shape) != (self.num_kv_heads, 256, self.block_dim):
            raise ValueError(f"codebook must be [num_kv_heads, 256, {self.block_dim}] or "
                             f"[256, {self.block_dim}], got {tuple(cb.shape)}")
        return cb.to(self.device).contiguous()

    def append(self, k, v) -> None:
        """Encode the tokens of ``k`` and ``v`` [S, H_kv, D] (or [H_kv, D]) into the
        slots that the page table opens for them.  The slots are planned on the
        host, so a captured append would write the same ones on every replay:
        it raises, and the cache stays as it is."""
        torch = _torch()
        _require_gpu(k, "PagedCodeKVCache.append")
        _require_gpu(v, "PagedCodeKVCache.append")
        if k.dim() == 2:
            k, v = k.unsqueeze(0), v.unsqueeze(0)
        want = (self.num_kv_heads, self.head_dim)
        if k.dim() != 3 or tuple(k.shape[1:]) != want or k.shape != v.shape:
            raise ValueError(f"k and v must be [S, {want[0]}, {want[1]}] of one shape")
        n = k.shape[0]
        if n == 0:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedCodeKVCache.append plans its slots on the host and cannot be "
                               "captured: capture ojasx_kv_encode_append_device with a device slot "
                               "mapping")
        self.total_tokens_seen += n
        slots = self.table.plan(n)
        if n <= 64:                      # the slots travel with the launch
            name, at = "ojasx_kv_encode_append_host_slots", slots.ctypes.data
        else:
            slots = torch.from_numpy(slots).to(self.device)
            name, at = "ojasx_kv_encode_append_device", slots.data_ptr()
        k = k.to(torch.float32).contiguous()
        v = v.to(torch.float32).contiguous()
        cbk = None if self.scalar_codes else _vp(self.k_codebook)
        cbv = None if self.scalar_codes else _vp(self.v_codebook)
        rc = getattr(_lib.lib(), name)(
            _vp(k), _vp(v), n, self.num_kv_heads, self.head_dim, self.block_dim, cbk, cbv,
            at, self.page_size, self.max_resident_pages, _vp(self.k_codes),
            _vp(self.k_scales), _vp(self.v_codes), _vp(self.v_scales), _stream())
        _lib.check(rc, name)

    @property
    def seq_len(self) -> int:
        return self.table.seq_len

    resident_tokens = seq_len

    def block_table(self):
        """Device int32 block table of the resident pages, in logical order."""
        torch = _torch()
        table = self.table
        if self._bt_opened != table.opened:
            n = len(table.pages)
            self._bt[:n].copy_(torch.from_numpy(table.ids[:n]))
            self._bt_opened = table.opened
        return self._bt

    def decode(self, q, scale_factor: float = -1.0, out=None):
        """Attention of q [num_q_heads, head_dim] (fp32) over the resident
        tokens; q head j reads kv head j // (num_q_heads // num_kv_heads).
        ``scale_factor <= 0`` means 1/sqrt(head_dim).  An empty cache gives 0."""
        torch = _torch()
        _require_gpu(q, "PagedCodeKVCache.decode")
        q = q.to(torch.float32).contiguous()
        Hq = q.shape[0]
        if q.dim() != 2 or q.shape[1] != self.head_dim or Hq % self.num_kv_heads:
            raise ValueError("q must be [num_q_heads, head_dim], num_q_heads a multiple of "
                             "num_kv_heads")
        T = self.seq_len
        if out is None:                  # written whole unless the cache is empty
            new = torch.empty if T else torch.zeros
            out = new(Hq, self.head_dim, dtype=torch.float32, device=q.device)
        if T:
            rc = _lib.lib().ojasx_kv_decode_paged_device(
                _vp(q), _vp(self.k_codes), _vp(self.k_scales), _vp(self.v_codes),
                _vp(self.v_scales), _vp(self.k_codebook), _vp(self.v_codebook),
                _vp(self.block_table()), T, self.page_size, Hq, self.num_kv_heads,
                self.head_dim, self.block_dim, float(scale_factor), _vp(out), _stream())
            _lib.check(rc, "ojasx_kv_decode_paged_device")
        return out

    @property
    def storage_bytes(self) -> int:
        """Codes and scales of the resident tokens (K and V)."""
        G = self.head_dim // self.block_dim
        return 2 * self.seq_len * self.num_kv_heads * (G + 4)


# The calls below serve single tokens, where the host's time is the call's: their checks
# read each property once, and hold devices by index.
_MOST_INT = 0x7fffffff      # the entry points' counts are C ints: a larger one would lose its high bits
_INFERENCE_TAGS = {}        # dtype -> (C-ABI tag, torch's forward-mode module)


def _inference_tag(what, *tensors):
    """(C-ABI tag, device index) of tensors of one dtype on one GPU, without a gradient, reverse
    or forward."""
    dtype, index = tensors[0].dtype, tensors[0].get_device()
    for u in tensors:
        if u.dtype != dtype or u.get_device() != index or index < 0:
            _require_gpu(u, what)
            raise ValueError(f"{what}: tensors of {dtype} on {tensors[0].device} and of {u.dtype} on {u.device}")
        if u.requires_grad and _torch().is_grad_enabled():
            raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or with detached "
                               "tensors")
    known = _INFERENCE_TAGS.get(dtype)
    if known is None:
        tag = _attn_tag(dtype)
        if tag is None or tag == _lib.DTYPE_F64:
            raise TypeError(f"{what}: unsupported dtype {dtype}: float32, bfloat16 or float16")
        known = _INFERENCE_TAGS[dtype] = tag, _torch().autograd.forward_ad
    tag, forward_ad = known
    if forward_ad._current_level >= 0 and _torch()._C._is_fwd_grad_enabled() and \
            any(forward_ad.unpack_dual(u).tangent is not None for u in tensors):
        raise RuntimeError(f"{what} has no forward-mode gradient: call it with the primal tensors or under "
                           "torch.inference_mode()")
    return tag, index


def _new_like(t):
    """An uninitialised contiguous tensor of t's shape, dtype and device."""
    torch = _torch()
    if t.is_contiguous():
        return torch.empty_like(t)      # takes half the time of torch.empty with a device
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _aligned_rows(t, es):
    """(t [n, heads, D] itself where its rows are contiguous and 16-byte aligned, else a
    contiguous copy; its address, its token and its head stride).  es: bytes per element."""
    ts, hs, ds = t.stride()
    at = t.data_ptr()
    if ds != 1 or (at | ts * es | hs * es) & 15:
        n, heads, D = t.shape
        # torch calls a tensor contiguous whatever stride a dimension of one entry has: the
        # packed one there
        if n <= 1:
            ts = heads * D
        if heads <= 1:
            hs = D
        if ds != 1 or (at | ts * es | hs * es) & 15:
            t = t.clone(memory_format=_torch().contiguous_format)
            ts, hs, at = heads * D, D, t.data_ptr()
    return t, at, ts, hs


def _lengths_tensor(t, n, index, what):
    if t.dtype != _torch().int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or \
            t.get_device() != index:
        raise ValueError(f"{what} must be a contiguous int32 tensor of {n} entries on cuda:{index}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _launch(index, what, *args):
    """The entry point ``what`` on the device's current stream, the device made current
    where another is."""
    torch = _torch()
    call = getattr(_lib.lib(), what)
    if torch.cuda.current_device() == index:
        rc = call(*args, _lib.raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _lib.raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _rotation(head_dim, rotary_dim, rope_theta, inv_freq):
    """(rotary_dim, the frequencies in turns per position or None) of a cache's arguments."""
    torch = _torch()
    if inv_freq is None and rope_theta is None:
        if rotary_dim:
            raise ValueError("rotary_dim without rope_theta or inv_freq")
        rotary_dim = 0
    elif rotary_dim is None:
        rotary_dim = head_dim
    if rotary_dim < 0 or rotary_dim > head_dim or rotary_dim % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim, got {rotary_dim}")
    if not rotary_dim:
        return 0, None
    if inv_freq is None:
        if not 0.0 < float(rope_theta) < math.inf:
            raise ValueError(f"rope_theta must be positive and finite, got {rope_theta}")
        inv_freq = float(rope_theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64)
                                         / rotary_dim)
    inv_freq = torch.as_tensor(inv_freq).detach().to(device="cpu", dtype=torch.float64)
    if tuple(inv_freq.shape) != (rotary_dim // 2,) or not torch.isfinite(inv_freq).all():
        raise ValueError(f"inv_freq must hold {rotary_dim // 2} finite values, got "
                         f"{tuple(inv_freq.shape)}")
    return rotary_dim, inv_freq / (2.0 * math.pi)


class PagedInt4KVCache:
    """Paged KV cache of one attention layer for ``num_sequences`` sequences, in
    4 bits, on the GPU.

    Of a token's key or value row of one head, each group of ``group_size``
    dimensions is held as its smallest value lo and the step s = (largest - lo)
    / 15 in fp16 and 4-bit codes, for the values lo + s * code: 4 + 32 /
    group_size bits per value.  A group with an infinity or a NaN reads back as
    NaN.

    Tokens fill pages of ``page_size`` (a power of two from 16).  A sequence
    keeps at most ``max_resident_pages`` of them: opening one more evicts the
    oldest after the ``sink_pages`` first ones.  Its page j sits in entry e = j
    < sink_pages ? j : sink_pages + (j - sink_pages) % (max_resident_pages -
    sink_pages) of its row of ``block_table`` (int32 [num_sequences,
    max_resident_pages], physical pages): by default every sequence has pages
    of its own.  With ``num_pages`` given, the pool has that many pages and the
    table starts as -1, no page; the caller fills it in (sequences may share
    pages that none of them writes).

    Keys, and queries given to ``append``, are rotated by their positions:
    dimensions (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with ``interleaved``,
    by the angle position * inv_freq[i], inv_freq[i] = rope_theta ** (-2 i /
    rotary_dim) unless ``inv_freq`` (rotary_dim / 2 values) is given;
    ``rope_theta=None`` without ``inv_freq``: no rotation.  Angles are held in
    64 bits.

    The sequences' lengths are the caller's: int32 tensors on the cache's
    device, one for all layers, that a captured graph advances itself.  Calls
    on one cache write its pages: order them on one stream."""

    def __init__(self, num_kv_heads: int, head_dim: int = 128, *, num_sequences: int = 1,
                 page_size: int = 16, max_resident_pages: int = 2048, sink_pages: int = 2,
                 group_size: int = 32, rope_theta: Optional[float] = 1e6, inv_freq=None,
                 rotary_dim: Optional[int] = None, interleaved: bool = False,
                 num_pages: Optional[int] = None, device="cuda") -> None:
        torch = _torch()
        if head_dim not in (64, 128, 256) or group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError(f"head_dim must be 64, 128 or 256 and group_size 32, 64 or 128, at most "
                             f"head_dim: got {head_dim} and {group_size}")
        if not 16 <= page_size <= 32768 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 32768, got {page_size}")
        if num_kv_heads <= 0 or num_sequences <= 0 or sink_pages < 0 or \
                max_resident_pages <= sink_pages or (num_pages is not None and num_pages <= 0):
            raise ValueError("Invalid page configuration for PagedInt4KVCache")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedInt4KVCache runs on the GPU only")
        rotary_dim, turns = _rotation(head_dim, rotary_dim, rope_theta, inv_freq)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        dev = self.device
        self._index = dev.index
        if turns is not None:
            turns = turns.to(dev)
        self.num_kv_heads, self.head_dim, self.group_size = num_kv_heads, head_dim, group_size
        self.num_sequences, self.page_size = num_sequences, page_size
        self.max_resident_pages, self.sink_pages = max_resident_pages, sink_pages
        self.rotary_dim, self.interleaved = rotary_dim, bool(interleaved)
        self.num_pages = num_sequences * max_resident_pages if num_pages is None else num_pages
        rows = self.num_pages * num_kv_heads * page_size
        self._k_codes = torch.zeros(rows * head_dim // 2, dtype=torch.uint8, device=dev)
        self._v_codes = torch.zeros_like(self._k_codes)
        self._k_steps = torch.zeros(rows * head_dim // group_size * 2, dtype=torch.float16, device=dev)
        self._v_steps = torch.zeros_like(self._k_steps)
        if num_pages is None:
            table = torch.arange(self.num_pages, dtype=torch.int32, device=dev)
        else:
            table = torch.full((num_sequences * max_resident_pages,), -1, dtype=torch.int32, device=dev)
        self._block_table = table.view(num_sequences, max_resident_pages)
        self._turns = turns
        self._c = _lib.KV4Cache(_vp(self.k_codes), _vp(self.v_codes), _vp(self.k_steps),
                                _vp(self.v_steps), _vp(table),
                                _vp(turns) if turns is not None else None, num_sequences,
                                max_resident_pages, sink_pages, page_size, self.num_pages,
                                num_kv_heads, head_dim, group_size, rotary_dim, int(self.interleaved))
        self._ref = ctypes.addressof(self._c)
        self._workspace_bytes = {}       # (query heads, max_seen) -> bytes

    # The kernels hold these tensors by address: they are filled in, never replaced.
    k_codes = property(lambda self: self._k_codes, doc="Codes of the keys, as csrc/kv4.h lays them out.")
    v_codes = property(lambda self: self._v_codes, doc="Codes of the values.")
    k_steps = property(lambda self: self._k_steps, doc="Steps and smallest values of the keys' groups.")
    v_steps = property(lambda self: self._v_steps, doc="Steps and smallest values of the values' groups.")

    @property
    def block_table(self):
        """The table itself: the kernels read this tensor, so it is filled in, never replaced."""
        return self._block_table

    @property
    def capacity(self) -> int:
        """Tokens of one sequence that its pages hold at most."""
        return self.max_resident_pages * self.page_size

    @property
    def storage_bytes(self) -> int:
        """Bytes of the pool: codes, steps and block table."""
        return sum(t.numel() * t.element_size() for t in
                   (self.k_codes, self.v_codes, self.k_steps, self.v_steps, self.block_table))

    def _check_rows(self, t, n, heads, name):
        shape = t.shape
        if len(shape) != 3 or shape[0] != n or shape[2] != self.head_dim or \
                (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [{n}, {heads or 'heads'}, {self.head_dim}], got "
                             f"{tuple(shape)}")

    def _tag(self, what, *tensors):
        tag, index = _inference_tag(what, *tensors)
        if index != self._index:
            raise ValueError(f"{what}: tensors on {tensors[0].device}, the cache on {self.device}")
        return tag

    def _packed(self, n, start, cu_seqlens):
        B = self.num_sequences
        at = _lengths_tensor(start, B, self._index, "start")
        if cu_seqlens is None:
            if n != B:
                raise ValueError(f"{n} tokens: without cu_seqlens each of the {B} sequences gets one")
            return at, None
        return at, _lengths_tensor(cu_seqlens, B + 1, self._index, "cu_seqlens")

    def append(self, key, value, start, cu_seqlens=None, *, query=None, return_key: bool = False):
        """Rotate and append ``key`` and ``value`` [N, num_kv_heads, head_dim]
        (float32, bfloat16 or float16, any strides): rows cu_seqlens[b] ..
        cu_seqlens[b + 1] - 1 are sequence b's tokens at positions start[b],
        start[b] + 1, ...; without ``cu_seqlens`` row b is sequence b's one
        token.  ``start`` (int32 [num_sequences]) is read, not advanced.

        Returns (query rotated by the same positions or None, the rotated key
        before its encoding or None without ``return_key``), contiguous, in
        their dtype; rows that belong to no sequence are zeros there."""
        what = "PagedInt4KVCache.append"
        tag = self._tag(what, key, value) if query is None else self._tag(what, key, value, query)
        n = key.shape[0] if key.dim() else 0
        if n > _MOST_INT:
            raise ValueError(f"{what}: {n} tokens")
        self._check_rows(key, n, self.num_kv_heads, "key")
        self._check_rows(value, n, self.num_kv_heads, "value")
        at, cu = self._packed(n, start, cu_seqlens)
        es = 4 if tag == _lib.DTYPE_F32 else 2
        k, ka, kt, kh = _aligned_rows(key, es)
        v, va, vt, vh = _aligned_rows(value, es)
        qo = ko = qa = qp = kp = None
        heads = qt = qh = 0
        if query is not None:
            self._check_rows(query, n, None, "query")
            heads = query.shape[1]
            q, qa, qt, qh = _aligned_rows(query, es)
            qo = _new_like(q)
            qp = qo.data_ptr()
        if return_key:
            ko = _new_like(k)
            kp = ko.data_ptr()
        _launch(self._index, "ojasx_kv4_append_device", self._ref, qa, qt, qh, heads, qp, ka, kt, kh, kp, va,
                vt, vh, n, tag, at, cu)
        return qo, ko

    def read(self, start, cu_seqlens=None, num_tokens: Optional[int] = None, *, seen=None, dtype=None):
        """The held keys (rotated) and values of tokens addressed as in
        ``append``: (k, v), each [num_tokens, num_kv_heads, head_dim] in
        ``dtype`` (float32 unless given).  ``seen`` (int32 [num_sequences]): the
        tokens of each sequence so far, where that is more than the last one
        read; a token its sequence has evicted reads as 0 (as a key it would
        take weight: leave such rows out of an attention over them)."""
        torch = _torch()
        dtype = torch.float32 if dtype is None else dtype
        tag = _attn_tag(dtype)
        if tag is None or tag == _lib.DTYPE_F64:
            raise TypeError(f"unsupported dtype {dtype}: float32, bfloat16 or float16")
        if num_tokens is None:
            if cu_seqlens is not None:
                raise ValueError("give num_tokens with cu_seqlens: the rows of the result")
            num_tokens = self.num_sequences
        if num_tokens < 0:
            raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
        at, cu = self._packed(num_tokens, start, cu_seqlens)
        sp = None if seen is None else _lengths_tensor(seen, self.num_sequences, self._index, "seen")
        k = torch.empty(num_tokens, self.num_kv_heads, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _launch(self._index, "ojasx_kv4_read_device", self._ref, at, cu, sp, num_tokens, k.data_ptr(),
                v.data_ptr(), tag)
        return k, v

    def decode(self, query, seen, scale_factor: float = -1.0, *, max_seen: int = 0, out=None):
        """Attention of one query token per sequence, ``query``
        [num_sequences, num_q_heads, head_dim] (rotated; float32, bfloat16 or
        float16), over the resident ones of the ``seen[b]`` tokens (int32
        [num_sequences], the current one included) of each sequence; q head j
        reads kv head j // (num_q_heads // num_kv_heads).  ``scale_factor <= 0``
        means 1/sqrt(head_dim); a sequence without tokens gives 0, one whose
        tokens all score -inf NaN.  Scores and sums are float32; for bfloat16
        outputs a softmax weight is rounded to 11 bits in the product with the
        values.  ``out`` may be the query itself.
        ``max_seen``, a bound on ``seen`` where the caller knows one, keeps the
        launch of short sequences as small as they are."""
        torch = _torch()
        tag = self._tag("PagedInt4KVCache.decode", query)
        self._check_rows(query, self.num_sequences, None, "query")
        heads = query.shape[1]
        if heads == 0 or heads % self.num_kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {self.num_kv_heads} kv heads")
        if max_seen < 0:
            raise ValueError(f"max_seen must not be negative, got {max_seen}")
        sp = _lengths_tensor(seen, self.num_sequences, self._index, "seen")
        need = self._workspace_bytes.get((heads, max_seen))
        if need is None:
            need = _lib.lib().ojasx_kv4_decode_workspace(self._ref, heads, max_seen)
            if need < 0:
                _lib.check(need, "ojasx_kv4_decode_workspace")
            if len(self._workspace_bytes) > 64:
                self._workspace_bytes.clear()
            self._workspace_bytes[(heads, max_seen)] = need
        if out is None:
            out = _new_like(query)
        elif out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or \
                not out.is_contiguous():
            raise ValueError("out must be contiguous and of the query's shape, dtype and device")
        q = query if query.is_contiguous() else query.contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        _launch(self._index, "ojasx_kv4_decode_device", self._ref, q.data_ptr(), heads, tag, sp, max_seen,
                scale_factor, out.data_ptr(), ws.data_ptr(), need)
        return out


class PagedEvictingKVCache:
    """Paged KV cache of one attention layer for ``num_sequences`` sequences, on
    the GPU, that counts the attention its tokens get and can drop those that
    get least: long generations in bounded memory, with the tokens kept that
    the model looks at, where the other caches keep the first and newest pages.

    Token slot t of a sequence lies in slot t % page_size (a power of two from
    16) of page ``block_table[sequence, t // page_size]`` (int32 [num_sequences,
    max_pages]): by default every sequence has pages of its own.  With
    ``num_pages`` given, the pool has that many pages and the table starts as
    -1, no page; the caller fills it in.  ``keys`` and ``values`` [num_pages,
    num_kv_heads, page_size, head_dim] hold ``dtype`` (float32, bfloat16 or
    float16), ``weights`` (float32) and ``positions`` (int32) [num_pages,
    num_kv_heads, page_size] a token's attention so far and where it stands.
    The caller may fill these tensors in, too.

    Keys, and queries given to ``append``, are rotated by their positions as
    PagedInt4KVCache does it (rope_theta, inv_freq, rotary_dim, interleaved);
    ``rope_theta=None`` without ``inv_freq``: no rotation.

    The sequences' lengths are the caller's: int32 tensors on the cache's
    device, one for all layers, that a captured graph advances itself.  Calls on
    one cache write its pages: order them on one stream.  A page may stand in
    the table more than once only where nothing writes it: no append, no
    eviction, and decode with ``count=False``."""

    def __init__(self, num_kv_heads: int, head_dim: int = 128, *, num_sequences: int = 1,
                 page_size: int = 16, max_pages: int = 512, rope_theta: Optional[float] = 1e6,
                 inv_freq=None, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 num_pages: Optional[int] = None, dtype=None, device="cuda") -> None:
        torch = _torch()
        dtype = torch.bfloat16 if dtype is None else dtype
        tag = _attn_tag(dtype)
        if tag is None or tag == _lib.DTYPE_F64:
            raise TypeError(f"unsupported dtype {dtype}: float32, bfloat16 or float16")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if not 16 <= page_size <= 32768 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 32768, got {page_size}")
        if num_kv_heads <= 0 or num_sequences <= 0 or max_pages <= 0 or \
                (num_pages is not None and num_pages <= 0):
            raise ValueError("Invalid page configuration for PagedEvictingKVCache")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedEvictingKVCache runs on the GPU only")
        rotary_dim, turns = _rotation(head_dim, rotary_dim, rope_theta, inv_freq)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        dev = self.device
        self._index = dev.index
        if turns is not None:
            turns = turns.to(dev)
        self.num_kv_heads, self.head_dim, self.dtype = num_kv_heads, head_dim, dtype
        self.num_sequences, self.page_size, self.max_pages = num_sequences, page_size, max_pages
        self.rotary_dim, self.interleaved = rotary_dim, bool(interleaved)
        self.num_pages = num_sequences * max_pages if num_pages is None else num_pages
        slots = (self.num_pages, num_kv_heads, page_size)
        self._keys = torch.zeros(*slots, head_dim, dtype=dtype, device=dev)
        self._values = torch.zeros_like(self._keys)
        self._weights = torch.zeros(slots, dtype=torch.float32, device=dev)
        self._positions = torch.zeros(slots, dtype=torch.int32, device=dev)
        if num_pages is None:
            table = torch.arange(self.num_pages, dtype=torch.int32, device=dev)
        else:
            table = torch.full((num_sequences * max_pages,), -1, dtype=torch.int32, device=dev)
        self._block_table = table.view(num_sequences, max_pages)
        self._turns = turns
        self._c = _lib.KVECache(_vp(self._keys), _vp(self._values), _vp(self._weights),
                                _vp(self._positions), _vp(table),
                                _vp(turns) if turns is not None else None, num_sequences, max_pages,
                                page_size, self.num_pages, num_kv_heads, head_dim, tag, rotary_dim,
                                int(self.interleaved))
        self._ref = ctypes.addressof(self._c)
        self._workspace_bytes = {}       # arguments of a workspace's size -> bytes

    # The kernels hold these tensors by address: they are filled in, never replaced.
    keys = property(lambda self: self._keys, doc="Keys, rotated.")
    values = property(lambda self: self._values, doc="Values.")
    weights = property(lambda self: self._weights, doc="The softmax weights that each token got, summed.")
    positions = property(lambda self: self._positions, doc="The tokens' positions.")
    block_table = property(lambda self: self._block_table, doc="The pages of each sequence.")

    @property
    def capacity(self) -> int:
        """Tokens of one sequence that its pages hold at most."""
        return self.max_pages * self.page_size

    @property
    def storage_bytes(self) -> int:
        """Bytes of the pool: keys, values, weights, positions and block table."""
        return sum(t.numel() * t.element_size() for t in
                   (self._keys, self._values, self._weights, self._positions, self._block_table))

    def _check(self, what, *tensors):
        """The cache's dtype and device, and no gradient."""
        tag, index = _inference_tag(what, *tensors)
        if index != self._index or tag != self._c.dtype:
            raise ValueError(f"{what}: tensors of {tensors[0].dtype} on {tensors[0].device}, the cache of "
                             f"{self.dtype} on {self.device}")

    def _check_rows(self, t, n, heads, name):
        shape = t.shape
        if len(shape) != 3 or shape[0] != n or shape[2] != self.head_dim or \
                (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [{n}, {heads or 'heads'}, {self.head_dim}], got "
                             f"{tuple(shape)}")

    def _workspace(self, name, *args):
        """An uninitialised workspace of the size that the entry point ``name`` gives, and its bytes."""
        key = (name, *args)
        need = self._workspace_bytes.get(key)
        if need is None:
            need = getattr(_lib.lib(), name)(self._ref, *args)
            if need < 0:
                _lib.check(need, name)
            if len(self._workspace_bytes) > 64:
                self._workspace_bytes.clear()
            self._workspace_bytes[key] = need
        return _torch().empty(need, dtype=_torch().uint8, device=self.device), need

    def append(self, key, value, start, cu_seqlens=None, *, position=None, query=None, weight=None):
        """Rotate ``key`` and write it with ``value`` [N, num_kv_heads, head_dim]
        (the cache's dtype, any strides): rows cu_seqlens[b] .. cu_seqlens[b +
        1] - 1 go to sequence b's slots start[b], start[b] + 1, ...; without
        ``cu_seqlens`` row b is sequence b's one token.  They stand at positions
        position[b], position[b] + 1, ... (int32 [num_sequences]; ``start``
        unless given, right as long as nothing has been evicted).  ``start`` and
        ``position`` are read, not advanced.  ``weight`` (float32 [N,
        num_kv_heads]) is the attention that the tokens got already, 0 unless
        given.  Slots past the sequence's pages are not written.

        Returns the query [N, heads, head_dim] rotated by the same positions, in
        its dtype (zeros in rows that belong to no sequence), or None."""
        what = "PagedEvictingKVCache.append"
        if query is None:
            self._check(what, key, value)
        else:
            self._check(what, key, value, query)
        n, B = key.shape[0] if key.dim() else 0, self.num_sequences
        if n > _MOST_INT:
            raise ValueError(f"{what}: {n} tokens")
        self._check_rows(key, n, self.num_kv_heads, "key")
        self._check_rows(value, n, self.num_kv_heads, "value")
        at = _lengths_tensor(start, B, self._index, "start")
        pa = None if position is None else _lengths_tensor(position, B, self._index, "position")
        cu = None
        if cu_seqlens is not None:
            cu = _lengths_tensor(cu_seqlens, B + 1, self._index, "cu_seqlens")
        elif n != B:
            raise ValueError(f"{n} tokens: without cu_seqlens each of the {B} sequences gets one")
        wa = None
        if weight is not None:
            if weight.dtype != _torch().float32 or tuple(weight.shape) != (n, self.num_kv_heads) or \
                    weight.get_device() != self._index or not weight.is_contiguous():
                raise ValueError(f"weight must be contiguous float32 [{n}, {self.num_kv_heads}] on "
                                 f"{self.device}, got {weight.dtype} {tuple(weight.shape)} on {weight.device}")
            _inference_tag(what, weight)
            wa = weight.data_ptr()
        es = 4 if self._c.dtype == _lib.DTYPE_F32 else 2
        k, ka, kt, kh = _aligned_rows(key, es)
        v, va, vt, vh = _aligned_rows(value, es)
        qo = qa = qp = None
        heads = qt = qh = 0
        if query is not None:
            self._check_rows(query, n, None, "query")
            heads = query.shape[1]
            q, qa, qt, qh = _aligned_rows(query, es)
            qo = _new_like(q)
            qp = qo.data_ptr()
        _launch(self._index, "ojasx_kve_append_device", self._ref, qa, qt, qh, heads, qp, ka, kt, kh, va, vt,
                vh, wa, n, at, pa, cu)
        return qo

    def decode(self, query, held, scale_factor: float = -1.0, *, max_held: int = 0, count: bool = True,
               out=None):
        """Attention of one query token per sequence, ``query``
        [num_sequences, num_q_heads, head_dim] (rotated; the cache's dtype),
        over the first ``held[b]`` slots (int32 [num_sequences], the current
        token included) of each sequence; q head j reads kv head j //
        (num_q_heads // num_kv_heads), at most 128 of them one kv head.
        ``scale_factor <= 0`` means 1/sqrt(head_dim); a sequence without tokens
        gives 0, one whose tokens all score -inf NaN.  With ``count`` each
        token's softmax weights, summed over the query heads of its kv head, are
        added to its entry of ``weights``.  Scores, sums and counted weights are
        float32; for the product with bfloat16 and float16 values a softmax
        weight is the sum of two numbers of that type (to 2^-14 of it;
        float16: 2^-20 of it or 2^-40 of the largest).  ``out`` may be the query
        itself.  ``max_held``, a bound on ``held`` where the caller knows one,
        keeps launch and workspace as small as the sequences are; of a longer
        one the first ``max_held`` tokens are attended."""
        self._check("PagedEvictingKVCache.decode", query)
        self._check_rows(query, self.num_sequences, None, "query")
        heads = query.shape[1]
        if heads == 0 or heads % self.num_kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {self.num_kv_heads} kv heads")
        if not 0 <= max_held <= _MOST_INT:
            raise ValueError(f"max_held must not be negative, got {max_held}")
        hp = _lengths_tensor(held, self.num_sequences, self._index, "held")
        count = 1 if count else 0
        ws, need = self._workspace("ojasx_kve_decode_workspace", heads, max_held, count)
        if out is None:
            out = _new_like(query)
        elif out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or \
                not out.is_contiguous() or out.data_ptr() & 15:
            raise ValueError("out must be contiguous, 16-byte aligned and of the query's shape, dtype and "
                             "device")
        q = query if query.is_contiguous() else query.contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
        _launch(self._index, "ojasx_kve_decode_device", self._ref, q.data_ptr(), heads, hp, max_held,
                scale_factor, count, out.data_ptr(), ws.data_ptr(), need)
        return out

    def evict(self, held, budget: int, *, sink_tokens: int = 4, recent_tokens: int = 0,
              max_held: int = 0) -> None:
        """Of each sequence and kv head that holds more than ``budget`` tokens
        (``held``, int32 [num_sequences]), keep ``budget``: those at positions
        below ``sink_tokens``, those of the ``recent_tokens`` newest positions,
        and of the others the ones of largest weight, ties to the lowest slot
        (NaN last).  A kept token from behind the budget takes the place of a
        dropped one before it, the i-th of them the i-th place, with its weight
        and position; nothing else is written.  Slots of a page that is not there
        go first, but are places all the same: a token whose place lies in such
        a page is lost, so the pages of the first ``budget`` slots should be
        there.  The caller then holds min(held, budget) tokens; ``held`` is read,
        not changed, so that the layers of a model can share it.  ``max_held`` as
        in ``decode``."""
        budget, sink_tokens, recent_tokens = int(budget), int(sink_tokens), int(recent_tokens)
        if min(sink_tokens, recent_tokens, max_held) < 0 or max(budget, max_held) > _MOST_INT or \
                not 0 < budget >= sink_tokens + recent_tokens:
            raise ValueError(f"budget {budget} for {sink_tokens} sink and {recent_tokens} recent tokens, "
                             f"max_held {max_held}")
        hp = _lengths_tensor(held, self.num_sequences, self._index, "held")
        ws, need = self._workspace("ojasx_kve_evict_workspace", budget, max_held)
        _launch(self._index, "ojasx_kve_evict_device", self._ref, hp, budget, sink_tokens, recent_tokens,
                max_held, ws.data_ptr(), need)


class PackedPromptAttention:
    """Attention of packed prompts: the queries of every sequence over its own
    keys, in one launch.  float32, bfloat16 or float16; head_dim a multiple of
    8 up to 256; scores times ``scale`` (1/sqrt(head_dim) unless given).
    Scores, the softmax's maxima and sums and the outputs' sums are float32;
    the softmax's weights are rounded to bfloat16 or float16 inputs' type for
    the product with the values, as the output is once more.  Where
    OnlineSoftmaxBlockAttention is exact (fp64) over one sequence's tiles, this
    is the batch's prefill at the speed of the inputs' own type."""

    def __init__(self, num_heads: int, num_kv_heads: Optional[int] = None, head_dim: int = 128, *,
                 causal: bool = True, scale: Optional[float] = None) -> None:
        self.num_heads = int(num_heads)
        self.num_kv_heads = self.num_heads if num_kv_heads is None else int(num_kv_heads)
        self.head_dim = int(head_dim)
        if self.num_heads <= 0 or self.num_kv_heads <= 0 or self.num_heads % self.num_kv_heads:
            raise ValueError(f"num_heads ({self.num_heads}) must be divisible by num_kv_heads "
                             f"({self.num_kv_heads})")
        if self.head_dim <= 0 or self.head_dim > 256 or self.head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {self.head_dim}")
        self.causal = bool(causal)
        self.scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        if not 0.0 < self.scale < math.inf:
            raise ValueError(f"scale must be positive and finite, got {scale}")

    def _check(self, t, heads, name):
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [tokens, {heads}, {self.head_dim}], got {tuple(shape)}")
        return shape[0]

    def forward(self, query, key, value, cu_seqlens, cu_seqlens_kv=None, *, out=None,
                return_lse: bool = False):
        """``query`` [N, num_heads, head_dim] over ``key`` and ``value`` [M,
        num_kv_heads, head_dim] (any strides): rows cu_seqlens[b] ..
        cu_seqlens[b + 1] - 1 (int32 [B + 1] on the device) are sequence b's.
        With ``cu_seqlens_kv`` its keys are those rows instead, and query i of
        Lq sees keys j <= i + Lk - Lq: a prompt's last rows over keys that
        begin earlier.  A row that sees no key is 0; one whose keys all score
        -inf is NaN.  What a row does not see reaches it in no way; an infinity
        or NaN that it sees, or scores past 2^20, cost its call a second pass
        over the keys (about 2.3 times the time; 5 times where all values are
        infinite or NaN).

        Returns the output [N, num_heads, head_dim] in the query's dtype, or
        (output, lse float32 [N, num_heads]) with ``return_lse``.  Rows of no
        sequence are 0 (lse -inf); in a given ``out`` they stay as they are.
        ``out`` may be the query itself, and shares no memory with the keys and
        values."""
        tag, dev = _inference_tag("PackedPromptAttention", query, key, value)
        n = self._check(query, self.num_heads, "query")
        m = self._check(key, self.num_kv_heads, "key")
        if self._check(value, self.num_kv_heads, "value") != m:
            raise ValueError(f"{m} keys and {value.shape[0]} values")
        B = cu_seqlens.numel() - 1
        if B < 1:
            raise ValueError(f"cu_seqlens must hold the B + 1 bounds of B sequences, got "
                             f"{tuple(cu_seqlens.shape)}")
        if m > _MOST_INT or B > _MOST_INT:
            raise ValueError(f"{m} keys, {B} sequences")
        cq = ck = _lengths_tensor(cu_seqlens, B + 1, dev, "cu_seqlens")
        if cu_seqlens_kv is not None:
            ck = _lengths_tensor(cu_seqlens_kv, B + 1, dev, "cu_seqlens_kv")
        elif m != n:
            raise ValueError(f"{n} queries and {m} keys without cu_seqlens_kv")
        fresh = out is None
        if fresh:
            out = _new_like(query)
        elif out.shape != query.shape or out.dtype != query.dtype or out.get_device() != dev or \
                not out.is_contiguous() or out.data_ptr() & 15:
            raise ValueError("out must be contiguous, 16-byte aligned and of the query's shape, dtype and "
                             "device")
        es = 4 if tag == _lib.DTYPE_F32 else 2
        q, qa, qt, qh = _aligned_rows(query, es)
        k, ka, kt, kh = _aligned_rows(key, es)
        v, va, vt, vh = _aligned_rows(value, es)
        lse = la = None
        if return_lse:
            torch = _torch()
            lse = torch.empty(n, self.num_heads, dtype=torch.float32, device=query.device)
            la = lse.data_ptr()
            if not fresh:
                lse.fill_(-math.inf)
        _launch(dev, "ojasx_prompt_attention_device", qa, qt, qh, ka, kt, kh, va, vt, vh, tag, n, m,
                self.num_heads, self.num_kv_heads, self.head_dim, cq, ck, B, self.causal, self.scale, fresh,
                out.data_ptr(), la)
        return (out, lse) if return_lse else out

    __call__ = forward
