"""Serving many sequences from one paged cache.

* :func:`qk_norm_rope` -- per-head q/k norm, rotation and cache append of a
  ragged batch of new tokens, in one pass over ``[q | k | v]``
* :func:`paged_attention` -- attention of the new tokens over the cache, with a
  sliding window and first tokens that stay visible
* :func:`update_pages`, :func:`compact_pages` -- drop, fork, extend (copy on
  write) and compact the sequences' pages
* :func:`sample_tokens` -- temperature, top-k, top-p and min-p from given
  uniform numbers
* :class:`PagedKVCache` -- a pool with its page tables, for all of the above

The reference keeps one sequence in a contiguous cache and does this work on
the host: QK-norm, RoPE, KV write and (sliding) attention in
runtime/cpp/src/model.cpp:196-216, 315-370, sampling in
runtime/py/sampler.py:3-50.

All tensors are torch CUDA tensors on one device; outputs are written in place
and the work is stream-ordered on that device's current stream.  Lengths, page
tables and counts are read on the device when a kernel runs, never on the
host, so a step can be captured in a CUDA graph and replayed while they
change.  A bad page, length or slot found there is skipped and reported by the
next ``context(device).sync_status()``.
"""
from __future__ import annotations

import ctypes
import math

from ._lib import BF16, F32, context

try:
    import torch
except Exception:  # pragma: no cover
    torch = None

_i32, _i64, _f32, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


class _Paged(ctypes.Structure):
    """alv_paged"""
    _fields_ = [("k", _vp), ("v", _vp), ("page_stride", _i64), ("head_stride", _i64), ("row_stride", _i64),
                ("pages", _i32), ("kv_heads", _i32), ("page_size", _i32), ("head_dim", _i32), ("table", _vp),
                ("table_stride", _i64), ("q_start", _vp), ("kv_lens", _vp), ("table_width", _i32), ("batch", _i32),
                ("tokens", _i32), ("reserved", _i32)]


class _NormRope(ctypes.Structure):
    """alv_qk_norm_rope_args"""
    _fields_ = [("qkv", _vp), ("qkv_stride", _i64), ("q_out", _vp), ("q_token_stride", _i64), ("q_head_stride", _i64),
                ("rope", _vp), ("q_weight", _vp), ("k_weight", _vp), ("qkv_dtype", _i32), ("rope_dtype", _i32),
                ("heads", _i32), ("rot", _i32), ("max_pos", _i32), ("eps", _f32)]


class _Attention(ctypes.Structure):
    """alv_attention_args"""
    _fields_ = [("q", _vp), ("q_token_stride", _i64), ("q_head_stride", _i64), ("out", _vp),
                ("out_token_stride", _i64), ("out_head_stride", _i64), ("heads", _i32), ("max_q_len", _i32),
                ("window", _i32), ("sinks", _i32), ("scale", _f32), ("reserved", _i32)]


class _Pages(ctypes.Structure):
    """alv_pages"""
    _fields_ = [("k", _vp), ("v", _vp), ("layer_stride", _i64), ("page_stride", _i64), ("page_bytes", _i64),
                ("table", _vp), ("lens", _vp), ("refs", _vp), ("table_stride", _i64), ("layers", _i32),
                ("pages", _i32), ("page_size", _i32), ("slots", _i32), ("table_width", _i32), ("reserved", _i32)]


class _Sample(ctypes.Structure):
    """alv_sample_args"""
    _fields_ = [("logits", _vp), ("logits_stride", _i64), ("u", _vp), ("tokens", _vp), ("logprobs", _vp),
                ("temperature_rows", _vp), ("top_p_rows", _vp), ("min_p_rows", _vp), ("top_k_rows", _vp),
                ("logits_dtype", _i32), ("rows", _i32), ("vocab", _i32), ("top_k", _i32), ("temperature", _f32),
                ("top_p", _f32), ("min_p", _f32), ("reserved", _i32)]


# ---------------------------------------------------------------------------
# checks
# ---------------------------------------------------------------------------
def _need(t, name: str, device: int, dtype, ndim: int):
    """A CUDA tensor of this type and rank on the call's device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if t.device.index != device:
        raise ValueError(f"{name} is on cuda:{t.device.index}, the call is on cuda:{device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")


def _device(t, name: str) -> int:
    if torch is None or not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a torch CUDA tensor")
    return t.device.index


def _rows(t, name: str, device: int, ndim: int):
    """A tensor of any supported activation type; the type's code."""
    code = F32 if t.dtype == torch.float32 else BF16 if t.dtype == torch.bfloat16 else None
    if code is None:
        raise TypeError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    _need(t, name, device, t.dtype, ndim)
    return code


def _unit(t, name: str) -> None:
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def _vector(t, name: str, device: int, dtype, n: int) -> int:
    """Pointer of a contiguous vector of n values."""
    _need(t, name, device, dtype, 1)
    if t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n}")
    return t.data_ptr()


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _paged(device: int, k_pages, v_pages, page_table, q_start, kv_lens, tokens: int) -> _Paged:
    _need(k_pages, "k_pages", device, torch.bfloat16, 4)
    _need(v_pages, "v_pages", device, torch.bfloat16, 4)
    _need(page_table, "page_table", device, torch.int32, 2)
    _need(q_start, "q_start", device, torch.int32, 1)
    _need(kv_lens, "kv_lens", device, torch.int32, 1)
    shape, strides = k_pages.shape, k_pages.stride()
    if v_pages.shape != shape or v_pages.stride() != strides:
        raise ValueError("k_pages and v_pages must have the same shape and strides")
    batch = kv_lens.shape[0]
    if page_table.shape[0] != batch or q_start.shape[0] != batch + 1:
        raise ValueError(f"page_table and q_start must have {batch} and {batch + 1} rows (kv_lens has {batch})")
    if strides[3] != 1 or page_table.stride(1) != 1 or not q_start.is_contiguous() or not kv_lens.is_contiguous():
        raise ValueError("pages and page_table must be contiguous in their last dimension, q_start and kv_lens whole")
    width = page_table.shape[1]
    return _Paged(k_pages.data_ptr(), v_pages.data_ptr(), strides[0], strides[1], strides[2], shape[0], shape[1],
                  shape[2], shape[3], page_table.data_ptr(), max(page_table.stride(0), width), q_start.data_ptr(),
                  kv_lens.data_ptr(), width, batch, tokens, 0)


# ---------------------------------------------------------------------------
# q/k norm + rotation + append, attention
# ---------------------------------------------------------------------------
def qk_norm_rope(qkv, q_out, k_pages, v_pages, page_table, q_start, kv_lens, rope, *, q_weight=None, k_weight=None,
                 eps: float = 1e-6) -> None:
    """Rotate (and, with a weight, RMS-normalise first) every query and key head
    of the new tokens; q goes to ``q_out``, k and v to their cache slots.

    qkv      (tokens, (heads + 2 kv_heads) * head_dim) float32 or bfloat16: q | k | v
    q_out    (tokens, heads, head_dim) bfloat16
    k_pages, v_pages  (pages, kv_heads, page_size, head_dim) bfloat16, one layer
    page_table        (batch, width) int32: page of positions [i page_size, (i + 1) page_size)
    q_start           (batch + 1,) int32: first token of each sequence, then the token count
    kv_lens           (batch,) int32: positions in the cache, the new tokens' included
    rope     (max_pos, 2 rot) float32 or bfloat16: cos (rot) | sin (rot) of each
             position (:func:`alveare_b200.llama.rope_table`); pairs are (i, i + rot / 2)
    q_weight, k_weight  (head_dim,) float32 or None (no norm)
    """
    device = _device(qkv, "qkv")
    qd = _rows(qkv, "qkv", device, 2)
    _need(q_out, "q_out", device, torch.bfloat16, 3)
    rd = _rows(rope, "rope", device, 2)
    tokens, heads, hd = q_out.shape
    c = _paged(device, k_pages, v_pages, page_table, q_start, kv_lens, tokens)
    if c.head_dim != hd or qkv.shape != (tokens, (heads + 2 * c.kv_heads) * hd):
        raise ValueError(f"qkv must be ({tokens}, {(heads + 2 * c.kv_heads) * c.head_dim}) for q_out "
                         f"{tuple(q_out.shape)} and {c.kv_heads} kv heads of {c.head_dim}")
    if rope.shape[1] % 2 or not rope.is_contiguous():
        raise ValueError("rope must be contiguous rows of cos | sin")
    _unit(qkv, "qkv")
    _unit(q_out, "q_out")
    qw = None if q_weight is None else _vector(q_weight, "q_weight", device, torch.float32, hd)
    kw = None if k_weight is None else _vector(k_weight, "k_weight", device, torch.float32, hd)
    a = _NormRope(qkv.data_ptr(), max(qkv.stride(0), qkv.shape[1]), q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
                  rope.data_ptr(), qw, kw, qd, rd, heads, rope.shape[1] // 2, rope.shape[0], eps)
    ctx = context(device)
    ctx.check(ctx.lib.alv_qk_norm_rope(ctx.ptr, ctypes.byref(c), ctypes.byref(a), _stream(device)), "alv_qk_norm_rope")


def paged_attention(q, out, k_pages, v_pages, page_table, q_start, kv_lens, *, max_q_len: int,
                    scale: float | None = None, window: int = 0, sinks: int = 0) -> None:
    """out = softmax(scale q k^T) v of the new tokens over the paged cache.

    The token at position p sees the positions j <= p, with ``window`` > 0 only
    those with j > p - window or j < sinks.  Consecutive query heads share a kv
    head.  A token that sees nothing gives zeros.

    q, out   (tokens, heads, head_dim) bfloat16; the cache as in
             :func:`qk_norm_rope` (head_dim 64, 128 or 256)
    max_q_len  no sequence has more new tokens than this (a host number: it
             chooses the kernel and its grid)
    scale    1 / sqrt(head_dim) by default
    """
    device = _device(q, "q")
    _need(q, "q", device, torch.bfloat16, 3)
    _need(out, "out", device, torch.bfloat16, 3)
    tokens, heads, hd = q.shape
    c = _paged(device, k_pages, v_pages, page_table, q_start, kv_lens, tokens)
    if c.head_dim != hd or out.shape != q.shape:
        raise ValueError(f"q and out must both be (tokens, heads, {c.head_dim})")
    _unit(q, "q")
    _unit(out, "out")
    if window < 0 or sinks < 0 or max_q_len < 0:
        raise ValueError("window, sinks and max_q_len must not be negative")
    a = _Attention(q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), heads,
                   min(max_q_len, tokens), window, sinks, 1.0 / math.sqrt(hd) if scale is None else scale, 0)
    ctx = context(device)
    ctx.check(ctx.lib.alv_paged_attention(ctx.ptr, ctypes.byref(c), ctypes.byref(a), _stream(device)),
              "alv_paged_attention")


# ---------------------------------------------------------------------------
# page bookkeeping
# ---------------------------------------------------------------------------
def _pool(device: int, k_pool, v_pool, page_table, lens, refs) -> _Pages:
    _need(k_pool, "k_pool", device, torch.bfloat16, 5)
    _need(v_pool, "v_pool", device, torch.bfloat16, 5)
    _need(page_table, "page_table", device, torch.int32, 2)
    layers, pages, nkv, ps, hd = k_pool.shape
    st = k_pool.stride()
    if v_pool.shape != k_pool.shape or v_pool.stride() != st:
        raise ValueError("k_pool and v_pool must have the same shape and strides")
    if st[2:] != (ps * hd, hd, 1) or page_table.stride(1) != 1:
        raise ValueError("a page must be contiguous, and page_table in its last dimension")
    slots, width = page_table.shape
    lp = None if lens is None else _vector(lens, "lens", device, torch.int32, slots)
    return _Pages(k_pool.data_ptr(), v_pool.data_ptr(), st[0] * 2, st[1] * 2, nkv * ps * hd * 2, page_table.data_ptr(),
                  lp, _vector(refs, "refs", device, torch.int32, pages), max(page_table.stride(0), width), layers,
                  pages, ps, slots, width, 0)


def _list(t, name: str, device: int, pairs: bool):
    if t is None:
        return None, 0
    _need(t, name, device, torch.int32, 2 if pairs else 1)
    if not t.is_contiguous() or (pairs and t.shape[1] != 2):
        raise ValueError(f"{name} must be a contiguous " + ("(n, 2) list of pairs" if pairs else "list"))
    return (t.data_ptr() or None) if t.shape[0] else None, t.shape[0]


def update_pages(k_pool, v_pool, page_table, lens, refs, *, free=None, fork=None, extend=None, info=None) -> None:
    """One scheduler turn on a pool's page tables, in this order:

    free    (n,) int32 slots to drop
    fork    (n, 2) int32 (parent, child): the child becomes a copy that shares
            the parent's pages (what it held is dropped)
    extend  (n, 2) int32 (slot, positions): room for that many more positions;
            a partly filled last page that others share is first copied, in
            every layer, to a page of the slot's own

    New pages are the free ones of lowest id, in list order; the first extend
    that does not fit, and all after it, change nothing.

    k_pool, v_pool  (layers, pages, kv_heads, page_size, head_dim) bfloat16
    page_table      (slots, width) int32, -1 where a slot has no page
    lens, refs      (slots,) positions held; (pages,) table entries naming the page
    info            (4,) int32 or None: receives free pages left, pages handed
                    out, pages copied, index of the first extend that did not
                    fit (-1: all did)
    """
    device = _device(k_pool, "k_pool")
    if lens is None:
        raise TypeError("lens must be a torch CUDA tensor")
    p = _pool(device, k_pool, v_pool, page_table, lens, refs)
    fr, n_fr = _list(free, "free", device, False)
    fo, n_fo = _list(fork, "fork", device, True)
    ex, n_ex = _list(extend, "extend", device, True)
    ip = None if info is None else _vector(info, "info", device, torch.int32, 4)
    ctx = context(device)
    ctx.check(ctx.lib.alv_pages_update(ctx.ptr, ctypes.byref(p), fr, n_fr, fo, n_fo, ex, n_ex, ip, _stream(device)),
              "alv_pages_update")


def compact_pages(k_pool, v_pool, page_table, refs, table_out, refs_out, *, info=None) -> None:
    """Move the n pages in use to ids 0 .. n - 1 (the i-th one past them to the
    i-th free id below n), in every layer.  The renumbered table and counts go
    to ``table_out`` and ``refs_out``, which may be ``page_table`` and ``refs``
    themselves.  info: (2,) int32 or None, receives pages in use and moved."""
    device = _device(k_pool, "k_pool")
    p = _pool(device, k_pool, v_pool, page_table, None, refs)
    _need(table_out, "table_out", device, torch.int32, 2)
    if table_out.shape != page_table.shape or not table_out.is_contiguous():
        raise ValueError("table_out must be contiguous and shaped as page_table")
    ro = _vector(refs_out, "refs_out", device, torch.int32, refs.shape[0])
    ip = None if info is None else _vector(info, "info", device, torch.int32, 2)
    ctx = context(device)
    ctx.check(ctx.lib.alv_pages_compact(ctx.ptr, ctypes.byref(p), table_out.data_ptr(), ro, ip, _stream(device)),
              "alv_pages_compact")


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def _param(v, name: str, device: int, dtype, rows: int, default):
    """(pointer of per-row values or None, scalar)"""
    if isinstance(v, torch.Tensor):
        return _vector(v, name, device, dtype, rows), default
    return None, v


def sample_tokens(logits, u, tokens, logprobs=None, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> None:
    """One token per row of ``logits`` from the given uniform numbers.

    The weights exp((l - max) / temperature) are cut to the ``top_k`` largest
    (ties: lowest index first; 0: all), these to the shortest prefix that holds
    ``top_p`` of their mass, these to weights of at least ``min_p`` of the
    largest; the token is the first, in index order, whose running mass passes
    u * total.  temperature 0 takes the largest logit.  A row with nothing above
    -inf gives -1.  The same inputs give the same tokens on every run.

    logits    (rows, vocab) float32 or bfloat16
    u         (rows,) float32 in [0, 1)
    tokens    (rows,) int32; logprobs (rows,) float32 or None: log of the
              token's share of the kept mass
    temperature, top_k, top_p, min_p   numbers, or one per row: (rows,) float32
              (top_k: int32) CUDA tensors
    """
    device = _device(logits, "logits")
    ld = _rows(logits, "logits", device, 2)
    _unit(logits, "logits")
    rows, vocab = logits.shape
    up = _vector(u, "u", device, torch.float32, rows)
    tp = _vector(tokens, "tokens", device, torch.int32, rows)
    lp = None if logprobs is None else _vector(logprobs, "logprobs", device, torch.float32, rows)
    t_rows, t = _param(temperature, "temperature", device, torch.float32, rows, 1.0)
    k_rows, k = _param(top_k, "top_k", device, torch.int32, rows, 0)
    p_rows, p = _param(top_p, "top_p", device, torch.float32, rows, 1.0)
    m_rows, m = _param(min_p, "min_p", device, torch.float32, rows, 0.0)
    a = _Sample(logits.data_ptr(), max(logits.stride(0), vocab), up, tp, lp, t_rows, p_rows, m_rows, k_rows, ld, rows,
                vocab, max(0, min(k, vocab)), t, p, m, 0)
    ctx = context(device)
    ctx.check(ctx.lib.alv_sample(ctx.ptr, ctypes.byref(a), _stream(device)), "alv_sample")


# ---------------------------------------------------------------------------
# a pool with its tables
# ---------------------------------------------------------------------------
class PagedKVCache:
    """A pool of cache pages for every layer of a model, with the page tables,
    lengths and reference counts of ``slots`` sequences (all on the GPU).

    :meth:`update` reserves room for a step's new tokens (and drops or forks
    sequences); :meth:`batch` then gives the tensors that
    :func:`qk_norm_rope` and :func:`paged_attention` take for those slots."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, *, page_size: int = 16, slots: int = 64,
                 max_len: int = 4096, device: int = 0):
        dev = torch.device("cuda", device)
        self.device, self.page_size = device, page_size
        self.k = torch.zeros(layers, pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device=dev)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((slots, -(-max_len // page_size)), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.info = torch.zeros(4, dtype=torch.int32, device=dev)

    def _ids(self, v, pairs: bool):
        if v is None or isinstance(v, torch.Tensor):
            return v
        t = torch.tensor(v, dtype=torch.int32).to(torch.device("cuda", self.device))
        return t.reshape(-1, 2) if pairs else t

    def update(self, free=None, fork=None, extend=None) -> None:
        """:func:`update_pages` on this pool; lists of ids (or pairs) or int32 CUDA tensors."""
        update_pages(self.k, self.v, self.table, self.lens, self.refs, free=self._ids(free, False),
                     fork=self._ids(fork, True), extend=self._ids(extend, True), info=self.info)

    def check(self) -> dict:
        """What the last :meth:`update` reported (synchronises)."""
        keys = ("free_pages", "handed_out", "copied", "first_unmet")
        return dict(zip(keys, self.info.tolist()))

    def compact(self) -> None:
        compact_pages(self.k, self.v, self.table, self.refs, self.table, self.refs)

    def batch(self, slots, q_lens) -> dict:
        """Tensors of a step in which ``slots[i]`` gets ``q_lens[i]`` new tokens
        (already reserved by :meth:`update`): page_table, q_start, kv_lens."""
        dev = torch.device("cuda", self.device)
        idx = torch.tensor(list(slots), dtype=torch.int64).to(dev)
        start = [0]
        for n in q_lens:
            start.append(start[-1] + int(n))
        return dict(page_table=self.table[idx], q_start=torch.tensor(start, dtype=torch.int32).to(dev),
                    kv_lens=self.lens[idx])
