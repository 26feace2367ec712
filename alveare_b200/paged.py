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
and the work is ordered on that device's current stream.  Attention and page
bookkeeping use one work area per device (as the Q4 products do), so calls on
one device come from one thread at a time and must not overlap: before a call
on another stream, or beside a replayed graph that holds such calls, make the
stream wait (``wait_stream``, an event).  Lengths, page tables and counts are
read on the device when a kernel runs, never on the host, so a step can be
captured in a CUDA graph and replayed while they change; run it once before,
since a call that needs a larger work area than any before it allocates, which
a capture does not allow.  A bad page, length or slot found on the device is
skipped and reported by the next ``context(device).sync_status()``.
"""
from __future__ import annotations

import math
import struct

from ._lib import BF16, F32, context

try:
    import torch
except Exception:  # pragma: no cover
    torch = None

_INT_MAX = 2 ** 31 - 1

# The C structures, packed (a call costs a few microseconds of host time; the
# ctypes.Structure form alone would take as long again).
_PAGED = struct.Struct("@PPqqqiiiiPqPPiiii")             # alv_paged
_NORM_ROPE = struct.Struct("@PqPqqPPPiiiiif")            # alv_qk_norm_rope_args
_ATTENTION = struct.Struct("@PqqPqqiiiifi")              # alv_attention_args
_PAGES = struct.Struct("@PPqqqPPPqiiiiii")               # alv_pages
_SAMPLE = struct.Struct("@PqPPPPPPPiiiifffi")            # alv_sample_args


# ---------------------------------------------------------------------------
# checks
# ---------------------------------------------------------------------------
def _need(t, name: str, device: int, dtype, ndim: int) -> None:
    """A CUDA tensor of this type and rank on the call's device."""
    try:
        if t.get_device() == device and t.dtype is dtype and t.dim() == ndim and device >= 0:
            return
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if t.get_device() != device:
        raise ValueError(f"{name} is on cuda:{t.get_device()}, the call is on cuda:{device}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")


def _device(t, name: str) -> int:
    if torch is None or not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a torch CUDA tensor")
    return t.get_device()


def _rows(t, name: str, device: int, ndim: int) -> int:
    """A tensor of either activation type; the type's code."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    code = F32 if t.dtype is torch.float32 else BF16 if t.dtype is torch.bfloat16 else None
    if code is None:
        raise TypeError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    _need(t, name, device, t.dtype, ndim)
    return code


def _vector(t, name: str, device: int, dtype, n: int) -> int:
    """Pointer of a contiguous vector of n values."""
    _need(t, name, device, dtype, 1)
    if t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n}")
    return t.data_ptr()


def _step(stride: int, rows: int, width: int) -> int:
    """Elements between a matrix's rows: its own stride (0 where one row is
    broadcast); of a single row, whose stride may be anything, its width."""
    return stride if rows > 1 else width


def _apart(strides, tokens: int, heads: int, hd: int, name: str) -> None:
    """An output's tokens and heads do not share memory."""
    if (strides[0] < hd and tokens > 1) or (strides[1] < hd and heads > 1):
        raise ValueError(f"{name}'s tokens and heads must not share memory (it is written)")


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


if torch is not None and hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _stream = torch._C._cuda_getCurrentRawStream  # noqa: F811  (the same handle, without the Stream object)


def _paged(device: int, k_pages, v_pages, page_table, q_start, kv_lens, tokens: int):
    """alv_paged, the kv heads and the head size."""
    bf16, i32 = torch.bfloat16, torch.int32
    _need(k_pages, "k_pages", device, bf16, 4)
    _need(v_pages, "v_pages", device, bf16, 4)
    _need(page_table, "page_table", device, i32, 2)
    _need(q_start, "q_start", device, i32, 1)
    _need(kv_lens, "kv_lens", device, i32, 1)
    shape, strides = k_pages.shape, k_pages.stride()
    if v_pages.shape != shape or v_pages.stride() != strides:
        raise ValueError("k_pages and v_pages must have the same shape and strides")
    batch = kv_lens.shape[0]
    rows, width = page_table.shape
    if rows != batch or q_start.shape[0] != batch + 1:
        raise ValueError(f"page_table and q_start must have {batch} and {batch + 1} rows (kv_lens has {batch})")
    ts = page_table.stride()
    if strides[3] != 1 or ts[1] != 1 or not q_start.is_contiguous() or not kv_lens.is_contiguous():
        raise ValueError("pages and page_table must be contiguous in their last dimension, q_start and kv_lens whole")
    pages, heads, ps, hd = shape
    return _PAGED.pack(k_pages.data_ptr(), v_pages.data_ptr(), strides[0], strides[1], strides[2], pages, heads, ps, hd,
                       page_table.data_ptr(), _step(ts[0], rows, width), q_start.data_ptr(), kv_lens.data_ptr(), width, batch,
                       tokens, 0), heads, hd


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
    q_start           (batch + 1,) int32: first token of each sequence, then one past the
                      last (rows from there on are left alone)
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
    c, kv_heads, cache_hd = _paged(device, k_pages, v_pages, page_table, q_start, kv_lens, tokens)
    cols = (heads + 2 * kv_heads) * hd
    if cache_hd != hd or qkv.shape[0] != tokens or qkv.shape[1] != cols:
        raise ValueError(f"qkv must be ({tokens}, {(heads + 2 * kv_heads) * cache_hd}) for q_out "
                         f"{tuple(q_out.shape)} and {kv_heads} kv heads of {cache_hd}")
    max_pos, width = rope.shape
    if width % 2 or not rope.is_contiguous():
        raise ValueError("rope must be contiguous rows of cos | sin")
    xs, qs = qkv.stride(), q_out.stride()
    if xs[1] != 1 or qs[2] != 1:
        raise ValueError("qkv and q_out must be contiguous in their last dimension")
    _apart(qs, tokens, heads, hd, "q_out")
    qw = 0 if q_weight is None else _vector(q_weight, "q_weight", device, torch.float32, hd)
    kw = 0 if k_weight is None else _vector(k_weight, "k_weight", device, torch.float32, hd)
    a = _NORM_ROPE.pack(qkv.data_ptr(), _step(xs[0], tokens, cols), q_out.data_ptr(), qs[0], qs[1], rope.data_ptr(), qw, kw, qd,
                        rd, heads, width // 2, max_pos, eps)
    ctx = context(device)
    rc = ctx.lib.alv_qk_norm_rope(ctx.ptr, c, a, _stream(device))
    if rc:
        ctx.check(rc, "alv_qk_norm_rope")


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
    tokens, heads, hd = shape = q.shape
    c, _, cache_hd = _paged(device, k_pages, v_pages, page_table, q_start, kv_lens, tokens)
    if cache_hd != hd or out.shape != shape:
        raise ValueError(f"q and out must both be (tokens, heads, {cache_hd})")
    qs, os = q.stride(), out.stride()
    if qs[2] != 1 or os[2] != 1:
        raise ValueError("q and out must be contiguous in their last dimension")
    _apart(os, tokens, heads, hd, "out")
    if window < 0 or sinks < 0 or max_q_len < 0:
        raise ValueError("window, sinks and max_q_len must not be negative")
    a = _ATTENTION.pack(q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], heads, min(max_q_len, tokens),
                        min(window, _INT_MAX), min(sinks, _INT_MAX), hd ** -0.5 if scale is None else scale, 0)
    ctx = context(device)
    rc = ctx.lib.alv_paged_attention(ctx.ptr, c, a, _stream(device))
    if rc:
        ctx.check(rc, "alv_paged_attention")


# ---------------------------------------------------------------------------
# page bookkeeping
# ---------------------------------------------------------------------------
def _pool(device: int, k_pool, v_pool, page_table, lens, refs) -> bytes:
    _need(k_pool, "k_pool", device, torch.bfloat16, 5)
    _need(v_pool, "v_pool", device, torch.bfloat16, 5)
    _need(page_table, "page_table", device, torch.int32, 2)
    layers, pages, nkv, ps, hd = k_pool.shape
    st, ts = k_pool.stride(), page_table.stride()
    if v_pool.shape != k_pool.shape or v_pool.stride() != st:
        raise ValueError("k_pool and v_pool must have the same shape and strides")
    if st[2:] != (ps * hd, hd, 1) or ts[1] != 1:
        raise ValueError("a page must be contiguous, and page_table in its last dimension")
    slots, width = page_table.shape
    step = _step(ts[0], slots, width)
    if step < width:
        raise ValueError("page_table's rows must not overlap (it is written)")
    lp = 0 if lens is None else _vector(lens, "lens", device, torch.int32, slots)
    return _PAGES.pack(k_pool.data_ptr(), v_pool.data_ptr(), st[0] * 2, st[1] * 2, nkv * ps * hd * 2,
                       page_table.data_ptr(), lp, _vector(refs, "refs", device, torch.int32, pages), step,
                       layers, pages, ps, slots, width, 0)


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
    lens, refs      (slots,) positions held; (pages,) table entries naming the page.
                    lens may be lowered between calls (rejected tokens): the pages
                    past it are the slot's until it is dropped or forked onto, or an
                    extend reaches their entries and drops them for new ones
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
    rc = ctx.lib.alv_pages_update(ctx.ptr, p, fr, n_fr, fo, n_fo, ex, n_ex, ip, _stream(device))
    if rc:
        ctx.check(rc, "alv_pages_update")


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
    rc = ctx.lib.alv_pages_compact(ctx.ptr, p, table_out.data_ptr(), ro, ip, _stream(device))
    if rc:
        ctx.check(rc, "alv_pages_compact")


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def _param(v, name: str, device: int, dtype, rows: int, default):
    """(pointer of per-row values or 0, scalar)"""
    if isinstance(v, torch.Tensor):
        return _vector(v, name, device, dtype, rows), default
    return 0, v


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
    rows, vocab = logits.shape
    stride = logits.stride()
    if stride[1] != 1:
        raise ValueError("logits must be contiguous in their last dimension")
    up = _vector(u, "u", device, torch.float32, rows)
    tp = _vector(tokens, "tokens", device, torch.int32, rows)
    lp = 0 if logprobs is None else _vector(logprobs, "logprobs", device, torch.float32, rows)
    t_rows, t = _param(temperature, "temperature", device, torch.float32, rows, 1.0)
    k_rows, k = _param(top_k, "top_k", device, torch.int32, rows, 0)
    p_rows, p = _param(top_p, "top_p", device, torch.float32, rows, 1.0)
    m_rows, m = _param(min_p, "min_p", device, torch.float32, rows, 0.0)
    a = _SAMPLE.pack(logits.data_ptr(), _step(stride[0], rows, vocab), up, tp, lp, t_rows, p_rows, m_rows, k_rows, ld, rows,
                     vocab, max(0, min(k, vocab)), t, p, m, 0)
    ctx = context(device)
    rc = ctx.lib.alv_sample(ctx.ptr, a, _stream(device))
    if rc:
        ctx.check(rc, "alv_sample")


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

    def check_slots(self, slots) -> None:
        """ValueError unless all of these (host numbers) are slots of this pool."""
        n = self.lens.shape[0]
        if not all(0 <= s < n for s in slots):
            raise ValueError(f"slots must be in [0, {n})")

    def update(self, free=None, fork=None, extend=None) -> None:
        """:func:`update_pages` on this pool; lists of ids (or pairs) or int32 CUDA tensors."""
        update_pages(self.k, self.v, self.table, self.lens, self.refs, free=self._ids(free, False),
                     fork=self._ids(fork, True), extend=self._ids(extend, True), info=self.info)

    def check(self) -> dict:
        """What the last :meth:`update` reported (synchronises)."""
        keys = ("free_pages", "handed_out", "copied", "first_unmet")
        return dict(zip(keys, self.info.tolist()))

    def snapshot(self):
        """Copies of the tables, lengths and counts, for :meth:`restore`."""
        return self.table.clone(), self.lens.clone(), self.refs.clone()

    def restore(self, state) -> None:
        """Undo the updates since a :meth:`snapshot` (the pages themselves keep
        what was written; those in use then are untouched by updates)."""
        for t, old in zip((self.table, self.lens, self.refs), state):
            t.copy_(old)

    def compact(self) -> None:
        """:func:`compact_pages` on this pool, in place."""
        compact_pages(self.k, self.v, self.table, self.refs, self.table, self.refs)

    def batch(self, slots, q_lens) -> dict:
        """Tensors of a step in which ``slots[i]`` gets ``q_lens[i]`` new tokens
        (already reserved by :meth:`update`): page_table, q_start, kv_lens."""
        dev = torch.device("cuda", self.device)
        slots, q_lens = [int(s) for s in slots], [int(n) for n in q_lens]
        self.check_slots(slots)
        if len(slots) != len(q_lens) or min(q_lens, default=0) < 0:
            raise ValueError("batch: every slot needs a number of new tokens")
        idx = torch.tensor(slots, dtype=torch.int64).to(dev)
        start = [0]
        for n in q_lens:
            start.append(start[-1] + n)
        return dict(page_table=self.table[idx], q_start=torch.tensor(start, dtype=torch.int32).to(dev),
                    kv_lens=self.lens[idx])
