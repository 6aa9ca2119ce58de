"""Serving over a paged cache on MI355X (gfx950 HIP kernels via the C ABI).

The whole-sequence operators (``flash_hca_forward`` and its parts, ``flash_sparse/hca.py:54-95``) serve prefill and
training.  A serving step has a ragged batch of new tokens instead, one for each request in a decode step or a chunk of a
prompt, and the earlier ones in a cache:

* :func:`paged_plan` — block tables and cache slots from the requests' lengths, on the GPU;
* :func:`paged_write` — the new tokens' rows into their slots;
* :func:`paged_compress` — the compressed entries that the new tokens complete (``flash_sparse/reference.py:176-272``);
* :func:`paged_attn_fwd` — attention of the new tokens over the cache.

:func:`streamindex_amd.hca.flash_hca_paged_forward` runs them for an HCA layer.  The reference has no counterpart.

A cache is ``[pages, page_size, width]``; a page holds consecutive entries of one request, ``block_table[r, i]`` is the
page of request r's entries ``i * page_size`` and on (negative where there is none), and ``slot = page * page_size +
offset`` names a row of the cache.  Lengths, tables and plans are read on the GPU alone, so a step can be captured into a
graph and replayed with other lengths.  Lengths stay below 2^31.  None of these has a gradient.
"""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .quant import _dtype_code
from .sparse_attn import SUPPORTED_D, _aligned, _check_device

__all__ = ["PagedPlan", "paged_plan", "paged_write", "paged_compress", "paged_attn_fwd"]


class PagedPlan(NamedTuple):
    """The rows of a step (new tokens, or new compressed entries) of R requests."""

    cu: torch.Tensor  # [R + 1] int32: request r has rows cu[r] .. cu[r + 1] - 1
    seq_lens: torch.Tensor  # [R] int32: entries of each request after the step
    slots: torch.Tensor  # [num_rows] int64: cache slot of each row, -1 where it has none
    request: torch.Tensor  # [num_rows] int32: request of each row, -1 behind the last
    positions: torch.Tensor  # [num_rows] int32: position of each row in its request, -1 behind the last
    free_next: torch.Tensor  # [1] int32: position in the free list after this step


def _int32(t: torch.Tensor, name: str, n: int) -> torch.Tensor:
    assert t.dim() == 1 and t.shape[0] == n, f"{name} must be [{n}], got {list(t.shape)}"
    if t.dtype is not torch.int32:
        if t.dtype is not torch.int64:
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _table_stride(table: torch.Tensor, name: str, R: int) -> int:
    """Stride of the rows of a ``[R, P]`` block table."""
    if table.dtype is not torch.int32:
        raise ValueError(f"{name} must be int32, got {table.dtype}")
    assert table.dim() == 2 and table.shape[0] == R, f"{name} must be [{R}, P], got {list(table.shape)}"
    s, one = table.stride()
    if one != 1 and table.shape[1] > 1:
        raise ValueError(f"{name} needs contiguous rows")
    return s if R > 1 else table.shape[1]


def _check_slots(slots: torch.Tensor, n: int) -> torch.Tensor:
    if slots.dtype is not torch.int64:
        raise ValueError(f"slots must be int64, got {slots.dtype}")
    assert slots.dim() == 1 and slots.shape[0] == n, f"slots must be [{n}], got {list(slots.shape)}"
    return slots if slots.is_contiguous() else slots.contiguous()


def _cache_strides(cache: torch.Tensor, name: str):
    """Page, row and element stride, with those that a size of one leaves free as for packed rows."""
    assert cache.dim() == 3, f"{name} must be [pages, page_size, width]"
    n, p, w = cache.shape
    if p < 1:
        raise ValueError(f"{name} needs a page size of at least 1")
    s = cache.stride()
    if n > 1 and p > 1 and w > 1:
        return s
    sw = s[2] if w > 1 else 1
    sp = s[1] if p > 1 else w
    return (s[0] if n > 1 else sp * p, sp, sw)


def _check_apart(strides, pages: int, page_size: int, width: int) -> None:
    """A cache that is written: no two rows share memory."""
    sp, sr, se = strides
    if se != 1 or sr < width or (pages > 1 and sp < sr * (page_size - 1) + width):
        raise ValueError("the cache's rows must be contiguous and apart")


def paged_plan(ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               page_size: int, num_rows: int, *, ratio: int = 1,
               free_start: Optional[torch.Tensor] = None) -> PagedPlan:
    """Rows, cache slots and new pages of a step that adds ``new_lens[r]`` tokens to request r's ``ctx_lens[r]``.

    Args:
      ctx_lens, new_lens: ``[R]`` int32 / int64 (negative counts as 0).
      block_table: ``[R, P]`` int32, updated in place: a request whose entries reach new pages takes them from
        ``free_pages`` in request order; other entries stay as they are.
      free_pages: ``[F]`` int32 list of unused pages; ``free_start``: optional ``[1]`` int32 position of the first one to
        take (default 0).  ``free_next`` of the result is the position after the last: past ``F``, the list was too
        short, and the pages it lacked are -1 in ``block_table`` and their rows' slots.
      page_size: entries of a page.
      num_rows: length of the row lists, at least the sum of the new rows in use; rows past it are cut, last requests
        first, and ``cu`` and ``seq_lens`` say so.
      ratio: plan the compressed entries, one for ``ratio`` tokens: entry i is new if this step completes it.
        ``num_rows = N // ratio + R`` holds the entries of N new tokens.
    A position past the table's width has slot -1.
    """
    assert ctx_lens.is_cuda
    dev = ctx_lens.device
    at = dev.index
    if not (new_lens.get_device() == block_table.get_device() == free_pages.get_device() == at
            and (free_start is None or free_start.get_device() == at)):
        _check_device(dev, new_lens=new_lens, block_table=block_table, free_pages=free_pages, free_start=free_start)
    assert ctx_lens.dim() == 1 and free_pages.dim() == 1
    R, F = ctx_lens.shape[0], free_pages.shape[0]
    ctx, new = _int32(ctx_lens, "ctx_lens", R), _int32(new_lens, "new_lens", R)
    stride, P = _table_stride(block_table, "block_table", R), block_table.shape[1]
    free_pages = _int32(free_pages, "free_pages", F)
    if free_start is not None:
        free_start = _int32(free_start, "free_start", 1)
    if page_size < 1 or ratio < 1 or num_rows < 0:
        raise ValueError(f"page_size and ratio must be positive and num_rows not negative, got {page_size}, {ratio}, {num_rows}")
    L = _lib.load()
    with _lib.on_device(dev):
        # (one allocation for the five int32 lists: each is 2 us)
        lists = torch.empty(2 * (R + 1 + num_rows), dtype=torch.int32, device=dev)
        cu, seq, nxt, req, pos = torch.unsafe_split_with_sizes(lists, [R + 1, R, 1, num_rows, num_rows])
        slots = torch.empty(num_rows, dtype=torch.int64, device=dev)
        rc = L.si_paged_plan(ctx.data_ptr(), new.data_ptr(), R, ratio, block_table.data_ptr(), stride, P,
                             free_pages.data_ptr(), F, None if free_start is None else free_start.data_ptr(), page_size,
                             num_rows, cu.data_ptr(), seq.data_ptr(), slots.data_ptr(), req.data_ptr(), pos.data_ptr(),
                             nxt.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc)
    return PagedPlan(cu, seq, slots, req, pos, nxt)


def paged_write(rows: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """``cache[slots[t] // page_size, slots[t] % page_size] = rows[t]``; returns ``cache``, written in place.

    ``rows [N, width]`` of the cache's type and not part of it, ``slots [N]`` int64; a slot outside the cache (-1) writes
    nothing.  Slots are distinct, as a plan's are: of a slot given twice each 16-byte piece is one of the two rows'.
    """
    assert rows.is_cuda
    dev = rows.device
    if not cache.get_device() == slots.get_device() == dev.index:
        _check_device(dev, cache=cache, slots=slots)
    st = _cache_strides(cache, "cache")
    pages, ps, width = cache.shape
    assert rows.dim() == 2 and rows.shape[1] == width, "rows must be [N, width of the cache]"
    if rows.dtype is not cache.dtype:
        raise ValueError(f"rows and cache must share one type, got {rows.dtype} and {cache.dtype}")
    N = rows.shape[0]
    slots = _check_slots(slots, N)
    _check_apart(st, pages, ps, width)
    rs, one = rows.stride()
    if (one != 1 and width > 1) or rs < 0:
        rows = rows.contiguous()
        rs = width
    size = cache.element_size()
    L = _lib.load()
    with _lib.on_device(dev):
        rc = L.si_paged_write(rows.data_ptr(), rs * size, slots.data_ptr(), N, width * size, cache.data_ptr(), st[0] * size,
                              st[1] * size, pages, ps, _lib.stream_ptr(dev))
    _lib.check(rc)
    return cache


def paged_compress(c_a: torch.Tensor, z_a: torch.Tensor, b_a: torch.Tensor, block_table: torch.Tensor,
                   request: torch.Tensor, positions: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, *,
                   c_b: Optional[torch.Tensor] = None, z_b: Optional[torch.Tensor] = None,
                   b_b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Compressed entries of paged streams: :func:`streamindex_amd.compressor.token_compressor` entry by entry.

    Entry ``positions[e]`` of request ``request[e]`` pools the request's tokens ``m * positions[e]`` and on, ``m`` of
    them, and goes to ``slots[e]`` of ``cache``, which is returned, written in place.

    Args:
      c_a, z_a: ``[pages, page_size, C]`` content and gate streams (views of wider rows are fine); ``b_a [m, C]``.
      block_table: ``[R, P]`` int32 pages of the streams.  Tokens without a page count as absent; an entry without any
        token is zero.
      request, positions: ``[E]`` int32, slots: ``[E]`` int64, as a plan with ``ratio=m`` gives them; an entry without
        request or slot is left out.
      cache: ``[entry_pages, entry_page_size, C]`` of the streams' type (fp32, bf16 or fp16).
      c_b, z_b, b_b: the second streams of overlapping entries, whose entry i also pools block i - 1 of these.
    Sums in fp32, one rounding at the end.
    """
    assert c_a.is_cuda
    dev = c_a.device
    if not (z_a.get_device() == b_a.get_device() == block_table.get_device() == request.get_device()
            == positions.get_device() == cache.get_device() == slots.get_device() == dev.index):
        _check_device(dev, z_a=z_a, b_a=b_a, block_table=block_table, request=request, positions=positions, cache=cache,
                      slots=slots)
    dtype = c_a.dtype
    dt = _dtype_code(c_a)
    overlap = c_b is not None
    if overlap != (z_b is not None) or overlap != (b_b is not None):
        raise ValueError("overlapping entries need c_b, z_b and b_b")
    if overlap:
        _check_device(dev, c_b=c_b, z_b=z_b, b_b=b_b)
    st = [_cache_strides(c_a, "c_a")]
    pages, ps, C = c_a.shape
    for n, t in (("z_a", z_a), ("c_b", c_b), ("z_b", z_b)):
        if t is not None:
            if t.shape != c_a.shape or t.dtype is not dtype:
                raise ValueError(f"{n} must match c_a")
            st.append(_cache_strides(t, n))
    st.append(_cache_strides(cache, "cache"))
    epages, eps, width = cache.shape
    if cache.dtype is not dtype or width != C:
        raise ValueError("cache must have the streams' type and width")
    if any(s[2] != 1 for s in st):
        raise ValueError("the streams and the cache need a contiguous last dimension")
    _check_apart(st[-1], epages, eps, C)
    m = b_a.shape[0]
    if b_a.dim() != 2 or b_a.shape[1] != C or m < 1 or (overlap and b_b.shape != b_a.shape):
        raise ValueError(f"biases must be [m, {C}]")
    E, R = request.shape[0], block_table.shape[0]
    request, positions = _int32(request, "request", E), _int32(positions, "positions", E)
    slots = _check_slots(slots, E)
    stride = _table_stride(block_table, "block_table", R)
    ba = b_a if b_a.dtype is torch.float32 else b_a.float()
    ba = ba if ba.is_contiguous() else ba.contiguous()
    bb = b_b.float().contiguous() if overlap else None
    st = [_lib.stride_array(s) for s in st]
    L = _lib.load()
    with _lib.on_device(dev):
        rc = L.si_paged_compress(
            c_a.data_ptr(), st[0], z_a.data_ptr(), st[1], ba.data_ptr(), c_b.data_ptr() if overlap else None,
            st[2] if overlap else None, z_b.data_ptr() if overlap else None, st[3] if overlap else None,
            bb.data_ptr() if overlap else None, dt, pages, ps, C, m, block_table.data_ptr(), stride, R,
            block_table.shape[1], request.data_ptr(), positions.data_ptr(), slots.data_ptr(), E, cache.data_ptr(), st[-1],
            epages, eps, _lib.stream_ptr(dev))
    _lib.check(rc)
    return cache


def paged_attn_fwd(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor,
                   seq_lens: torch.Tensor, attn_sink: torch.Tensor, softmax_scale: Optional[float] = None, *,
                   window: Optional[int] = None, kv2_cache: Optional[torch.Tensor] = None,
                   block_table2: Optional[torch.Tensor] = None, ratio: Optional[int] = None
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """MQA attention with sink of new tokens over their requests' paged caches (forward only).

    The tokens of request r are rows ``cu_q[r] .. cu_q[r + 1] - 1`` of ``q``, at its last positions: the last one is at
    position ``seq_lens[r] - 1``.  A token at position p attends to entries k of the first cache with
    ``p - window < k <= p`` and, with a second cache, to its entries i with ``ratio * (i + 1) - 1 <= p``, in one softmax.

    Args:
      q: ``[N, H, D]`` bf16 or fp16.  kv_cache: ``[pages, page_size, D]`` of q's type (the new tokens' rows included), one
        row for key and value, shared by the heads; rows 16-byte aligned, within 64 GiB of the first.
      block_table: ``[R, P]`` int32.  Keys whose page is negative, past the cache or past the table are masked: pages
        that the window has left may be given back.
      cu_q: ``[R + 1]`` int32, ascending (if it descends anywhere, no request has rows); seq_lens: ``[R]`` int32;
        attn_sink: ``[H]`` fp32.
      softmax_scale: defaults to ``D ** -0.5``.
      window: earlier tokens seen, the token itself included (None: all).
      kv2_cache, block_table2, ratio: the compressed entries, one for ``ratio`` tokens.
    Returns:
      ``(o [N, H, D] in q's type, lse [N, H] fp32)``.  A row without a key, those of no request among them, gets
      ``o = 0`` and ``lse = sink`` (or ``-1e30`` if the sink is ``-inf``).  A value that is not finite reaches the rows that
      see its key and no others.  Scores are fp32: one below its range weighs nothing, one above it makes its row NaN.
    """
    assert q.is_cuda
    dev = q.device
    if not (kv_cache.get_device() == block_table.get_device() == cu_q.get_device() == seq_lens.get_device()
            == attn_sink.get_device() == dev.index):
        _check_device(dev, kv_cache=kv_cache, block_table=block_table, cu_q=cu_q, seq_lens=seq_lens, attn_sink=attn_sink)
    assert q.dim() == 3, "q must be [N, H, D]"
    N, H, D = q.shape
    dtype = q.dtype
    assert dtype is torch.bfloat16 or dtype is torch.float16, f"q must be bf16 or fp16, got {dtype}"
    assert attn_sink.dtype is torch.float32 and attn_sink.dim() == 1 and attn_sink.shape[0] == H, "attn_sink must be [H] fp32"
    if D not in SUPPORTED_D:
        raise ValueError(f"D ({D}) must be one of {SUPPORTED_D}")
    if window is not None and window < 1:
        raise ValueError(f"window must be positive, got {window}")
    two = kv2_cache is not None
    if two != (block_table2 is not None) or two != (ratio is not None):
        raise ValueError("a second cache needs kv2_cache, block_table2 and ratio")
    if two and not kv2_cache.get_device() == block_table2.get_device() == dev.index:
        _check_device(dev, kv2_cache=kv2_cache, block_table2=block_table2)
    if two and ratio < 1:
        raise ValueError(f"ratio must be positive, got {ratio}")
    R = block_table.shape[0]

    def cache_args(cache, table, name):
        assert cache.dtype is dtype and cache.shape[-1] == D, f"{name}_cache must have q's type and width"
        s = _cache_strides(cache, f"{name}_cache")
        p = cache.data_ptr()
        if s[2] != 1 or (s[0] | s[1]) % 8 or p % 16:
            raise ValueError(f"{name}_cache needs a contiguous last dimension and rows that start at multiples of 16 bytes")
        pages, ps, _ = cache.shape
        return (p, _lib.stride_array(s), pages, ps, table.data_ptr(), _table_stride(table, f"{name}'s block table", R),
                table.shape[1])

    c1 = cache_args(kv_cache, block_table, "kv")
    c2 = cache_args(kv2_cache, block_table2, "kv2") if two else (None, None, 0, 1, None, 0, 0)
    cu, lens = _int32(cu_q, "cu_q", R + 1), _int32(seq_lens, "seq_lens", R)
    q = q if _aligned(q) else _lib.packed(q)
    attn_sink = attn_sink if attn_sink.is_contiguous() else attn_sink.contiguous()
    window, ratio = window or 0, ratio or 0
    L = _lib.load()
    with _lib.on_device(dev):
        o = torch.empty((N, H, D), dtype=dtype, device=dev)
        lse = torch.empty((N, H), dtype=torch.float32, device=dev)
        scratch, nscratch = _lib.scratch(_attn_scratch(N, H, D, R, window, c1[3] * c1[6], c2[3] * c2[6]), dev)
        rc = L.si_paged_attn_fwd(q.data_ptr(), _lib.strides(q), *c1, *c2, window, ratio, cu.data_ptr(), lens.data_ptr(),
                                 attn_sink.data_ptr(), N, H, D, R, D ** -0.5 if softmax_scale is None else float(softmax_scale),
                                 _lib.qkv_dtype(q), o.data_ptr(), lse.data_ptr(),
                                 None if scratch is None else scratch.data_ptr(), nscratch, _lib.stream_ptr(dev))
    _lib.check(rc)
    return o, lse


@functools.lru_cache(maxsize=1024)
def _attn_scratch(*sizes) -> int:
    return _lib.load().si_paged_attn_fwd_scratch_bytes(*sizes)
