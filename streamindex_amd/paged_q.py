"""Serving over a paged cache held in 8 bits on MI355X (gfx950 HIP kernels via the C ABI).

A cache in 8 bits is ``[pages, page_size, width]`` e4m3 codes (``torch.float8_e4m3fn``) and ``[pages, blocks]`` fp32 scales; a
scale is shared by ``page_size // blocks`` consecutive tokens of a page, one by default of a server that can spare 4 bytes a
token, a page of them at most.  An entry is its code times its scale.  Tables, plans and lengths are those of
:mod:`streamindex_amd.paged`:

* :func:`paged_write_q` — the new tokens' rows into their slots;
* :func:`paged_attn_q_fwd` — attention of the new tokens over such caches.

The reference has no counterpart.  None of these has a gradient.
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from . import _lib
from .paged import _cache_strides, _check_apart, _check_slots, _int32, _table_stride
from .quant import _dtype_code
from .sparse_attn import SUPPORTED_D, _aligned, _check_device

__all__ = ["paged_write_q", "paged_attn_q_fwd"]

F8 = torch.float8_e4m3fn


def _check_scales(cache: torch.Tensor, scales: torch.Tensor, name: str) -> Tuple[int, int]:
    """Tokens of a block, and the stride of the pages' scales."""
    if cache.dtype is not F8 or scales.dtype is not torch.float32:
        raise ValueError(f"{name} must be float8_e4m3fn with fp32 scales, got {cache.dtype} and {scales.dtype}")
    assert cache.dim() == 3 and scales.dim() == 2, f"{name} must be [pages, page_size, width] and its scales [pages, blocks]"
    pages, ps, _ = cache.shape
    n, blocks = scales.shape
    if n != pages or blocks < 1 or ps % blocks:
        raise ValueError(f"the scales of {name} must be [{pages}, a divisor of {ps}], got {list(scales.shape)}")
    s, one = scales.stride()
    if one != 1 and blocks > 1:
        raise ValueError(f"the scales of {name} need contiguous rows")
    return ps // blocks, s if n > 1 else blocks


def paged_write_q(rows: torch.Tensor, cache: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Quantises ``rows[t]`` into slot ``slots[t]`` of a cache in 8 bits; returns ``(cache, scales)``, written in place.

    Args:
      rows: ``[N, width]`` fp32, bf16 or fp16.  cache: ``[pages, page_size, width]`` float8_e4m3fn, rows contiguous and apart.
      scales: ``[pages, blocks]`` fp32, ``blocks`` a divisor of the page size: one scale for ``page_size // blocks`` tokens.
      slots: ``[N]`` int64; one outside the cache (-1) writes nothing.  Slots are distinct and the rows of one block follow each
        other in rising order, as a plan's do, with fewer than 64 rows without a slot between two of them; otherwise what that
        block holds is undefined.
    A block's scale becomes the smallest power of two (at least 2^-64) that holds its new rows within e4m3's 448, unless that of its
    earlier tokens, those before the first new one, is larger and stays, a power of two or not.  A block written from its first token on
    starts anew, and an earlier scale that is not positive and finite counts as none (the codes stay).
    Where the scale grows, the earlier codes are rounded to it.  New codes are the nearest (ties to even) to ``x / scale``.
    Infinities and NaN become NaN and do not count for the scale.  Tokens of the block behind its first new row that are not written
    again lose their meaning: their codes stay and their scale is the new one.
    """
    assert rows.is_cuda
    dev = rows.device
    if not cache.get_device() == scales.get_device() == slots.get_device() == dev.index:
        _check_device(dev, cache=cache, scales=scales, slots=slots)
    block, sstride = _check_scales(cache, scales, "cache")
    st = _cache_strides(cache, "cache")
    pages, ps, width = cache.shape
    assert rows.dim() == 2 and rows.shape[1] == width, "rows must be [N, width of the cache]"
    dt = _dtype_code(rows)
    N = rows.shape[0]
    slots = _check_slots(slots, N)
    _check_apart(st, pages, ps, width)
    rs, one = rows.stride()
    if (one != 1 and width > 1) or rs < 0:
        rows = rows.contiguous()
        rs = width
    if width == 0:
        return cache, scales
    L = _lib.load()
    with _lib.on_device(dev):
        rc = L.si_paged_write_q(rows.data_ptr(), rs, dt, slots.data_ptr(), N, width, cache.data_ptr(), st[0], st[1],
                                scales.data_ptr(), sstride, pages, ps, block, _lib.stream_ptr(dev))
    _lib.check(rc)
    return cache, scales


def paged_attn_q_fwd(q: torch.Tensor, kv_cache: torch.Tensor, kv_scales: torch.Tensor, block_table: torch.Tensor,
                     cu_q: torch.Tensor, seq_lens: torch.Tensor, attn_sink: torch.Tensor,
                     softmax_scale: Optional[float] = None, *, window: Optional[int] = None,
                     kv2_cache: Optional[torch.Tensor] = None, kv2_scales: Optional[torch.Tensor] = None,
                     block_table2: Optional[torch.Tensor] = None, ratio: Optional[int] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`streamindex_amd.paged.paged_attn_fwd` over caches in 8 bits: an entry is its code times its block's scale.

    Args:
      q: ``[N, H, D]`` bf16 or fp16.
      kv_cache, kv2_cache: ``[pages, page_size, D]`` float8_e4m3fn, rows 16-byte aligned, within 64 GiB of the first.
      kv_scales, kv2_scales: ``[pages, blocks]`` fp32, ``blocks`` a divisor of the page size; of either sign, zero or from 2^-64 (the
        least that :func:`paged_write_q` sets) to 2^100.
      The others: as there.
    Returns:
      ``(o [N, H, D] in q's type, lse [N, H] fp32)``.  Weights times scales are rounded to q's type: in fp16 those below 2^-25 of a
      row's largest lose bits, and below 2^-36 they are lost; in bf16 those of scales outside the range above leave fp32's.
      A row without a key gets ``o = 0`` and ``lse = sink`` (or ``-1e30`` if the sink is ``-inf``).  A code of NaN reaches the
      rows that see its key and no others; so does a scale that is not finite.  Scores are fp32, as are q's products with the codes
      before their scale: one below its range weighs nothing, one above it makes its row NaN.
    """
    assert q.is_cuda
    dev = q.device
    if not (kv_cache.get_device() == kv_scales.get_device() == block_table.get_device() == cu_q.get_device()
            == seq_lens.get_device() == attn_sink.get_device() == dev.index):
        _check_device(dev, kv_cache=kv_cache, kv_scales=kv_scales, block_table=block_table, cu_q=cu_q, seq_lens=seq_lens,
                      attn_sink=attn_sink)
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
    if two != (block_table2 is not None) or two != (ratio is not None) or two != (kv2_scales is not None):
        raise ValueError("a second cache needs kv2_cache, kv2_scales, block_table2 and ratio")
    if two and not kv2_cache.get_device() == kv2_scales.get_device() == block_table2.get_device() == dev.index:
        _check_device(dev, kv2_cache=kv2_cache, kv2_scales=kv2_scales, block_table2=block_table2)
    if two and ratio < 1:
        raise ValueError(f"ratio must be positive, got {ratio}")
    R = block_table.shape[0]

    def cache_args(cache, scales, table, name):
        block, sstride = _check_scales(cache, scales, f"{name}_cache")
        assert cache.shape[-1] == D, f"{name}_cache must have q's width"
        s = _cache_strides(cache, f"{name}_cache")
        p = cache.data_ptr()
        if s[2] != 1 or (s[0] | s[1] | p) % 16:
            raise ValueError(f"{name}_cache needs a contiguous last dimension and rows that start at multiples of 16 bytes")
        pages, ps, _ = cache.shape
        return (p, _lib.stride_array(s), scales.data_ptr(), sstride, block, pages, ps, table.data_ptr(),
                _table_stride(table, f"{name}'s block table", R), table.shape[1])

    c1 = cache_args(kv_cache, kv_scales, block_table, "kv")
    c2 = cache_args(kv2_cache, kv2_scales, block_table2, "kv2") if two else (None, None, None, 0, 1, 0, 1, None, 0, 0)
    cu, lens = _int32(cu_q, "cu_q", R + 1), _int32(seq_lens, "seq_lens", R)
    q = q if _aligned(q) else _lib.packed(q)
    attn_sink = attn_sink if attn_sink.is_contiguous() else attn_sink.contiguous()
    window, ratio, dt = window or 0, ratio or 0, _lib.qkv_dtype(q)
    L = _lib.load()
    with _lib.on_device(dev):
        o = torch.empty((N, H, D), dtype=dtype, device=dev)
        lse = torch.empty((N, H), dtype=torch.float32, device=dev)
        scratch, nscratch = _lib.scratch(_attn_scratch(N, H, D, R, window, c1[6] * c1[9], c2[6] * c2[9]), dev)
        rc = L.si_paged_attn_q_fwd(q.data_ptr(), _lib.strides(q), *c1, *c2, window, ratio, cu.data_ptr(), lens.data_ptr(),
                                   attn_sink.data_ptr(), N, H, D, R, D ** -0.5 if softmax_scale is None else float(softmax_scale),
                                   dt, o.data_ptr(), lse.data_ptr(), None if scratch is None else scratch.data_ptr(), nscratch,
                                   _lib.stream_ptr(dev))
    _lib.check(rc)
    return o, lse


@functools.lru_cache(maxsize=1024)
def _attn_scratch(*sizes) -> int:
    return _lib.load().si_paged_attn_q_fwd_scratch_bytes(*sizes)
