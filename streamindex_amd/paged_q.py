"""Serving over a paged cache held in 8 bits on MI355X (gfx950 HIP kernels via the C ABI).

A cache in 8 bits is ``[pages, page_size, width]`` e4m3 codes (``torch.float8_e4m3fn``) and ``[pages, blocks]`` fp32 scales; a
scale is shared by ``page_size // blocks`` consecutive tokens of a page, one by default of a server that can spare 4 bytes a
token, a page of them at most.  An entry is its code times its scale.  Tables, plans and lengths are those of
:mod:`streamindex_amd.paged`:

* :func:`paged_write_q` — the new tokens' rows into their slots.

The reference has no counterpart.  None of these has a gradient.
"""

from __future__ import annotations

from typing import Tuple

import torch

from . import _lib
from .paged import _cache_strides, _check_apart, _check_slots
from .quant import _dtype_code
from .sparse_attn import _check_device

__all__ = ["paged_write_q"]

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
    A block's scale becomes the smallest power of two (at least 2^-64) that holds its new rows within e4m3's 448, and no smaller
    than the scale of its earlier tokens, those before the first new one: a block written from its first token on starts anew.
    Where the scale grows, the earlier codes are rounded to it.  New codes are the nearest (ties to even) to ``x / scale``.
    Infinities and NaN become NaN and do not count for the scale.
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
