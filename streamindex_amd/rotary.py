"""Rotary positions of the heads' rows, alone and behind their norm, on MI355X (gfx950 HIP kernels via the C ABI).

Queries and keys come to the attention "RoPE-rotated" (``flash_sparse/csa.py:184``), as the reference's operators take them:

* :func:`rotary` — the rotation, of neighbouring dimensions or of halves, of the whole head or a part of it;
* :func:`norm_rotary` — each head's row over its root mean square, by a weight, then the rotation, in one pass;
* :func:`rotary_freqs` — the frequencies, stretched for long contexts or not.

Both have gradients, in x and the weight, of the first order and backward; forward-mode derivatives raise.  Angles are 64-bit, everything else fp32, rounded once to x's type.  The reference has
no counterpart.
"""

from __future__ import annotations

import functools
import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .quant import _DT, _dtype_code
from .sparse_attn import _check_device

__all__ = ["rotary", "norm_rotary", "rotary_freqs"]

MOST_D = 1024


def rotary_freqs(dims: int, base: float = 10000.0, *, factor: float = 1.0, original_length: int = 4096, fast: float = 32.0,
                 slow: float = 1.0, device="cuda") -> torch.Tensor:
    """Radians a position of each pair, ``base ** (-2 i / dims)``, ``[dims / 2]`` fp64.

    ``factor > 1`` stretches a context of ``original_length`` tokens, as the interpolation by parts of YaRN does (Peng, Quesnelle,
    Fan and Shippole, 2023): pairs that turn fewer than ``slow`` times in it are divided by ``factor``, those that turn more than
    ``fast`` times stay, and between them the share goes in a straight line over the pairs.  ``base`` is above 1 then.
    """
    if (dims < 0 or dims % 2 or not 0 < base < math.inf or not 1 <= factor < math.inf or original_length < 1 or not fast > slow > 0
            or (factor > 1 and base <= 1)):
        raise ValueError(f"bad frequencies: dims={dims}, base={base}, factor={factor}, original_length={original_length}, "
                         f"fast={fast}, slow={slow}")
    f = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if factor > 1:
        def pair(turns):  # that turns so often in original_length
            return dims * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dims - 1), pair(slow)
        share = [1.0 if i >= last else min(1.0, max(0.0, (i - lo) / max(hi - lo, 1))) for i in range(dims // 2)]
        f = [x * (1 - s) + x / factor * s for x, s in zip(f, share)]
    return torch.tensor(f, dtype=torch.float64, device=device)


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, interleaved: bool = True,
           start: Optional[int] = None, magnitude: float = 1.0, inverse: bool = False) -> torch.Tensor:
    """Rotates pairs of dimensions of every head by the token's position: with t = position * freqs[i],
    ``(a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t)``.

    Args:
      x: ``[..., H, D]`` fp32, bf16 or fp16, ``D <= 1024``.
      positions: int32 or int64, the sizes of x in front of the heads or the last of them (``[S]`` for ``[B, S, H, D]``);
        negative ones turn backwards.
      freqs: ``[dims / 2]`` radians a position (:func:`rotary_freqs`; fp32 ones are taken as they are, in 64 bits).
      interleaved: pairs of neighbours ``(2i, 2i + 1)`` (True) or of halves ``(i, i + dims / 2)``.
      start: the first of the ``dims`` rotary dimensions, those before and behind stay (default: the last of the head).
      magnitude: of the rotary dimensions, as stretched contexts scale them.
      inverse: turn the other way, as attention outputs are turned back.
    Returns a new tensor of x's type and shape.  Gradient in x.
    """
    return _apply(x, positions, freqs, None, None, interleaved, start, magnitude, inverse)


def norm_rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                eps: float = 1e-6, interleaved: bool = True, start: Optional[int] = None, magnitude: float = 1.0,
                inverse: bool = False) -> torch.Tensor:
    """``rotary(x * (mean(x ** 2) + eps) ** -0.5 * weight, ...)``, the mean over each head's D, in one pass.

    Squares are summed in fp32: values beyond about 2^60 overflow them and their row becomes 0; with an ``eps`` below 2^-120, rows of
    values below about 2^-60 lose bits, and then everything.
    ``weight``: ``[D]``, None for ones; the other arguments are :func:`rotary`'s.  Gradients in x and the weight (the same
    bits every time).  A step with its backward can be captured into a graph; results of eager calls on the same leaves have to be
    gone by then, since autograd ties the leaves to the stream of the first.
    """
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _apply(x, positions, freqs, weight, float(eps), interleaved, start, magnitude, inverse)


def _apply(x, positions, freqs, weight, eps, interleaved, start, magnitude, inverse):
    assert x.is_cuda, "x must be on the GPU"
    at_device = x.get_device()
    if not (positions.get_device() == freqs.get_device() == at_device and (weight is None or weight.get_device() == at_device)):
        _check_device(x.device, positions=positions, freqs=freqs, weight=weight)
    dt = _DT.get(x.dtype)
    if dt is None:
        dt = _dtype_code(x)
    shape = x.shape
    lead = len(shape) - 2
    if lead < 0:
        raise ValueError(f"x must be [..., H, D], got {list(shape)}")
    D = shape[-1]
    ft = freqs.dtype
    if freqs.dim() != 1 or not (ft is torch.float64 or ft.is_floating_point) or freqs.requires_grad:
        raise ValueError("freqs must be [dims / 2] floating point without gradient")
    dims = 2 * freqs.shape[0]
    at = D - dims if start is None else start
    if D < 1 or D > MOST_D or at < 0 or at + dims > D:
        raise ValueError(f"the head needs 1 to {MOST_D} dimensions and the rotary ones within it, got {D} and {at} to {at + dims}")
    n = positions.dim()
    pt = positions.dtype
    if pt is not torch.int64 and pt is not torch.int32:
        raise ValueError(f"positions must be int32 or int64, got {pt}")
    if n > lead or positions.shape != shape[lead - n:lead]:
        raise ValueError(f"positions must be {list(shape[:lead])} or its last sizes, got {list(positions.shape)}")
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != D):
        raise ValueError(f"weight must be [{D}], got {list(weight.shape)}")
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if ft is not torch.float64 or not freqs.is_contiguous():
        freqs = freqs.double().contiguous()
    args = (eps, not interleaved, at, float(magnitude), bool(inverse), dt)
    if ((x.requires_grad or (weight is not None and weight.requires_grad)) and torch.is_grad_enabled()) or _forward_mode():
        return _RotaryFunc.apply(x, weight, positions, freqs, args)
    return _forward(x, weight, positions, freqs, args)


def _forward_mode() -> bool:
    """Whether tensors may carry tangents, which autograd's function refuses and a kernel would drop."""
    return forward_ad._current_level >= 0


def _rows(x: torch.Tensor):
    """``x [..., H, D]`` as rows of a contiguous last dimension: the tensor to read (x itself where it can be), the strides of its
    tokens and heads."""
    H, D = x.shape[-2:]
    if x.is_contiguous():
        return x, _lib.stride_array((H * D, D))
    x = x.reshape(-1, H, D)
    s = x.stride()
    if s[2] != 1 and D > 1:
        x = x.contiguous()
        s = (H * D, D)
    return x, _lib.stride_array(s[:2])


def _fp32(weight: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if weight is None:
        return None
    w = weight if weight.dtype is torch.float32 else weight.float()
    return w if w.is_contiguous() else w.contiguous()


def _forward(x, weight, positions, freqs, args):
    eps, halves, start, magnitude, inverse, dt = args
    dev = x.device
    H, D = x.shape[-2:]
    n = x.numel()
    L = _lib.load()
    with _lib.on_device(dev):
        if x.is_contiguous():
            y, rows, strides = torch.empty_like(x), x, _lib.stride_array((H * D, D))
        else:
            y = torch.empty(x.shape, dtype=x.dtype, device=dev)
            rows, strides = _rows(x) if n else (x, None)
        if n == 0:
            return y
        w = _fp32(weight)
        rc = L.si_norm_rotary(rows.data_ptr(), strides, eps is not None, None if w is None else w.data_ptr(), eps or 0.0,
                              positions.data_ptr(), positions.dtype is torch.int64, positions.numel(), freqs.data_ptr(),
                              freqs.shape[0], start, halves, magnitude, inverse, n // (H * D), H, D, dt, y.data_ptr(),
                              _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    return y


@functools.lru_cache(maxsize=1024)
def _workspace(*sizes) -> int:
    return _lib.load().si_norm_rotary_bwd_workspace_bytes(*sizes)


def _backward(ctx, dy):
    if _forward_mode() and forward_ad.unpack_dual(dy).tangent is not None:
        raise NotImplementedError("the gradients of rotary and norm_rotary have no forward-mode derivative")
    positions, freqs, *saved = ctx.saved_tensors
    eps, halves, start, magnitude, inverse, dt = ctx.args
    if not saved:
        return _forward(dy, None, positions, freqs, (None, halves, start, magnitude, not inverse, dt)), None, None, None, None
    x, weight = saved[0], saved[1] if len(saved) > 1 else None
    need_w = weight is not None and ctx.needs_input_grad[1]
    dev = x.device
    L = _lib.load()
    with _lib.on_device(dev):
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        n = x.numel()
        H, D = x.shape[-2:]
        dw = torch.empty(D, dtype=torch.float32, device=dev) if need_w else None
        if n == 0:
            return dx, None if dw is None else dw.zero_().to(weight.dtype), None, None, None
        (rows, strides), (drows, dstrides), w = _rows(x), _rows(dy), _fp32(weight)
        T = n // (H * D)
        size = _workspace(T, H, D, freqs.shape[0]) if need_w else 0
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if need_w else None
        rc = L.si_norm_rotary_bwd(drows.data_ptr(), dstrides, rows.data_ptr(), strides, None if w is None else w.data_ptr(), eps,
                                  positions.data_ptr(), positions.dtype is torch.int64, positions.numel(), freqs.data_ptr(),
                                  freqs.shape[0], start, halves, magnitude, inverse, T, H, D, dt, dx.data_ptr(),
                                  None if dw is None else dw.data_ptr(), None if ws is None else ws.data_ptr(), size,
                                  _lib.stream_ptr(dev))
    _lib.check(rc)
    return dx, None if dw is None else dw if weight.dtype is torch.float32 else dw.to(weight.dtype), None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


class _RotaryFunc(torch.autograd.Function):
    """Norm (with ``eps``) and rotation; the backward keeps x for the norm and nothing for the rotation alone."""

    @staticmethod
    def forward(ctx, x, weight, positions, freqs, args):
        if args[0] is None:
            ctx.save_for_backward(positions, freqs)
        elif weight is None:
            ctx.save_for_backward(positions, freqs, x)
        else:
            ctx.save_for_backward(positions, freqs, x, weight)
        ctx.args = args
        return _forward(x, weight, positions, freqs, args)

    @staticmethod
    def backward(ctx, dy):
        # (a second derivative is an error; without one asked for, nothing has to see to that: 10 us)
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)
