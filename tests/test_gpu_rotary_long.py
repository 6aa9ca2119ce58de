"""Norm and rotation of training sequences so long that a workgroup fills its table of cosines and sines several times, from rows that
begin inside a token: every value of y, dx and dw against 64-bit floats.

Tolerances of y and dx as in ``test_gpu_rotary``.  dw: 2^-17 of each term, and along a path at most 223 additions in a register, 3
between lanes, 2 between waves, 32 and 16 between workgroups: 276 2^-24 < 2^-15.8, together below 2^-15 of sum |d n|.
"""

from __future__ import annotations

import pytest
import torch

from streamindex_amd import norm_rotary, rotary_freqs

from tests.test_gpu_rotary import BF, DEV, F32, HF, turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,T,H,D,dims,halves", [
    (BF, 15000, 64, 128, 128, False), (BF, 27405, 64, 576, 64, False), (HF, 14000, 64, 128, 128, True), (F32, 60000, 5, 64, 64, True),
    (BF, 60000, 5, 64, 64, False), (BF, 11000, 6, 128, 128, False), (F32, 12806, 64, 128, 128, False), (BF, 5001, 24, 128, 64, True)])
def test_every_row(dtype, T, H, D, dims, halves):
    g = torch.Generator(device=DEV).manual_seed(T + D)
    x, dy = (torch.randn(T, H, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    w = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).requires_grad_()
    pos, freqs, start, m, eps = torch.arange(T, device=DEV) + 1000, rotary_freqs(dims), D - dims, 1.1, 1e-6
    x.requires_grad_()
    y = norm_rotary(x, pos, freqs, w, eps=eps, interleaved=not halves, magnitude=m)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    only, = torch.autograd.grad(norm_rotary(x, pos, freqs, eps=eps, interleaved=not halves, magnitude=m), [x], dy)  # without a weight
    u, small = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    want_dw, mag_dw = torch.zeros(2, D, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 25) // (H * D))
    for at in range(0, T, step):
        part = slice(at, at + step)
        a, b = x[part].detach().double(), dy[part].double()
        r = (a.square().mean(-1, keepdim=True) + eps) ** -0.5
        n = a * r
        d, dmag = turn(b, pos[part], freqs, halves, start, m, -1)
        want_dw += (d * n).sum((0, 1))
        mag_dw += (dmag * n.abs()).sum((0, 1))
        for weight, gy, gx in ((w.detach().double(), y, dx), (1.0, None, only)):
            if gy is not None:
                want, mag = turn(n * weight, pos[part], freqs, halves, start, m, 1)
                assert ((gy[part].detach().double() - want).abs() <= u * want.abs() + 2.0 ** -18 * mag + small).all(), ("y", at)
            e = d * weight
            emag = dmag * abs(weight)
            want = r * (e - n * (e * n).mean(-1, keepdim=True))
            mag = r * (emag + n.abs() * (emag * n.abs()).mean(-1, keepdim=True))
            err = (gx[part].double() - want).abs() - (u * want.abs() + 2.0 ** -17 * mag + small)
            assert (err <= 0).all(), ("dx", at, int((err > 0).sum()), float(err.max()))
    assert ((dw.double() - want_dw).abs() <= 2.0 ** -15 * mag_dw).all()
