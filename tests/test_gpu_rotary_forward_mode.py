"""Forward-mode derivatives of the norm and rotation are refused: a result without its tangent would be a derivative of zero."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from streamindex_amd import norm_rotary, rotary, rotary_freqs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make():
    g = torch.Generator().manual_seed(3)
    x, v, w = torch.randn(2, 5, 2, 64, generator=g)[0].to(DEV), torch.randn(5, 2, 64, generator=g).to(DEV), torch.rand(64, generator=g).to(DEV)
    return x, v, w, torch.arange(5, device=DEV), rotary_freqs(32)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dual_tensors_raise(dtype, grad):
    x, v, w, pos, f = make()
    x, v = x.to(dtype), v.to(dtype)
    plain, normed = rotary(x, pos, f), norm_rotary(x, pos, f, w)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dx, dw, df = forward_ad.make_dual(x, v), forward_ad.make_dual(w, torch.ones_like(w)), forward_ad.make_dual(f, torch.ones_like(f))
        for call in (lambda: rotary(dx, pos, f), lambda: norm_rotary(dx, pos, f), lambda: norm_rotary(dx, pos, f, w),
                     lambda: norm_rotary(x, pos, f, dw), lambda: rotary(x, pos, df), lambda: norm_rotary(x, pos, df, w)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        # tensors without a tangent: as outside
        assert torch.equal(rotary(x, pos, f), plain) and torch.equal(norm_rotary(x, pos, f, w), normed)
    assert torch.equal(norm_rotary(x, pos, f, w), normed)


@pytest.mark.parametrize("norm", [True, False])
def test_jvp_and_a_dual_gradient_raise(norm):
    x, v, w, pos, f = make()
    call = (lambda t: norm_rotary(t, pos, f, w)) if norm else (lambda t: rotary(t, pos, f))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(call, (x,), (v,))
    leaf = x.clone().requires_grad_()
    want, = torch.autograd.grad(call(leaf), [leaf], v)
    with forward_ad.dual_level():
        y = call(leaf)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.autograd.grad(y, [leaf], forward_ad.make_dual(v, x), retain_graph=True)
        assert torch.equal(torch.autograd.grad(y, [leaf], v)[0], want)
