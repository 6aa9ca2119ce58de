"""Writes beside earlier tokens whose scale is no power of two, as another program may have set it: the scale stays where it is large
enough, and every code, new or rescaled, is the one e4m3 rounding of the exact quotient or product, to the bit.

The values stand where a rounding to fp32 in between would be seen: within 2^-23 of the middle between two e4m3 values.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_write_q import BF, DEV, F32, F8, HF, Cache, make_rows, plan_slots

pytestmark = pytest.mark.gpu


def ulps(x, k):
    """fp32 values k steps from x > 0."""
    return (x.float().view(torch.int32) + k).view(torch.float32)


def middles():
    """The middles between e4m3 values from 2^-10 to 200."""
    v = torch.arange(256, dtype=torch.uint8).view(F8).float()[:0x7f].double()
    m = (v[1:] + v[:-1]) / 2
    return m[m < 200]


@pytest.mark.parametrize("D", [64, 36, 7])
@pytest.mark.parametrize("power", [0, -60, 90])
def test_new_codes_fp32(D, power):
    """Blocks of two tokens with scales of 24 bits; the new row's values within two fp32 steps of a middle times the scale."""
    g = torch.Generator().manual_seed(D + power)
    n = 200
    c = Cache(n, 2, 2, D, seed=1)
    scale = (0.5 + torch.rand(n, generator=g)) * 2.0 ** power
    m = middles()[torch.randint(0, len(middles()), (n, D), generator=g)]
    x = ulps(m * scale[:, None].double(), torch.randint(-2, 3, (n, D), generator=g).to(torch.int32))
    x *= torch.randint(0, 2, (n, D), generator=g) * 2 - 1
    c.scales[:, 0] = scale.to(DEV)
    was = c.codes.view(torch.uint8).clone()
    c.check(x.to(DEV), torch.arange(n, device=DEV) * 2 + 1)
    assert torch.equal(c.scales[:, 0].cpu(), scale) and torch.equal(c.codes.view(torch.uint8)[:, 0], was[:, 0])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_new_codes_16_bits(dtype):
    """The scales chosen for one value of each row: x / scale within two fp32 steps of a middle."""
    g = torch.Generator().manual_seed(2)
    n, D = 800, 64
    m = middles()
    m = m[m > 0.01][torch.randint(0, int((m > 0.01).sum()), (n,), generator=g)]
    x = torch.randn(n, D, generator=g).clamp(-3, 3).to(dtype)
    x[:, 5] = (0.5 + torch.rand(n, generator=g)).to(dtype)
    scale = ulps(x[:, 5].double() / m, torch.randint(-2, 3, (n,), generator=g).to(torch.int32))
    x = torch.minimum(x.abs().double(), 200 * scale.double()[:, None]).to(dtype).copysign(x)
    c = Cache(n, 2, 2, D, seed=1)
    c.scales[:, 0] = scale.to(DEV)
    c.check(x.to(DEV), torch.arange(n, device=DEV) * 2 + 1)
    assert torch.equal(c.scales[:, 0].cpu(), scale)


@pytest.mark.parametrize("power", [0, -70, 60])
def test_rescaled_codes(power):
    """Earlier codes times old / new within two fp32 steps of a middle, where the new row makes the scale a larger power of two."""
    c8 = torch.arange(8, 16).double() / 8
    tie = (torch.arange(17, 32, 2).double() / 16)
    old = (tie[:, None] / c8).reshape(-1)
    old = torch.cat([ulps(old, torch.tensor(k, dtype=torch.int32)) for k in range(-2, 3)])
    n = len(old)
    codes = torch.arange(256, dtype=torch.uint8).view(F8)
    codes = torch.where(codes.float().isnan(), 0.0, codes.float()).to(F8)
    for up in (2, 3, 6, 9, 14):
        c = Cache(n, 2, 2, 256)
        c.codes[:, 0] = codes.to(DEV)
        c.scales[:, 0] = (old * 2.0 ** power).to(DEV)
        row = torch.zeros(n, 256, device=DEV)
        row[:, 3] = 448 * 2.0 ** (power + up)
        c.check(row, torch.arange(n, device=DEV) * 2 + 1)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("page,block,D", [(64, 64, 576), (16, 4, 64), (100, 25, 500), (6, 3, 1), (8, 8, 1028), (8, 8, 4100)])
def test_steps(page, block, D, dtype):
    """Ragged chunks beside such scales, large enough and too small ones; rows without a slot between; and the next step."""
    lens = [(5, 1), (63, 70), (2, 9), (31, 1), (70, 200)]
    pages = sum(-(-(a + b) // page) for a, b in lens) + 2
    slots = plan_slots(lens, page, pages, pad=3)
    slots[75] = -1  # (rows 1 .. 70 and 71 .. 79 are two requests')
    c = Cache(pages, page, block, D, seed=D)
    c.scales *= 1.37 * torch.rand(c.scales.shape, generator=torch.Generator().manual_seed(3)).to(DEV) + 0.01
    for k in range(2):
        c.check(make_rows(len(slots), D, dtype, seed=k), slots)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_largest_scales(dtype):
    """Earlier scales next to fp32's largest value, whose reciprocal is below its normal range."""
    g = torch.Generator().manual_seed(4)
    top = torch.tensor([2.0 ** 126, 2.0 ** 127, 1.5 * 2.0 ** 126, 1.3 * 2.0 ** 127, torch.finfo(torch.float32).max])
    c = Cache(len(top), 2, 2, 64, seed=1)
    c.scales[:, 0] = top.to(DEV)
    x = (torch.rand(len(top), 64, generator=g) * 2 - 1) * torch.exp2(torch.randint(90, 128, (len(top), 64), generator=g).float())
    c.check(x.to(dtype).to(DEV), torch.arange(len(top), device=DEV) * 2 + 1)
    assert torch.equal(c.scales[:, 0].cpu(), top)
