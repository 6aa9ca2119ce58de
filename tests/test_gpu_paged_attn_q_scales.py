"""The attention over 8-bit caches with scales at both ends of the range that it serves, in each of its loops.  The softmax scale
brings the scores back to ordinary ones, normal ones of a deviation of at most 2: they differ by less than 20, so that weights stay
above 2^-30 of a row's largest and no product with a scale leaves fp32's range.  Tolerances as in ``test_gpu_paged_attn_q``."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_attn_q import BF, DEV, HF, Step, every

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H,lens", [(128, 16, [(200, 3), (70, 1)]), (576, 64, [(5000, 1), (20, 2)]), (576, 64, [(200, 300)]),
                                      (32, 8, [(2000, 2)])])
@pytest.mark.parametrize("dtype,power", [(BF, -64), (BF, 96), (HF, -64), (HF, 0)])
def test_ends_of_the_range(D, H, lens, dtype, power):
    s = Step(lens, H, D, page=16, block=4, dtype=dtype)
    g = torch.Generator().manual_seed(1)
    sign = torch.where(torch.rand(s.sc.shape, generator=g) < 0.3, -1.0, 1.0)
    s.sc = (torch.exp2(torch.randint(0, 5, s.sc.shape, generator=g).float() + power) * sign).to(DEV)
    s.sc[::3, 1] = 0
    scale = 2.0 ** (-power - 9) * D ** -0.5
    s.check(s.run(softmax_scale=scale), scale=scale, skip=every(s, 6, 3) if s.N > 100 else ())
    assert float(s.sc.abs().max()) <= 2.0 ** 100 and (s.sc.abs()[s.sc != 0] >= 2.0 ** -64).all()
