"""The attention over 8-bit caches where two workgroups share a CU (D >= 512 and more than 256 row blocks: tiles of 32 keys, a loop of
its own), in the situations that ``test_gpu_paged_attn_q`` meets with few row blocks: keys split over workgroups and joined, missing
pages, pages that end inside a tile, values that are not finite.  Tolerances as there."""

from __future__ import annotations

import math

import pytest
import torch

from streamindex_amd import _lib

import tests.test_gpu_paged_attn_q as base
from tests.test_gpu_paged_attn_q import BF, DEV, HF, Step, every, same

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [BF, HF])


@pytest.fixture(params=[True, False], ids=["split", "whole"])
def scratch(request, monkeypatch):
    """With and without room for the shares of a row block's keys."""
    sizes = []
    take = _lib.scratch

    def note(n, d):
        sizes.append(n)
        return take(n, d) if request.param else (None, 0)

    monkeypatch.setattr(_lib, "scratch", note)
    yield sizes
    assert sizes and min(sizes) > 0  # every call here has row blocks to split


@BOTH
@pytest.mark.parametrize("D,H,lens", [
    (576, 64, [(5000 - 700 * (r // 60) if r % 60 == 7 else r % 90, 1) for r in range(300)]),  # the shares by every thread, R > 64
    (512, 64, [(6100 if r in (0, 599) else r % 50, 1) for r in range(600)]),  # more row blocks than run at once
    (576, 64, [(6000, 300), (20, 5), (0, 1)]),  # by every wave for itself
    (512, 100, [(3, 1), (4500, 250)]),  # row blocks that begin inside a token
    (576, 128, [(2500 if r % 16 == 3 else 10, 3) for r in range(64)]),
])
def test_split_keys(D, H, lens, dtype, scratch):
    s = Step(lens, H, D, dtype=dtype, page=64, block=16, pad=2)
    s.check(s.run(), skip=every(s, 7, 3) if s.N > 200 else ())


@BOTH
@pytest.mark.parametrize("D", [512, 576])
def test_split_hca(D, dtype, scratch):
    s = Step([(9000, 260), (700, 30), (0, 3)], 64, D, window=128, ratio=3, page=64, page2=16, block=64, block2=1, dtype=dtype, pad=1)
    s.check(s.run(), skip=every(s, 5, 2))


@pytest.mark.parametrize("page,block", [(1, 1), (3, 3), (7, 1), (33, 11), (96, 3), (512, 128)])
def test_pages_that_end_inside_a_tile(page, block):
    for D, dtype in ((512, BF), (576, HF)):
        s = Step([(150, 260), (40, 31), (0, 3)], 64, D, window=50, ratio=4, page=page, page2=page, block=block, block2=page, dtype=dtype, pad=1)
        s.check(s.run(), skip=every(s, 6, 5))
        s = Step([(150, 270)], 64, D, page=page, block=block, dtype=dtype)
        s.check(s.run(), skip=every(s, 6, 1))


@BOTH
@pytest.mark.parametrize("D", [512, 576])
@pytest.mark.parametrize("long", [0, 6000])
def test_missing_pages(D, long, dtype):
    """Pages that are not there, in one part of a tile, a whole one, all of them; what they would be read from is not finite."""
    s = Step([(200 + long, 300), (90, 2)], 64, D, page=16, block=16, window=None if long else 100, ratio=None if long else 8, page2=4, block2=2,
             dtype=dtype)
    for col in (8, 12, 13, 14, 17):
        s.table[0, col] = -1 if col != 12 else s.kv.shape[0]
    s.table[1, 5] = -2**31
    if s.ratio:
        s.table2[0, 3] = 2**31 - 1
        s.table2[1, :] = -1
    s.check(s.run(), skip=every(s, 6, 1))
    used = set(s.table.flatten().tolist()) | {0}
    for p in range(s.kv.shape[0]):
        if p not in used or not (s.table == p).any():
            s.kv.view(torch.uint8)[p] = 0x7f
            s.sc[p] = math.nan
    s.check(s.run(), skip=every(s, 6, 1))
    s.table[:] = -1
    if s.ratio:
        s.table2[:] = -1
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, s.sink.expand_as(lse))


@pytest.mark.parametrize("bad", ["code 0x7f", "code 0xff", "scale nan", "scale inf", "scale -inf"])
@pytest.mark.parametrize("D", [512, 576])
def test_not_finite(bad, D):
    """Masked keys in a chunk of 300 tokens, before the window, between the tokens, behind the end."""
    base.test_not_finite(bad, D, 64, [(60, 300), (5, 2)])


@BOTH
@pytest.mark.parametrize("bad", ["code", "scale"])
def test_not_finite_and_split(bad, dtype, scratch):
    """One late key of a long context: the tokens before it are as without it, to the bit, those that see it NaN."""
    s = Step([(6000, 300), (30, 2)], 64, 576, page=16, dtype=dtype)
    clean = s.run()
    at = 6123
    if bad == "code":
        s.kv.view(torch.uint8)[int(s.table[0, at // 16]), at % 16, 7] = 0xff
    else:
        s.sc[int(s.table[0, at // 16]), at % 16] = math.inf
    end = 6300  # behind the request's last key, in its last page
    s.kv.view(torch.uint8)[int(s.table[0, end // 16]), end % 16:] = 0x7f
    o, lse = s.run()
    assert torch.equal(o[:123], clean[0][:123]) and torch.equal(lse[:123], clean[1][:123])
    assert o[123:300, :, 7].isnan().all()
    assert torch.equal(o[300:], clean[0][300:]) and torch.equal(lse[300:], clean[1][300:])


@BOTH
@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("split", [True, False])
def test_many_small_weights(monkeypatch, dtype, last, split):
    base.test_many_small_weights(monkeypatch, dtype, 576, 64, 300, 1 << 14, last, split)


@BOTH
def test_scales_of_very_different_values(dtype):
    """Blocks of scales apart by 2^12, negative ones and zeros among them, queries of very different size."""
    g = torch.Generator().manual_seed(1)
    s = Step([(200, 300), (2100, 4)], 64, 576, page=16, block=4, dtype=dtype)
    s.sc = torch.exp2(torch.randint(-14, -2, s.sc.shape, generator=g).float()).to(DEV) * torch.where(torch.rand(s.sc.shape, generator=g) < 0.3, -1.0, 1.0).to(DEV)
    s.sc[::3, 1] = 0
    s.q *= torch.exp2(torch.randint(-12, 3, s.q.shape, generator=g).to(DEV))
    s.q[3] = 0
    s.check(s.run(), skip=every(s, 6, 3))


def test_in_a_graph_and_the_same_bits():
    """Captured and replayed with other queries, codes, tables and lengths, eager calls between the replays, on another stream too."""
    lens = [[(3000, 1)] * 3 + [(r % 70, 1) for r in range(297)], [(r % 40, 1) for r in range(295)] + [(2900, 1)] * 5]
    steps = [Step(v, 64, 576, page=64, block=16, seed=k) for k, v in enumerate(lens)]
    pages = max(s.kv.shape[0] for s in steps)
    wide = max(s.table.shape[1] for s in steps)
    for s in steps:
        grow = pages - s.kv.shape[0]
        s.kv = torch.cat([s.kv.view(torch.uint8), s.kv.view(torch.uint8).new_zeros(grow, *s.kv.shape[1:])]).view(s.kv.dtype)
        s.sc = torch.cat([s.sc, s.sc.new_zeros(grow, s.sc.shape[1])])
        s.table = torch.cat([s.table, s.table.new_full((300, wide - s.table.shape[1]), -1)], 1)
    names = ("q", "kv", "sc", "table", "cu", "seq", "sink")
    held = Step(lens[0], 64, 576, page=64, block=16)
    for n in names:
        setattr(held, n, getattr(steps[0], n).clone())
    held.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = held.run()
    side = torch.cuda.Stream()
    for i in (1, 0, 1):
        for n in names:
            getattr(held, n).copy_(getattr(steps[i], n))
        graph.replay()
        with torch.cuda.stream(side):
            other = steps[i].run()
        want = steps[i].run()
        torch.cuda.synchronize()
        same(out, want)
        same(other, want)
    steps[1].check(out, skip=every(steps[1], 4, 2))
