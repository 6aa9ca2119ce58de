"""GPU results of the write into a paged cache in 8 bits: the definition's own codes and scales, to the bit.

Every step is exact but the one rounding to e4m3, which the oracle does in 64 bits from its definition: steps of 2^(e - 3) from
2^e on, of 2^-9 below 2^-6, ties to even.
"""

from __future__ import annotations

import math

import pytest
import torch

from streamindex_amd import paged_plan, paged_write_q

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def e4m3(v):
    """The nearest e4m3 value of ``|v| <= 464`` in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def oracle(codes, scales, rows, slots, block):
    """``(codes, scales)`` in 64 bits behind a write of rows in the plan's order."""
    codes, scales = codes.double(), scales.double()
    pages, ps, D = codes.shape
    flat, sc = codes.view(-1, D), scales.reshape(-1)
    rows = rows.double()
    t, n = 0, rows.shape[0]
    slots = slots.tolist()
    while t < n:
        s = slots[t]
        if not 0 <= s < pages * ps:
            t += 1
            continue
        b = s // block
        here, k = [t], t + 1  # rows of the run: those without a slot do not matter
        while k < n and k - here[-1] <= 64 and (not 0 <= slots[k] < pages * ps or (slots[k] // block == b and slots[k] > slots[here[-1]])):
            if 0 <= slots[k] < pages * ps:
                here.append(k)
            k += 1
        x = rows[here]
        most = float(x.abs()[x.isfinite()].max()) if x.isfinite().any() else 0.0
        e = -64
        while 448 * 2.0 ** e < most:
            e += 1
        scale, first = 2.0 ** e, s % block
        if first:
            old = float(sc[b])
            scale = max(scale, old)
            flat[b * block: s] = e4m3(flat[b * block: s] * (old / scale))
        sc[b] = scale
        x = torch.where(x.isfinite(), x, math.nan)
        flat[[slots[i] for i in here]] = e4m3(x / scale)
        t = here[-1] + 1
    return codes, sc.view(scales.shape)


class Cache:
    def __init__(self, pages, page, block, D, seed=0, pad=0):
        g = torch.Generator().manual_seed(seed)
        wide = (torch.randn(pages, page, D + pad, generator=g) * 100).clamp(-448, 448).to(F8)
        self.block = block
        self.codes = wide.to(DEV)[..., :D]
        self.scales = torch.exp2(torch.randint(-9, -4, (pages, page // block), generator=g).float()).to(DEV)

    def check(self, rows, slots):
        want, sc = oracle(self.codes.cpu().float(), self.scales.cpu(), rows.cpu().float(), slots.cpu(), self.block)
        got = paged_write_q(rows, self.codes, self.scales, slots)
        assert got[0] is self.codes and got[1] is self.scales
        assert torch.equal(self.scales.cpu().double(), sc)
        a = self.codes.cpu().float().double()
        assert ((a == want) | (a.isnan() & want.isnan())).all(), int((a != want).sum())


def plan_slots(lens, page, pages, pad=0, seed=0):
    """Slots of new tokens of requests ``(earlier, new)`` in pages of a random order, `pad` rows without one behind them."""
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    out, at = [], 0
    for ctx, n in lens:
        mine = perm[at: at + -(-(ctx + n) // page)]
        at += len(mine)
        out += [mine[p // page] * page + p % page for p in range(ctx, ctx + n)]
    assert at <= pages
    return torch.tensor(out + [-1] * pad, dtype=torch.int64, device=DEV)


def make_rows(n, D, dtype, seed=0, spread=0.8):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, D, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))).to(dtype).to(DEV)


LENS = [[(0, 1)], [(5, 1), (63, 1), (64, 1), (1, 1)], [(0, 200), (3, 130), (127, 5), (64, 64)], [(17, 700)], [(100, 1)] * 40]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("page,block,D", [(64, 1, 576), (64, 64, 576), (64, 16, 512), (16, 4, 64), (100, 25, 500), (32, 2, 7), (6, 3, 1),
                                          (128, 128, 33), (8, 8, 1028)])
def test_values(page, block, D, lens, dtype):
    pages = sum(-(-(a + b) // page) for a, b in lens) + 2
    slots = plan_slots(lens, page, pages, pad=3)
    c = Cache(pages, page, block, D, seed=D)
    for k in range(2):  # the second time the scales are those of the first
        c.check(make_rows(len(slots), D, dtype, seed=k), slots)


@pytest.mark.parametrize("block", [1, 16, 64])
def test_steps_of_a_request(block):
    """A request written token by token, then in chunks: the scale grows as its block fills."""
    c = Cache(4, 64, block, 128)
    for k, (ctx, n) in enumerate([(i, 1) for i in range(20)] + [(20, 30), (50, 100), (150, 1)]):
        c.check(make_rows(n, 128, BF, seed=k, spread=2.0), plan_slots([(ctx, n)], 64, 4))


def test_many_rows():
    """More rows than workgroups: several blocks begin in one's share, and blocks go over its end."""
    for block, n in ((8, 9001), (32, 9001), (64, 70000)):
        pages = n // 64 + 3
        slots = plan_slots([(40, n)], 64, pages)
        c = Cache(pages, 64, block, 16)
        rows = make_rows(n, 16, BF)
        c.check(rows, slots)
    lens = [(i % 70, 1 + i % 9) for i in range(900)]
    slots = plan_slots(lens, 64, 1900)
    Cache(1900, 64, 32, 64).check(make_rows(len(slots), 64, BF), slots)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_every_exponent(dtype):
    """Maxima next to 448 times every power of two, from below the least scale to the type's largest value."""
    fi = torch.finfo(dtype)
    tops = [m * 2.0 ** e for e in range(-140, 128) for m in (0.875, 0.87890625, 0.8828125, 1.0, 0.5)]
    tops = [t for t in tops if t <= fi.max] + [fi.max, 0.0]
    g = torch.Generator().manual_seed(1)
    rows = torch.tensor(tops, dtype=torch.float64)[:, None] * torch.cat([torch.ones(1), torch.rand(15, generator=g) * 2 - 1])
    rows = rows.to(dtype).to(DEV)
    n = rows.shape[0]
    for block in (1, 2):
        c = Cache(n, block, block, 16)
        slots = torch.arange(n, device=DEV) * block
        c.check(rows, slots)
        if block == 2:
            c.check(rows.flip(0), slots + 1)  # beside an earlier token whose scale it may lift far


def test_every_code_is_rescaled():
    codes = torch.arange(256, dtype=torch.uint8).view(F8).float()
    codes = torch.where(codes.isnan(), 0.0, codes)
    for up in range(0, 20):
        c = Cache(1, 2, 2, 256)
        c.codes[0, 0] = codes.to(F8).to(DEV)
        c.scales[0, 0] = 0.5
        row = torch.zeros(1, 256, device=DEV)
        row[0, 0] = 448 * 0.5 * 2.0 ** up
        c.check(row, torch.tensor([1], device=DEV))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("block", [1, 4])
def test_not_finite(block, dtype):
    c = Cache(10, 4, block, 64)
    rows = make_rows(20, 64, dtype)
    rows[3, 5], rows[4, 0], rows[9, 63], rows[12] = math.nan, math.inf, -math.inf, math.nan
    c.check(rows, plan_slots([(2, 20)], 4, 10))


def test_a_cache_that_held_something_else():
    """A block begun anew takes nothing from the scale and the codes that its page held; a scale that is none counts as none."""
    for bad in (math.nan, math.inf, 0.0, -1.0):
        c = Cache(2, 8, 8, 32)
        c.scales[:] = bad
        rows = make_rows(3, 32, BF)
        got = paged_write_q(rows, c.codes, c.scales, torch.tensor([0, 1, 2], device=DEV))
        want, sc = oracle(torch.zeros(2, 8, 32), torch.ones(2, 1), rows.cpu().float(), torch.tensor([0, 1, 2]), 8)
        assert torch.equal(got[0][0, :3].float().cpu().double(), want[0, :3]) and float(got[1][0, 0]) == float(sc[0, 0])
        was = c.codes[1].view(torch.uint8).clone()
        paged_write_q(rows, c.codes, c.scales, torch.tensor([11, 12, 13], device=DEV))
        assert torch.equal(c.codes[1, :3].view(torch.uint8), was[:3]) and float(c.scales[1, 0]) == float(sc[0, 0])
        assert torch.equal(c.codes[1, 3:6].float().cpu().double(), want[0, :3])


def test_slots_outside_and_rows_behind():
    c = Cache(4, 8, 4, 64)
    before, sc = c.codes.view(torch.uint8).clone(), c.scales.clone()
    slots = torch.tensor([-1, 32, 1 << 40, -(1 << 62), 2**31], device=DEV)
    paged_write_q(make_rows(5, 64, BF), c.codes, c.scales, slots)
    assert torch.equal(c.codes.view(torch.uint8), before) and torch.equal(c.scales, sc)
    c.check(make_rows(8, 64, BF), torch.tensor([-1, 4, 5, -1, 6, 9, 31, -1], device=DEV))


@pytest.mark.parametrize("gap", [1, 5, 63])
def test_rows_without_a_slot_within_a_block(gap):
    for block, D in ((8, 64), (64, 7)):
        g = torch.Generator().manual_seed(gap)
        slots = plan_slots([(3, 200), (60, 90)], 64, 8).tolist()
        out = []
        for s in slots:
            out += [s] + [-1] * int(torch.randint(0, gap + 1, (1,), generator=g))
        c = Cache(8, 64, block, D)
        c.check(make_rows(len(out), D, BF, seed=gap, spread=1.5), torch.tensor(out, device=DEV))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides(dtype):
    """Rows that are a part of wider ones or at odd places, caches that are, scales of wider rows."""
    for D, pad in ((576, 16), (64, 3), (128, 8)):
        slots = plan_slots([(3, 50)], 16, 8)
        rows = make_rows(50, 3 * D + 1, dtype)
        for r in (rows[:, D:2 * D], rows[:, 1:D + 1], make_rows(D, 50, dtype).t(), make_rows(1, D, dtype).expand(50, D)):
            for block in (1, 16):
                c = Cache(8, 16, block, D, pad=pad)
                c.scales = torch.cat([c.scales, c.scales], 1)[:, : c.scales.shape[1]]
                c.check(r, slots)
                want = c.codes.float()
                other = c.codes.new_zeros(8, 16, D + pad).view(torch.uint8)
                assert c.codes.stride() == other.stride() and want.isfinite().all()


@pytest.mark.parametrize("block", [1, 16])
def test_far_offsets(block):
    """Cache rows past 2^32 bytes, scales past 2^31, rows past 2^31 values: as near ones."""
    slots = plan_slots([(3, 40), (70, 9)], 16, 10, seed=2)
    rows = make_rows(len(slots), 64, BF)
    c = Cache(10, 16, block, 64)
    far = torch.empty(6 << 30, dtype=torch.uint8, device=DEV).view(F8).as_strided((10, 16, 64), ((6 << 30) // 10 // 16 * 16, 64, 1))
    far.view(torch.uint8).copy_(c.codes.view(torch.uint8))
    scales = torch.empty((10 << 30) // 4, device=DEV).as_strided((10, 16 // block), ((10 << 30) // 40, 1))
    scales.copy_(c.scales)
    wide = torch.empty((len(slots) + 1) * (1 << 26), dtype=BF, device=DEV).as_strided((len(slots), 64), (1 << 26, 1))
    wide.copy_(rows)
    paged_write_q(wide, far, scales, slots)
    c.check(rows, slots)
    assert torch.equal(far.contiguous().view(torch.uint8), c.codes.view(torch.uint8)) and torch.equal(scales.contiguous(), c.scales)


def test_nothing_between_rows_is_written():
    wide = torch.full((4, 8, 100), 7, dtype=torch.uint8, device=DEV)
    cache = wide.view(F8)[..., 20:84]
    paged_write_q(make_rows(9, 64, BF), cache, torch.ones(4, 2, device=DEV), torch.arange(5, 14, device=DEV))
    assert (wide[..., :20] == 7).all() and (wide[..., 84:] == 7).all()
    flat = wide.view(-1, 100)
    assert (flat[:5] == 7).all() and (flat[14:] == 7).all()


def test_of_a_plan_and_captured():
    """Plan and write captured, replayed for step after step, against the same steps one by one."""
    R, page, block, D = 5, 16, 8, 64
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    ctx, new = i32([0, 3, 15, 16, 40]), i32([1, 1, 1, 1, 1])
    free = torch.randperm(60, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(DEV)
    table, start = torch.full((R, 8), -1, dtype=torch.int32, device=DEV), i32([0])
    warm = paged_plan(i32([0] * R), ctx, table, free, page, 200, free_start=start)
    c, d = Cache(60, page, block, D), Cache(60, page, block, D)
    first = make_rows(200, D, BF, seed=9)
    start.copy_(warm.free_next)
    c.check(first, warm.slots)
    paged_write_q(first, d.codes, d.scales, warm.slots)
    rows = make_rows(R, D, BF)

    def step(cache, t, f):
        p = paged_plan(ctx, new, t, free, page, R, free_start=f)
        paged_write_q(rows, cache.codes, cache.scales, p.slots)
        return p

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(Cache(60, page, block, D), table.clone(), start)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    mine, at = table.clone(), start.clone()
    with torch.cuda.graph(graph):
        p = step(c, mine, at)
        at.copy_(p.free_next)
        ctx += 1
    for k in range(12):
        rows.copy_(make_rows(R, D, BF, seed=20 + k, spread=1.5))
        torch.cuda.synchronize()
        q = step(d, table, start)
        start.copy_(q.free_next)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.codes.view(torch.uint8), d.codes.view(torch.uint8)) and torch.equal(c.scales, d.scales)
        assert torch.equal(mine, table)


def test_refusals():
    rows, slots = make_rows(2, 64, BF), torch.tensor([0, 1], device=DEV)
    cache, scales = torch.zeros(2, 4, 64, device=DEV).to(F8), torch.ones(2, 4, device=DEV)
    for call in (
            lambda: paged_write_q(rows, cache.float(), scales, slots), lambda: paged_write_q(rows, cache, scales.double(), slots),
            lambda: paged_write_q(rows, cache, scales[:, :3], slots), lambda: paged_write_q(rows, cache, scales[:1], slots),
            lambda: paged_write_q(rows, cache, scales[:, :0], slots), lambda: paged_write_q(rows, cache, scales, slots.int()),
            lambda: paged_write_q(rows.double(), cache, scales, slots), lambda: paged_write_q(rows, cache, torch.ones(4, 2, device=DEV).t(), slots),
            lambda: paged_write_q(rows, cache[:, :1].expand(2, 4, 64), scales, slots),
            lambda: paged_write_q(rows, cache, scales[:1].expand(2, 4), slots)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: paged_write_q(rows[:, :63], cache, scales, slots), lambda: paged_write_q(rows, cache, scales, slots[:1]),
                 lambda: paged_write_q(rows, cache, scales.cpu(), slots), lambda: paged_write_q(rows, cache[0], scales, slots)):
        with pytest.raises(AssertionError):
            call()
