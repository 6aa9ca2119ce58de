"""GPU parity of the attention over a paged cache in 8 bits against 64-bit floats, over codes times scales.

Tolerances: u |ref| + (u + 2 E) sum p |v| / l (1 + 2 u), u = eps / 2 of q's type: the roundings of the output and of a weight times its
scale.  fp16: such a product keeps its 11 bits down to 2^-25 of its row's largest (that is at 2^11 to 2^15, normal values reach
2^-14); below, it is off by 2^-25, half a subnormal step, so by 2^-36 of the largest, for every key: + 2^-36 max_k p_k s_k / l sum |c|,
codes c.  E bounds the error of a score: D fp32 products and sums
(D 2^-24 scale |q|.|k|) and the exponential (2^-20).  lse: E + 2^-20 (1 + |lse|).
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from streamindex_amd import (_lib, norm_rotary, paged_attn_fwd, paged_attn_q_fwd, paged_compress, paged_plan, paged_write,
                             paged_write_q, rotary, rotary_freqs)

from tests.test_gpu_paged import EVERY, half_step, i32, make_table

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16


class Step:
    """A step of requests (earlier, new tokens) with random caches in 8 bits."""

    def __init__(self, lens, H, D, *, window=None, ratio=None, page=16, page2=16, block=1, block2=1, dtype=BF, pad=0, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed + 17)
        self.lens, self.H, self.D, self.window, self.ratio, self.dtype = lens, H, D, window, ratio, dtype
        self.N = sum(n for _, n in lens) + pad
        self.table, pages = make_table([(max(0, c + 1 - (window or EVERY)), c + n) for c, n in lens], page, seed)
        self.kv, self.sc = self.cache(pages, page, block, spread, g)
        self.kv2 = self.sc2 = self.table2 = None
        if ratio:
            self.table2, pages2 = make_table([(0, (c + n) // ratio) for c, n in lens], page2, seed + 1)
            self.kv2, self.sc2 = self.cache(pages2, page2, block2, spread, g)
        self.q = torch.randn(self.N, H, D, generator=g).to(dtype).to(DEV)
        self.sink = torch.randn(H, generator=g).to(DEV)
        cu = [0]
        for _, n in lens:
            cu.append(cu[-1] + n)
        self.cu, self.seq = i32(cu), i32([c + n for c, n in lens])

    def cache(self, pages, page, block, spread, g):
        """Rows of about ``spread``, blocks of scales from 2^-9 to 2^-5 of it, not all powers of two."""
        e = torch.randint(-9, -5, (pages, page // block), generator=g).float()
        scales = torch.exp2(e) * (1 + 0.37 * (torch.rand(pages, page // block, generator=g) < 0.3))
        codes = torch.randn(pages, page, self.D, generator=g) * 64
        return codes.clamp(-448, 448).to(F8).to(DEV), (scales * spread).to(DEV)

    def run(self, **kw):
        more = {"kv2_cache": self.kv2, "kv2_scales": self.sc2, "block_table2": self.table2, "ratio": self.ratio} if self.ratio else {}
        return paged_attn_q_fwd(self.q, self.kv, self.sc, self.table, self.cu, self.seq, self.sink, window=self.window, **more, **kw)

    def keys(self, r, p, scales=False):
        """Entries that the token of request r at position p sees, and their scales."""
        out, of = [], []
        for cache, sc, table, ks in ((self.kv, self.sc, self.table, range(max(0, p + 1 - (self.window or EVERY)), p + 1)),
                                     (self.kv2, self.sc2, self.table2, range((p + 1) // self.ratio if self.ratio else 0))):
            if len(ks) == 0:
                continue
            k = torch.tensor(ks, device=DEV)
            page = cache.shape[1]
            block = page // sc.shape[1]
            col = k // page
            pg = torch.where(col < table.shape[1], table[r].long()[col.clamp(max=table.shape[1] - 1)], -1) if table.shape[1] else col * 0 - 1
            ok = (pg >= 0) & (pg < cache.shape[0])
            at, off = pg[ok], (k % page)[ok]
            of.append(sc[at, off // block].double())
            out.append(cache.view(torch.uint8)[at, off].view(F8).double() * of[-1][:, None])
        k = torch.cat(out) if out else torch.zeros(0, self.D, dtype=torch.float64, device=DEV)
        return (k, torch.cat(of) if of else k[:, 0]) if scales else k

    def check(self, got, scale=None, skip=(), more=0.0):
        """Compares with the definition in 64 bits, token by token; ``more``: of sums over very many keys."""
        o, lse = got
        u, scale = half_step(self.dtype), self.D ** -0.5 if scale is None else scale
        assert o.dtype == self.dtype and o.shape == self.q.shape and lse.shape == (self.N, self.H)
        t = 0
        for r, (c, n) in enumerate(self.lens):
            for p in range(c, c + n):
                if t in skip:
                    t += 1
                    continue
                (k, s), q = self.keys(r, p, True), self.q[t].double()
                sink = self.sink.double()
                if len(k):
                    x = q @ k.t() * scale
                    E = self.D * 2.0**-24 * abs(scale) * (q.abs() @ k.abs().t()).amax(1) + 2.0**-20 + more
                    top = torch.maximum(x.amax(1), sink)
                else:
                    x, E, top = q.new_zeros(self.H, 0), torch.zeros(self.H, device=DEV), sink
                e = torch.exp(x - top[:, None])
                l = e.sum(1) + torch.exp(sink - top)
                ref, mag = e @ k / l[:, None], e @ k.abs() / l[:, None]
                tol = u * ref.abs() + (u + 2 * E[:, None]) * mag * (1 + 2 * u) + torch.finfo(self.dtype).smallest_normal
                if self.dtype is HF and len(k):
                    codes = torch.where(s[:, None] != 0, k / s[:, None], 0.0).abs().sum(0)
                    tol = tol + 2.0**-36 * ((e * s.abs()).amax(1) / l)[:, None] * codes
                err = (o[t].double() - ref).abs()
                assert (err <= tol).all(), (r, p, float((err - tol).max()), float(err.max()))
                rl = top + torch.log(l)
                el = (lse[t].double() - rl).abs()
                assert (el <= E + 2.0**-20 * (1 + rl.abs())).all(), (r, p, float(el.max()))
                t += 1
        assert not o[t:].any()
        assert torch.equal(lse[t:], self.sink.expand(self.N - t, self.H))


def every(s, k, at):
    """All tokens but every k-th from ``at`` on, to be skipped."""
    return set(t for t in range(s.N) if t % k != at)


def same(a, b):
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 128, 256, 512, 576])
@pytest.mark.parametrize("H", [1, 16, 24, 64, 100])
def test_shapes(D, H, dtype):
    """A ragged batch of every kind of request: a first token, a decode step, chunks; full and HCA."""
    lens = [(0, 1), (37, 1), (0, 5), (200, 9), (31, 2)]
    s = Step(lens, H, D, dtype=dtype, pad=3, block=4)
    s.check(s.run())
    s = Step(lens, H, D, dtype=dtype, window=32, ratio=8, page=7, page2=5, block=7, seed=5)
    s.check(s.run())


@pytest.mark.parametrize("page,block", [(1, 1), (2, 1), (3, 3), (16, 8), (33, 11), (64, 1), (64, 64), (100, 25), (4096, 512), (96, 3)])
def test_page_and_block_sizes(page, block):
    s = Step([(150, 3), (64, 1), (0, 40)], 16, 64, window=50, ratio=4, page=page, page2=page, block=block, block2=page, pad=1)
    s.check(s.run())
    s = Step([(150, 3), (300, 1)], 16, 576, page=page, block=block)
    s.check(s.run())


@pytest.mark.parametrize("lens", [
    [(0, 1)], [(31, 1)], [(63, 1)], [(64, 1)], [(127, 2)], [(0, 200)], [(5000, 1)], [(3000, 33), (0, 1), (700, 70)],
    [(0, 0), (10, 0), (5, 1), (0, 0)], [(i * 7 % 50, 1) for i in range(300)], [(9000, 1)] + [(20, 1)] * 70,
])
@pytest.mark.parametrize("window,ratio", [(None, None), (1, None), (128, 128), (40, 3)])
def test_lengths(lens, window, ratio):
    s = Step(lens, 20, 64, window=window, ratio=ratio, block=8, pad=2)
    s.check(s.run())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,H,n", [(576, 64, 4), (576, 128, 1), (512, 16, 3), (256, 16, 2), (128, 8, 1), (64, 4, 40), (32, 8, 2)])
def test_long(D, H, n, dtype):
    """Thousands of keys: rows split over workgroups, far from each other in length."""
    s = Step([(12000, n), (3, 1), (2500, 1)], H, D, page=64, block=16, dtype=dtype)
    s.check(s.run())


def test_long_hca():
    s = Step([(40000, 2), (900, 1)], 64, 576, window=128, ratio=8, page=64, page2=64, block=64, block2=4)
    s.check(s.run())


def test_split_is_joined(monkeypatch):
    """With and without scratch: the same definition."""
    s = Step([(20000, 1), (100, 2)], 64, 576, page=64, block=16)
    s.check(s.run())
    monkeypatch.setattr(_lib, "scratch", lambda n, d: (None, 0))
    s.check(s.run())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,H,lens", [
    (576, 64, [(1000, 200), (0, 150), (77, 1)]), (512, 32, [(40, 700)]), (576, 100, [(0, 170), (333, 31)]),
    (256, 64, [(500, 900), (3, 200)]), (128, 128, [(700, 600), (0, 250)]), (128, 24, [(90, 4400)]),
])
@pytest.mark.parametrize("window,ratio", [(None, None), (60, 8)])
def test_many_rows(D, H, lens, window, ratio, dtype):
    """More row blocks than run at once; every ninth token is compared."""
    s = Step(lens, H, D, window=window, ratio=ratio, dtype=dtype, pad=3, spread=2.0, block=4)
    s.check(s.run(), skip=every(s, 9, 4))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30, None])
def test_softmax_scales(scale, dtype):
    s = Step([(90, 3), (5, 1)], 16, 128, dtype=dtype, block=2)
    s.check(s.run(softmax_scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 576])
def test_queries_of_very_different_values(D, dtype):
    """Rows with a value far above their others, rows of the least and largest values, rows of zeros."""
    s = Step([(150, 40)], 8, D, dtype=dtype, block=16)
    g = torch.Generator().manual_seed(1)
    s.q *= torch.exp2(torch.randint(-12, 4, s.q.shape, generator=g).to(DEV))
    s.q[3, :, 5] = 300.0
    s.q[4] *= 2.0**-100 if dtype is BF else 2.0**-10
    s.q[5] = 0
    s.q[6, 2] = torch.finfo(dtype).smallest_normal
    s.check(s.run())
    s.q[7] *= 2.0**100 if dtype is BF else 2.0**8
    s.check(s.run(), skip={7})


def test_scales_of_very_different_values():
    """Blocks of scales from 2^-60 to 2^30, zero and negative ones; queries that bring the scores back to some."""
    s = Step([(200, 3), (70, 1)], 16, 128, page=16, block=4)
    g = torch.Generator().manual_seed(1)
    s.sc = torch.exp2(torch.randint(-30, 3, s.sc.shape, generator=g).float()).to(DEV) * torch.where(torch.rand(s.sc.shape, generator=g) < 0.3, -1.0, 1.0).to(DEV)
    s.sc[::3, 1] = 0
    s.check(s.run())
    for power in (-60, 80):
        s = Step([(200, 3), (5000, 1)], 64, 576, page=16, block=4)
        s.sc *= 2.0**power
        s.q *= 2.0**-power
        s.check(s.run())


def test_missing_pages():
    s = Step([(200, 4), (90, 2)], 16, 64, page=16, window=100, ratio=8, page2=4, block=16, block2=2)
    s.table[0, 8] = -1
    s.table[0, 12] = s.kv.shape[0]  # past the cache
    s.table[1, 4] = -2**31
    s.table2[0, 3] = 2**31 - 1
    s.table2[1, :] = -1
    s.check(s.run())
    s.kv.view(torch.uint8)[0] = 0x7f  # what a missing page reads instead must not matter
    s.sc[0] = math.nan
    keep = [r for r in range(2) if 0 not in s.table[r].tolist()]
    if keep:
        s.check(s.run(), skip=set(range(4) if 0 not in keep else range(4, 6)))
    s.table[:] = -1  # no key at all in the first cache
    s.table2[0] = -1
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, s.sink.expand_as(lse))
    s.sink[3] = -math.inf
    o, lse = s.run()
    assert not o.any() and (lse[:, 3] == -1e30).all() and torch.equal(lse[:, :3], s.sink[:3].expand(6, 3))


def test_narrow_table():
    """Keys past the table's width are masked."""
    s = Step([(200, 2)], 16, 64, page=16)
    s.table = s.table[:, :9].contiguous()
    s.check(s.run())
    s.table = torch.empty(1, 0, dtype=torch.int32, device=DEV)
    o, lse = s.run()
    assert not o.any()
    s.kv, s.sc = torch.empty(0, 16, 64, dtype=F8, device=DEV), torch.empty(0, 16, device=DEV)
    s.table = i32([[0] * 13])
    o, lse = s.run()
    assert not o.any()


@pytest.mark.parametrize("bad", ["code 0x7f", "code 0xff", "scale nan", "scale inf", "scale -inf"])
@pytest.mark.parametrize("D,H,lens", [(64, 16, [(60, 8), (33, 3)]), (576, 64, [(60, 8), (20000, 1)]), (32, 8, [(60, 8), (9000, 2)]),
                                      (128, 64, [(60, 300), (5, 2)]), (512, 64, [(60, 8), (5, 2)]), (256, 64, [(60, 8), (5, 2)])])
def test_not_finite(bad, D, H, lens):
    """A code or scale that is not finite reaches the rows that see its key and no other, wherever the key is masked: past the end
    of the request, before the window, between the tokens of a chunk, in an unused page."""
    for dtype in (BF, HF):
        s = Step(lens, H, D, window=20, ratio=8, page=16, page2=4, dtype=dtype)
        clean = s.run()

        def spoil(page, at, dim=slice(None)):
            if bad.startswith("code"):
                s.kv.view(torch.uint8)[page, at, dim] = int(bad[5:], 16)
            else:
                s.sc[page, at] = float(bad[6:])

        used = set(s.table[s.table >= 0].tolist())
        for p in range(s.kv.shape[0]):
            if p not in used:
                spoil(p, slice(None))  # nobody's page
        for r, (c, n) in enumerate(s.lens):
            if (c + n) % 16:  # behind the request's end in its last page
                spoil(int(s.table[r, (c + n) // 16]), slice((c + n) % 16, 16))
            first = max(0, c + 1 - 20)
            if first % 16:  # before the first token's window, in its first page
                spoil(int(s.table[r, first // 16]), slice(0, first % 16))
        same(s.run(), clean)
        # position 64 of request 0: seen by the tokens at 64 .. 83
        n = min(lens[0][1], 24)
        spoil(int(s.table[0, 4]), 0, 3)
        o, lse = s.run()
        assert torch.equal(o[:4], clean[0][:4]) and torch.equal(lse[:4], clean[1][:4])
        assert o[4:n, :, 3].isnan().all()
        assert torch.equal(o[24:], clean[0][24:]) if lens[0][1] > 24 else torch.equal(o[lens[0][1]:], clean[0][lens[0][1]:])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_queries_that_are_not_finite(bad, dtype):
    """They make their own row NaN, and a row without a key stays one."""
    for D, lens in ((64, [(60, 8), (33, 3)]), (576, [(20000, 1), (70, 2)])):
        s = Step(lens, 16, D, dtype=dtype, pad=1)
        o, lse = s.run()
        s.q[0, 3, D - 1] = bad
        s.q[-1] = bad
        o2, lse2 = s.run()
        keep = torch.ones(s.N, 16, dtype=torch.bool, device=DEV)
        keep[0, 3] = False
        assert torch.equal(o2[keep], o[keep]) and torch.equal(lse2[keep], lse[keep])
        assert o2[0, 3].isnan().all() and lse2[0, 3].isnan()
        s.table[:] = -1
        o3, lse3 = s.run()
        assert not o3.any() and torch.equal(lse3, s.sink.expand_as(lse3))


def test_scores_out_of_range():
    """A score below fp32's range weighs nothing, one above it makes its row NaN."""
    s = Step([(40, 2), (9, 1)], 4, 64, page=16)
    s.q.abs_()
    s.kv.view(torch.uint8)[int(s.table[0, 0]), 3] = 0xfe  # -448
    s.sc[int(s.table[0, 0]), 3] = 2.0**120
    got = s.run()
    full = s.kv.clone()
    keys = s.keys
    def seen(r, p, scales):
        k, sc = keys(r, p, True)
        keep = ~(k < -1e30).all(1)
        return k[keep], sc[keep]

    s.keys = seen
    s.check(got)
    s.kv = full
    s.kv.view(torch.uint8)[int(s.table[0, 0]), 3] = 0x7e  # 448
    o, lse = s.run()
    assert o[:2].isnan().all() and torch.equal(o[2], got[0][2])


def test_strides():
    """q as a slice of wider rows, caches as slices of wider ones with pages apart, tables and scales as views."""
    s = Step([(100, 3), (40, 1)], 8, 64, window=30, ratio=4, page=16, page2=8, block=4)
    want = s.run()
    wide = torch.randn(s.N, 10, 3 * 64, device=DEV).to(s.dtype)
    wide[:, 1:9, 64:128] = s.q
    s.q = wide[:, 1:9, 64:128]
    big = torch.full((s.kv.shape[0], 20, 192), 0x7f, dtype=torch.uint8, device=DEV).view(F8)
    big.view(torch.uint8)[:, 2:18, 64:128] = s.kv.view(torch.uint8)
    s.kv = big[:, 2:18, 64:128]
    more = torch.full((s.sc.shape[0], 9), math.nan, device=DEV)
    more[:, 3:7] = s.sc
    s.sc = more[:, 3:7]
    t = torch.zeros(2, 50, dtype=torch.int32, device=DEV)
    t[:, 5:5 + s.table.shape[1]] = s.table
    s.table = t[:, 5:5 + s.table.shape[1]]
    s.cu, s.seq = s.cu.long(), s.seq.long()
    same(s.run(), want)
    odd = torch.randn(s.N, 8, 65, device=DEV).to(s.dtype)  # rows at odd places
    odd[..., 1:] = s.q
    s.q = odd[..., 1:]
    same(s.run(), want)


def test_far_offsets():
    """Cache rows past 2^32 bytes and 2^35, scales past 2^31."""
    s = Step([(20, 2)], 4, 64, page=16, block=16)
    want = s.run()
    store = torch.empty((9 << 30) + (1 << 20), dtype=torch.uint8, device=DEV).view(F8)
    n = s.kv.shape[0]
    far = store.as_strided((n, 16, 64), ((9 << 30) // n // 16 * 16, 64, 1))
    far.view(torch.uint8).copy_(s.kv.view(torch.uint8))
    s.kv = far
    same(s.run(), want)
    scales = torch.empty((10 << 30) // 4, device=DEV).as_strided((n, 1), ((10 << 30) // 4 // n, 1))
    scales.copy_(s.sc)
    s.sc = scales
    same(s.run(), want)


def test_lengths_that_do_not_fit():
    """Fewer entries than new tokens: those before position 0 see nothing; nothing is read out of range."""
    s = Step([(0, 4), (10, 2)], 4, 64)
    s.seq = i32([2, 12])
    o, lse = s.run()
    assert not o[:2].any() and torch.equal(lse[:2], s.sink.expand(2, 4))
    s.seq = i32([-3, 2**31 - 1])
    o, _ = s.run()
    assert not o[:4].any()
    s.cu = i32([0, 100, 3])  # past q, descending
    s.run()
    torch.cuda.synchronize()


def test_positions_near_the_largest():
    """Positions up to 2^31 - 2 under a block table that names 2^31 keys: the tile past the last key is not looked up."""
    for D, H, lens, window in ((32, 16, [(2**31 - 4, 3), (2**31 - 70, 1)], 100), (64, 64, [(2**31 - 130, 129)], 2000),
                               (576, 64, [(2**31 - 66, 2)], 1)):
        s = Step(lens, H, D, window=window, page=2**18, block=2**18)
        s.check(s.run(), skip=every(s, 97, 5) if s.N > 100 else ())


def test_no_rows():
    s = Step([(5, 1)], 4, 64)
    o, lse = paged_attn_q_fwd(s.q[:0], s.kv, s.sc, s.table, i32([0, 0]), s.seq, s.sink)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    o, lse = paged_attn_q_fwd(s.q, s.kv, s.sc, s.table[:0], i32([0]), i32([]), s.sink)
    assert not o.any() and torch.equal(lse, s.sink.expand(1, 4))


@pytest.mark.parametrize("R", [64, 65, 257, 600])
def test_many_requests(R):
    """One long request among short ones, its keys split over workgroups: each way of working out the shares."""
    s = Step([(5000, 1) if r == R // 2 else (r % 40, r % 2) for r in range(R)], 4, 64, seed=R, block=16)
    s.check(s.run())


def test_rows_in_front():
    """Rows before the first request are rows without a key, as those behind the last."""
    s = Step([(300, 3), (0, 2)], 4, 64)
    want = s.run()
    q = torch.cat([torch.full_like(s.q[:2], math.nan), s.q, torch.full_like(s.q[:1], math.nan)])
    o, lse = paged_attn_q_fwd(q, s.kv, s.sc, s.table, s.cu + 2, s.seq, s.sink)
    assert torch.equal(o[2:7], want[0]) and torch.equal(lse[2:7], want[1])
    rest = [0, 1, 7]
    assert not o[rest].any() and torch.equal(lse[rest], s.sink.expand(3, 4))


@pytest.mark.parametrize("R", [3, 70, 300])
def test_descending_rows(R):
    """Requests whose rows overlap (cu_q descends) would have more row blocks than the call has room for: none has any."""
    s = Step([(4000, 1)] * R, 64, 64)
    s.cu = i32([0, R] * (R // 2 + 1))[:R + 1]
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, s.sink.expand(R, 64))


def test_shared_pages():
    """Requests that share their pages, by equal table rows and by one row expanded."""
    s = Step([(70, 2), (70, 2), (70, 2)], 8, 128, window=50, ratio=4, block=16)
    s.table[1:] = s.table[0]
    s.table2[1:] = s.table2[0]
    s.q[2:] = s.q[:2].repeat(2, 1, 1)
    o, lse = s.run()
    assert torch.equal(o[:2], o[2:4]) and torch.equal(o[:2], o[4:]) and torch.equal(lse[:2], lse[4:])
    s.check((o, lse))
    s.table, s.table2 = s.table[:1].expand(3, -1), s.table2[:1].expand(3, -1)
    same(s.run(), (o, lse))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,H,N,keys,last", [(64, 4, 1, 1 << 17, False), (64, 4, 1, 1 << 17, True), (576, 64, 1, 1 << 20, False),
                                             (128, 64, 1600, 1 << 14, False), (256, 64, 1100, 1 << 13, False)])
@pytest.mark.parametrize("split", [True, False])
def test_many_small_weights(monkeypatch, dtype, D, H, N, keys, last, split):
    """One key far above all others, first or last: weights of 2^-25 of the largest count, however many keys share the page.  fp32
    sums of one addition a tile of 32 keys add (keys / 32) 2^-24 to the error, twice."""
    if not split:
        monkeypatch.setattr(_lib, "scratch", lambda n, d: (None, 0))
    page = 64
    low = torch.ones(page, D, dtype=torch.float64)
    low[0::2, 0], low[1::2, 0] = -1.125, -1.0  # times 16: 18 and 16 below the top
    low[1::2, 1] = -0.5
    at = page - 1 if last else 0
    one = low.clone()
    one[at] = 0
    kv = torch.stack([one, low]).to(F8).to(DEV)
    q = torch.zeros(N, H, D, dtype=dtype, device=DEV)
    q[..., 0] = 16
    table = torch.ones(1, keys // page, dtype=torch.int32, device=DEV)
    table[0, -1 if last else 0] = 0
    sink = torch.full((H,), -math.inf, device=DEV)
    o, lse = paged_attn_q_fwd(q, kv, torch.ones(2, 1, device=DEV), table, i32([0, N]), i32([keys]), sink, 1.0)
    p = torch.arange(keys - N, keys, dtype=torch.float64)
    w0 = (p == keys - 1).double() if last else torch.ones_like(p)
    even = torch.floor(p / 2) + 1 - (0 if last else 1)
    odd = torch.floor((p + 1) / 2) - (w0 if last else 0)
    we, wo = even * math.exp(-18), odd * math.exp(-16)
    l = w0 + we + wo
    ref = torch.ones(N, D, dtype=torch.float64) * ((we + wo) / l)[:, None]
    mag = ref.clone()
    ref[:, 0], mag[:, 0] = (-1.125 * we - wo) / l, (1.125 * we + wo) / l
    ref[:, 1], mag[:, 1] = (we - 0.5 * wo) / l, (we + 0.5 * wo) / l
    # (fp16: a weight of e^-18 is at 2^-15 or above where the largest is at 2^11 or above: off by half a subnormal step, 2^-25, 2^-10 of it)
    u, w, E, a = half_step(dtype), 2.0**-8 if dtype is BF else 2.0**-10, D * 2.0**-24 * 18 + 2.0**-20, keys / 32 * 2.0**-24
    err = (o.double().cpu() - ref[:, None]).abs()
    tol = u * ref.abs() + (w + 2 * E + 2 * a) * mag
    assert (err <= tol[:, None]).all(), float((err / tol[:, None]).max())
    el = (lse.double().cpu() - torch.log(l)[:, None]).abs()
    assert (el <= E + a + 2.0**-20 * (1 + torch.log(l).abs()[:, None])).all(), float(el.max())


@pytest.mark.parametrize("H", [7, 24, 40, 100])
@pytest.mark.parametrize("lens,kw", [
    ([(3000, 9), (5, 4)], {"window": 31, "ratio": 2}), ([(4000, 12)], {"window": 700}), ([(2000, 3), (900, 30)], {"window": 96, "ratio": 8}),
])
def test_row_blocks_that_begin_inside_a_token(H, lens, kw):
    """Head counts that do not divide 64, with split keys: a row block spans one token more than its rows need."""
    s = Step(lens, H, 128, block=8, **kw)
    s.check(s.run())


@pytest.mark.parametrize("D,H,lens", [(64, 8, [(40, 2), (9, 1)]), (576, 64, [(12000, 1), (100, 2)]), (32, 8, [(9000, 2)])])
def test_sinks_at_the_ends_of_their_range(D, H, lens):
    f32 = torch.finfo(torch.float32)
    s = Step(lens, H, D, pad=2)
    s.sink[:6] = torch.tensor([f32.min, -math.inf, f32.max, 2.5e38, -2.5e38, 1.5])
    empty = torch.where(s.sink == -math.inf, -1e30, s.sink)
    o, lse = want = s.run()
    assert torch.equal(lse[-2:], empty.expand(2, H)) and not o[-2:].any()
    inner = lse.clone()
    inner[-2:] = s.sink  # (check() compares rows of no request with the sinks themselves)
    s.check((o, inner))
    s.sink[0] = -math.inf  # the lowest value weighs as little beside a key
    got = s.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][:-2], want[1][:-2])
    s.sink[0], s.table[:] = f32.min, -1
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, empty.expand(s.N, H))
    s.sink[:2] = torch.tensor([math.inf, math.nan])
    o, lse = s.run()
    assert not o[:, 0].any() and (lse[:, 0] == math.inf).all() and lse[:, 1].isnan().all()


@pytest.mark.parametrize("D,H,n,low,high", [(64, 4, 6000, -130, -86), (576, 16, 9000, -128, -85), (32, 8, 300, -87, -87)])
def test_small_beside_the_sink(D, H, n, low, high):
    """Scores that begin far below the sink and rise: their weights are in fp32's range, the difference of the first one from the
    sink is not."""
    s = Step([(n, 1)], H, D, page=64, block=1)
    s.q.zero_()
    s.q[..., 0] = 1
    s.sink.zero_()
    k = torch.arange(n + 1, device=DEV)
    page = s.table[0].long()[k // 64]
    s.kv.view(torch.uint8)[page, k % 64, 0] = 0xf8  # -256
    s.sc[page, k % 64] = -(low + (high - low) * k / n) / 256
    got = s.run(softmax_scale=1.0)
    s.check(got, scale=1.0)
    assert got[0].any(-1).all()


def test_in_a_graph():
    """A captured call, replayed with other lengths, tables, codes and queries; eager work between the replays."""
    steps = [Step([(c, 1) for c in lens], 64, 576, window=128, ratio=16, page=64, page2=64, block=16, seed=k)
             for k, lens in enumerate([[3000, 10, 500], [64, 20000, 129], [0, 1, 2]])]
    wide = max(s.table.shape[1] for s in steps), max(s.table2.shape[1] for s in steps)
    pages = max(s.kv.shape[0] for s in steps), max(s.kv2.shape[0] for s in steps)

    def grown(s):
        def rows(t, n):
            return torch.cat([t.view(torch.uint8), t.new_zeros(n - t.shape[0], *t.shape[1:]).view(torch.uint8)]).view(t.dtype)

        pad = lambda t, n: torch.cat([t, t.new_full((t.shape[0], n - t.shape[1]), -1)], 1)  # noqa: E731
        s.table, s.table2 = pad(s.table, wide[0]), pad(s.table2, wide[1])
        s.kv, s.sc, s.kv2, s.sc2 = rows(s.kv, pages[0]), rows(s.sc, pages[0]), rows(s.kv2, pages[1]), rows(s.sc2, pages[1])
        return s

    steps = [grown(s) for s in steps]
    names = ("q", "kv", "sc", "table", "kv2", "sc2", "table2", "cu", "seq", "sink")
    held = Step(steps[0].lens, 64, 576, window=128, ratio=16, page=64, page2=64, block=16)
    for n in names:
        setattr(held, n, getattr(steps[0], n).clone())
    held.run()
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = held.run()
    with torch.cuda.graph(second):
        out2 = held.run()
    for i in (1, 2, 0, 1):
        for n in names:
            getattr(held, n).copy_(getattr(steps[i], n))
        graph.replay()
        second.replay()
        want = steps[i].run()
        torch.cuda.synchronize()
        same(out, want)
        same(out2, want)
        steps[i].check(out)


def test_two_streams():
    """Calls on two streams at once do not share anything."""
    steps = [Step([(3000, 2), (10, 1)], 64, 128, seed=i, page=64, block=4) for i in range(2)]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(steps[i].run())
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            same(g, want[i])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,D,page,block", [(64, 576, 64, 16), (8, 64, 8, 8), (20, 128, 6, 1)])
def test_serving_together(H, D, page, block, dtype):
    """Norm and rotation of queries and keys, plan, write in 8 bits and attention, chunk by chunk and token by token: every output
    against 64-bit arithmetic over the cache as it stands, and the cache against the keys, half an e4m3 step each."""
    R, total = 3, [150, 3, 70]
    g = torch.Generator().manual_seed(D)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    q, x, weight = [rnd(t, H, D) for t in total], [rnd(t, 1, D) for t in total], (1 + 0.1 * torch.randn(D, generator=g)).to(DEV)
    freqs, sink = rotary_freqs(32, factor=4.0), torch.randn(H, generator=g).to(DEV)
    pages = 100
    cache = torch.full((pages, page, D), 0x7f, dtype=torch.uint8, device=DEV).view(F8)  # recycled pages hold anything
    scales = torch.full((pages, page // block), math.nan, device=DEV)
    free, at = torch.randperm(pages, generator=g).to(torch.int32).to(DEV), i32([0])
    table, ctx = torch.full((R, 160 // page + 1), -1, dtype=torch.int32, device=DEV), i32([0] * R)
    done, rng = [0] * R, random.Random(D)
    while any(done[r] < total[r] for r in range(R)):
        new = [min(total[r] - done[r], rng.choice([0, 1, 1, 1, 40])) for r in range(R)]
        if not any(new):
            continue
        cut = lambda t: torch.cat([t[r][done[r]:done[r] + new[r]] for r in range(R)] + [rnd(2, *t[0].shape[1:])])  # noqa: E731
        qs, xs = cut(q), cut(x)
        plan = paged_plan(ctx, i32(new), table, free, page, len(qs), free_start=at)
        ctx, at = plan.seq_lens, plan.free_next
        turned = norm_rotary(qs, plan.positions, freqs)
        rows = norm_rotary(xs, plan.positions, freqs, weight)[:, 0]
        paged_write_q(rows, cache, scales, plan.slots)
        o, lse = paged_attn_q_fwd(turned, cache, scales, table, plan.cu, plan.seq_lens, sink)
        back = rotary(o, plan.positions, freqs, inverse=True)
        assert back.shape == o.shape
        s = Step([(done[r], new[r]) for r in range(R)], H, D, page=page, dtype=dtype, pad=2)
        s.q, s.kv, s.sc, s.table, s.sink = turned, cache, scales, table, sink
        s.check((o, lse))
        t = 0
        for r in range(R):
            for p in range(done[r], done[r] + new[r]):
                # (a block's later scales round its earlier codes again: the newest token's is one rounding)
                if p == done[r] + new[r] - 1:
                    got, sc = s.keys(r, p)[-1], scales[int(table[r, p // page]), p % page // block].double()
                    want = rows[t].double()
                    assert ((got - want).abs() <= 2.0**-4 * want.abs() + sc * 2.0**-10).all()
                t += 1
            done[r] += new[r]


@pytest.mark.parametrize("H,d,m,n_win,page,block", [(64, 576, 16, 24, 64, 16), (8, 64, 8, 20, 6, 1)])
def test_hca_serving_together(H, d, m, n_win, page, block):
    """An HCA layer over caches in 8 bits, in chunks and single tokens: rows and compressed entries quantised as they come, every output
    against 64-bit arithmetic over the caches as they stand, and each new entry against the compressor's, half an e4m3 step."""
    R, total, pages = 3, [5 * m + 3, 2, 4 * m], 60
    g = torch.Generator().manual_seed(m)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).to(DEV)  # noqa: E731
    q, x = [rnd(t, H, d) for t in total], [rnd(t, 3 * d) for t in total]
    bias, sink = torch.randn(m, d, generator=g).to(DEV), torch.randn(H, generator=g).to(DEV)
    kv, ents = (torch.full((pages, page, d), 0x7f, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2))
    sc, esc = (torch.full((pages, page // block), math.nan, device=DEV) for _ in range(2))
    streams = torch.full((pages, page, 2 * d), math.nan, dtype=BF, device=DEV)  # compressor content and gate
    free, efree = (torch.randperm(pages, generator=g).to(torch.int32).to(DEV) for _ in range(2))
    table, etable = (torch.full((R, max(total) // page + 1), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    ctx, at, eat = i32([0] * R), i32([0]), i32([0])
    done, rng = [0] * R, random.Random(m)
    while any(done[r] < total[r] for r in range(R)):
        new = [min(total[r] - done[r], rng.choice([0, 1, 1, m + 2])) for r in range(R)]
        if not any(new):
            continue
        cut = lambda t: torch.cat([t[r][done[r]:done[r] + new[r]] for r in range(R)] + [rnd(1, *t[0].shape[1:])])  # noqa: E731
        qs, xs = cut(q), cut(x)
        N = len(qs)
        tok = paged_plan(ctx, i32(new), table, free, page, N, free_start=at)
        ent = paged_plan(ctx, i32(new), etable, efree, page, N // m + R, ratio=m, free_start=eat)
        ctx, at, eat = tok.seq_lens, tok.free_next, ent.free_next
        paged_write_q(xs[:, :d], kv, sc, tok.slots)
        paged_write(xs[:, d:], streams, tok.slots)
        E = len(ent.slots)
        made = torch.zeros(1, E, d, dtype=BF, device=DEV)
        paged_compress(streams[..., :d], streams[..., d:], bias, table, ent.request, ent.positions, made,
                       torch.where(ent.slots >= 0, torch.arange(E, device=DEV), -1))
        paged_write_q(made[0], ents, esc, ent.slots)
        got = paged_attn_q_fwd(qs, kv, sc, table, tok.cu, tok.seq_lens, sink, window=n_win, kv2_cache=ents, kv2_scales=esc, block_table2=etable,
                               ratio=m)
        s = Step([(done[r], new[r]) for r in range(R)], H, d, window=n_win, ratio=m, page=page, pad=1)
        s.q, s.kv, s.sc, s.table, s.kv2, s.sc2, s.table2, s.sink = qs, kv, sc, table, ents, esc, etable, sink
        s.check(got)
        for i, slot in enumerate(ent.slots.tolist()):
            if slot >= 0:
                scale = esc.view(-1)[slot // block].double()
                want, have = made[0, i].double(), ents.view(-1, d)[slot].double() * scale
                assert ((have - want).abs() <= 2.0**-4 * want.abs() + scale * 2.0**-10).all()
        done = [done[r] + new[r] for r in range(R)]


def test_close_to_16_bits():
    """Over values that both caches hold exactly, the two attentions differ by their own roundings alone."""
    s = Step([(300, 5), (2000, 1)], 64, 576, page=64, block=16)
    s.sc = torch.exp2(torch.floor(torch.log2(s.sc)))
    kv = (s.kv.float() * s.sc.repeat_interleave(16, 1)[..., None]).to(BF)
    o, lse = s.run()
    o16, lse16 = paged_attn_fwd(s.q, kv, s.table, s.cu, s.seq, s.sink)
    assert (lse - lse16).abs().max() < 2.0**-15
    assert (o.float() - o16.float()).norm() < 2.0**-7 * o16.float().norm()


def test_refusals():
    s = Step([(20, 2)], 4, 64, ratio=4, window=9)
    args = (s.q, s.kv, s.sc, s.table, s.cu, s.seq, s.sink)
    two = {"kv2_cache": s.kv2, "kv2_scales": s.sc2, "block_table2": s.table2, "ratio": 4}
    put = lambda i, t: args[:i] + (t,) + args[i + 1:]  # noqa: E731
    paged_attn_q_fwd(*args, **two)
    for a, kw in (
            (put(1, s.kv.to(BF)), {}), (put(2, s.sc.double()), {}), (put(2, s.sc[:, :3]), {}), (put(2, s.sc[:-1]), {}),
            (put(1, torch.cat([s.kv.view(torch.uint8)] * 2, 2)[..., 8:72].view(F8)), {}), (put(3, s.table.long()), {}), (args, {"window": 0}),
            (args, {**two, "ratio": 0}), (args, {k: v for k, v in two.items() if k != "kv2_scales"}), (args, {"ratio": 4}),
            (args, {**two, "kv2_scales": s.sc2[:, :3]}), (put(4, s.cu.float()), {}),
            ((s.q[..., :33],) + args[1:], {}), (put(1, s.kv.transpose(0, 1)), {})):
        with pytest.raises((ValueError, AssertionError)):
            paged_attn_q_fwd(*a, **kw)
    for a in (put(0, s.q.float()), put(0, s.q[0]), put(6, s.sink[:3]), put(6, s.sink.cpu()), put(2, s.sc.cpu()), put(1, s.kv[..., :32])):
        with pytest.raises(AssertionError):
            paged_attn_q_fwd(*a)
