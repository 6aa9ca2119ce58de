"""GPU parity of the paged serving operators against their definitions in Python integers and 64-bit floats.

Tolerances (u = eps / 2 of the type, half a rounding step relative to the value):
* a plan and a write are exact;
* a compressed entry is one rounding of fp32 sums: u |ref| + 2^-18 sum |v| w / sum w (exponentials of arguments below 2^5
  to 2^-19 and at most 2^5 additions of 2^-24 each along a path, twice);
* attention rounds P (u of each weight) and the output: u |ref| + (u + 2 E) sum p |v| / l, where E bounds the error of a
  score, D fp32 products and sums (D 2^-24 scale |q|.|k|) and its exponential (2^-20); lse: E + 2^-20 (1 + |lse|).
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from streamindex_amd import (flash_hca_forward, flash_hca_paged_forward, paged_attn_fwd, paged_compress, paged_plan,
                             paged_write)
from streamindex_amd.compressor import token_compressor

pytestmark = pytest.mark.gpu
DEV = "cuda"
EVERY = 1 << 30


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def half_step(t):
    return torch.finfo(t).eps / 2


def make_table(spans, page, seed, width=None, spare=2):
    """Random pages for each request's entries [first, end), and their number."""
    rng = random.Random(seed)
    width = max([width or 1] + [-(-e // page) for _, e in spans])
    table = [[-1] * width for _ in spans]
    need = [(r, i) for r, (b, e) in enumerate(spans) for i in range(b // page, -(-e // page) if e > b else b // page)]
    pages = list(range(len(need) + spare))
    rng.shuffle(pages)
    for p, (r, i) in zip(pages, need):
        table[r][i] = p
    return i32(table).view(len(spans), width), len(need) + spare


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
def plan_ref(ctx, new, table, free, page, rows, ratio, start):
    table = [list(r) for r in table]
    P = len(table[0]) if table else 0
    cu, seq, slots, req, pos, nxt = [0], [], [], [], [], max(start, 0)
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        old = c // ratio
        take = min((c + n) // ratio - old, rows - cu[-1])
        have, need = min(-(-old // page), P), min(-(-(old + take) // page), P)
        for i in range(have, need):
            table[r][i] = free[nxt] if nxt < len(free) else -1
            nxt += 1
        for p in range(old, old + take):
            pg = table[r][p // page] if p // page < P else -1
            slots.append(pg * page + p % page if pg >= 0 else -1)
            req.append(r)
            pos.append(p)
        cu.append(cu[-1] + take)
        seq.append(old + take)
    rest = rows - len(req)
    return cu, seq, slots + [-1] * rest, req + [-1] * rest, pos + [-1] * rest, [nxt], table


PLANS = [
    # R, ctx, new, page, ratio, extra rows (negative: cut), free pages short by, start, width of the table cut by
    (1, 0, 1, 16, 1, 0, 0, 0, 0),
    (1, 5, 0, 16, 1, 3, 0, None, 0),
    (64, 3000, 1, 64, 1, 0, 0, 5, 0),
    (64, 3000, 1, 1, 1, 7, 0, 0, 0),
    (7, 300, 90, 16, 1, -25, 0, 0, 0),
    (300, 60, 40, 100, 1, 50, 0, 2, 0),
    (300, 200, 40, 16, 4, 9, 0, 0, 0),
    (700, 900, 300, 8, 128, 20, 0, 0, 0),
    (1500, 20, 3, 4, 1, 0, 10, 0, 0),
    (20, 100, 60, 16, 1, 0, 4, 3, 0),
    (20, 100, 60, 16, 1, 5, 0, 0, 3),
    (5, 100, 60, 16, 1, -100000, 0, 0, 0),
]


@pytest.mark.parametrize("R,ctx_hi,new_hi,page,ratio,extra,short,start,narrow", PLANS)
def test_plan(R, ctx_hi, new_hi, page, ratio, extra, short, start, narrow):
    rng = random.Random(R * 1000 + page)
    ctx = [rng.randint(0, ctx_hi) for _ in range(R)]
    new = [rng.randint(0, new_hi) if rng.random() < 0.8 else 0 for _ in range(R)]
    if R > 3:
        ctx[1], new[2] = -4, -1  # count as none
    P = max(1, max(-(-((max(c, 0) + max(n, 0)) // ratio) // page) for c, n in zip(ctx, new)) - narrow)
    pages = 0
    table = [[-1] * P for _ in range(R)]
    for r in range(R):
        for i in range(min(P, -(-(max(ctx[r], 0) // ratio) // page))):
            table[r][i] = pages
            pages += 1
    total = sum((max(c, 0) + max(n, 0)) // ratio - max(c, 0) // ratio for c, n in zip(ctx, new))
    want = sum(max(0, min(P, -(-((max(c, 0) + max(n, 0)) // ratio) // page)) - min(P, -(-(max(c, 0) // ratio) // page)))
               for c, n in zip(ctx, new))
    rows = max(0, total + extra)
    begin = start or 0
    free = list(range(pages, pages + max(0, want + begin - short)))
    rng.shuffle(free)
    dev_table = torch.full((R, P + 3), -7, dtype=torch.int32, device=DEV)  # a view: rows apart
    view = dev_table[:, :P]
    view.copy_(i32(table).view(R, P))
    plan = paged_plan(i32(ctx), torch.tensor(new, device=DEV), view, i32(free).view(-1), page, rows, ratio=ratio,
                      free_start=None if start is None else i32([start]))
    ref = plan_ref(ctx, new, table, free, page, rows, ratio, begin)
    for got, want_, name in zip([*plan, view], ref, ("cu", "seq_lens", "slots", "request", "positions", "free_next", "table")):
        assert got.tolist() == want_, name
    assert (dev_table[:, P:] == -7).all()
    assert plan.slots.dtype == torch.int64 and plan.cu.dtype == torch.int32


def test_plan_without_requests():
    plan = paged_plan(i32([]), i32([]), torch.empty(0, 3, dtype=torch.int32, device=DEV), i32([1]), 16, 5)
    assert plan.cu.tolist() == [0] and plan.slots.tolist() == [-1] * 5 and plan.free_next.tolist() == [0]


def test_plan_largest_lengths():
    """Positions near 2^31 have no page in a narrow table, and nothing overflows."""
    table = i32([[3, 4], [5, -1]])
    plan = paged_plan(i32([2**31 - 5, 15]), i32([4, 2]), table, i32([9]), 16, 6)
    assert plan.seq_lens.tolist() == [2**31 - 1, 17]
    assert plan.slots.tolist() == [-1] * 4 + [5 * 16 + 15, 9 * 16]
    assert table.tolist() == [[3, 4], [5, 9]]


# ---------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("N,width,page", [(1, 576, 64), (64, 1728, 64), (301, 100, 16), (33, 7, 5), (1000, 64, 1), (5, 1, 3)])
def test_write(dtype, N, width, page):
    g = torch.Generator().manual_seed(N + width)
    pages = N // page + 3
    raw = torch.randint(0, 256, (pages, page, width * dtype.itemsize), generator=g, dtype=torch.uint8)
    rows = torch.randint(0, 256, (N, width * dtype.itemsize), generator=g, dtype=torch.uint8)
    slots = torch.randperm(pages * page, generator=g)[:N]
    slots[1::7] = pages * page + slots[1::7]  # past the cache
    slots[::5] = -1
    want = raw.clone().view(pages * page, -1)
    ok = (slots >= 0) & (slots < pages * page)
    want[slots[ok]] = rows[ok]
    # any bits, NaN among them (copied as bytes); rows and cache inside wider buffers, at odd places
    size = dtype.itemsize
    wide = torch.zeros(pages, page + 1, (width + 3) * size, dtype=torch.uint8, device=DEV)
    inner = wide[:, :page, size:(width + 1) * size]
    inner.copy_(raw)
    src = torch.zeros(N, (width + 5) * size, dtype=torch.uint8, device=DEV)
    src[:, 2 * size:(width + 2) * size] = rows.to(DEV)
    cache = wide.view(dtype)[:, :page, 1:width + 1]
    out = paged_write(src.view(dtype)[:, 2:width + 2], cache, slots.to(DEV))
    assert out is cache
    assert torch.equal(inner.cpu().reshape(pages * page, -1), want)
    inner.zero_()
    assert not wide.any()  # nothing beside the cache
    # packed, as a whole
    packed = raw.to(DEV).view(dtype).clone()
    paged_write(rows.to(DEV).view(dtype), packed, slots.to(DEV))
    assert torch.equal(packed.view(torch.uint8).cpu().view(pages * page, -1), want)


def test_write_nothing():
    cache = torch.ones(2, 4, 8, device=DEV)
    paged_write(torch.zeros(0, 8, device=DEV), cache, torch.zeros(0, dtype=torch.int64, device=DEV))
    paged_write(torch.zeros(3, 8, device=DEV), cache, torch.tensor([-1, 8, 1 << 40], device=DEV))
    paged_write(torch.zeros(1, 8, device=DEV), torch.empty(0, 4, 8, device=DEV), torch.tensor([0], device=DEV))
    assert (cache == 1).all()


def test_write_far_offsets():
    """Row offsets past 2^32 bytes."""
    store = torch.empty((3 << 30) + 64, dtype=torch.bfloat16, device=DEV)  # 6 GiB
    cache = store.as_strided((2, 2, 8), (3 << 30, 8, 1))
    cache.zero_()
    rows = torch.arange(16, device=DEV).view(2, 8).bfloat16()
    paged_write(rows, cache, torch.tensor([3, 0], device=DEV))
    assert torch.equal(cache[1, 1], rows[0]) and torch.equal(cache[0, 0], rows[1]) and not cache[0, 1].any()


# ---------------------------------------------------------------------------
# compress
# ---------------------------------------------------------------------------
COMPRESS = [
    # C, m, overlap, page, entries of each request (first, end), page of the entries
    (576, 128, False, 64, [(0, 2), (3, 4), (5, 5)], 64),
    (576, 4, True, 16, [(0, 9), (2, 3)], 16),
    (64, 100, False, 7, [(1, 3)], 3),
    (500, 8, True, 100, [(0, 3), (7, 12), (0, 1)], 2),
    (33, 5, False, 4, [(0, 6), (9, 10)], 1),
    (8, 1, True, 3, [(0, 5), (1, 2)], 4),
    (128, 200, True, 64, [(0, 1), (1, 3)], 64),
    (576, 128, False, 64, [(0, 300), (5, 160), (3, 3)], 64),
    (500, 50, True, 16, [(0, 90), (1, 61)], 7),
    (100, 20, True, 32, [(0, 7), (4, 9)], 5),
    (72, 33, False, 10, [(0, 400)], 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C,m,overlap,page,spans,epage", COMPRESS)
def test_compress(dtype, C, m, overlap, page, spans, epage):
    g = torch.Generator().manual_seed(C + m)
    n = 2 if overlap else 1
    tok = [(max(0, b - 1) * m, e * m) for b, e in spans]
    table, pages = make_table(tok, page, 3)
    width = 2 * n * C
    x = torch.randn(pages, page, width, generator=g).to(dtype).to(DEV)
    bias = [torch.randn(m, C, generator=g).to(DEV) for _ in range(n)]
    etable, epages = make_table(spans, epage, 4)
    cache = torch.full((epages, epage, C), 7.0, dtype=dtype, device=DEV)
    req = [r for r, (b, e) in enumerate(spans) for _ in range(b, e)]
    ent = [i for b, e in spans for i in range(b, e)]
    slots = [int(etable[r, i // epage]) * epage + i % epage for r, i in zip(req, ent)]
    # one entry without a slot, one whose first page is gone, padding behind
    slots[0] = -1
    gone = len(req) - 1
    r, i = req[gone], ent[gone]
    table[r, (i * m) // page] = -1
    args = (x[..., :C], x[..., C:2 * C], bias[0], table, i32(req + [-1, -1]), i32(ent + [-1, 0]), cache,
            torch.tensor(slots + [-1, 3], device=DEV))
    kw = {"c_b": x[..., 2 * C:3 * C], "z_b": x[..., 3 * C:], "b_b": bias[1]} if overlap else {}
    assert paged_compress(*args, **kw) is cache
    want = torch.full((epages * epage, C), 7.0, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(want)
    for r, i, s in zip(req, ent, slots):
        if s < 0:
            continue
        v, z = [], []
        for blk, o in ((i - 1, 2 * C), (i, 0)) if overlap else ((i, 0),):
            for j in range(m):
                p = blk * m + j
                if blk < 0 or int(table[r, p // page]) < 0:
                    continue
                row = x[int(table[r, p // page]), p % page].double()
                v.append(row[o:o + C])
                z.append(row[o + C:o + 2 * C] + bias[1 if o else 0][j].double())
        if not v:
            want[s] = 0
            continue
        v, w = torch.stack(v), torch.softmax(torch.stack(z), 0)
        want[s] = (w * v).sum(0)
        tol[s] = half_step(dtype) * want[s].abs() + 2.0**-18 * (w * v.abs()).sum(0) + torch.finfo(dtype).smallest_normal
    err = (cache.view(-1, C).double() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())


def test_compress_is_the_token_compressor():
    """Pages in order: the whole-sequence compressor's entries."""
    C, m, S, page = 64, 4, 203, 16
    g = torch.Generator().manual_seed(1)
    x = torch.randn(208 // page, page, 4 * C, generator=g).to(DEV)
    b = [torch.randn(m, C, generator=g).to(DEV) for _ in range(2)]
    flat = x.view(1, -1, 4 * C)[:, :S]
    want = token_compressor(flat[..., :C], flat[..., C:2 * C], b[0], m, c_b=flat[..., 2 * C:3 * C], z_b=flat[..., 3 * C:],
                            b_b=b[1], overlap=True)
    n = S // m
    cache = torch.zeros(4, 16, C, device=DEV)
    paged_compress(x[..., :C], x[..., C:2 * C], b[0], torch.arange(13, device=DEV, dtype=torch.int32).view(1, -1),
                   torch.zeros(n, dtype=torch.int32, device=DEV), torch.arange(n, dtype=torch.int32, device=DEV), cache,
                   torch.arange(n, device=DEV), c_b=x[..., 2 * C:3 * C], z_b=x[..., 3 * C:], b_b=b[1])
    torch.testing.assert_close(cache.view(-1, C)[:n], want[0], rtol=2.0**-17, atol=2.0**-17)


def test_compress_values_that_are_not_finite():
    """A gate of -inf weighs nothing, one of +inf or NaN makes its channel NaN, as in a softmax."""
    x = torch.zeros(1, 4, 16, device=DEV)
    x[0, :, :8] = torch.arange(4, device=DEV)[:, None].float()
    x[0, 1:, 8] = -math.inf  # channel 0: token 0 alone
    x[0, 2, 9] = math.inf
    x[0, 3, 10] = math.nan
    cache = torch.zeros(1, 1, 8, device=DEV)
    paged_compress(x[..., :8], x[..., 8:], torch.zeros(4, 8, device=DEV), i32([[0]]), i32([0]), i32([0]), cache,
                   torch.tensor([0], device=DEV))
    out = cache.view(-1)
    assert out[0] == 0 and out[1:3].isnan().all() and (out[3:] == 1.5).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class Step:
    """A step of requests (earlier, new tokens) with random caches."""

    def __init__(self, lens, H, D, *, window=None, ratio=None, page=16, page2=16, dtype=torch.bfloat16, pad=0, seed=0,
                 spread=1.0):
        g = torch.Generator().manual_seed(seed + 17)
        self.lens, self.H, self.D, self.window, self.ratio, self.dtype = lens, H, D, window, ratio, dtype
        self.N = sum(n for _, n in lens) + pad
        self.table, pages = make_table([(max(0, c + 1 - (window or EVERY)), c + n) for c, n in lens], page, seed)
        self.kv = (torch.randn(pages, page, D, generator=g) * spread).to(dtype).to(DEV)
        self.kv2 = self.table2 = None
        if ratio:
            self.table2, pages2 = make_table([(0, (c + n) // ratio) for c, n in lens], page2, seed + 1)
            self.kv2 = (torch.randn(pages2, page2, D, generator=g) * spread).to(dtype).to(DEV)
        self.q = torch.randn(self.N, H, D, generator=g).to(dtype).to(DEV)
        self.sink = torch.randn(H, generator=g).to(DEV)
        cu = [0]
        for _, n in lens:
            cu.append(cu[-1] + n)
        self.cu, self.seq = i32(cu), i32([c + n for c, n in lens])

    def run(self, **kw):
        more = {"kv2_cache": self.kv2, "block_table2": self.table2, "ratio": self.ratio} if self.ratio else {}
        return paged_attn_fwd(self.q, self.kv, self.table, self.cu, self.seq, self.sink, window=self.window, **more, **kw)

    def keys(self, r, p):
        """Rows that the token of request r at position p sees."""
        out = []
        for cache, table, ks in ((self.kv, self.table, range(max(0, p + 1 - (self.window or EVERY)), p + 1)),
                                 (self.kv2, self.table2, range((p + 1) // self.ratio if self.ratio else 0))):
            if len(ks) == 0:
                continue
            k = torch.tensor(ks, device=DEV)
            page = cache.shape[1]
            col = k // page
            pg = torch.where(col < table.shape[1], table[r].long()[col.clamp(max=table.shape[1] - 1)], -1)
            ok = (pg >= 0) & (pg < cache.shape[0])
            out.append(cache[pg[ok], (k % page)[ok]].double())
        return torch.cat(out) if out else torch.zeros(0, self.D, dtype=torch.float64, device=DEV)

    def check(self, got, scale=None, skip=()):
        """Compares with the definition in 64 bits, token by token."""
        o, lse = got
        u, scale = half_step(self.dtype), self.D ** -0.5 if scale is None else scale
        assert o.dtype == self.dtype and o.shape == self.q.shape and lse.shape == (self.N, self.H)
        t = 0
        for r, (c, n) in enumerate(self.lens):
            for p in range(c, c + n):
                if t in skip:
                    t += 1
                    continue
                k, q = self.keys(r, p), self.q[t].double()
                x = q @ k.t() * scale
                E = self.D * 2.0**-24 * abs(scale) * (q.abs() @ k.abs().t()).amax(1) + 2.0**-20 if len(k) else torch.zeros(self.H, device=DEV)
                sink = self.sink.double()
                top = torch.maximum(x.amax(1), sink) if len(k) else sink
                w = torch.exp(x - top[:, None])
                l = w.sum(1) + torch.exp(sink - top)
                ref, mag = w @ k / l[:, None], w @ k.abs() / l[:, None]
                tol = u * ref.abs() + (u + 2 * E[:, None]) * mag * (1 + 2 * u) + torch.finfo(self.dtype).smallest_normal
                err = (o[t].double() - ref).abs()
                assert (err <= tol).all(), (r, p, float((err - tol).max()), float(err.max()))
                rl = top + torch.log(l)
                el = (lse[t].double() - rl).abs()
                assert (el <= E + 2.0**-20 * (1 + rl.abs())).all(), (r, p, float(el.max()))
                t += 1
        assert not o[t:].any()
        assert torch.equal(lse[t:], self.sink.expand(self.N - t, self.H))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 128, 256, 512, 576])
@pytest.mark.parametrize("H", [1, 16, 24, 64, 100])
def test_attn_shapes(D, H, dtype):
    """A ragged batch of every kind of request: a first token, a decode step, chunks; full and HCA."""
    lens = [(0, 1), (37, 1), (0, 5), (200, 9), (31, 2)]
    s = Step(lens, H, D, dtype=dtype, pad=3)
    s.check(s.run())
    s = Step(lens, H, D, dtype=dtype, window=32, ratio=8, page=7, page2=5, seed=5)
    s.check(s.run())


@pytest.mark.parametrize("page", [1, 2, 3, 16, 33, 64, 100, 4096])
def test_attn_page_sizes(page):
    s = Step([(150, 3), (64, 1), (0, 40)], 16, 64, window=50, ratio=4, page=page, page2=page, pad=1)
    s.check(s.run())


@pytest.mark.parametrize("lens", [
    [(0, 1)], [(31, 1)], [(32, 1)], [(127, 2)], [(0, 200)], [(5000, 1)], [(3000, 33), (0, 1), (700, 70)],
    [(0, 0), (10, 0), (5, 1), (0, 0)], [(i * 7 % 50, 1) for i in range(300)], [(9000, 1)] + [(20, 1)] * 70,
])
@pytest.mark.parametrize("window,ratio", [(None, None), (1, None), (128, 128), (40, 3)])
def test_attn_lengths(lens, window, ratio):
    s = Step(lens, 20, 64, window=window, ratio=ratio, pad=2)
    s.check(s.run())


@pytest.mark.parametrize("D,H,n", [(576, 64, 4), (576, 128, 1), (512, 16, 3), (128, 8, 1), (64, 4, 40)])
def test_attn_long(D, H, n):
    """Thousands of keys: rows split over workgroups, far from each other in length."""
    s = Step([(12000, n), (3, 1), (2500, 1)], H, D, page=64)
    s.check(s.run())


def test_attn_long_hca():
    s = Step([(70000, 1), (130000, 2), (100, 1)], 64, 576, window=128, ratio=16, page=64, page2=64)
    s.check(s.run())


def test_attn_split_is_joined(monkeypatch):
    """Without scratch a call runs unsplit: the same up to the roundings of P."""
    from streamindex_amd import _lib

    s = Step([(8000, 2)], 64, 128, page=64)
    got = s.run()
    monkeypatch.setattr(_lib, "scratch", lambda n, d: (None, 0))
    s.check(s.run())
    assert torch.equal(s.run()[0], s.run()[0])
    monkeypatch.undo()
    assert torch.equal(got[0], s.run()[0]) and torch.equal(got[1], s.run()[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attn_large_scores(dtype):
    """Maxima that rise by more than the range between two rescales."""
    s = Step([(400, 3), (1000, 1)], 16, 64, dtype=dtype, spread=0.02, page=16)
    for i in range(0, 400, 40):  # rising along the request
        p = int(s.table[0, i // 16])
        s.kv[p, i % 16] = s.q[0, 0] * (0.2 * (1 + i // 40))
    s.check(s.run())
    s.check(s.run(softmax_scale=-0.3), scale=-0.3)
    s.check(s.run(softmax_scale=0.0), scale=0.0)


def test_attn_missing_pages():
    s = Step([(200, 4), (90, 2)], 16, 64, page=16, window=100, ratio=8, page2=4)
    s.table[0, 8] = -1
    s.table[0, 12] = s.kv.shape[0]  # past the cache
    s.table[1, 4] = -2**31
    s.table2[0, 3] = 2**31 - 1
    s.table2[1, :] = -1
    s.check(s.run())
    s.table[:] = -1  # no key at all in the first cache
    s.table2[0] = -1
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, s.sink.expand_as(lse))
    s.sink[3] = -math.inf
    o, lse = s.run()
    assert not o.any() and (lse[:, 3] == -1e30).all() and torch.equal(lse[:, :3], s.sink[:3].expand(6, 3))


def test_attn_narrow_table():
    """Keys past the table's width are masked."""
    s = Step([(200, 2)], 16, 64, page=16)
    s.table = s.table[:, :9].contiguous()
    s.check(s.run())
    s.table = torch.empty(1, 0, dtype=torch.int32, device=DEV)
    o, lse = s.run()
    assert not o.any()
    s.kv = torch.empty(0, 16, 64, dtype=s.dtype, device=DEV)
    s.table = i32([[0] * 13])
    o, lse = s.run()
    assert not o.any()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 576])
def test_attn_values_that_are_not_finite(value, D):
    """They reach the rows that see their key and no other, wherever the key is masked: past the end of the request, before
    the window, between the tokens of a chunk, in an unused page."""
    s = Step([(60, 8), (33, 3)], 16, D, window=20, ratio=8, page=16, page2=4)
    clean = s.run()
    used = set(s.table[s.table >= 0].tolist())
    for p in range(s.kv.shape[0]):
        if p not in used:
            s.kv[p] = value  # nobody's page
    for r, (c, n) in enumerate(s.lens):
        for p in range((c + n) % 16, 16):  # behind the request's end in its last page
            if (c + n) % 16:
                s.kv[int(s.table[r, (c + n) // 16]), p] = value
        first = max(0, c + 1 - 20)
        for p in range(first // 16 * 16, first):  # before the first token's window, in its first page
            s.kv[int(s.table[r, p // 16]), p % 16] = value
    got = s.run()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # position 64 of request 0: seen by the tokens at 64 .. 67, rows 4 .. 7
    s.kv[int(s.table[0, 4]), 0, 3] = value
    o, lse = s.run()
    assert torch.equal(o[:4], clean[0][:4]) and torch.equal(o[8:], clean[0][8:]) and torch.equal(lse[8:], clean[1][8:])
    assert o[4:8, :, 3].isnan().all()


def test_attn_lowest_values():
    """Keys of the type's lowest value and sinks that outweigh every key."""
    s = Step([(40, 2)], 4, 64)
    s.kv[int(s.table[0, 0]), 3] = torch.finfo(torch.bfloat16).min / 2**20
    s.q.abs_()
    s.sink.copy_(torch.tensor([80.0, -80.0, -math.inf, 0.0]))
    s.check(s.run())


def test_attn_strides():
    """q as a slice of wider rows, caches as slices of wider ones with pages apart, tables as views."""
    s = Step([(100, 3), (40, 1)], 8, 64, window=30, ratio=4, page=16, page2=8)
    want = s.run()
    wide = torch.randn(s.N, 10, 3 * 64, device=DEV).to(s.dtype)
    wide[:, 1:9, 64:128] = s.q
    s.q = wide[:, 1:9, 64:128]
    big = torch.full((s.kv.shape[0], 20, 192), math.nan, dtype=s.dtype, device=DEV)
    big[:, 2:18, 64:128] = s.kv
    s.kv = big[:, 2:18, 64:128]
    t = torch.zeros(2, 50, dtype=torch.int32, device=DEV)
    t[:, 5:5 + s.table.shape[1]] = s.table
    s.table = t[:, 5:5 + s.table.shape[1]]
    s.cu, s.seq = s.cu.long(), s.seq.long()
    got = s.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.randn(s.N, 8, 65, device=DEV).to(s.dtype)  # rows at odd places
    odd[..., 1:] = s.q
    s.q = odd[..., 1:]
    assert torch.equal(s.run()[0], want[0])


def test_attn_far_offsets():
    """Cache rows past 2^32 bytes."""
    s = Step([(20, 2)], 4, 64, page=16)
    store = torch.empty((3 << 30) * 2 + 4096, dtype=s.dtype, device=DEV)
    far = store.as_strided((s.kv.shape[0], 16, 64), ((3 << 30) // 2, 64, 1))
    far.copy_(s.kv)
    want = s.run()
    s.kv = far
    got = s.run()
    assert torch.equal(got[0], want[0])


def test_attn_lengths_that_do_not_fit():
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


def test_attn_no_rows():
    s = Step([(5, 1)], 4, 64)
    o, lse = paged_attn_fwd(s.q[:0], s.kv, s.table, i32([0, 0]), s.seq, s.sink)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    o, lse = paged_attn_fwd(s.q, s.kv, s.table[:0], i32([0]), i32([]), s.sink)
    assert not o.any() and torch.equal(lse, s.sink.expand(1, 4))


@pytest.mark.parametrize("R", [64, 65, 257, 600])
def test_attn_many_requests(R):
    """One long request among short ones, its keys split over workgroups: each way of working out the shares."""
    s = Step([(5000, 1) if r == R // 2 else (r % 40, r % 2) for r in range(R)], 4, 64, seed=R)
    s.check(s.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,lens", [
    (576, 64, [(1000, 200), (0, 150), (77, 1)]), (512, 32, [(40, 700)]), (576, 100, [(0, 170), (333, 31)]),
    (256, 64, [(500, 900), (3, 200)]), (128, 128, [(700, 600), (0, 250)]), (128, 24, [(90, 4400)]),
])
@pytest.mark.parametrize("window,ratio", [(None, None), (60, 8)])
def test_attn_many_rows(D, H, lens, window, ratio, dtype):
    """More row blocks than run at once; every ninth token is compared."""
    s = Step(lens, H, D, window=window, ratio=ratio, dtype=dtype, pad=3, spread=3.0)
    t = torch.arange(s.N)
    s.check(s.run(), skip=set(t[t % 9 != 4].tolist()))


@pytest.mark.parametrize("D,n", [(576, 400), (256, 1200), (128, 1700)])
def test_attn_many_rows_missing_and_not_finite(D, n):
    """Pages that are missing and a value that is not finite, where there are more row blocks than run at once."""
    s = Step([(150, n)], 64, D, page=16)
    s.table[0, 3:7] = -1
    s.table[0, 20] = s.kv.shape[0]
    o, lse = got = s.run()
    t = torch.arange(n)
    s.check(got, skip=set(t[t % 9 != 4].tolist()))
    k = 150 + n // 2
    s.kv[s.table[0, k // 16].long(), k % 16, 5] = math.inf
    o2, lse2 = s.run()
    assert torch.equal(o2[: n // 2], o[: n // 2]) and torch.equal(lse2[: n // 2], lse[: n // 2])
    assert torch.isnan(o2[n // 2:]).any(-1).all()


def test_attn_rows_in_front():
    """Rows before the first request are rows without a key, as those behind the last."""
    s = Step([(300, 3), (0, 2)], 4, 64)
    want = s.run()
    q = torch.cat([torch.full_like(s.q[:2], math.nan), s.q, torch.full_like(s.q[:1], math.nan)])
    o, lse = paged_attn_fwd(q, s.kv, s.table, s.cu + 2, s.seq, s.sink)
    assert torch.equal(o[2:7], want[0]) and torch.equal(lse[2:7], want[1])
    rest = [0, 1, 7]
    assert not o[rest].any() and torch.equal(lse[rest], s.sink.expand(3, 4))


@pytest.mark.parametrize("R", [3, 70, 300])
def test_attn_descending_rows(R):
    """Requests whose rows overlap (cu_q descends) would have more row blocks than the call has room for: none has any."""
    s = Step([(4000, 1)] * R, 64, 64)
    s.cu = i32([0, R] * (R // 2 + 1))[:R + 1]
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, s.sink.expand(R, 64))


def test_attn_shared_pages():
    """Requests that share their pages, by equal table rows and by one row expanded; lengths as int64 and strided."""
    s = Step([(70, 2), (70, 2), (70, 2)], 8, 128, window=50, ratio=4)
    s.table[1:] = s.table[0]
    s.table2[1:] = s.table2[0]
    s.q[2:] = s.q[:2].repeat(2, 1, 1)
    o, lse = s.run()
    assert torch.equal(o[:2], o[2:4]) and torch.equal(o[:2], o[4:]) and torch.equal(lse[:2], lse[4:])
    s.check((o, lse))
    s.table, s.table2 = s.table[:1].expand(3, -1), s.table2[:1].expand(3, -1)
    s.cu, s.seq = s.cu.long(), torch.stack([s.seq.long(), s.seq.long() * 0], 1)[:, 0]
    o2, lse2 = s.run()
    assert torch.equal(o2, o) and torch.equal(lse2, lse)


def test_write_views():
    """Rows expanded, every other slot of a list, a cache that is a slice of wider rows."""
    g = torch.Generator().manual_seed(8)
    wide = torch.zeros(5, 8, 96, dtype=torch.bfloat16, device=DEV)
    row = torch.randn(1, 32, generator=g).to(torch.bfloat16).to(DEV)
    slots = torch.randperm(40, generator=g).to(DEV)
    paged_write(row.expand(20, 32), wide[..., 32:64], slots[::2])
    want = torch.zeros(40, 96, dtype=torch.bfloat16, device=DEV)
    want[slots[::2], 32:64] = row
    assert torch.equal(wide.view(40, 96), want)


def test_compress_twice_the_same_and_shared():
    """An entry given twice, to two slots, and requests that share their pages: the same bits each."""
    g = torch.Generator().manual_seed(9)
    C, m, page = 64, 8, 16
    x = torch.randn(4, page, 2 * C, generator=g).to(torch.bfloat16).to(DEV)
    bias = torch.randn(m, C, generator=g).to(DEV)
    table = i32([[2, 0, 3]]).expand(3, -1)
    cache = torch.zeros(2, 8, C, dtype=torch.bfloat16, device=DEV)
    paged_compress(x[..., :C], x[..., C:], bias, table, torch.tensor([0, 1, 2, 0], device=DEV), i32([4, 4, 4, 4]), cache,
                   torch.tensor([1, 9, 4, 14], device=DEV))
    out = cache.view(16, C)
    assert out[1].any() and all(torch.equal(out[1], out[i]) for i in (9, 4, 14))
    rest = [i for i in range(16) if i not in (1, 4, 9, 14)]
    assert not out[rest].any()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class Server:
    """An HCA layer served step by step."""

    def __init__(self, R, pages, page, epage, d, m, n_win, dtype, bias, sink, most):
        self.m, self.n_win, self.bias, self.sink, self.page, self.epage = m, n_win, bias, sink, page, epage
        self.rows = torch.full((pages, page, 3 * d), math.nan, dtype=dtype, device=DEV)
        self.ents = torch.full((pages, epage, d), math.nan, dtype=dtype, device=DEV)
        g = torch.Generator().manual_seed(5)
        self.free, self.efree = (torch.randperm(pages, generator=g).to(torch.int32).to(DEV) for _ in range(2))
        self.at, self.eat = i32([0]), i32([0])
        self.table = torch.full((R, most // page + 1), -1, dtype=torch.int32, device=DEV)
        self.etable = torch.full((R, most // m // epage + 1), -1, dtype=torch.int32, device=DEV)
        self.ctx = torch.zeros(R, dtype=torch.int32, device=DEV)

    def step(self, q, x, new):
        N, R = q.shape[0], len(self.ctx)
        tok = paged_plan(self.ctx, new, self.table, self.free, self.page, N, free_start=self.at)
        ent = paged_plan(self.ctx, new, self.etable, self.efree, self.epage, N // self.m + R, ratio=self.m, free_start=self.eat)
        self.ctx.copy_(tok.seq_lens)
        self.at.copy_(tok.free_next)
        self.eat.copy_(ent.free_next)
        return flash_hca_paged_forward(q, x, self.bias, self.sink, self.rows, self.table, tok, self.ents, self.etable, ent,
                                       n_win=self.n_win)


@pytest.mark.parametrize("H,d,m,n_win,page", [(64, 576, 128, 128, 64), (8, 64, 8, 20, 7)])
def test_serving_equals_prefill(H, d, m, n_win, page):
    """Prompts given in chunks, then decode steps in a padded batch: each token's output is flash_hca_forward's over the
    whole sequence, up to the roundings of P and of the output in both (2 u each)."""
    dtype, R = torch.bfloat16, 3
    g = torch.Generator().manual_seed(3)
    total = [3 * m + 5, m - 1, 2 * m]
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    q, x = [rnd(t, H, d) for t in total], [rnd(t, 3 * d) for t in total]
    bias, sink = torch.randn(m, d, generator=g).to(DEV), torch.randn(H, generator=g).to(DEV)
    srv = Server(R, 120, page, 4, d, m, n_win, dtype, bias, sink, max(total))
    got = [[] for _ in range(R)]
    done = [0] * R
    rng = random.Random(1)
    while any(done[r] < total[r] for r in range(R)):
        new = [min(total[r] - done[r], rng.choice([0, 1, 1, m // 2 + 3])) for r in range(R)]
        pad = rng.choice([0, 2])
        qs = torch.cat([q[r][done[r]:done[r] + new[r]] for r in range(R)] + [rnd(pad, H, d)])
        xs = torch.cat([x[r][done[r]:done[r] + new[r]] for r in range(R)] + [rnd(pad, 3 * d)])
        if len(qs) == 0:
            continue
        o, at = srv.step(qs, xs, i32(new)), 0
        for r in range(R):
            got[r].append(o[at:at + new[r]])
            at += new[r]
            done[r] += new[r]
        assert not o[at:].any()
    u = half_step(dtype)
    for r in range(R):
        kv, c, z = (t[None].contiguous() for t in x[r].split(d, 1))
        comp = token_compressor(c, z, bias, m, overlap=False)
        want = flash_hca_forward(q[r][None], kv, comp, sink, n_win=n_win, m_prime=m)[0].double()
        mag = flash_hca_forward(q[r][None], kv, comp, sink, n_win=n_win, m_prime=m).double().abs().amax()
        # both entries round the compressed rows once from fp32 sums (u more of a weight's value where they differ)
        err = (torch.cat(got[r]).double() - want).abs()
        top = max(float(kv.abs().max()), float(comp.abs().max()) if comp.numel() else 0.0)
        assert float(err.max()) <= 6 * u * top and float(err.mean()) <= u * float(mag), (float(err.max()), float(err.mean()))


def test_serving_in_a_graph():
    """A captured decode step, replayed with other lengths, tokens and pages; eager work between the replays."""
    H, d, m, n_win, page, R = 8, 64, 4, 12, 8, 4
    g = torch.Generator().manual_seed(9)
    bias, sink = torch.randn(m, d, generator=g).to(DEV), torch.randn(H, generator=g).to(DEV)
    mk = lambda: Server(R, 200, page, 4, d, m, n_win, torch.bfloat16, bias, sink, 200)  # noqa: E731
    eager, graphed = mk(), mk()
    q, x, new = (torch.zeros(R + 2, H, d, dtype=torch.bfloat16, device=DEV),
                 torch.zeros(R + 2, 3 * d, dtype=torch.bfloat16, device=DEV), i32([1] * R))
    graphed.step(q, x, new)  # warm up, then start anew
    state = mk()
    for n in ("rows", "ents", "at", "eat", "table", "etable", "ctx"):
        getattr(graphed, n).copy_(getattr(state, n))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.step(q, x, new)
    for n in ("rows", "ents", "at", "eat", "table", "etable", "ctx"):
        getattr(graphed, n).copy_(getattr(state, n))
    rng = random.Random(2)
    for i in range(25):
        counts = [rng.choice([0, 1, 1, 1, 2]) for _ in range(R)]
        while sum(counts) > R + 2:
            counts[rng.randrange(R)] = 0
        q.copy_(torch.randn(q.shape, generator=g))
        x.copy_(torch.randn(x.shape, generator=g))
        new.copy_(i32(counts))
        graph.replay()
        want = eager.step(q, x, new)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(graphed.table, eager.table) and torch.equal(graphed.ctx, eager.ctx)


def test_two_streams():
    """Calls on two streams at once do not share anything."""
    steps = [Step([(3000, 2), (10, 1)], 64, 128, seed=i, page=64) for i in range(2)]
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
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])
