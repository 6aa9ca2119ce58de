"""GPU parity of the paged serving operators at values far from the usual ones, against 64-bit floats.

Tolerances (u = eps / 2 of the type):
* a compressed entry: u |ref| + 2^-18 sum w |v| / sum w.  The gates are chosen so that gate + bias is exact in fp32; their
  differences from the maximum are then exact or off by 2^-24 of themselves, and a weight e^-d by d e^-d 2^-24 < 2^-25 and an
  exponential's 2^-22.  The rest is fp32 sums, at most 2^5 additions along a path, twice.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from streamindex_amd import _lib, flash_hca_paged_forward, paged_attn_fwd, paged_compress, paged_plan

from tests.test_gpu_paged import Server, Step

pytestmark = pytest.mark.gpu
DEV = "cuda"


def half_step(t):
    return torch.finfo(t).eps / 2


# ---------------------------------------------------------------------------
# compress
# ---------------------------------------------------------------------------
def gate_masks(E, n):
    """Tokens ``[E, n]`` to mask: some of an entry's first, all, all but one, every other one, every fourth kept."""
    j, e = torch.arange(n), torch.arange(E)[:, None] % 7
    kinds = [j < n // 2, j < 4, j >= 0, j < n - 1, j % 2 == 0, j % 4 != 3, j >= 1]
    return torch.stack([torch.where(e[:, 0] == i, 1, 0)[:, None] * k[None] for i, k in enumerate(kinds)]).sum(0).bool()


def check_gates(dtype, C, m, overlap, E, make):
    """``make(z [E, tokens, C]) -> z``: the gates of each entry's tokens, the block before first, before the bias."""
    g = torch.Generator().manual_seed(m + E)
    page, epage, k = 16, 8, 2 if overlap else 1
    S = E * m
    pages = -(-S // page)
    x = torch.zeros(pages * page, 2 * k * C, dtype=dtype)
    bias = [(torch.randn(m, C, generator=g) * 64).round() / 64 for _ in range(k)]
    for s in range(k):  # content and gate of stream a, then of b
        x[:S, 2 * s * C:(2 * s + 1) * C] = torch.randn(S, C, generator=g).to(dtype)
        z = make((torch.randn(E, m, C, generator=g) * 64).round() / 64)
        x[:S, (2 * s + 1) * C:(2 * s + 2) * C] = z.reshape(S, C).to(dtype)
    perm = torch.randperm(pages, generator=g)
    store = torch.empty(pages, page, 2 * k * C, dtype=dtype)
    store[perm] = x.view(pages, page, -1)
    store, x, bias = store.to(DEV), x.to(DEV), [b.to(DEV) for b in bias]
    cache = torch.zeros(-(-E // epage), epage, C, dtype=dtype, device=DEV)
    ent = torch.arange(E, device=DEV)
    more = {"c_b": store[..., 2 * C:3 * C], "z_b": store[..., 3 * C:], "b_b": bias[1]} if overlap else {}
    paged_compress(store[..., :C], store[..., C:2 * C], bias[0], perm.to(torch.int32).to(DEV).view(1, -1),
                   torch.zeros(E, dtype=torch.int32, device=DEV), ent.to(torch.int32), cache, ent, **more)
    v, z = x[:S, :C].view(E, m, C).double(), x[:S, C:2 * C].view(E, m, C).double() + bias[0].double()
    if overlap:
        vb, zb = x[:S, 2 * C:3 * C].view(E, m, C).double(), x[:S, 3 * C:].view(E, m, C).double() + bias[1].double()
        v = torch.cat([torch.cat([vb[:1] * 0, vb[:-1]]), v], 1)
        z = torch.cat([torch.cat([torch.full_like(zb[:1], -math.inf), zb[:-1]]), z], 1)
    w = torch.softmax(z, 1)
    want, mag = (w * v).sum(1), (w * v.abs()).sum(1)
    err = (cache.view(-1, C)[:E].double() - want).abs()
    tol = half_step(dtype) * want.abs() + 2.0**-18 * mag + torch.finfo(dtype).smallest_normal
    ok = (err <= tol) | (want.isnan() & err.isnan())  # (every gate -inf: NaN, as a softmax's)
    assert ok.all(), (int((~ok).sum()), float((err - tol).nan_to_num(nan=math.inf).max()))
    return want


# few tokens an entry; some; many of few entries; many of many entries
GATES = [(72, 8, False, 40), (33, 4, True, 50), (100, 50, False, 20), (64, 16, True, 30), (576, 128, False, 30), (128, 200, True, 9),
         (576, 64, False, 600), (500, 100, False, 700)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C,m,overlap,E", GATES)
@pytest.mark.parametrize("value", ["lowest", "lowest and -inf"])
def test_compress_masked_gates(dtype, C, m, overlap, E, value):
    """Gates masked with the type's lowest value weigh nothing beside others, and all the same where an entry has no others."""
    masked = gate_masks(E, m)[..., None].expand(E, m, C)

    def make(z):
        z = torch.where(masked, torch.finfo(dtype).min, z)
        if value != "lowest":
            z[:, ::3] = -math.inf
        return z

    want = check_gates(dtype, C, m, overlap, E, make)
    assert not want.isnan().any() or value != "lowest"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C,m,overlap,E", GATES)
@pytest.mark.parametrize("offset", [32, -1000, 10000])
def test_compress_gates_far_from_zero(dtype, C, m, overlap, E, offset):
    """A common offset changes nothing but what the type can hold of the gates."""
    check_gates(dtype, C, m, overlap, E, lambda z: z + offset)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("D,H,lens,window", [
    (32, 16, [(2**31 - 4, 3), (2**31 - 40, 1), (2**31 - 2**18 - 2, 5)], 100), (32, 1, [(2**31 - 2, 1), (2**31 - 33, 1)], 1),
    (64, 64, [(2**31 - 130, 129)], 2000), (128, 64, [(2**31 - 1601, 1600)], 60),
])
def test_attn_positions_near_the_largest(D, H, lens, window):
    """Positions up to 2^31 - 2 under a block table that names 2^31 keys: the tile past the last key is not looked up."""
    s = Step(lens, H, D, window=window, page=2**18)
    t = torch.arange(s.N)
    s.check(s.run(), skip=set(t[(t % 97 != 5) & (s.N > 200)].tolist()))


class Lowest(Step):
    """Keys of the type's lowest value, at the positions ``at`` of each request and the entries ``at2``, and queries whose fp32
    scores with them are -inf: they weigh nothing."""

    def __init__(self, *args, at=(), at2=(), **kw):
        super().__init__(*args, **kw)
        self.q.abs_()
        lowest = torch.finfo(self.dtype).min
        for r, (c, n) in enumerate(self.lens):
            self.lower(self.kv, self.table[r], at, c + n, lowest)
            if self.ratio:
                self.lower(self.kv2, self.table2[r], at2, (c + n) // self.ratio, lowest)

    @staticmethod
    def lower(cache, pages, at, end, lowest):
        for p in {p % end for p in at} if end else ():
            page = int(pages[p // cache.shape[1]])
            if page >= 0:
                cache[page, p % cache.shape[1]] = lowest

    def keys(self, r, p):
        k = super().keys(r, p)
        return k[~(k == torch.finfo(self.dtype).min).all(1)]


# positions: whole tiles, the tile that the chunk's rows see in part, the window's edge (counted from the end)
@pytest.mark.parametrize("D,H,lens,kw", [
    (64, 16, [(40, 9), (3, 1), (70, 2)], {}), (576, 64, [(40, 9), (100, 3)], {"window": 20, "ratio": 4, "page2": 8}),
    (128, 24, [(9000, 2), (300, 1)], {}), (32, 1, [(200, 70)], {"window": 33}), (256, 64, [(90, 5)], {"ratio": 2}),
    (128, 64, [(150, 1600)], {"window": 100}), (512, 64, [(150, 300)], {}), (576, 64, [(100, 300)], {"window": 40, "ratio": 8}),
])
def test_attn_keys_of_the_lowest_value(D, H, lens, kw):
    """A finite key whose score leaves fp32 downwards weighs nothing, in tiles that every row sees whole and in others."""
    s = Lowest(lens, H, D, at=(2, 33, -1, -4, -15, -19, -21, -36), at2=(0, 3, -1, -2), **kw)
    t = torch.arange(s.N)
    s.check(s.run(), skip=set(t[(t % 11 != 5) & (s.N > 200)].tolist()))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,H,lens", [(64, 16, [(60, 8), (33, 3)]), (576, 64, [(20000, 1), (70, 2)]), (128, 8, [(9000, 2)])])
def test_attn_unused_rows_not_finite(value, D, H, lens):
    """Values behind the last row and the last entry in their pages, in calls of one launch and where keys are split: nobody's."""
    for kw in ({"window": 20, "ratio": 8}, {}):
        s = Step(lens, H, D, page=48, page2=48, **kw)
        want = s.run()
        for cache, table, ends in ((s.kv, s.table, [c + n for c, n in lens]),
                                   *([(s.kv2, s.table2, [(c + n) // 8 for c, n in lens])] if kw else [])):
            for r, end in enumerate(ends):
                if end % 48:
                    cache[int(table[r, end // 48]), end % 48:] = value
        got = s.run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,H,n", [(64, 16, 8), (576, 64, 300), (128, 64, 1700)])
def test_attn_entry_not_finite(value, D, H, n):
    """An entry that is not finite reaches the tokens from its last one on, whose earlier ones share its tile."""
    s = Step([(60, n)], H, D, window=20, ratio=8)
    want = s.run()
    e = (60 + n // 2) // 8
    s.kv2[int(s.table2[0, e // 16]), e % 16, 7] = value
    o, lse = s.run()
    first = 8 * (e + 1) - 1 - 60
    assert torch.equal(o[:first], want[0][:first]) and torch.equal(lse[:first], want[1][:first])
    assert o[first:, :, 7].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,N,keys,last", [
    (64, 4, 1, 1 << 17, False), (64, 4, 1, 1 << 17, True), (576, 64, 1, 1 << 20, False), (128, 16, 3, 1 << 18, True),
    (128, 64, 1600, 1 << 14, False), (256, 64, 1100, 1 << 13, False), (576, 64, 300, 1 << 15, False),
])
@pytest.mark.parametrize("split", [True, False])
def test_attn_many_small_weights(monkeypatch, dtype, D, H, N, keys, last, split):
    """One key far above all others, first or last: weights of 2^-25 of the largest count, however many keys share the page.

    u |ref| + (u + 2 E + 2 a) sum p |v| / l: P keeps u of each of these weights, E as for any scores, and a bounds fp32 sums of
    one addition a tile of 32 keys, (keys / 32) 2^-24."""
    if not split:
        monkeypatch.setattr(_lib, "scratch", lambda n, d: (None, 0))
    page = 64
    low = torch.ones(page, D, dtype=torch.float64)
    low[0::2, 0], low[1::2, 0] = -1.0625, -1.0  # times 16: 17 and 16 below the top
    low[1::2, 1] = -0.5
    top = torch.zeros(1, D, dtype=torch.float64)
    at = page - 1 if last else 0
    one = torch.cat([low[:at], top, low[at + 1:]])
    kv = torch.stack([one, low]).to(dtype).to(DEV)
    q = torch.zeros(N, H, D, dtype=dtype, device=DEV)
    q[..., 0] = 16
    table = torch.ones(1, keys // page, dtype=torch.int32, device=DEV)
    table[0, -1 if last else 0] = 0
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    sink = torch.full((H,), -math.inf, device=DEV)
    o, lse = paged_attn_fwd(q, kv, table, i32([0, N]), i32([keys]), sink, 1.0)
    p = torch.arange(keys - N, keys, dtype=torch.float64)
    # the top is every token's where it is first, the last token's alone where it is last
    w0 = (p == keys - 1).double() if last else torch.ones_like(p)
    even = torch.floor(p / 2) + 1 - (0 if last else 1)  # keys at even and odd places that the token at p sees, without the top
    odd = torch.floor((p + 1) / 2) - (w0 if last else 0)
    we, wo = even * math.exp(-17), odd * math.exp(-16)
    l = w0 + we + wo
    ref = torch.ones(N, D, dtype=torch.float64) * ((we + wo) / l)[:, None]
    mag = ref.clone()
    ref[:, 0], mag[:, 0] = (-1.0625 * we - wo) / l, (1.0625 * we + wo) / l
    ref[:, 1], mag[:, 1] = (we - 0.5 * wo) / l, (we + 0.5 * wo) / l
    u, E, a = half_step(dtype), D * 2.0**-24 * 17 + 2.0**-20, keys / 32 * 2.0**-24
    err = (o.double().cpu() - ref[:, None]).abs()
    tol = u * ref.abs() + (u + 2 * E + 2 * a) * mag
    assert (err <= tol[:, None]).all(), float((err / tol[:, None]).max())
    el = (lse.double().cpu() - torch.log(l)[:, None]).abs()
    assert (el <= E + a + 2.0**-20 * (1 + torch.log(l).abs()[:, None])).all(), float(el.max())


@pytest.mark.parametrize("H", [7, 24, 40, 100])
@pytest.mark.parametrize("lens,kw", [
    ([(3000, 9), (5, 4)], {"window": 31, "ratio": 2}), ([(4000, 12)], {"window": 700}), ([(2000, 3), (900, 30)], {"window": 96, "ratio": 8}),
])
def test_attn_row_blocks_that_begin_inside_a_token(H, lens, kw):
    """Head counts that do not divide 64, with split keys: a row block spans one token more than its rows need."""
    s = Step(lens, H, 128, **kw)
    s.check(s.run())


@pytest.mark.parametrize("D,H,lens", [(64, 8, [(40, 2), (9, 1)]), (576, 64, [(12000, 1), (100, 2)]), (128, 64, [(300, 1600)]), (32, 8, [(9000, 2)])])
def test_attn_sinks_at_the_ends_of_their_range(D, H, lens):
    """Sinks of fp32's lowest and largest values and infinite ones, for rows with keys, without any (no page) and of no request."""
    f32 = torch.finfo(torch.float32)
    s = Step(lens, H, D, pad=2)
    s.sink[:6] = torch.tensor([f32.min, -math.inf, f32.max, 2.5e38, -2.5e38, 1.5])
    t = torch.arange(s.N)
    skip = set(t[(t % 97 != 5) & (s.N > 200) & (t < s.N - 2)].tolist())
    empty = torch.where(s.sink == -math.inf, -1e30, s.sink)

    def check(o, lse):
        assert torch.equal(lse[-2:], empty.expand(2, H)) and not o[-2:].any()
        inner = lse.clone()
        inner[-2:] = s.sink  # (check() compares rows of no request with the sinks themselves)
        s.check((o, inner), skip=skip)

    check(*s.run())
    want = s.run()
    s.sink[0] = -math.inf  # the lowest value weighs as little beside a key
    same = s.run()
    assert torch.equal(same[0], want[0]) and torch.equal(same[1][:-2], want[1][:-2])
    s.sink[0], s.table[:] = f32.min, -1
    o, lse = s.run()
    assert not o.any() and torch.equal(lse, empty.expand(s.N, H))
    s.sink[:2] = torch.tensor([math.inf, math.nan])
    o, lse = s.run()
    assert not o[:, 0].any() and (lse[:, 0] == math.inf).all() and lse[:, 1].isnan().all()


# ---------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------
def test_refused_step_writes_nothing():
    """Each argument that the layer's last operator would refuse is refused before the first one writes."""
    d, H, m, N = 64, 4, 4, 6
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    bf, f32 = torch.bfloat16, torch.float32
    ones = lambda *s, t=bf: torch.ones(s, dtype=t, device=DEV)  # noqa: E731

    def args(**kw):
        table, etable = i32([[-1, -1], [-1, -1]]), i32([[-1], [-1]])
        tok = paged_plan(i32([0, 0]), i32([4, 2]), table, i32([0, 1, 2]), 4, N)
        ent = paged_plan(i32([0, 0]), i32([4, 2]), etable, i32([0, 1]), 4, 3, ratio=m)
        a = dict(q=ones(N, H, d), rows=ones(N, 3 * d), bias=ones(m, d, t=f32), attn_sink=ones(H, t=f32),
                 row_cache=ones(3, 4, 3 * d) * 0, block_table=table, tokens=tok, entry_cache=ones(2, 4, d) * 0,
                 entry_table=etable, entries=ent, n_win=3)
        a.update(kw)
        return a

    good = args()
    assert flash_hca_paged_forward(**good).any() and good["row_cache"].any() and good["entry_cache"].any()
    odd = torch.zeros(3, 4, 3 * d + 4, dtype=bf, device=DEV)[..., :3 * d]
    for kw in ({"n_win": 0}, {"q": ones(N, H, d, t=f32)}, {"q": ones(N + 1, H, d)}, {"q": ones(N, H, 96)}, {"attn_sink": ones(H + 1, t=f32)},
               {"attn_sink": ones(H)}, {"entry_cache": ones(2, 4, d + 8) * 0}, {"entry_cache": ones(2, 4, d, t=torch.float16) * 0},
               {"entry_table": i32([[0]])}, {"row_cache": odd}, {"row_cache": ones(3, 4, 2 * d) * 0}):
        a = args(**kw)
        with pytest.raises(ValueError):
            flash_hca_paged_forward(**a)
        assert not a["row_cache"].any() and not a["entry_cache"].any(), kw


@pytest.mark.parametrize("H,d,m,n_win,page,dtype", [
    (64, 576, 16, 24, 64, torch.bfloat16), (8, 64, 8, 20, 7, torch.bfloat16), (24, 128, 5, 1, 3, torch.float16),
])
def test_serving_steps_against_the_definition(H, d, m, n_win, page, dtype):
    """Chunks and decode steps of three requests: every entry and every output against 64-bit arithmetic over the tokens' own
    rows, with the tolerances of an entry and of the attention (whose keys are the entries as they are cached)."""
    R, total = 3, [5 * m + 3, 2, 4 * m]
    g = torch.Generator().manual_seed(m)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    bias, sink = torch.randn(m, d, generator=g).to(DEV), torch.randn(H, generator=g).to(DEV)
    srv = Server(R, 150, page, 4, d, m, n_win, dtype, bias, sink, max(total))
    q, x = [rnd(t, H, d) for t in total], [rnd(t, 3 * d) for t in total]
    done, rng, u, scale = [0] * R, random.Random(m), half_step(dtype), d ** -0.5
    while any(done[r] < total[r] for r in range(R)):
        new = [min(total[r] - done[r], rng.choice([0, 1, 1, m + 2])) for r in range(R)]
        if not any(new):
            continue
        o = srv.step(torch.cat([q[r][done[r]:done[r] + new[r]] for r in range(R)] + [rnd(1, H, d)]),
                     torch.cat([x[r][done[r]:done[r] + new[r]] for r in range(R)] + [rnd(1, 3 * d)]),
                     torch.tensor(new, dtype=torch.int32, device=DEV))
        t = 0
        for r in range(R):
            rows = x[r].double()
            ends = (done[r] + new[r]) // m
            ents = [srv.ents[int(srv.etable[r, i // 4]), i % 4].double() for i in range(ends)]
            for i in range(done[r] // m, ends):
                v, z = rows[i * m:(i + 1) * m, d:2 * d], rows[i * m:(i + 1) * m, 2 * d:] + bias.double()
                w = torch.softmax(z, 0)
                tol = u * (w * v).sum(0).abs() + 2.0**-18 * (w * v.abs()).sum(0) + torch.finfo(dtype).smallest_normal
                assert ((ents[i] - (w * v).sum(0)).abs() <= tol).all()
            for p in range(done[r], done[r] + new[r]):
                k = torch.cat([rows[max(0, p + 1 - n_win):p + 1, :d], *(e[None] for e in ents[:(p + 1) // m])])
                qd = q[r][p].double()
                s = qd @ k.t() * scale
                E = d * 2.0**-24 * scale * (qd.abs() @ k.abs().t()).amax(1) + 2.0**-20
                w = torch.softmax(torch.cat([s, sink.double()[:, None]], 1), 1)[:, :-1]
                ref, mag = w @ k, w @ k.abs()
                tol = u * ref.abs() + (u + 2 * E[:, None]) * mag * (1 + 2 * u) + torch.finfo(dtype).smallest_normal
                assert ((o[t].double() - ref).abs() <= tol).all(), (r, p)
                t += 1
            done[r] += new[r]
        assert not o[t:].any()


def scored(s, score):
    """Queries of one and keys whose scores are ``score(r, k)``, for entries ``score(r, -1 - i)``, with sinks of zero."""
    s.q.zero_()
    s.q[..., 0] = 1
    s.sink.zero_()
    for r, (c, n) in enumerate(s.lens):
        for cache, table, at in ((s.kv, s.table, range(c + n)), (s.kv2, s.table2, range((c + n) // s.ratio if s.ratio else 0))):
            if len(at):
                k = torch.tensor(at, device=DEV)
                page = table[r, k // cache.shape[1]].long()
                x = torch.tensor([score(r, i if cache is s.kv else -1 - i) for i in at], device=DEV, dtype=s.dtype)
                cache[page[page >= 0], (k % cache.shape[1])[page >= 0], 0] = x[page >= 0]
    return s


@pytest.mark.parametrize("D,H,lens,kw,low,high", [
    (64, 4, [(40, 3), (9, 1)], {"window": 1, "ratio": 8}, -90, -47), (576, 64, [(100, 300)], {"window": 2, "ratio": 4}, -90, -47),
    (128, 64, [(100, 1600)], {"window": 1, "ratio": 16}, -90, -47), (512, 16, [(70, 2)], {"window": 3, "ratio": 4}, -89, -45.5),
    (256, 8, [(50, 1)], {"window": 1, "ratio": 8}, -94, -86.5), (32, 8, [(20, 1)], {"window": 1, "ratio": 8}, -87, -87),
    (64, 4, [(6000, 1)], {}, -130, -86), (576, 16, [(9000, 2)], {}, -128, -85),
])
def test_attn_small_beside_the_sink(D, H, lens, kw, low, high):
    """Scores that begin far below the sink and rise by less than moves the reference: their weights are in fp32's range, whole
    and joined, the difference of the first one from the sink is not."""
    s = Step(lens, H, D, **kw)
    end = lens[0][0] + lens[0][1]
    scored(s, (lambda r, k: low if k >= 0 else high) if kw else lambda r, k: low + (high - low) * k / end)
    t = torch.arange(s.N)
    o, lse = s.run(softmax_scale=1.0)
    s.check((o, lse), scale=1.0, skip=set(t[(t % 17 != 5) & (s.N > 200)].tolist()))
    assert o.any(-1).all()


@pytest.mark.parametrize("D,H,lens", [(64, 16, [(70, 3), (0, 2)]), (576, 64, [(5000, 1)]), (128, 64, [(40, 1600)])])
@pytest.mark.parametrize("power", [-80, 90])
def test_attn_small_and_large_values(D, H, lens, power):
    """bf16 rows of about 2^power, with queries that bring their scores back to some."""
    s = Step(lens, H, D)
    s.kv *= 2.0**power
    s.q *= 2.0**-power
    t = torch.arange(s.N)
    s.check(s.run(), skip=set(t[(t % 17 != 5) & (s.N > 200)].tolist()))
