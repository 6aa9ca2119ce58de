"""Serving operators over a paged cache: the calls a user makes of them, their plain forms and what a pass cannot do without.

A serving step of an HCA layer takes a ragged batch of new tokens (a decode step has one for each request, a chunk of a
prompt has many) through four operators:

  plan      paged_plan: from the requests' lengths the block tables, the cache row of each new token, its request and position
  write     paged_write: the new tokens' rows into their pages
  compress  paged_compress: the compressed entries that the new tokens complete, pooled from the pages
  attn      paged_attn_fwd: attention of the new tokens over a paged cache; with a window and a second cache of compressed
            entries (HCA), or over every earlier token

A page holds ``page`` consecutive tokens (or entries) of one request; a block table row names a request's pages in order, -1
where there is none.  Sizes are those of this package's layers (64 heads, D = 576, a window of 128, one entry per 128 tokens)
and ranges around them.
"""

import math
import random

import torch

own = False  # False: the plain forms; True: the package's operators

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EVERY = 1 << 30  # a window that holds every earlier token


# ---------------------------------------------------------------------------
# The cases.  R requests with ctx_lo .. ctx_hi earlier tokens and new_lo .. new_hi new ones; `mix` seeds these lengths.
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 requests: the smallest call, a launch's latency
        {"name": "plan_decode_64", "op": "plan", "R": 64, "ctx_lo": 1, "ctx_hi": 131072, "new_lo": 1, "new_hi": 1, "page": 64, "ratio": 1,
         "pad": 0, "mix": 1},
        # a batch of prompts in small pages, the token buffer longer than the tokens
        {"name": "plan_prompts", "op": "plan", "R": 301, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 0, "new_hi": 513, "page": 16, "ratio": 1,
         "pad": 1001, "mix": 2},
        # the rows of one decode step: key/value, content and gate of a token side by side
        {"name": "write_decode_64", "op": "write", "R": 64, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 1, "new_hi": 1, "page": 64, "D": 1728,
         "pad": 0, "dtype": "bf16", "mix": 3},
        # the rows of several chunks, padded
        {"name": "write_chunks", "op": "write", "R": 17, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 200, "new_hi": 2000, "page": 64, "D": 576,
         "pad": 300, "dtype": "bf16", "mix": 4},
        # a decode step of 256 requests, of which few complete an entry
        {"name": "compress_decode_256", "op": "compress", "R": 256, "ctx_lo": 128, "ctx_hi": 4096, "new_lo": 1, "new_hi": 1, "page": 64,
         "C": 576, "ratio": 128, "overlap": False, "dtype": "bf16", "mix": 5},
        # the entries of a 64K-token prompt given as four ragged chunks
        {"name": "compress_64k", "op": "compress", "R": 4, "ctx_lo": 1, "ctx_hi": 2048, "new_lo": 15000, "new_hi": 17000, "page": 64,
         "C": 576, "ratio": 128, "overlap": False, "dtype": "bf16", "mix": 6},
        # one new token of one request: latency
        {"name": "hca_decode_1", "op": "attn", "R": 1, "ctx_lo": 4096, "ctx_hi": 4096, "new_lo": 1, "new_hi": 1, "H": 64, "D": 576,
         "window": 128, "ratio": 128, "page": 64, "pad": 0, "dtype": "bf16", "mix": 7},
        # one decode step of 64 requests of very different lengths
        {"name": "hca_decode_64", "op": "attn", "R": 64, "ctx_lo": 2000, "ctx_hi": 131072, "new_lo": 1, "new_hi": 1, "H": 64, "D": 576,
         "window": 128, "ratio": 128, "page": 64, "pad": 0, "dtype": "bf16", "mix": 8},
        # one decode step of four requests of a million tokens
        {"name": "hca_decode_1m", "op": "attn", "R": 4, "ctx_lo": 1000000, "ctx_hi": 1048575, "new_lo": 1, "new_hi": 1, "H": 64, "D": 576,
         "window": 128, "ratio": 128, "page": 64, "pad": 0, "dtype": "bf16", "mix": 9},
        # decode over every earlier token, few heads, small pages, fp16
        {"name": "full_decode_32", "op": "attn", "R": 32, "ctx_lo": 1000, "ctx_hi": 16384, "new_lo": 1, "new_hi": 1, "H": 16, "D": 128,
         "window": 0, "ratio": 0, "page": 16, "pad": 0, "dtype": "f16", "mix": 10},
        # ragged chunks of four long prompts
        {"name": "hca_chunks", "op": "attn", "R": 4, "ctx_lo": 8000, "ctx_hi": 65536, "new_lo": 700, "new_hi": 2048, "H": 64, "D": 576,
         "window": 128, "ratio": 128, "page": 64, "pad": 100, "dtype": "bf16", "mix": 11},
        # a chunk of a prompt over every earlier token
        {"name": "full_chunk", "op": "attn", "R": 1, "ctx_lo": 7000, "ctx_hi": 8192, "new_lo": 1024, "new_hi": 1024, "H": 32, "D": 256,
         "window": 0, "ratio": 0, "page": 64, "pad": 0, "dtype": "bf16", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above.  No drawn case costs more than the largest listed one."""
    op = rng.choice(["plan", "write", "compress", "attn", "attn", "attn"])
    mix = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 100, 128])
    if op == "plan":
        R = _log_int(rng, 1, 1024)
        ratio = rng.choice([1, 1, 4, 128])
        return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": _log_int(rng, 100, 32768), "new_lo": 0, "new_hi": _log_int(rng, 1, max(1, 65536 // R)),
                "page": page, "ratio": ratio, "pad": rng.choice([0, 7, 200]), "mix": mix}
    if op == "write":
        R = _log_int(rng, 1, 256)
        return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 1, "new_hi": _log_int(rng, 1, max(1, 16384 // R)), "page": page,
                "D": rng.choice([64, 128, 500, 576, 1152, 1728]), "pad": rng.choice([0, 5, 129]), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "mix": mix}
    if op == "compress":
        R = _log_int(rng, 1, 128)
        overlap = rng.random() < 0.4
        return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 1, "new_hi": _log_int(rng, 1, max(1, 40000 // R)), "page": page,
                "C": rng.choice([64, 128, 500, 576]), "ratio": rng.choice([4, 8]) if overlap else rng.choice([32, 100, 128]),
                "overlap": overlap, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "mix": mix}
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if rng.random() < 0.5:  # HCA
        H, D = rng.choice([16, 64, 64, 128]), rng.choice([512, 576])
        if rng.random() < 0.6:  # a decode step, a few tokens each at times
            ctx = _log_int(rng, 500, 500000)
            return {"op": op, "R": _log_int(rng, 1, 100), "ctx_lo": max(1, ctx // 20), "ctx_hi": ctx, "new_lo": 1, "new_hi": rng.choice([1, 1, 4]),
                    "H": H, "D": D, "window": 128, "ratio": 128, "page": page, "pad": rng.choice([0, 3]), "dtype": dtype, "mix": mix}
        R = _log_int(rng, 1, 8)
        new = _log_int(rng, 16, 3000 // R)
        return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": _log_int(rng, 100, 60000), "new_lo": max(1, new // 2), "new_hi": new, "H": rng.choice([16, 64]),
                "D": D, "window": 128, "ratio": 128, "page": page, "pad": rng.choice([0, 31]), "dtype": dtype, "mix": mix}
    H, D = rng.choice([1, 8, 16, 24, 64]), rng.choice([32, 64, 128, 256, 576])
    window = rng.choice([0, 0, 0, 512])
    if rng.random() < 0.6:
        ctx = _log_int(rng, 100, 16384)
        return {"op": op, "R": _log_int(rng, 1, 64), "ctx_lo": max(1, ctx // 8), "ctx_hi": ctx, "new_lo": 1, "new_hi": rng.choice([1, 1, 3]), "H": H,
                "D": D, "window": window, "ratio": 0, "page": page, "pad": rng.choice([0, 3]), "dtype": dtype, "mix": mix}
    R = _log_int(rng, 1, 4)
    new = _log_int(rng, 16, 1024 // R)
    return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": _log_int(rng, 100, 8192), "new_lo": max(1, new // 2), "new_hi": new, "H": min(H, 24), "D": D,
            "window": window, "ratio": 0, "page": page, "pad": rng.choice([0, 17]), "dtype": dtype, "mix": mix}


def _lens(c):
    """Earlier and new tokens of each request."""
    rng = random.Random(c["mix"])
    return [(_log_int(rng, c["ctx_lo"], c["ctx_hi"]), rng.randint(c["new_lo"], c["new_hi"])) for _ in range(c["R"])]


def _entries(c, r):
    """Entries that (ctx, new) completes."""
    return (r[0] + r[1]) // c["ratio"] - r[0] // c["ratio"]


def _rows(c):
    """Rows of the token (or entry) buffer: the new ones and the padding."""
    if c["op"] == "compress":
        return sum(new // c["ratio"] + 1 for _, new in _lens(c))
    return max(1, sum(_entries(c, r) if c["op"] == "plan" else r[1] for r in _lens(c)) + c["pad"])


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(spans, page, g, spare=0):
    """A block table that gives each request's tokens [first, end) pages, in an order drawn from `g`, the rest -1; and the
    number of pages, some of them unused."""
    width = max(1, spare + max(-(-end // page) for _, end in spans))
    first = torch.tensor([s[0] // page for s in spans])
    count = torch.tensor([-(-s[1] // page) for s in spans]) - first
    base = torch.cumsum(count, 0) - count
    pages = int(count.sum()) + 3
    col = torch.arange(width)
    at = base[:, None] + col - first[:, None]
    there = (col >= first[:, None]) & (col < (first + count)[:, None])
    perm = torch.randperm(pages, generator=g, device="cuda")
    table = torch.where(there.cuda(), perm[at.clamp(0, pages - 1).cuda()], -1)
    return table.to(torch.int32), pages, perm[pages - 3:]


def _slots(c, lens, table, rows):
    """The cache row of each new token, -1 for the padding."""
    req = [r for r, (_, n) in enumerate(lens) for _ in range(n)]
    pos = [ctx + j for ctx, n in lens for j in range(n)]
    req, pos = torch.tensor(req, device="cuda"), torch.tensor(pos, device="cuda")
    slots = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    slots[: len(req)] = table.long()[req, pos // c["page"]] * c["page"] + pos % c["page"]
    return slots


def _store(pages, page, width, dtype, g):
    """A cache of random rows, and one page behind it that the plain forms write what belongs nowhere to."""
    return torch.randn(pages + 1, page, width, generator=g, device="cuda", dtype=dtype)


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    lens, page, s = _lens(c), c["page"], {"case": c, "rows": _rows(c)}
    if c["op"] == "plan":
        m = c["ratio"]
        s["table"], pages, _ = _table([(0, ctx // m) for ctx, _ in lens], page, g, spare=max(-(-_entries(c, r) // page) + 1 for r in lens))
        more = sum(-(-_entries(c, r) // page) + 1 for r in lens)
        s["free"] = (pages + torch.randperm(more, generator=g, device="cuda")).to(torch.int32)
        s["ctx"], s["new"] = _int32([r[0] for r in lens]), _int32([r[1] for r in lens])
        return s
    dt = DTYPES[c["dtype"]]
    if c["op"] == "write":
        table, pages, _ = _table([(0, ctx + n) for ctx, n in lens], page, g)
        s["store"] = _store(pages, page, c["D"], dt, g)
        s["slots"] = _slots(c, lens, table, s["rows"])
        s["new"] = torch.randn(s["rows"], c["D"], generator=g, device="cuda", dtype=dt)
        return s
    if c["op"] == "compress":
        m, C, n = c["ratio"], c["C"], 2 if c["overlap"] else 1
        # content and gate stay in the pages until their entry is made
        s["table"], pages, _ = _table([(max(0, ctx // m - 1) * m, ctx + new) for ctx, new in lens], page, g)
        s["streams"] = torch.randn(pages, page, 2 * n * C, generator=g, device="cuda", dtype=dt)
        s["bias"] = [torch.randn(m, C, generator=g, device="cuda") for _ in range(n)]
        table2, pages2, _ = _table([(ctx // m, (ctx + new) // m) for ctx, new in lens], page, g)
        s["store"] = _store(pages2, page, C, dt, g)
        req = [r for r, x in enumerate(lens) for _ in range(_entries(c, x))]
        ent = [x[0] // m + j for x in lens for j in range(_entries(c, x))]
        rest = s["rows"] - len(req)
        s["request"], s["entry"] = _int32(req + [-1] * rest), _int32(ent + [-1] * rest)
        r, e = s["request"].long(), s["entry"].long()
        s["slots"] = torch.where(r >= 0, table2.long()[r, e.clamp(0) // page] * page + e % page, -1)
        return s
    total = [ctx + n for ctx, n in lens]
    window = c["window"] or EVERY
    s["table"], pages, _ = _table([(max(0, ctx + 1 - window), ctx + n) for ctx, n in lens], page, g)
    s["kv"] = torch.randn(pages, page, c["D"], generator=g, device="cuda", dtype=dt)
    s["longest"] = max(min(ctx + n, n + window - 1) for ctx, n in lens)  # keys of a request's chunk
    if c["ratio"]:
        s["table2"], pages2, _ = _table([(0, t // c["ratio"]) for t in total], page, g)
        s["kv2"] = torch.randn(pages2, page, c["D"], generator=g, device="cuda", dtype=dt)
        s["longest2"] = max(total) // c["ratio"]
    s["most"] = max(n for _, n in lens)
    s["q"] = torch.randn(s["rows"], c["H"], c["D"], generator=g, device="cuda", dtype=dt)
    s["sink"] = torch.randn(c["H"], generator=g, device="cuda")
    s["lens"] = _int32(total)
    s["cu"] = torch.cat([_int32([0]), torch.cumsum(_int32([n for _, n in lens]), 0, dtype=torch.int32)])
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _plan_plain(s):
    c, P, F = s["case"], s["table"].shape[1], s["free"].shape[0]
    m, page, rows = c["ratio"], c["page"], s["rows"]
    ctx, new, table, free = s["ctx"].long(), s["new"].long(), s["table"], s["free"].long()
    old = ctx // m
    cu = torch.cumsum((ctx + new) // m - old, 0).clamp(max=rows)
    cu = torch.cat([cu.new_zeros(1), cu])
    n = cu[1:] - cu[:-1]
    have = ((old + page - 1) // page).clamp(max=P)
    more = (((old + n + page - 1) // page).clamp(max=P) - have).clamp(min=0)
    base = torch.cumsum(more, 0) - more
    col = torch.arange(P, device="cuda")
    fresh = (col >= have[:, None]) & (col < (have + more)[:, None])
    at = base[:, None] + col - have[:, None]
    pages = torch.where(at < F, free[at.clamp(0, F - 1)], -1)
    table.copy_(torch.where(fresh, pages, table))
    row = torch.arange(rows, device="cuda")
    real = row < cu[-1]
    req = torch.searchsorted(cu[1:].contiguous(), row, right=True).clamp(max=c["R"] - 1)
    pos = old[req] + row - cu[req]
    page_of = table.long()[req, (pos // page).clamp(0, P - 1)]
    slots = torch.where(real & (pos // page < P) & (page_of >= 0), page_of * page + pos % page, -1)
    i32 = torch.int32
    return [cu.to(i32), (old + n).to(i32), slots, torch.where(real, req, -1).to(i32), torch.where(real, pos, -1).to(i32),
            more.sum().reshape(1).to(i32), table]


def _write_plain(s):
    flat = s["store"].view(-1, s["store"].shape[2])
    spare = flat.shape[0] - 1  # a row of the page behind the cache
    flat.index_copy_(0, torch.where(s["slots"] >= 0, s["slots"], spare), s["new"])
    return s["store"][:-1]


def _gather(cache, table, at):
    """fp32 rows `at` ([R, L] positions) of each request, and whether they are there."""
    page, width = cache.shape[1], table.shape[1]
    col = at // page
    page_of = torch.gather(table.long(), 1, col.clamp(0, width - 1))
    there = (at >= 0) & (col < width) & (page_of >= 0)
    return cache[page_of.clamp(min=0), at.clamp(min=0) % page].float(), there


def _compress_plain(s):
    c = s["case"]
    m, C = c["ratio"], c["C"]
    real = s["request"] >= 0
    table = s["table"][s["request"].long().clamp(min=0)]
    first = torch.where(real, s["entry"].long(), 0)[:, None] * m
    at = first + torch.arange(-m if c["overlap"] else 0, m, device="cuda")
    x, there = _gather(s["streams"], table, at)
    v, z = x[..., :C], x[..., C:2 * C] + s["bias"][0].repeat(2 if c["overlap"] else 1, 1)
    if c["overlap"]:  # the block before comes from the second pair of streams
        before = (torch.arange(-m, m, device="cuda") < 0)[:, None]
        v = torch.where(before, x[..., 2 * C:3 * C], v)
        z = torch.where(before, x[..., 3 * C:] + s["bias"][1].repeat(2, 1), z)
    z = z.masked_fill(~there[..., None], -math.inf)
    w = torch.exp(z - z.amax(1, keepdim=True))
    out = ((w * v).sum(1) / w.sum(1)).to(s["store"].dtype)
    flat = s["store"].view(-1, C)
    flat.index_copy_(0, torch.where(s["slots"] >= 0, s["slots"], flat.shape[0] - 1), out)
    return s["store"][:-1]


def _attn_plain(s):
    c, N = s["case"], s["rows"]
    H, D, R, Q = c["H"], c["D"], c["R"], s["most"]
    cu, lens = s["cu"].long(), s["lens"].long()
    n = cu[1:] - cu[:-1]
    j = torch.arange(Q, device="cuda")
    row = torch.where(j < n[:, None], cu[:-1, None] + j, N)  # [R, Q], N: no token
    pos = (lens - n)[:, None] + j
    window = c["window"] or EVERY
    at = (lens - n + 1 - window).clamp(min=0)[:, None] + torch.arange(s["longest"], device="cuda")
    keys, there = _gather(s["kv"], s["table"], at)
    legal = there[:, None] & (at[:, None] <= pos[:, :, None]) & (at[:, None] > pos[:, :, None] - window)
    if c["ratio"] and s["longest2"]:
        at = torch.arange(s["longest2"], device="cuda").expand(R, -1)
        keys2, there = _gather(s["kv2"], s["table2"], at)
        keys = torch.cat([keys, keys2], 1)
        legal = torch.cat([legal, there[:, None] & ((at[:, None] + 1) * c["ratio"] <= pos[:, :, None] + 1)], 2)
    q = torch.cat([s["q"], s["q"].new_zeros(1, H, D)])[row].float().view(R, Q * H, D)
    x = torch.bmm(q, keys.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(R, Q, H, -1)
    x.masked_fill_(~legal[:, :, None], -math.inf)
    top = torch.maximum(x.amax(-1), s["sink"])
    x.sub_(top[..., None]).exp_()
    total = x.sum(-1) + torch.exp(s["sink"] - top)
    o = torch.bmm(x.view(R, Q * H, -1), keys).view(R, Q, H, D) / total[..., None]
    out = torch.zeros(N + 1, H, D, device="cuda")  # a row without a token has no key
    lse = s["sink"].expand(N + 1, H).clone()
    out.index_copy_(0, row.view(-1), o.view(R * Q, H, D))
    lse.index_copy_(0, row.view(-1), (top + torch.log(total)).view(R * Q, H))
    return [out[:N].to(s["q"].dtype), lse[:N]]


def run(s):
    c = s["case"]
    if own:
        from streamindex_amd import paged_attn_fwd, paged_compress, paged_plan, paged_write

        if c["op"] == "plan":
            return [*paged_plan(s["ctx"], s["new"], s["table"], s["free"], c["page"], s["rows"], ratio=c["ratio"]), s["table"]]
        if c["op"] == "write":
            return paged_write(s["new"], s["store"][:-1], s["slots"])
        if c["op"] == "compress":
            C, x, b = c["C"], s["streams"], s["bias"]
            more = {"c_b": x[..., 2 * C:3 * C], "z_b": x[..., 3 * C:], "b_b": b[1]} if c["overlap"] else {}
            return paged_compress(x[..., :C], x[..., C:2 * C], b[0], s["table"], s["request"], s["entry"], s["store"][:-1], s["slots"], **more)
        more = {"kv2_cache": s["kv2"], "block_table2": s["table2"], "ratio": c["ratio"]} if c["ratio"] else {}
        return list(paged_attn_fwd(s["q"], s["kv"], s["table"], s["cu"], s["lens"], s["sink"], window=c["window"] or None, **more))
    return {"plan": _plan_plain, "write": _write_plain, "compress": _compress_plain, "attn": _attn_plain}[c["op"]](s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c, lens, rows = case, _lens(case), _rows(case)
    if c["op"] == "plan":  # two lengths a request, the new pages read and written, three values a row
        new = sum(-(-((a + b) // c["ratio"]) // c["page"]) + (-(a // c["ratio"]) // c["page"]) for a, b in lens)
        return {"bytes": 16 * c["R"] + 8 * new + 16 * rows, "flops": 0}
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] == "write":
        n = sum(r[1] for r in lens)
        return {"bytes": 2 * n * c["D"] * size + 8 * rows, "flops": 0}
    if c["op"] == "compress":
        m, C = c["ratio"], c["C"]
        n, k = sum(_entries(c, r) for r in lens), 2 if c["overlap"] else 1
        return {"bytes": (n * m * 2 * k + n) * C * size + k * m * C * 4 + 16 * rows, "flops": 6 * n * m * k * C}
    window, m = c["window"] or EVERY, c["ratio"]
    keys = sum(min(a + b, b + window - 1) + ((a + b) // m if m else 0) for a, b in lens)
    pairs = sum(sum(min(p + 1, window) + ((p + 1) // m if m else 0) for p in range(a, a + b)) for a, b in lens)
    H, D = c["H"], c["D"]
    return {"bytes": (keys * D + 2 * rows * H * D) * size + 4 * rows * H, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, request by request
# ---------------------------------------------------------------------------
def _rows_of(cache, table_row, first, end):
    """Rows [first, end) of one request in 64 bits; the cases' tables hold the pages of every legal key."""
    page = cache.shape[1]
    pages = table_row[first // page: -(-end // page)].long()
    x = cache[pages].reshape(-1, cache.shape[2])
    return x[first - first // page * page:][: end - first].double()


def exact(case, seed):
    c, lens = case, _lens(case)
    if c["op"] == "plan":
        return None
    s = prepare(case, seed)
    if c["op"] == "write":
        out = s["store"][:-1].double()
        rows = out.view(-1, c["D"])
        n = sum(r[1] for r in lens)
        rows[s["slots"][:n]] = s["new"][:n].double()
        return out
    if c["op"] == "compress":
        out = s["store"][:-1].double()
        rows, m, C, k = out.view(-1, c["C"]), c["ratio"], c["C"], 0
        for r, x in enumerate(lens):
            for e in range(x[0] // m, (x[0] + x[1]) // m):
                y = _rows_of(s["streams"], s["table"][r], e * m, (e + 1) * m)
                v, z = y[:, :C], y[:, C:2 * C] + s["bias"][0].double()
                if c["overlap"] and e > 0:
                    y = _rows_of(s["streams"], s["table"][r], (e - 1) * m, e * m)
                    v = torch.cat([v, y[:, 2 * C:3 * C]])
                    z = torch.cat([z, y[:, 3 * C:] + s["bias"][1].double()])
                rows[s["slots"][k]] = (torch.softmax(z, 0) * v).sum(0)
                k += 1
        return out
    H, D, m = c["H"], c["D"], c["ratio"]
    window, at = c["window"] or EVERY, 0
    out = torch.zeros(s["rows"], H, D, device="cuda", dtype=torch.float64)
    lse = s["sink"].double().expand(s["rows"], H).clone()
    for r, (ctx, n) in enumerate(lens):
        for a in range(0, n, 128):
            b = min(n, a + 128)
            pos = torch.arange(ctx + a, ctx + b, device="cuda")
            first, end = max(0, ctx + a + 1 - window), ctx + b
            keys, at1 = _rows_of(s["kv"], s["table"][r], first, end), torch.arange(first, end, device="cuda")
            legal = (at1 <= pos[:, None]) & (at1 + window > pos[:, None])
            if m and end // m:
                keys = torch.cat([keys, _rows_of(s["kv2"], s["table2"][r], 0, end // m)])
                legal = torch.cat([legal, (torch.arange(end // m, device="cuda") * m + m - 1) <= pos[:, None]], 1)
            x = torch.matmul(s["q"][at + a: at + b].double(), keys.t()) * D ** -0.5
            x = torch.where(legal[:, None], x, -math.inf)
            x = torch.cat([x, s["sink"].double().expand(b - a, H)[..., None]], 2)
            lse[at + a: at + b] = torch.logsumexp(x, 2)
            out[at + a: at + b] = torch.matmul(torch.softmax(x, 2)[..., :-1], keys)
        at += n
    return [out, lse]
