"""From a layer's projections to attention over a cache in 8 bits: the calls a user makes, their plain forms and what a pass cannot
do without.

  norm    norm_rotary: each head's row over its root mean square, by a weight, then its rotary dimensions turned by the token's
          position; for training with its gradients
  rotary  rotary: the rotation alone, for training with its gradient
  write   paged_write_q: the new tokens' rows into the pages of a cache held in 8 bits, a power of two as scale for each block of
          tokens
  attn    paged_attn_q_fwd: attention of the new tokens over such caches: with a window and a second cache of compressed entries
          (HCA), or over every earlier token

Sizes are those of this package's layers (64 heads, D = 576 with 64 rotary dimensions, a window of 128, one entry per 128
tokens) and ranges around them.  A page holds ``page`` consecutive tokens (or entries) of one request, a block ``block`` of them;
a block table row names a request's pages in order, -1 where there is none.
"""

import math
import random

import torch

own = False  # False: the plain forms; True: the package's operators

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
EVERY = 1 << 30  # a window that holds every earlier token
EPS = 1e-6
LEAST = -64  # exponent of the smallest scale


# ---------------------------------------------------------------------------
# The cases.  norm, rotary: x is [B, S, H, D] at positions from `at` on, `dims` of each head's D turned (the last ones), in pairs
# of neighbours or of halves.  write, attn: R requests with ctx_lo .. ctx_hi earlier tokens and new_lo .. new_hi new ones; `mix`
# seeds these lengths.
# ---------------------------------------------------------------------------
def listed():
    return [
        # the queries of a decode step of 64 requests: the smallest call, a launch's latency
        {"name": "norm_q_decode", "op": "norm", "B": 64, "S": 1, "H": 64, "D": 576, "dims": 64, "halves": False, "weight": False, "at": 100000,
         "factor": 1.0, "train": False, "dtype": "bf16"},
        # the queries of a chunk of a prompt far into its context
        {"name": "norm_q_chunk", "op": "norm", "B": 1, "S": 4096, "H": 64, "D": 576, "dims": 64, "halves": False, "weight": False, "at": 1000000,
         "factor": 16.0, "train": False, "dtype": "bf16"},
        # the queries of a training step, with gradients
        {"name": "norm_q_train", "op": "norm", "B": 1, "S": 4096, "H": 64, "D": 576, "dims": 64, "halves": False, "weight": True, "at": 0,
         "factor": 1.0, "train": True, "dtype": "bf16"},
        # a small odd model in 32 bits, every dimension turned
        {"name": "norm_odd_train", "op": "norm", "B": 2, "S": 1001, "H": 6, "D": 100, "dims": 100, "halves": True, "weight": True, "at": 0,
         "factor": 1.0, "train": True, "dtype": "f32"},
        # the rotation alone, halves, whole heads, a context stretched to a million tokens
        {"name": "rotary_long", "op": "rotary", "B": 1, "S": 16001, "H": 24, "D": 128, "dims": 128, "halves": True, "weight": False, "at": 900000,
         "factor": 32.0, "train": False, "dtype": "f16"},
        # the same in training
        {"name": "rotary_train", "op": "rotary", "B": 4, "S": 2048, "H": 16, "D": 128, "dims": 128, "halves": True, "weight": False, "at": 0,
         "factor": 1.0, "train": True, "dtype": "bf16"},
        # the rows of one decode step of 256 requests, into blocks with earlier tokens
        {"name": "write_decode_256", "op": "write", "R": 256, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 1, "new_hi": 1, "page": 64, "block": 16,
         "D": 576, "pad": 0, "dtype": "bf16", "mix": 1},
        # the rows of long prompts given as ragged chunks, padded
        {"name": "write_64k", "op": "write", "R": 9, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 3000, "new_hi": 12000, "page": 64, "block": 64,
         "D": 576, "pad": 300, "dtype": "bf16", "mix": 2},
        # one HCA decode step of 64 requests of very different lengths
        {"name": "hca_decode_64", "op": "attn", "R": 64, "ctx_lo": 2000, "ctx_hi": 131072, "new_lo": 1, "new_hi": 1, "H": 64, "D": 576,
         "window": 128, "ratio": 128, "page": 64, "block": 1, "pad": 0, "dtype": "bf16", "mix": 3},
        # decode over every earlier token
        {"name": "full_decode_32", "op": "attn", "R": 32, "ctx_lo": 4096, "ctx_hi": 65536, "new_lo": 1, "new_hi": 1, "H": 64, "D": 576,
         "window": 0, "ratio": 0, "page": 64, "block": 16, "pad": 0, "dtype": "bf16", "mix": 4},
        # ragged HCA chunks of four long prompts
        {"name": "hca_chunks", "op": "attn", "R": 4, "ctx_lo": 8000, "ctx_hi": 65536, "new_lo": 700, "new_hi": 2048, "H": 64, "D": 576,
         "window": 128, "ratio": 128, "page": 64, "block": 64, "pad": 100, "dtype": "bf16", "mix": 5},
        # a chunk of a prompt over every earlier token, small pages, fp16
        {"name": "full_chunk_f16", "op": "attn", "R": 1, "ctx_lo": 7000, "ctx_hi": 8192, "new_lo": 1000, "new_hi": 1000, "H": 32, "D": 256,
         "window": 0, "ratio": 0, "page": 16, "block": 16, "pad": 0, "dtype": "f16", "mix": 6},
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges above.  No drawn case costs more than the largest listed one."""
    op = rng.choice(["norm", "norm", "rotary", "write", "write", "attn", "attn", "attn"])
    mix = rng.randrange(1 << 20)
    if op in ("norm", "rotary"):
        D = rng.choice([64, 96, 100, 128, 256, 512, 576])
        dims = rng.choice([D, D // 2 // 2 * 2, 64, 64])
        train = rng.random() < 0.5
        H = rng.choice([1, 1, 5, 8, 32, 64])
        B = rng.choice([1, 1, 2, 3])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = (20 if train else 60) * 1000000 // (B * H * D)
        return {"op": op, "B": B, "S": _log_int(rng, 1, max(1, min(65536, most))), "H": H, "D": D, "dims": dims, "halves": rng.random() < 0.5,
                "weight": op == "norm" and rng.random() < 0.6, "at": rng.choice([0, 0, 5000, 2000000]), "factor": rng.choice([1.0, 1.0, 8.0]),
                "train": train, "dtype": dtype}
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([1, 1, 16, page])
    if op == "write":
        R = _log_int(rng, 1, 256)
        return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": 4096, "new_lo": 1, "new_hi": _log_int(rng, 1, max(1, 30000 // R)), "page": page,
                "block": block, "D": rng.choice([64, 128, 500, 512, 576]), "pad": rng.choice([0, 5, 129]), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "mix": mix}
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16"])
    if rng.random() < 0.5:  # HCA
        H, D = rng.choice([16, 64, 64, 128]), rng.choice([512, 576])
        if rng.random() < 0.6:  # a decode step, a few tokens each at times
            ctx = _log_int(rng, 500, 500000)
            return {"op": op, "R": _log_int(rng, 1, 100), "ctx_lo": max(1, ctx // 20), "ctx_hi": ctx, "new_lo": 1, "new_hi": rng.choice([1, 1, 4]),
                    "H": H, "D": D, "window": 128, "ratio": 128, "page": page, "block": block, "pad": rng.choice([0, 3]), "dtype": dtype, "mix": mix}
        R = _log_int(rng, 1, 8)
        new = _log_int(rng, 16, 3000 // R)
        return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": _log_int(rng, 100, 60000), "new_lo": max(1, new // 2), "new_hi": new, "H": rng.choice([16, 64]),
                "D": D, "window": 128, "ratio": 128, "page": page, "block": block, "pad": rng.choice([0, 31]), "dtype": dtype, "mix": mix}
    H, D = rng.choice([1, 8, 16, 24, 64]), rng.choice([32, 64, 128, 256, 576])
    window = rng.choice([0, 0, 0, 512])
    if rng.random() < 0.6:
        ctx = _log_int(rng, 100, 32768)
        return {"op": op, "R": _log_int(rng, 1, 64), "ctx_lo": max(1, ctx // 8), "ctx_hi": ctx, "new_lo": 1, "new_hi": rng.choice([1, 1, 3]), "H": H,
                "D": D, "window": window, "ratio": 0, "page": page, "block": block, "pad": rng.choice([0, 3]), "dtype": dtype, "mix": mix}
    R = _log_int(rng, 1, 4)
    new = _log_int(rng, 16, 1024 // R)
    return {"op": op, "R": R, "ctx_lo": 1, "ctx_hi": _log_int(rng, 100, 8192), "new_lo": max(1, new // 2), "new_hi": new, "H": min(H, 24), "D": D,
            "window": window, "ratio": 0, "page": page, "block": block, "pad": rng.choice([0, 17]), "dtype": dtype, "mix": mix}


def _lens(c):
    """Earlier and new tokens of each request."""
    rng = random.Random(c["mix"])
    return [(_log_int(rng, c["ctx_lo"], c["ctx_hi"]), rng.randint(c["new_lo"], c["new_hi"])) for _ in range(c["R"])]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _freqs(dims, factor, base=10000.0, length=4096, fast=32.0, slow=1.0):
    """Radians a position of each pair.  Stretched by `factor`: those that turn fewer than `slow` times in `length` tokens are
    divided by it, those that turn more than `fast` times stay, those between go from one to the other in a straight line."""
    f = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if factor > 1:
        at = lambda turns: dims * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), dims - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(dims // 2)]
        f = [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)]
    return torch.tensor(f, dtype=torch.float64, device="cuda")


def _table(spans, page, g):
    """A block table that gives each request's tokens [first, end) pages, in an order drawn from `g`, the rest -1; and the
    number of pages, some of them unused."""
    width = max(1, max(-(-end // page) for _, end in spans))
    first = torch.tensor([s[0] // page for s in spans])
    count = torch.tensor([-(-s[1] // page) for s in spans]) - first
    base = torch.cumsum(count, 0) - count
    pages = int(count.sum()) + 3
    col = torch.arange(width)
    at = base[:, None] + col - first[:, None]
    there = (col >= first[:, None]) & (col < (first + count)[:, None])
    perm = torch.randperm(pages, generator=g, device="cuda")
    table = torch.where(there.cuda(), perm[at.clamp(0, pages - 1).cuda()], -1)
    return table.to(torch.int32), pages


def _codes(pages, page, block, width, g):
    """A cache in 8 bits of random rows, and its scales."""
    codes = (torch.randn(pages, page, width, generator=g, device="cuda", dtype=torch.bfloat16) * 90).clamp_(-448, 448).to(F8)
    scales = torch.exp2(torch.randint(-8, -5, (pages, page // block), generator=g, device="cuda").float())
    return codes, scales


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s, dt = {"case": c}, DTYPES[c["dtype"]]
    if c["op"] in ("norm", "rotary"):
        shape = (c["B"], c["S"], c["H"], c["D"])
        s["x"] = torch.randn(shape, generator=g, device="cuda", dtype=dt)
        if c["train"]:
            s["x"].requires_grad_()
            s["dy"] = torch.randn(shape, generator=g, device="cuda", dtype=dt)
        # one decode token of each request at a place of its own, or the tokens of a chunk one after the other
        far = torch.randint(0, 1 + c["at"], (c["B"], 1), generator=g, device="cuda")
        s["pos"] = (far if c["S"] == 1 else c["at"]) + torch.arange(c["S"], device="cuda").expand(c["B"], -1)
        s["freqs"] = _freqs(c["dims"], c["factor"])
        s["magnitude"] = 0.1 * math.log(c["factor"]) + 1.0
        s["weight"] = None
        if c["weight"]:
            s["weight"] = 1 + 0.2 * torch.randn(c["D"], generator=g, device="cuda")
            s["weight"].requires_grad_(c["train"])
        return s
    lens, page, block = _lens(c), c["page"], c["block"]
    s["rows"] = sum(r[1] for r in lens) + c["pad"]
    total = [ctx + n for ctx, n in lens]
    if c["op"] == "write":
        table, pages = _table([(0, t) for t in total], page, g)
        # (one page more, which the plain form writes what belongs nowhere to)
        s["codes"], s["scales"] = _codes(pages + 1, page, block, c["D"], g)
        req = torch.tensor([r for r, (_, n) in enumerate(lens) for _ in range(n)], device="cuda")
        pos = torch.tensor([ctx + j for ctx, n in lens for j in range(n)], device="cuda")
        s["slots"] = torch.full((s["rows"],), -1, dtype=torch.int64, device="cuda")
        s["slots"][: len(req)] = table.long()[req, pos // page] * page + pos % page
        size = torch.exp(0.7 * torch.randn(s["rows"], 1, generator=g, device="cuda"))  # tokens differ in size
        s["new"] = (torch.randn(s["rows"], c["D"], generator=g, device="cuda") * size).to(dt)
        s["first"] = torch.cumsum(torch.tensor([0] + [n for _, n in lens[:-1]], device="cuda"), 0)  # first row of each request
        return s
    window = c["window"] or EVERY
    s["table"], pages = _table([(max(0, ctx + 1 - window), ctx + n) for ctx, n in lens], page, g)
    s["kv"], s["scales"] = _codes(pages, page, block, c["D"], g)
    s["longest"] = max(min(ctx + n, n + window - 1) for ctx, n in lens)  # keys of a request's chunk
    if c["ratio"]:
        s["table2"], pages2 = _table([(0, t // c["ratio"]) for t in total], page, g)
        s["kv2"], s["scales2"] = _codes(pages2, page, block, c["D"], g)
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
def _turn(y, pos, freqs, magnitude, halves, sign):
    """The last 2 len(freqs) of y's dimensions turned by pos * freqs.  Angles of far positions need 64 bits."""
    angle = pos.double()[..., None, None] * freqs
    co, si = (magnitude * torch.cos(angle)).float(), (sign * magnitude * torch.sin(angle)).float()
    n = freqs.shape[0]
    rest, part = y[..., : y.shape[-1] - 2 * n], y[..., y.shape[-1] - 2 * n:]
    a, b = (part[..., :n], part[..., n:]) if halves else (part[..., 0::2], part[..., 1::2])
    a, b = a * co - b * si, a * si + b * co
    part = torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([rest, part], -1)


def _rotary_plain(s):
    c = s["case"]
    more = (s["pos"], s["freqs"], s["magnitude"], c["halves"])
    y = _turn(s["x"].detach().float(), *more, 1).to(s["x"].dtype)
    return [y, _turn(s["dy"].float(), *more, -1).to(y.dtype)] if c["train"] else y


def _norm_plain(s):
    c = s["case"]
    more = (s["pos"], s["freqs"], s["magnitude"], c["halves"])
    x = s["x"].detach().float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    w = s["weight"].detach() if c["weight"] else 1.0
    y = _turn(n * w, *more, 1).to(s["x"].dtype)
    if not c["train"]:
        return y
    d = _turn(s["dy"].float(), *more, -1)
    dn = d * w
    dx = (r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(y.dtype)
    return [y, dx, (d * n).sum((0, 1, 2))] if c["weight"] else [y, dx]


def _exponent(most):
    """Of the smallest power of two that 448 times is at least `most` (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(most)
    return torch.where(most > 0, torch.where(m > 0.875, e - 8, e - 9), LEAST).clamp(min=LEAST)


def _write_plain(s):
    c = s["case"]
    D, block, pages = c["D"], c["block"], s["codes"].shape[0]
    slots = torch.where(s["slots"] >= 0, s["slots"], (pages - 1) * c["page"])  # (the spare page)
    blk = slots // block
    new, old = s["new"].float(), s["scales"].view(-1)
    # of each block: what its new rows need, and its first new token
    e = torch.full_like(old, LEAST - 1, dtype=torch.int32).scatter_reduce_(0, blk, _exponent(new.abs().amax(1)), "amax")
    first = torch.full_like(old, block, dtype=torch.int64).scatter_reduce_(0, blk, slots % block, "amin")
    touched, kept = e >= LEAST, (first > 0) & (first < block)
    scale = torch.where(touched, torch.maximum(torch.exp2(e.float()), torch.where(kept, old, 0.0)), old)
    # earlier tokens of a block stand before a request's first row
    head = blk[s["first"]]
    codes = s["codes"].view(-1, block, D)
    before = codes[head]
    again = (before.float() * (old / scale)[head][:, None, None]).to(F8)
    ours = torch.arange(block, device="cuda") < first[head][:, None]
    flat = codes.view(torch.uint8)
    flat[head] = torch.where(ours[..., None], again.view(torch.uint8), before.view(torch.uint8))
    flat.view(-1, D).index_copy_(0, slots, (new / scale[blk][:, None]).to(F8).view(torch.uint8))
    old.copy_(scale)
    return [s["codes"][:-1], s["scales"][:-1]]


def _gather(cache, scales, table, at):
    """fp32 rows `at` ([R, L] positions) of each request, and whether they are there."""
    page, width = cache.shape[1], table.shape[1]
    col = at // page
    page_of = torch.gather(table.long(), 1, col.clamp(0, width - 1))
    there = (at >= 0) & (col < width) & (page_of >= 0)
    page_of, off = page_of.clamp(min=0), at.clamp(min=0) % page
    return cache[page_of, off].float() * scales[page_of, off // (page // scales.shape[1])][..., None], there


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
    keys, there = _gather(s["kv"], s["scales"], s["table"], at)
    legal = there[:, None] & (at[:, None] <= pos[:, :, None]) & (at[:, None] > pos[:, :, None] - window)
    if c["ratio"] and s["longest2"]:
        at = torch.arange(s["longest2"], device="cuda").expand(R, -1)
        keys2, there = _gather(s["kv2"], s["scales2"], s["table2"], at)
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
        import streamindex_amd as si

        if c["op"] == "rotary":
            y = si.rotary(s["x"], s["pos"], s["freqs"], interleaved=not c["halves"], magnitude=s["magnitude"])
            return [y.detach(), *torch.autograd.grad(y, [s["x"]], s["dy"])] if c["train"] else y
        if c["op"] == "norm":
            y = si.norm_rotary(s["x"], s["pos"], s["freqs"], s["weight"], eps=EPS, interleaved=not c["halves"], magnitude=s["magnitude"])
            leaves = [s["x"], s["weight"]] if c["weight"] else [s["x"]]
            return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])] if c["train"] else y
        if c["op"] == "write":
            return list(si.paged_write_q(s["new"], s["codes"][:-1], s["scales"][:-1], s["slots"]))
        more = {"kv2_cache": s["kv2"], "kv2_scales": s["scales2"], "block_table2": s["table2"], "ratio": c["ratio"]} if c["ratio"] else {}
        return list(si.paged_attn_q_fwd(s["q"], s["kv"], s["scales"], s["table"], s["cu"], s["lens"], s["sink"], window=c["window"] or None, **more))
    return {"norm": _norm_plain, "rotary": _rotary_plain, "write": _write_plain, "attn": _attn_plain}[c["op"]](s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] in ("norm", "rotary"):
        tokens = c["B"] * c["S"]
        n, turned = tokens * c["H"] * c["D"], tokens * c["H"] * c["dims"]
        each = {"norm": 4, "rotary": 0}[c["op"]]
        small = 8 * tokens + 4 * c["dims"] + (4 * c["D"] * (2 if c["train"] else 1) if c["weight"] else 0)
        if not c["train"]:
            return {"bytes": 2 * n * size + small, "flops": each * n + 3 * turned}
        # (a rotation's gradient needs no x)
        return {"bytes": 4 * n * size + small, "flops": 3 * each * n + 6 * turned}
    lens = _lens(c)
    rows = sum(r[1] for r in lens) + c["pad"]
    if c["op"] == "write":
        n = sum(r[1] for r in lens)
        blocks = sum(-(-(a + b) // c["block"]) - a // c["block"] for a, b in lens)
        return {"bytes": n * c["D"] * (size + 1) + 4 * blocks + 8 * rows, "flops": 2 * n * c["D"]}
    window, m = c["window"] or EVERY, c["ratio"]
    keys = sum(min(a + b, b + window - 1) + ((a + b) // m if m else 0) for a, b in lens)
    pairs = sum(sum(min(p + 1, window) + ((p + 1) // m if m else 0) for p in range(a, a + b)) for a, b in lens)
    H, D = c["H"], c["D"]
    return {"bytes": keys * D + 4 * keys // c["block"] + 2 * rows * H * D * size + 4 * rows * H, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _matrix(s, sign):
    """cos and sin of each token and pair, [B, S, 1, pairs]."""
    angle = torch.einsum("bs,i->bsi", s["pos"].double(), s["freqs"])[:, :, None]
    return s["magnitude"] * torch.cos(angle), sign * s["magnitude"] * torch.sin(angle)


def _turned(y, s, sign):
    c = s["case"]
    n, out = c["dims"] // 2, y.clone()
    base = c["D"] - c["dims"]
    i = torch.arange(n, device="cuda")
    first, second = (base + i, base + n + i) if c["halves"] else (base + 2 * i, base + 2 * i + 1)
    co, si = _matrix(s, sign)
    out[..., first] = co * y[..., first] - si * y[..., second]
    out[..., second] = si * y[..., first] + co * y[..., second]
    return out


def _e4m3(v):
    """The nearest value of 4 exponent and 3 fraction bits (ties to even): steps of 2^(e - 3) from 2^e on, of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _rows_of(cache, scales, table_row, first, end):
    """Rows [first, end) of one request in 64 bits; the cases' tables hold the pages of every legal key."""
    page = cache.shape[1]
    pages = table_row[first // page: -(-end // page)].long()
    x = cache[pages].double() * scales[pages].double().repeat_interleave(page // scales.shape[1], 1)[..., None]
    return x.reshape(-1, cache.shape[2])[first - first // page * page:][: end - first]


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] in ("norm", "rotary"):
        x = s["x"].detach().double()
        if c["op"] == "rotary":
            y = _turned(x, s, 1)
            return [y, _turned(s["dy"].double(), s, -1)] if c["train"] else y
        r = ((x ** 2).sum(-1, keepdim=True) / c["D"] + EPS) ** -0.5
        w = s["weight"].detach().double() if c["weight"] else torch.ones(c["D"], device="cuda", dtype=torch.float64)
        y = _turned(x * r * w, s, 1)
        if not c["train"]:
            return y
        d = _turned(s["dy"].double(), s, -1)
        dx = r * d * w - r ** 3 * x * (d * w * x).sum(-1, keepdim=True) / c["D"]
        return [y, dx, (d * x * r).reshape(-1, c["D"]).sum(0)] if c["weight"] else [y, dx]
    lens = _lens(c)
    if c["op"] == "write":
        codes, scales, at = s["codes"][:-1].double(), s["scales"][:-1].double(), 0
        rows, flat, B = codes.view(-1, c["D"]), scales.view(-1), c["block"]
        for ctx, n in lens:
            x, slots = s["new"][at: at + n].double(), s["slots"][at: at + n]
            at += n
            blk, inside = slots // B, slots % B
            start = torch.cat([torch.ones_like(blk[:1], dtype=torch.bool), blk[1:] != blk[:-1]])
            which = torch.cumsum(start, 0) - 1
            ids = blk[start]
            most = torch.zeros(len(ids), device="cuda", dtype=torch.float64).scatter_reduce_(0, which, x.abs().amax(1), "amax")
            need = torch.exp2(torch.ceil(torch.log2(most.clamp(min=448 * 2.0 ** LEAST) / 448)))
            k = int(inside[0])
            if k:  # the block of the first row holds k earlier tokens
                was = flat[ids[0]].clone()
                need[0] = torch.maximum(need[0], was)
                there = slice(int(ids[0]) * B, int(ids[0]) * B + k)
                rows[there] = _e4m3(rows[there] * (was / need[0]))
            flat[ids] = need
            rows[slots] = _e4m3(x / need[which][:, None])
        return [codes, scales]
    H, D, m = c["H"], c["D"], c["ratio"]
    window, at = c["window"] or EVERY, 0
    out = torch.zeros(s["rows"], H, D, device="cuda", dtype=torch.float64)
    lse = s["sink"].double().expand(s["rows"], H).clone()
    for r, (ctx, n) in enumerate(lens):
        for a in range(0, n, 128):
            b = min(n, a + 128)
            pos = torch.arange(ctx + a, ctx + b, device="cuda")
            first, end = max(0, ctx + a + 1 - window), ctx + b
            keys, there = _rows_of(s["kv"], s["scales"], s["table"][r], first, end), torch.arange(first, end, device="cuda")
            legal = (there <= pos[:, None]) & (there + window > pos[:, None])
            if m and end // m:
                keys = torch.cat([keys, _rows_of(s["kv2"], s["scales2"], s["table2"][r], 0, end // m)])
                legal = torch.cat([legal, (torch.arange(end // m, device="cuda") * m + m - 1) <= pos[:, None]], 1)
            x = torch.matmul(s["q"][at + a: at + b].double(), keys.t()) * D ** -0.5
            x = torch.where(legal[:, None], x, -math.inf)
            x = torch.cat([x, s["sink"].double().expand(b - a, H)[..., None]], 2)
            lse[at + a: at + b] = torch.logsumexp(x, 2)
            out[at + a: at + b] = torch.matmul(torch.softmax(x, 2)[..., :-1], keys)
        at += n
    return [out, lse]
