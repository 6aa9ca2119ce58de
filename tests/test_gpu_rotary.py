"""GPU parity of the rotation and of the norm with it, and of their gradients, against 64-bit floats.

Tolerances (u = eps / 2 of the type, m the magnitude, (a, b) a pair):
* y: u |y| for the rounding and 2^-18 of m (|a| + |b|) (of |y| where nothing is turned) for the fp32 before it: the sum of squares
  is off by at most 80 additions' 2^-24, its root by half of that, the reciprocal, four products and a cosine or sine by
  2^-22 together: below 2^-18.  Half a step of the smallest subnormal on top.
* dx: the same of r (|d w| + |n| mean |d w n|), 2^-17: a second sum and its product.
* dw: 2^-16 of sum |d n|: 2^-17 of each term and at most 128 additions along a path.
"""

from __future__ import annotations

import math

import pytest
import torch

from streamindex_amd import norm_rotary, rotary, rotary_freqs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def turn(y, pos, freqs, halves, start, m, sign):
    """The rotation of ``y [..., H, D]`` in 64 bits, and ``m (|a| + |b|)`` (``|y|`` outside)."""
    n = freqs.shape[0]
    angle = pos.double()[..., None, None] * freqs.double()
    co, si = m * torch.cos(angle), sign * m * torch.sin(angle)
    i = torch.arange(n, device=y.device)
    one, two = (start + i, start + n + i) if halves else (start + 2 * i, start + 2 * i + 1)
    out, mag = y.clone(), y.abs()
    a, b = y[..., one], y[..., two]
    out[..., one], out[..., two] = a * co - b * si, a * si + b * co
    mag[..., one] = mag[..., two] = abs(m) * (a.abs() + b.abs())
    return out, mag


class Problem:
    def __init__(self, lead, H, D, dims, dtype, halves=False, start=None, m=1.0, inverse=False, weight=True, norm=True, eps=1e-6, pos=None,
                 seed=0, freqs=None, pos_dtype=torch.int64):
        g = torch.Generator().manual_seed(seed + D)
        self.x = (torch.randn(*lead, H, D, generator=g) * torch.exp(torch.randn(*lead, H, 1, generator=g))).to(dtype).to(DEV)
        self.dy = torch.randn(*lead, H, D, generator=g).to(dtype).to(DEV)
        n = math.prod(lead)
        self.pos = (torch.randint(0, 5000, lead, generator=g) if pos is None else torch.tensor(pos).expand(n).reshape(lead)).to(pos_dtype).to(DEV)
        self.freqs = rotary_freqs(dims, device=DEV) if freqs is None else freqs
        self.weight = (1 + 0.3 * torch.randn(D, generator=g)).to(DEV) if weight and norm else None
        self.norm, self.eps = norm, eps
        self.kw = {"interleaved": not halves, "start": start, "magnitude": m, "inverse": inverse}
        self.args = (halves, D - dims if start is None else start, m, -1 if inverse else 1)

    def call(self, x=None, pos=None, weight=None):
        x, pos = self.x if x is None else x, self.pos if pos is None else pos
        if not self.norm:
            return rotary(x, pos, self.freqs, **self.kw)
        return norm_rotary(x, pos, self.freqs, self.weight if weight is None else weight, eps=self.eps, **self.kw)

    def grads(self, x=None, dy=None):
        x = (self.x if x is None else x).detach().requires_grad_()
        leaves = [x]
        w = None
        if self.weight is not None:
            w = self.weight.detach().clone().requires_grad_()
            leaves.append(w)
        return torch.autograd.grad(self.call(x, weight=w), leaves, self.dy if dy is None else dy)

    def want(self, x=None):
        """y and its tolerance; dx and dw and theirs."""
        halves, start, m, sign = self.args
        x, dy = (self.x if x is None else x).double(), self.dy.double()
        u, small = torch.finfo(self.x.dtype).eps / 2, torch.finfo(self.x.dtype).smallest_normal * torch.finfo(self.x.dtype).eps
        d, dmag = turn(dy, self.pos, self.freqs, halves, start, m, -sign)
        w = 1.0 if self.weight is None else self.weight.double()
        if self.norm:
            r = (x.square().mean(-1, keepdim=True) + self.eps) ** -0.5
            n = x * r
        else:
            n = x
        y, mag = turn(n * w, self.pos, self.freqs, halves, start, m, sign)
        out = [(y, u * y.abs() + 2.0 ** -18 * mag + small)]
        if not self.norm:
            return out + [(d, u * d.abs() + 2.0 ** -18 * dmag + small)]
        dx = r * (d * w - n * (d * w * n).mean(-1, keepdim=True))
        mag = r * (dmag * abs(w) + n.abs() * (dmag * abs(w) * n.abs()).mean(-1, keepdim=True))
        out.append((dx, u * dx.abs() + 2.0 ** -17 * mag + small))
        if self.weight is not None:
            D = x.shape[-1]
            out.append(((d * n).reshape(-1, D).sum(0), 2.0 ** -16 * (dmag * n.abs()).reshape(-1, D).sum(0) + 1e-30))
        return out

    def check(self, x=None, pos=None):
        got = [self.call(x, pos), *self.grads(x)]
        for name, g, (want, tol) in zip(("y", "dx", "dw"), got, self.want(x)):
            assert g.shape == want.shape and g.is_contiguous()
            err = (g.double() - want).abs() - tol
            assert not err.isnan().any() and (err <= 0).all(), (name, float(err.max()), int((err > 0).sum()))


SHAPES = [  # tokens, heads, D, rotary dimensions
    ((64,), 64, 576, 64), ((1,), 1, 576, 64), ((3, 50), 5, 512, 64), ((2, 33), 1, 128, 128), ((700,), 3, 64, 32), ((9,), 2, 96, 96),
    ((41,), 6, 100, 100), ((2, 3, 5), 7, 33, 6), ((130,), 1, 1, 0), ((5,), 2, 2, 2), ((17,), 2, 1024, 1024), ((300,), 1, 576, 576),
    ((11,), 1, 1023, 1022), ((40,), 4, 600, 8), ((1025,), 16, 32, 32), ((77,), 1, 256, 0), ((6,), 3, 8, 8),
]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("lead,H,D,dims", SHAPES)
def test_norm(lead, H, D, dims, halves, dtype):
    Problem(lead, H, D, dims, dtype, halves, weight=D % 3 != 0).check()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("lead,H,D,dims", SHAPES)
def test_rotation_alone(lead, H, D, dims, halves, dtype):
    Problem(lead, H, D, dims, dtype, halves, norm=False, m=1.25, inverse=D % 2 == 0).check()


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("D,dims,start", [(576, 64, 0), (576, 64, 256), (128, 32, 5), (100, 50, 25), (64, 24, 8), (96, 16, 80)])
def test_part_of_the_head(D, dims, start, halves):
    for dtype in (BF, F32):
        Problem((37,), 3, D, dims, dtype, halves, start=start, m=0.5, inverse=True).check()
        Problem((37,), 3, D, dims, dtype, halves, start=start, norm=False).check()


@pytest.mark.parametrize("pos,pos_dtype", [(0, torch.int32), (-1, torch.int32), (2**31 - 1, torch.int32), (-(2**31), torch.int32),
                                           (2**31 - 1, torch.int64), (1048575, torch.int64)])
def test_positions(pos, pos_dtype):
    """The angle keeps its fraction of a turn wherever the position."""
    for dtype in (F32, BF):
        Problem((9,), 4, 128, 128, dtype, True, pos=pos, pos_dtype=pos_dtype).check()
        Problem((9,), 1, 64, 64, dtype, pos=pos, pos_dtype=pos_dtype, norm=False).check()


def test_stretched_frequencies_and_fp32_ones():
    f = rotary_freqs(64, 500000.0, factor=16.0, original_length=8192)
    Problem((50,), 8, 576, 64, BF, freqs=f, m=0.1 * math.log(16.0) + 1, pos=100000).check()
    Problem((50,), 8, 128, 64, F32, freqs=f.float(), pos=70000).check()
    Problem((50,), 8, 128, 64, F32, freqs=torch.stack([f, f])[:, ::2].T.reshape(-1), pos=70000).check()


@pytest.mark.parametrize("place", ["heads last", "part of wider rows", "odd place", "every other token", "last dimension strided", "expanded"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides(place, dtype):
    for D, halves in ((128, True), (576, False)):
        p = Problem((2, 23), 4, D, 64, dtype, halves)
        x = p.x

        def like(t):
            if place == "heads last":
                return t.transpose(1, 2).contiguous().transpose(1, 2)
            if place == "part of wider rows":
                return torch.cat([t, t], -1)[..., :D]
            if place == "odd place":
                return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
            if place == "every other token":
                return torch.stack([t, t], 2)[:, :, 1]
            return torch.stack([t, t], -1)[..., 0]

        if place == "expanded":  # one head's row for all
            x = p.x[:, :, :1].expand_as(p.x)
            p.check(x)
            continue
        assert place == "odd place" or not like(x).is_contiguous()
        y, grads = p.call(), p.grads()
        assert torch.allclose(y.float(), p.call(like(x)).float(), rtol=2**-6, atol=1e-5)
        p.check(like(x))
        for a, b in zip(grads, p.grads(like(x), like(p.dy))):
            assert torch.allclose(a.float(), b.float(), rtol=2**-6, atol=2e-3)


def test_positions_of_the_last_sizes():
    p = Problem((3, 40), 4, 64, 64, F32)
    p.pos = p.pos[1].expand(3, 40)
    y, g = p.call(), p.grads()
    one = p.pos[0]
    assert torch.equal(y, p.call(pos=one)) and torch.equal(y, p.call(pos=one.to(torch.int32)))
    p.check(pos=one)
    p.pos = one
    for a, b in zip(g, p.grads()):
        assert torch.equal(a, b)
    p = Problem((5, 1), 2, 32, 32, F32)
    assert torch.equal(p.call(), p.call(pos=p.pos.reshape(5, 1)))


def test_one_position_for_all_and_no_sizes():
    x = torch.randn(3, 64, device=DEV)  # [H, D]: no sizes in front of the heads
    f = rotary_freqs(64)
    got = rotary(x, torch.tensor(7, device=DEV), f)
    want = rotary(x[None], torch.tensor([7], device=DEV), f)[0]
    assert torch.equal(got, want)


def test_empty():
    f = rotary_freqs(8)
    for shape in ((0, 3, 8), (4, 0, 8), (0, 5, 2, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        y = norm_rotary(x, torch.zeros(shape[:-2], dtype=torch.int64, device=DEV), f, w)
        dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
        assert y.shape == dx.shape == shape and (dw == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_value_stays_in_its_row(bad):
    p = Problem((40,), 5, 576, 64, BF)
    y, g = p.call(), p.grads()
    x = p.x.clone()
    x[17, 3, 100] = bad
    keep = torch.ones(40, 5, dtype=torch.bool, device=DEV)
    keep[17, 3] = False
    assert torch.equal(p.call(x)[keep], y[keep]) and torch.equal(p.grads(x)[0][keep], g[0][keep])
    assert p.call(x)[17, 3].isnan().any() and p.grads(x)[1].isnan().any()
    q = Problem((40,), 5, 128, 64, BF, norm=False)
    x = q.x.clone()
    x[17, 3, 100] = bad
    got, want = q.call(x), q.call()
    same = got.eq(want)
    same[17, 3, 100:102] = True
    assert same.all()


def test_zero_rows():
    p = Problem((6,), 2, 64, 64, F32)
    x = p.x.clone()
    x[2] = 0
    assert (p.call(x)[2] == 0).all()
    p.check(x)


def test_weight_types_and_gradients_asked_for():
    p = Problem((30,), 4, 128, 64, BF)
    w = p.weight.to(BF).requires_grad_()
    x = p.x.detach().requires_grad_()
    y = norm_rotary(x, p.pos, p.freqs, w, **p.kw)
    dx, dw = torch.autograd.grad(y, [x, w], p.dy)
    assert dw.dtype is BF and dx.dtype is BF
    p.weight = w.detach().float()
    a, b = p.grads()
    assert torch.equal(dx, a) and torch.equal(dw, b.to(BF))
    only = torch.autograd.grad(norm_rotary(p.x, p.pos, p.freqs, w, **p.kw), [w], p.dy)[0]
    assert torch.equal(only, dw)
    assert torch.equal(torch.autograd.grad(norm_rotary(x, p.pos, p.freqs, w.detach(), **p.kw), [x], p.dy)[0], dx)
    assert not norm_rotary(p.x, p.pos, p.freqs, w.detach(), **p.kw).requires_grad
    with torch.no_grad():
        assert torch.equal(norm_rotary(x, p.pos, p.freqs, w, **p.kw), y)


@pytest.mark.parametrize("norm", [True, False])
def test_gradient_against_differences(norm):
    """Along a direction v: (L(x + h v) - L(x - h v)) / 2h of L = sum dy y, against <dx, v>.  They differ by what the definition's own
    difference and derivative differ by in 64 bits, and by the roundings of L's terms over h and of dx."""
    p = Problem((6,), 3, 96, 64, F32, m=1.1, norm=norm)
    g = torch.Generator().manual_seed(5)
    h = 2.0 ** -7
    v, vw = torch.randn(p.x.shape, generator=g).to(DEV), torch.randn(96, generator=g).to(DEV)
    got = p.grads()

    def loss(f, x, w):
        old, p.weight = p.weight, None if p.weight is None else w
        y = f(x)
        p.weight = old
        return (p.dy.double() * y.double()).sum()

    ends = [(p.x + s * h * v, None if p.weight is None else p.weight + s * h * vw) for s in (1, -1)]
    diff = [(loss(f, *ends[0]) - loss(f, *ends[1])) / (2 * h) for f in (lambda x: p.call(x), lambda x: p.want(x)[0][0])]
    want = [w for w, _ in p.want()[1:]]
    slope = sum((a.double() * b.double()).sum() for a, b in zip(want, (v, vw)))
    mine = sum((a.double() * b.double()).sum() for a, b in zip(got, (v, vw)))
    tol = (p.want()[0][1] * p.dy.double().abs()).sum() * 2 / h + sum((t * b.double().abs()).sum() for (_, t), b in zip(p.want()[1:], (v, vw)))
    assert (diff[0] - mine).abs() <= (diff[1] - slope).abs() + tol
    assert (diff[1] - slope).abs() < 0.02 * sum(a.double().norm() * b.double().norm() for a, b in zip(want, (v, vw)))


def test_many_rows_and_the_same_bits_twice():
    p = Problem((5003,), 16, 64, 64, BF)
    p.check()
    for a, b in zip(p.grads(), p.grads()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lead,H,D,dims,halves", [
    ((43711,), 3, 64, 64, True), ((131079,), 1, 64, 64, False), ((8209,), 16, 100, 50, False), ((16387,), 8, 36, 12, True)])
def test_two_groups_of_rows(lead, H, D, dims, halves):
    """Enough rows that a workgroup takes two groups of them: with one table, with one for each group, past the last row."""
    Problem(lead, H, D, dims, BF, halves).check()
    Problem(lead, H, D, dims, HF, halves, norm=False).check()


def test_far_offsets():
    """Values past 2^31 of x and of the gradient, rows past 2^31, strides past 2^32 bytes: as the same rows near the front."""
    freqs = rotary_freqs(64)

    def last_as_alone(x, pos, f, tokens, norm, gradient):
        with torch.no_grad():
            call = (lambda a, b: norm_rotary(a, b, f)) if norm else (lambda a, b: rotary(a, b, f))
            y = call(x, pos)
            for at in (slice(0, tokens), slice(x.shape[0] - tokens, None)):
                want = call(x[at].clone(), pos[at])
                # (few rows have more lanes each: sums in another order, two roundings, each value else within 2^-18 of its terms,
                # below 4)
                assert norm or torch.equal(y[at], want)
                assert ((y[at].float() - want.float()).abs() <= 1.01 * 2.0 ** -7 * want.float().abs() + 2.0 ** -15).all()
            del y
        if not gradient:
            return
        dy = torch.empty_like(x).uniform_(-1, 1)
        x.requires_grad_()
        dx, = torch.autograd.grad(call(x, pos), [x], dy)
        for at in (slice(0, tokens), slice(x.shape[0] - tokens, None)):
            near = x[at].detach().clone().requires_grad_()
            want, = torch.autograd.grad(call(near, pos[at]), [near], dy[at].clone())
            # (as above: each within 2^-17 of its terms, r (|a| + |b|) (1 + |n| mean |n|) <= sqrt(3) 2 (1 + 1.74 * 0.87) < 9)
            assert ((dx[at].float() - want.float()).abs() <= 1.01 * 2.0 ** -7 * want.float().abs() + 2.0 ** -12).all()

    T = 2 ** 31 // (64 * 512) + 5
    last_as_alone(torch.empty(T, 64, 512, dtype=BF, device=DEV).uniform_(-1, 1), torch.arange(T, device=DEV), freqs, 3, True, True)
    T = 2 ** 31 + 300
    last_as_alone(torch.empty(T, 1, 2, dtype=BF, device=DEV).uniform_(-1, 1), (torch.arange(T, device=DEV) // 1000).int(),
                  rotary_freqs(2), 70, False, False)
    x = torch.empty(3 << 31, dtype=BF, device=DEV).as_strided((3, 2, 128), (1 << 31, 1 << 30, 1)).uniform_(-1, 1)
    pos = torch.arange(3, device=DEV)
    assert torch.equal(norm_rotary(x, pos, freqs), norm_rotary(x.contiguous(), pos, freqs))


def test_inverse_undoes():
    p = Problem((50,), 4, 576, 64, F32, norm=False, m=1.0)
    back = rotary(p.call(), p.pos, p.freqs, inverse=True)
    assert (back - p.x).abs().max() <= 2.0 ** -18 * 4 * p.x.abs().max()


def test_graph_and_stream():
    """Captured and replayed with other inputs, eager work between the replays; and on a stream of its own."""
    p = Problem((64,), 8, 576, 64, BF)
    x, w, pos = p.x.detach().clone().requires_grad_(), p.weight.detach().clone().requires_grad_(), p.pos.clone()

    def step():
        y = norm_rotary(x, pos, p.freqs, w, **p.kw)
        return [y.detach(), *torch.autograd.grad(y, [x, w], p.dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            first = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    del first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        q = Problem((64,), 8, 576, 64, BF, seed=100 + k)
        with torch.no_grad():
            x.copy_(q.x)
            w.copy_(q.weight)
        pos.copy_(q.pos)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_refusals():
    x, pos, f = torch.zeros(4, 2, 16, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV), rotary_freqs(16)
    for call in (
            lambda: rotary(x.double(), pos, f), lambda: rotary(x[0, 0], pos, f), lambda: rotary(x, pos[:3], f), lambda: rotary(x, pos.float(), f),
            lambda: rotary(x, pos, f[None]), lambda: rotary(x, pos, f, start=1), lambda: rotary(x, pos, f, start=-1),
            lambda: rotary(x, pos, rotary_freqs(18)), lambda: rotary(x, pos, f.long()), lambda: rotary(x, pos, f.clone().requires_grad_()),
            lambda: rotary(x, pos[None, :].expand(2, 4), f), lambda: norm_rotary(x, pos, f, torch.ones(15, device=DEV)),
            lambda: rotary(torch.zeros(1, 1, 1025, device=DEV), pos[:1], f)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: rotary(x, pos.cpu(), f), lambda: rotary(x, pos, f.cpu()), lambda: norm_rotary(x, pos, f, torch.ones(16))):
        with pytest.raises(AssertionError):
            call()
    y = norm_rotary(x.clone().requires_grad_(), pos, f)
    g = torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable], create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
