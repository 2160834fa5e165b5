"""The step of AdamW over many tensors on the GPU, and the optimizer on it, against plain implementations in 64 bits.

Tolerances count roundings; u = 2^-24.  The clipping's factor takes 4 of them, the gradient 1 more: dg = 5 u |g|.  m + c (g - m): the
difference, the product and the sum, c itself: 4 u (|m| + |g|) + c dg; v in the same way with g^2: 4 u (v + g^2) + 2 c |g| dg.  The
way of a parameter, rate m / (sqrt(v) root + eps): rate, root and eps are rounded, the root of v, two products, the sum and the
quotient: 12 u of it, the error of m and half the relative error of v on top; the decay and the sum 4 u (|p| + the way)."""
import copy
import math

import pytest
import torch

import fp8_gmm_amd as pkg
from fp8_gmm_amd import backend, moe

from helpers import gen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HYPER = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
BLOCK = 128


def assert_within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} are off, by up to {(off / tol)[bad].max().item():.3g} of what is allowed"


def blocks_max(t):
    t = t.reshape(-1)
    return torch.nn.functional.pad(t.abs(), (0, -t.numel() % BLOCK)).view(-1, BLOCK).amax(1)


def spread(scales, n):
    return scales.repeat_interleave(BLOCK)[:n]


class Problem:
    """Lists as a program has them, and the step in 64 bits."""

    def __init__(self, dev, sizes, t, g, bits, masters, seed, magnitude=1e-3):
        r = gen(seed)

        def normal(n, std):
            return (torch.randn(n, generator=r) * std).to(dev)

        self.bits, self.dev = bits, dev
        self.params = [normal(n, 0.05).to(TYPES[t]) for n in sizes]
        self.masters = [normal(n, 0.05) for n in sizes] if masters else None
        if masters:
            self.params = [m.to(TYPES[t]) for m in self.masters]
        self.grads = [normal(n, magnitude * (1 + i % 5)).to(TYPES[g]) for i, n in enumerate(sizes)]
        m = [normal(n, 0.3 * magnitude) for n in sizes]
        v = [normal(n, magnitude).square() for n in sizes]
        for t_ in v:
            t_[::7] = 0.0
        self.scales = None
        if bits == 8:
            self.scales = ([blocks_max(a) / 448 for a in m], [blocks_max(a.sqrt()) / 448 for a in v])
            self.m = [(a / spread(s, a.numel())).nan_to_num(0).clamp(-448, 448).to(torch.float8_e4m3fn) for a, s in zip(m, self.scales[0])]
            self.v = [(a.sqrt() / spread(s, a.numel())).nan_to_num(0).clamp(0, 448).to(torch.float8_e4m3fn) for a, s in zip(v, self.scales[1])]
        else:
            self.m, self.v = m, v

    def all(self):
        return self.params + self.m + self.v + (self.masters or []) + (self.scales[0] + self.scales[1] if self.scales else [])

    def values(self, i):
        n = self.params[i].numel()
        m, v = self.m[i].double().reshape(-1), self.v[i].double().reshape(-1)
        if self.bits == 8:
            m, v = m * spread(self.scales[0][i].double(), n), (v * spread(self.scales[1][i].double(), n)).square()
        return m, v

    def step(self, t, norm=None, max_norm=None, **kw):
        backend.multi_adamw(self.params, self.grads, self.m, self.v, t, **{**HYPER, **kw}, scales=self.scales, masters=self.masters, norm=norm,
                            max_norm=max_norm)

    def check(self, t, norm=None, max_norm=None, **kw):
        h = {**HYPER, **kw}
        before = [(*self.values(i), (self.masters or self.params)[i].double().clone()) for i in range(len(self.params))]
        factor = 1.0 if norm is None else min(1.0, max_norm / (norm.item() + 1e-6))
        self.step(t, norm, max_norm, **kw)
        c1, c2 = 1 - h["betas"][0], 1 - h["betas"][1]
        rate, root = h["lr"] / (1 - h["betas"][0] ** t), 1 / math.sqrt(1 - h["betas"][1] ** t)
        for i, (m, v, p) in enumerate(before):
            g = self.grads[i].double() * factor
            dg = 5 * U * g.abs()
            m1, v1 = m + c1 * (g - m), v + c2 * (g * g - v)
            e = 4 * U if self.bits == 32 else 12 * U   # of moments that come from codes, times their scales
            tol_m = e * (m.abs() + g.abs()) + c1 * dg + 1e-44
            tol_v = e * (v + g * g) + 2 * c2 * g.abs() * dg + 1e-44
            way = rate * m1 / (v1.sqrt() * root + h["eps"])
            # the root of a v that is nearly nothing has what its error leaves of it
            low = (v1 - tol_v).clamp(min=0).sqrt()
            tol_way = rate * (m1.abs() + tol_m) / (low * root + h["eps"]) * (1 + 12 * U) - way.abs()
            want = p - h["lr"] * h["weight_decay"] * p - way
            tol = tol_way + 4 * U * (p.abs() + way.abs())
            if self.masters is not None:
                assert_within(self.masters[i], want, tol, f"master {i}")
                assert torch.equal(self.params[i], self.masters[i].to(self.params[i].dtype))
            half = torch.finfo(self.params[i].dtype).eps / 2
            tiny = torch.finfo(self.params[i].dtype).smallest_normal * half
            assert_within(self.params[i], want, tol + half * (want.abs() + tol) + tiny, f"param {i}")
            if self.bits == 32:
                assert_within(self.m[i], m1, tol_m, f"m {i}")
                assert_within(self.v[i], v1, tol_v, f"v {i}")
            else:
                self.check_codes(i, t, m1, v1, tol_m, tol_v)

    def check_codes(self, i, t, m, v, tol_m, tol_v):
        n = m.numel()
        h = (torch.arange(n, device=self.dev) * 0x6A09E667 + t * 0x9E3779B9) & 0xFFFFFFFF
        for name, codes, scale, value, tol, u in (
                ("m", self.m[i], self.scales[0][i], m, tol_m, (h >> 12).double() * 2.0 ** -20),
                ("v", self.v[i], self.scales[1][i], v.sqrt(), tol_v / (2 * v.sqrt()).clamp(min=1e-30), ((h ^ 0x80000000) >> 8).double() * 2.0 ** -24)):
            most = blocks_max(value)
            assert_within(scale, most / 448, 4 * U * most / 448 + blocks_max(tol) / 448 + 1e-44, f"scale of {name} {i}")
            y = value.abs() / spread(most, n).clamp(min=1e-37) * 448
            # 8 roundings between the moment and y; what its own error makes of it
            dy = 8 * U * y + tol / spread(most, n).clamp(min=1e-37) * 448
            normal = y.clamp(min=2.0 ** -6)
            gap = normal / torch.frexp(normal).mantissa / 16   # (a power of two, exactly)
            low = torch.floor(y / gap) * gap
            high = low + gap
            if name == "m":
                way, up_from = (y - low) / gap, 1 - u
                slack = dy / gap + 2.0 ** -19
            else:
                way, up_from = (y - low) * (y + low) / (gap * (high + low)), u
                slack = (2 * dy * y / (gap * (high + low))) + 2.0 ** -19
            up = (way >= up_from) if name == "m" else (way > up_from)
            want = torch.where(up, high, low).clamp(max=448)
            if name == "v":
                want = torch.where((low == 0) & (y > 0), high, want)
            got = codes.double().reshape(-1)
            sure = ((way - up_from).abs() > slack) & ((y - low) > dy) & ((high - y) > dy)
            # (a v next to fp32's smallest number, 2^-149, has only a few bits: the 1e-44 of its tolerance is a share of it)
            clear = tol <= value.abs() * 2.0 ** -10
            assert n < 64 or clear.sum() < 64 or sure[clear].double().mean() > 0.9 or (m == 0).all()
            assert torch.equal(got.abs()[sure], want[sure]), f"{name} {i}: {int((got.abs()[sure] != want[sure]).sum())} codes"
            # the others: either neighbour, or one further where y itself is in doubt about its interval
            rest = ~sure
            assert ((got.abs() - y).abs()[rest] <= (gap + dy)[rest] * 1.0001).all(), f"{name} {i}"
            if name == "m":
                assert (torch.sign(got) * torch.sign(value) >= 0).all()
            else:
                assert (got[value > 2.0 ** -74] > 0).all() and (got >= 0).all()   # (a v below fp32's numbers is zero)


SIZES = [[1], [7, 0, 129], [128, 127, 1000, 8192, 1], [2048, 2047, 2049, 1024, 1023, 1025], [100003], [17] * 60 + [5000] * 60, [1 << 20, 3, (1 << 18) + 77]]


@pytest.mark.parametrize("sizes", SIZES, ids=[str(i) for i in range(len(SIZES))])
@pytest.mark.parametrize("t, g, masters", [("bf16", "bf16", False), ("bf16", "fp32", False), ("bf16", "bf16", True), ("bf16", "fp32", True),
                                           ("fp16", "fp16", False), ("fp16", "fp32", True), ("fp32", "fp32", False)])
@pytest.mark.parametrize("bits", [32, 8])
def test_against_64_bits(dev, sizes, t, g, masters, bits):
    p = Problem(dev, sizes, t, g, bits, masters, len(sizes) + bits)
    p.check(1)
    p.check(2, torch.full((), 4.0, device=dev), 1.0)
    p.check(1000, torch.full((1,), 0.5, device=dev), 1.0)   # within the bound
    if bits == 8 and all(n > 0 for n in sizes):
        assert all(torch.isfinite(a.float()).all() for a in p.all())


@pytest.mark.parametrize("magnitude", [1e-18, 1e-6, 1e4])
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_any_magnitude(dev, magnitude, bits):
    Problem(dev, [5000, 333], "fp32", "fp32", bits, False, 4, magnitude).check(3)


@pytest.mark.parametrize("bits", [32, 8])
def test_magnitudes_side_by_side(dev, bits):
    """Second moments below fp32's normal numbers among others of their block, alone in it, and with an eps that does not hide them."""
    for small, large in ((1e-22, 1e-3), (3e-20, 1e-18), (1e-21, 1e-21), (1e-6, 1e12)):
        for eps in (1e-8, 1e-12, 1e-24):
            p = Problem(dev, [3000, 77], "fp32", "fp32", bits, False, 8, 1.0)
            for g in p.grads:
                g *= torch.where(torch.arange(g.numel(), device=dev) % 3 == 0, large, small)
            for t in p.m + p.v + (p.scales[0] + p.scales[1] if bits == 8 else []):
                t.zero_()
            p.check(1, eps=eps)


def test_codes_have_the_moments_means(dev):
    """Over the thresholds of 4096 steps the codes' mean is m, the mean of their squares v: to a few of 1 / 4096 of a code's distance."""
    p = Problem(dev, [4096], "fp32", "fp32", 8, False, 5)
    start = [a.clone() for a in p.all()]
    m, v = p.values(0)
    g = p.grads[0].double()
    m, v = m + 0.1 * (g - m), v + 0.01 * (g * g - v)
    sums = [torch.zeros(4096, dtype=torch.float64, device=dev) for _ in range(2)]
    steps = 4096
    for t in range(1, steps + 1):
        for a, b in zip(p.all(), start):
            a.copy_(b)
        p.step(t)
        a, b = p.values(0)
        sums[0] += a
        sums[1] += b
    for total, value, exponent in ((sums[0], m, 1), (sums[1], v, 2)):
        most = spread(blocks_max(value), 4096)
        gap = torch.maximum(value.abs() * 2.0 ** -2.99 * exponent, most * (2.0 ** -9 / 448) ** exponent)   # between two codes' values, at most
        off = (total / steps - value).abs()
        # the thresholds' multiples of the golden ratio fall short of evenness by less than 2 + log2(steps) of `steps`; 20 bits of them
        ok = off <= gap * (16 / steps) + value.abs() * 16 * U
        lowest = (value > 0) & (value < most * (2.0 ** -9 / 448) ** 2) if exponent == 2 else torch.zeros_like(ok)   # never zero: above v
        assert ok[~lowest].all(), (off / gap)[~ok].max().item() * steps
        assert (total[lowest] / steps >= value[lowest]).all()


def test_shapes_and_strides(dev):
    g = gen(7)
    shapes = [(33, 17), (5, 4, 3), (), (2, 0, 3), (64,)]
    make = [lambda t: t, lambda t: t.transpose(-1, 0).contiguous().transpose(-1, 0) if t.dim() > 1 else t]
    for bits in (32, 8):
        for order in make:
            params = [order(torch.randn(s, generator=g).to(dev)) for s in shapes]
            grads = [order(torch.randn(s, generator=g).to(dev)) for s in shapes]
            other = [torch.empty(s + (2,), device=dev)[..., 0].copy_(t) for s, t in zip(shapes, grads)]   # with gaps
            states = [torch.float32] if bits == 32 else [torch.float8_e4m3fn]
            m = [torch.zeros_like(p, dtype=states[0]) for p in params]
            v = [torch.zeros_like(p, dtype=states[0]) for p in params]
            scales = None if bits == 32 else tuple([torch.zeros(-(-p.numel() // 128), device=dev) for p in params] for _ in range(2))
            lists = copy.deepcopy((params, m, v, scales))
            backend.multi_adamw(params, grads, m, v, 1, **HYPER, scales=scales)
            backend.multi_adamw(lists[0], other, lists[1], lists[2], 1, **HYPER, scales=lists[3])
            for a, b in zip(params + m + v, lists[0] + lists[1] + lists[2]):
                assert torch.equal(a.float(), b.float())
            negated = copy.deepcopy((params, m, v, scales))
            backend.multi_adamw(params, grads, m, v, 2, **HYPER, scales=scales)
            backend.multi_adamw(negated[0], [torch._neg_view(-t) for t in grads], negated[1], negated[2], 2, **HYPER, scales=negated[3])
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(params + m + v, negated[0] + negated[1] + negated[2]))
    # tensors at any element of a buffer, and what lies between them
    flat, gflat = (torch.randn(5000, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    params, grads = [flat[3:1000], flat[1001:4999]], [gflat[1:998], gflat[1002:5000]]
    apart = [t.clone() for t in params]
    gapart = [t.clone() for t in grads]
    kept = flat.clone()
    m, v = [torch.zeros(t.numel(), device=dev) for t in params], [torch.zeros(t.numel(), device=dev) for t in params]
    backend.multi_adamw(params, grads, m, v, 1, **HYPER)
    backend.multi_adamw(apart, gapart, [torch.zeros_like(t) for t in m], [torch.zeros_like(t) for t in v], 1, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(params, apart))
    assert torch.equal(flat[:3], kept[:3]) and flat[1000] == kept[1000] and flat[4999] == kept[4999]


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_what_is_no_number(dev, value):
    for bits in (32, 8):
        p = Problem(dev, [1000], "fp32", "fp32", bits, False, 3)
        p.grads[0][300] = value
        p.step(1)
        bad = ~torch.isfinite(p.params[0])
        assert bad[300] and bad.sum() == 1
        for values in p.values(0):
            off = ~torch.isfinite(values)
            assert off[300] or (value != value and bits == 8)
            assert not off[:256].any() and not off[384:].any()   # at most its block
    p = Problem(dev, [1000], "fp32", "fp32", 32, False, 3)
    before = p.params[0].clone()
    p.step(1, torch.full((), value, device=dev), 1.0)   # a norm that is infinite or none: gradients of zeros, or none
    assert torch.isfinite(p.params[0]).all() if value == float("inf") else p.params[0].isnan().all()
    assert not torch.equal(p.params[0], before)


def test_zero_moments_and_gradients(dev):
    for bits in (32, 8):
        p = Problem(dev, [500], "bf16", "bf16", bits, True, 3)
        for t in p.m + p.v + p.grads:
            t.zero_()
        before = p.masters[0].clone()
        p.step(1)
        assert not any(t.float().any() for t in p.m + p.v)
        assert torch.allclose(p.masters[0], before * (1 - 1e-4), rtol=1e-6)


def test_squares_that_fp32_does_not_hold(dev):
    """A second moment that is infinite leaves the decay alone; without eps, one that is zero sends a parameter to infinity."""
    for bits in (32, 8):
        p = Problem(dev, [500], "fp32", "fp32", bits, False, 3)
        p.grads[0][100], p.grads[0][101] = 1e25, -1e25
        before = p.params[0].clone()
        p.step(1)
        assert torch.isfinite(p.params[0]).all()
        decayed = before.double() * (1 - 1e-4)
        assert_within(p.params[0][100:102], decayed[100:102], 4 * U * decayed.abs()[100:102], "params")
        if bits == 32:
            assert p.v[0][100:102].isinf().all() and torch.isfinite(p.m[0]).all()
        q = Problem(dev, [500], "fp32", "fp32", bits, False, 3)
        for t in q.m + q.v:
            t.zero_()
        q.grads[0][1:4] = torch.tensor([0.0, 1e-25, -1e-25], device=dev)
        q.step(1, eps=0.0)
        assert q.params[0][1].isnan() and q.params[0][2] == -math.inf and q.params[0][3] == math.inf
        assert torch.isfinite(q.params[0][4:]).all()


def test_past_32_bits(dev):
    n = (1 << 31) + 12345
    tail = 4096 + 12345
    p = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    m, v = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    r = gen(3)
    p[-tail:], g[-tail:] = torch.randn(tail, generator=r).to(dev), torch.randn(tail, generator=r).to(dev)
    small = [t[-tail:].clone() for t in (p, g, m, v)]
    backend.multi_adamw([p], [g], [m], [v], 1, **HYPER)
    backend.multi_adamw(*[[t] for t in small], 1, **HYPER)
    assert all(torch.equal(a[-tail:], b) for a, b in zip((p, g, m, v), small)) and not p[:1 << 20].any()
    del m, v
    codes = [torch.zeros(n, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2)]
    scales = [torch.zeros(-(-n // 128), device=dev) for _ in range(2)]
    backend.multi_adamw([p], [g], [codes[0]], [codes[1]], 1, **HYPER, scales=([scales[0]], [scales[1]]))
    last = (n - 1) // 128
    part = codes[0][last * 128:].double() * scales[0][last].double()
    want = 0.1 * g[last * 128:].double()
    assert ((part - want).abs() <= want.abs().max() / 448 * 32).all()


def test_the_same_bits_alone_together_and_side_by_side(dev):
    a, b = Problem(dev, [5000, 77, 2048], "bf16", "bf16", 8, True, 3), Problem(dev, [5000, 77, 2048], "bf16", "bf16", 8, True, 3)
    a.step(5)
    for i in range(3):
        backend.multi_adamw([b.params[i]], [b.grads[i]], [b.m[i]], [b.v[i]], 5, **HYPER, scales=([b.scales[0][i]], [b.scales[1][i]]),
                            masters=[b.masters[i]])
    assert all(torch.equal(x.float(), y.float()) for x, y in zip(a.all(), b.all()))
    streams = [torch.cuda.Stream() for _ in range(2)]
    problems = [Problem(dev, [300000, 77], "fp32", "fp32", 32, False, s) for s in (1, 2)]
    twins = [Problem(dev, [300000, 77], "fp32", "fp32", 32, False, s) for s in (1, 2)]
    torch.cuda.synchronize()
    for s, p in zip(streams, problems):
        with torch.cuda.stream(s):
            for t in (1, 2, 3):
                p.step(t)
    torch.cuda.synchronize()
    for p in twins:
        for t in (1, 2, 3):
            p.step(t)
    assert all(torch.equal(x, y) for p, q in zip(problems, twins) for x, y in zip(p.all(), q.all()))


def test_step_and_rate_of_the_device(dev):
    """The rate takes another four roundings (the powers are good to 2^-30), the decay two."""
    for bits in (32, 8):
        for t in (1, 7, 100000):
            step, lr = torch.full((), t, dtype=torch.int64, device=dev), torch.full((1,), 1e-3, device=dev)
            a, *others = (Problem(dev, [3000, 11], "fp32", "fp32", bits, False, 3) for _ in range(4))
            start = [p.clone() for p in a.params]
            a.step(t)
            for other, args in zip(others, (dict(t=step, lr=lr), dict(t=step), dict(t=t, lr=lr))):
                other.step(**args)
                assert all(torch.equal(x.float(), y.float()) for x, y in zip(a.m + a.v, other.m + other.v))
                for x, y, p in zip(a.params, other.params, start):
                    assert_within(y, x.double(), 8 * U * (x - p).double().abs() + 4 * U * p.double().abs(), f"{args}")


def test_refusals(dev):
    def call(change):
        p = Problem(dev, [100, 200], "bf16", "bf16", 32, False, 1)
        args = dict(params=p.params, grads=p.grads, exp_avgs=p.m, exp_avg_sqs=p.v, step=1, lr=1e-3)
        args.update(change(p))
        backend.multi_adamw(**args)

    one = torch.ones(1, device=dev)
    changes = [lambda p: dict(params=[]), lambda p: dict(grads=p.grads[:1]), lambda p: dict(exp_avgs=p.m[:1]), lambda p: dict(step=0),
               lambda p: dict(lr=-1.0), lambda p: dict(lr=float("nan")), lambda p: dict(betas=(1.0, 0.9)), lambda p: dict(betas=(0.9, -0.1)),
               lambda p: dict(eps=-1.0), lambda p: dict(weight_decay=-0.1), lambda p: dict(norm=one), lambda p: dict(max_norm=1.0),
               lambda p: dict(norm=one, max_norm=-1.0), lambda p: dict(norm=one.cpu(), max_norm=1.0), lambda p: dict(norm=one.double(), max_norm=1.0),
               lambda p: dict(step=one), lambda p: dict(lr=one.double()), lambda p: dict(step=torch.ones(2, dtype=torch.int64, device=dev)),
               lambda p: dict(params=[t.cpu() for t in p.params]), lambda p: dict(params=[p.params[0], p.params[0]], grads=[p.grads[0]] * 2,
                                                                                 exp_avgs=[p.m[0]] * 2, exp_avg_sqs=[p.v[0]] * 2),
               lambda p: dict(exp_avgs=[t.bfloat16() for t in p.m]), lambda p: dict(exp_avgs=p.v),
               lambda p: dict(grads=[t.half() for t in p.grads]), lambda p: dict(grads=[t[:-1] for t in p.grads]),
               lambda p: dict(grads=[p.params[0], p.grads[1]]), lambda p: dict(masters=p.m[:1]),
               lambda p: dict(masters=[t.clone() for t in p.params]), lambda p: dict(scales=(p.m, p.v)),
               lambda p: dict(params=[t.requires_grad_() for t in p.params]),
               lambda p: dict(params=[t.double() for t in p.params]),
               lambda p: dict(params=[torch.zeros(200, dtype=torch.bfloat16, device=dev)[::2], p.params[1]]),
               lambda p: dict(params=[torch.zeros(1, dtype=torch.bfloat16, device=dev).expand(100), p.params[1]])]
    for i, change in enumerate(changes):
        with pytest.raises((RuntimeError, TypeError)):
            call(change)
            print(i)
    p = Problem(dev, [100, 200], "bf16", "bf16", 8, False, 1)
    for scales in ((p.scales[0][:1], p.scales[1]), ([s.double() for s in p.scales[0]], p.scales[1]), (p.scales[0], p.scales[0]),
                   ([torch.zeros(5, device=dev)] * 2, p.scales[1])):
        with pytest.raises(RuntimeError):
            backend.multi_adamw(p.params, p.grads, p.m, p.v, 1, 1e-3, scales=scales)
    fp32 = Problem(dev, [100], "fp32", "fp32", 32, False, 1)
    with pytest.raises(RuntimeError, match="its own master"):
        backend.multi_adamw(fp32.params, fp32.grads, fp32.m, fp32.v, 1, 1e-3, masters=[fp32.params[0].clone()])
    turned = torch.zeros(20, 10, dtype=torch.float32, device=dev)
    with pytest.raises(RuntimeError, match="order"):
        backend.multi_adamw([turned], [turned.clone()], [torch.zeros(10, 20, device=dev).t()], [turned.clone()], 1, 1e-3)
    with torch.inference_mode():
        inner = torch.zeros(100, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="inference"):
        backend.multi_adamw([inner], [p.grads[0]], [torch.zeros(100, device=dev)], [torch.zeros(100, device=dev)], 1, 1e-3)


# ---- the optimizer -------------------------------------------------------------------------------------------------------
def model(dev, dtype, seed=0):
    g = gen(seed)
    shapes = [(40, 30), (30,), (7, 5, 3), (1000,)]
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype).to(dev)) for s in shapes]


def set_grads(params, seed):
    g = gen(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=g) * 0.1).to(p.dtype).to(p.device)


def test_optimizer_against_torch_in_64_bits(dev):
    """Ten steps in fp32 against torch's optimizer in float64: every step adds at most 16 roundings of a way of at most 4 lr and 4 of p."""
    params = model(dev, torch.float32)
    twins = [torch.nn.Parameter(p.detach().double()) for p in params]
    hyper = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
    ours, theirs = pkg.AdamW([{"params": params[:2]}, {"params": params[2:], "lr": 3e-3}], **hyper), torch.optim.AdamW(
        [{"params": twins[:2]}, {"params": twins[2:], "lr": 3e-3}], **hyper)
    for t in range(10):
        set_grads(params, 50 + t)
        if t % 3 == 1:
            params[1].grad = None   # passed over: counts its own steps
        for p, q in zip(params, twins):
            q.grad = None if p.grad is None else p.grad.double()
        ours.step()
        theirs.step()
    for p, q in zip(params, twins):
        assert_within(p.detach(), q.detach(), 10 * (64 * U * 4e-2 + 4 * U * q.detach().abs()), "parameter")
    assert ours.state[params[1]]["step"] == 7 and ours.state[params[0]]["step"] == 10


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_clips_and_goes_on_from_a_checkpoint(dev, dtype, bits):
    params = model(dev, dtype)
    options = dict(lr=1e-2, state_bits=bits, master_weights=True, max_norm=0.5)
    opt = pkg.AdamW(params, **options)
    for t in range(3):
        set_grads(params, t)
        held = [p.grad.clone() for p in params]
        opt.step()
        assert all(torch.equal(p.grad, h) for p, h in zip(params, held))
        norm = math.sqrt(sum(h.double().square().sum().item() for h in held))
        assert abs(opt.grad_norm.item() - norm) <= 1e-6 * norm
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = pkg.AdamW(copies, **options)
    saved = copy.deepcopy(opt.state_dict())
    other.load_state_dict(saved)
    for p, q in zip(params, copies):
        assert {k: getattr(v, "dtype", type(v)) for k, v in opt.state[p].items()} == {k: getattr(v, "dtype", type(v)) for k, v in other.state[q].items()}
        assert ("master" in opt.state[p]) == (dtype != torch.float32)
    for t in range(3, 6):
        set_grads(params, t)
        set_grads(copies, t)
        opt.step()
        other.step()
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert v == other.state[q][k] if k == "step" else torch.equal(v.float(), other.state[q][k].float())
    assert not any(torch.equal(v.float(), saved["state"][0][k].float()) for k, v in opt.state[params[0]].items() if k != "step")


def test_optimizer_learns_with_8_bits(dev):
    """Moments in 8 bits: the ways of 300 steps together stay within a tenth of those in 32 bits."""
    ways = []
    for bits in (32, 8):
        params = model(dev, torch.float32)
        start = [p.detach().clone() for p in params]
        opt = pkg.AdamW(params, lr=1e-3, weight_decay=0.0, state_bits=bits)
        for t in range(300):
            for i, p in enumerate(params):   # a slope with noise on it
                slope = torch.randn(p.shape, generator=gen(i)).to(dev) * 0.1
                p.grad = slope + torch.randn(p.shape, generator=gen(1000 + 10 * t + i)).to(dev) * 0.1
            opt.step()
        ways.append(torch.cat([(p.detach() - s).flatten() for p, s in zip(params, start)]))
    assert (ways[0] - ways[1]).norm() < 0.1 * ways[0].norm()


def test_captured_steps_replay(dev):
    for bits in (32, 8):
        params, twins = model(dev, torch.bfloat16), model(dev, torch.bfloat16)
        lr = torch.full((), 1e-2, device=dev)
        options = dict(state_bits=bits, master_weights=True, max_norm=0.5)
        opt, eager = pkg.AdamW(params, lr=lr, capturable=True, **options), pkg.AdamW(twins, lr=lr, capturable=True, **options)
        for ps, o in ((params, opt), (twins, eager)):
            set_grads(ps, 0)
            o.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        for t in range(1, 5):
            for ps in (params, twins):
                g = gen(t)
                for p in ps:
                    p.grad.copy_((torch.randn(p.shape, generator=g) * 0.1).to(p.dtype))
            lr.fill_(1e-2 / t)
            graph.replay()
            torch.cuda.synchronize()
            eager.step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(params, twins))
            for p, q in zip(params, twins):
                assert all(torch.equal(v.float(), eager.state[q][k].float()) for k, v in opt.state[p].items())
        assert opt.param_groups[0]["steps"].item() == 5
        again = pkg.AdamW(model(dev, torch.bfloat16), lr=lr, capturable=True, **options)
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["steps"].item() == 5 and again.param_groups[0]["steps"] is not opt.param_groups[0]["steps"]


def test_captured_steps_that_cannot_replay_are_refused(dev):
    params = model(dev, torch.float32)
    set_grads(params, 0)
    for opt, match in ((pkg.AdamW(params), "capturable"), (pkg.AdamW(params, capturable=True), "ahead of the capture")):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=match):
            with torch.cuda.graph(graph):
                opt.step()
        torch.cuda.synchronize()


def test_a_training_step_of_a_routed_block(dev):
    """Embedding, residual stream, norm, routing, experts, loss, clipping and step, as they are used together: the loss's gradients
    reach every parameter, and every parameter moves by less than a few steps' way."""
    torch.manual_seed(3)
    from fp8_gmm_amd import moe_ops

    embed = pkg.Embedding(100, 64, device=dev)
    norm = pkg.RMSNorm(64, device=dev)
    layer = moe.Fp8MlpModule(64, 128, 8, 2, device=dev, routing=moe_ops.Routing("sigmoid", True, 4, 2, True))
    params = [*embed.parameters(), *norm.parameters(), *layer.parameters()]
    opt = pkg.AdamW(params, lr=1e-3, master_weights=True, max_norm=1.0, state_bits=8)
    ids = torch.randint(0, 100, (300,), generator=gen(1)).to(dev)
    with pkg.fp8_autocast(fp8_recipe=pkg.DelayedScaling(amax_history_len=4)):
        for _ in range(3):
            before = [p.detach().clone() for p in params]
            opt.zero_grad()
            stream = embed(ids)
            rows, stream = norm(layer.gating_network.weight.new_zeros(300, 64), stream)
            out = stream + layer(rows)
            out.float().square().mean().backward()
            assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in params)
            opt.step()
            load = layer.tokens_per_expert.float()
            layer.expert_bias += 1e-3 * torch.sign(load.mean() - load)
            # the first steps' ways are at most lr / (1 - beta1) of a root's worth; decay and bf16 on top
            assert all(((p.detach() - b).float().abs() <= 2e-2 + 2 ** -7 * b.float().abs()).all() for p, b in zip(params, before))
    assert torch.isfinite(opt.grad_norm) and sum(opt.state[p]["step"] for p in params) == 3 * len(params)
    assert int(layer.tokens_per_expert.sum()) == 600
