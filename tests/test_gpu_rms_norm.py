"""Root-mean-square norm, with the residual's addition, in 8 bits and with its gradients, on the GPU against plain implementations in
64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, h half a step of the result's type (``finfo.eps / 2``).  A sum of a row
is taken by at most 1024 threads, each over cols / threads elements (at most 32 where a row fits the registers), then by halving and
over at most 16 wavefronts: K(cols) = 64 + cols / 1024 additions bound its error by K u times the sum of the magnitudes, and a factor of 2
covers the products around it.  The squares are positive: r is off by at most k r, k = 2 K u."""
import pytest
import torch
import torch.utils.checkpoint

import fp8_gmm_amd as pkg
from fp8_gmm_amd import backend

from helpers import gen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAIRS = [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")]
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half a step of the type's subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def assert_within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} are off, by up to {(off / tol)[bad].max().item():.3g} of what is allowed"


def inputs(dev, rows, cols, t, p, seed):
    g = gen(seed)
    x = (torch.randn(rows, cols, generator=g) * 2 + torch.randn(1, cols, generator=g)).to(TYPES[t]).to(dev)
    residual = (torch.randn(rows, cols, generator=g) * 3).to(TYPES[t]).to(dev)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(TYPES[p]).to(dev)
    dy = (0.1 * torch.randn(rows, cols, generator=g)).to(TYPES[t]).to(dev)
    dh = (0.1 * torch.randn(rows, cols, generator=g)).to(TYPES[t]).to(dev)
    return x, residual, w, dy, dh


def reference(h, w, dy, dh, eps):
    """(y, dx, dw) in 64 bits, and the bound of each one's error in 32 bits (without the final rounding)."""
    h, w, dy = h.double(), w.double(), dy.double()
    rows, cols = h.shape
    k = 2 * (64 + cols / 1024) * U
    r = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    z = h * r
    y, g = z * w, dy * w
    m = (g * z).mean(1, keepdim=True)
    dx = r * (g - z * m) + (dh.double() if dh is not None else 0.0)
    tol_x = 3 * k * r * (g.abs() + z.abs() * (g * z).abs().mean(1, keepdim=True)) + 2 * U * (dx.abs() + (dh.double().abs() if dh is not None else 0.0))
    # rows: some per thread, in at least 64 slices where there are so many, then over the slices
    tol_w = (64 + rows / 64) * U * (dy * z).abs().sum(0) + k * (dy * z).abs().sum(0)
    return (y, dx, (dy * z).sum(0)), (k * y.abs() + 2 * U * y.abs(), tol_x, tol_w)


def check(x, residual, w, dy, dh, eps=1e-5, what=""):
    leaves = [t.detach().requires_grad_() for t in (x, w)] + ([residual.detach().requires_grad_()] if residual is not None else [])
    out = pkg.rms_norm(leaves[0], leaves[1], eps, leaves[2] if residual is not None else None)
    y, h = out if residual is not None else (out, None)
    with torch.no_grad():
        again = pkg.rms_norm(x, w, eps, residual)
        for a, b in zip((again,) if residual is None else again, (y, h)):
            assert torch.equal(a, b), f"{what}: inference differs from training"
    rows = x
    if residual is not None:
        rows = (x.float() + residual.float()).to(x.dtype)
        assert torch.equal(h, rows) and h.is_contiguous(), f"{what}: the sum"
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    outs, grads = ((y,), (dy,)) if residual is None or dh is None else ((y, h), (dy, dh))
    got = torch.autograd.grad(outs, leaves, grads)
    if residual is not None:
        assert torch.equal(got[0], got[2])
    flat = [t.reshape(-1, x.shape[-1]) for t in (rows, dy)]
    want, tol = reference(flat[0], w, flat[1], dh.reshape(flat[0].shape) if residual is not None and dh is not None else None, eps)
    for a, v, e, name in zip((y, got[0], got[1]), want, tol, ("y", "dx", "dw")):
        assert_within(a.detach().reshape(v.shape), v, e + half_step(a.dtype) * (v.abs() + e) + smallest(a.dtype), f"{what} {name}")
    return y.detach(), got[0], got[1]


SHAPES = [(1, 1), (3, 7), (5, 64), (40, 127), (17, 129), (33, 512), (7, 1000), (129, 1411), (65, 2048), (1531, 1024), (9, 4097),
          (300, 4096), (3, 8191), (5, 16384), (700, 768), (5000, 24), (2, 40000)]
# columns on both sides of where a row takes another number of threads, of pieces per thread, or another kernel
SHAPES += [(37, c + d) for c in (4, 8, 64, 128, 256, 384, 512, 768, 1024, 1536, 2048, 4096, 6144, 8192, 16384) for d in (-1, 0, 1, 8)]
SHAPES += [(1001, c) for c in (192, 193, 384, 385)] + [(70000, 129), (3, 32768)]


@pytest.mark.parametrize("rows, cols", SHAPES)
@pytest.mark.parametrize("t, p", PAIRS)
def test_against_64_bits(dev, rows, cols, t, p):
    x, residual, w, dy, dh = inputs(dev, rows, cols, t, p, 100 + rows + cols)
    with_residual = (rows + cols) % 3 != 0
    check(x, residual if with_residual else None, w, dy, dh if (rows + cols) % 2 else None, what=f"{rows} x {cols}")


@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (64, 4096), (129, 1411), (37, 2048), (5, 8192), (3, 16385), (2, 40000), (1531, 1024),
                                        (4001, 100), (33, 24)])
@pytest.mark.parametrize("t, p", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_in_8_bits(dev, rows, cols, t, p, fmt):
    x, residual, w, _, _ = inputs(dev, rows, cols, t, p, 7 + rows + cols)
    dtype, most = FP8[fmt], torch.finfo(FP8[fmt]).max
    for add in (None, residual):
        h = x if add is None else (x.float() + add.float()).to(x.dtype)
        (y, _, _), (tol, _, _) = reference(h, w, x, None, 1e-6)

        def check_codes(q, scaled, bound, what):
            want = scaled.clamp(-most, most)
            assert q.dtype == dtype and q.shape == x.shape
            assert_within(q, want, bound + half_step(dtype) * (want.abs() + bound) + smallest(dtype), f"{what} {rows} x {cols}")

        # by the tensor's scale, the largest values beyond what 8 bits hold
        largest = y.abs().max()
        scale = (1.5 * most / largest).float().reshape(1)
        amax = torch.zeros(3, device=dev)
        q, none, sum_ = pkg.rms_norm_fp8(x, w, 1e-6, add, scale, amax[1:2], dtype)
        assert none is None and (sum_ is None if add is None else torch.equal(sum_, h))
        check_codes(q, y * scale.double(), (tol + 2 * U * y.abs()) * scale.double(), "tensor")
        assert amax[0] == 0 and amax[2] == 0
        assert_within(amax[1], largest, tol.max(), "amax")
        before = (2 * largest).float()
        amax[1] = before   # only ever raised
        pkg.rms_norm_fp8(x, w, 1e-6, add, scale, amax[1:2], dtype)
        assert amax[1] == before
        assert torch.equal(pkg.rms_norm_fp8(x, w, 1e-6, add, scale, None, dtype)[0].float(), q.float())
        # by every row's
        q, inv, sum_ = pkg.rms_norm_fp8(x, w, 1e-6, add, dtype=dtype)
        assert inv.shape == (rows,) and inv.dtype == torch.float32 and (sum_ is None if add is None else torch.equal(sum_, h))
        exact = y.abs().max(1).values / most
        k = 2 * (64 + cols / 1024) * U
        assert_within(inv, exact, (k + 4 * U) * exact, "scale_inv")
        check_codes(q, y / exact[:, None], (2 * k + 8 * U) * (y / exact[:, None]).abs(), "rows")


def test_in_8_bits_feeds_a_product(dev):
    """Delayed scaling: the codes, their scale's inverse and a weight in 8 bits through this package's product."""
    x, residual, w, _, _ = inputs(dev, 96, 256, "bf16", "bf16", 3)
    weight = (torch.randn(128, 256, generator=gen(4)) * 0.05).to(dev)
    w8 = (weight * 1000).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale, amax = torch.full((1,), 50.0, device=dev), torch.zeros(1, device=dev)
    q, _, h = pkg.rms_norm_fp8(x, w, 1e-5, residual, scale, amax)
    out = torch.empty(96, 128, dtype=torch.bfloat16, device=dev)
    backend.cublas_fp8_gemm(q, w8, out, 1 / scale, torch.full((1,), 1e-3, device=dev))
    want = (q.double() / 50) @ (w8.double() / 1000).t()
    bound = (q.double().abs() / 50) @ (w8.double().abs() / 1000).t() * 256 * U
    assert_within(out, want, bound * 2 + (half_step(torch.bfloat16) * 1.01) * (want.abs() + bound), "product")
    y = pkg.rms_norm(h, w, 1e-5)
    assert abs(amax.item() - y.abs().max().item()) <= half_step(torch.bfloat16) * 1.01 * amax.item()


def test_rows_of_zeros_and_what_is_no_number(dev):
    x = torch.randn(6, 300, generator=gen(1)).to(dev)
    w = torch.ones(300, device=dev)
    x[1] = 0.0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    x[4] = 1e30   # squares past fp32
    y = pkg.rms_norm(x, w, 1e-5)
    assert torch.isfinite(y[[0, 1, 5]]).all() and not y[1].any() and y[3].isnan().all() and not y[4].any()
    assert y[2, 7].isnan() and not y[2, :7].any()
    q, inv, _ = pkg.rms_norm_fp8(x, w, 1e-5)
    assert not q[1].float().any() and 0 < inv[1] < 1e-30 and q[3].float().isnan().all() and not q[4].float().any()
    assert torch.isfinite(inv[[0, 1, 3, 4, 5]]).all()
    xs = x.requires_grad_()
    dx, = torch.autograd.grad(pkg.rms_norm(xs, w, 1e-5), xs, torch.ones_like(x))
    assert torch.isfinite(dx[[0, 1, 5]]).all()
    zero = torch.zeros(1, 64, device=dev)
    assert pkg.rms_norm(zero, torch.ones(64, device=dev), 0.0).isnan().all()


def test_views_and_their_gradients(dev):
    x, residual, w, dy, dh = inputs(dev, 24, 650, "bf16", "bf16", 7)
    want = check(x, residual, w, dy, dh)
    wide = torch.empty(24, 1301, dtype=x.dtype, device=dev)
    wide[:, 3:653] = x
    dwide = torch.empty(24, 900, dtype=x.dtype, device=dev)
    dwide[:, 1:651] = dy
    flat = torch.empty(24 * 650 + 1, dtype=x.dtype, device=dev)
    flat[1:] = residual.reshape(-1)
    cases = [("pitch", wide[:, 3:653], residual, dwide[:, 1:651], dh), ("at an odd element", x, flat[1:].view(24, 650), dy, dh),
             ("three dimensions", *(t.view(2, 12, 650) for t in (x, residual, dy, dh))),
             ("transposed", *(t.t().contiguous().t() for t in (x, residual, dy, dh)))]
    for name, *tensors in cases:
        got = check(tensors[0], tensors[1], w, tensors[2], tensors[3], what=name)
        for a, c in zip(got, want):
            assert torch.equal(a.reshape(c.shape), c), name
    for dv in (dy[:1].expand(24, 650), torch.full((1, 1), 0.5, dtype=x.dtype, device=dev).expand(24, 650)):
        check(x, residual, w, dv, dv, what="expanded")
    check(x, residual, w, torch._neg_view(-dy), torch._neg_view(-dh), what="negated")
    with torch.no_grad():
        a = pkg.rms_norm_fp8(wide[:, 3:653], w, 1e-5, flat[1:].view(24, 650))
        b = pkg.rms_norm_fp8(x, w, 1e-5, residual)
        assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


def test_without_rows_and_with_some_gradients(dev):
    x, residual, w, dy, dh = inputs(dev, 12, 96, "bf16", "fp32", 5)
    empty = x[:0].requires_grad_()
    ws = w.clone().requires_grad_()
    y, h = pkg.rms_norm(empty, ws, 1e-5, x[:0])
    assert y.shape == h.shape == (0, 96)
    dx, dw = torch.autograd.grad((y, h), (empty, ws), (x[:0], x[:0]))
    assert dx.shape == (0, 96) and not dw.any()
    q, inv, _ = pkg.rms_norm_fp8(x[:0], w)
    assert q.shape == (0, 96) and inv.shape == (0,)
    want = check(x, residual, w, dy, dh)
    xs, rs = x.clone().requires_grad_(), residual.clone().requires_grad_()
    y, h = pkg.rms_norm(x, w, 1e-5, rs)      # the residual alone
    assert torch.equal(torch.autograd.grad((y, h), rs, (dy, dh))[0], want[1])
    y, h = pkg.rms_norm(x, ws, 1e-5, residual)
    assert torch.equal(torch.autograd.grad(y, ws, dy)[0], want[2])
    y, h = pkg.rms_norm(xs, w, 1e-5, rs)     # the sum alone goes on
    assert all(torch.equal(g, dh) for g in torch.autograd.grad(h, (xs, rs), dh))
    y, h = pkg.rms_norm(xs, w, 1e-5, xs.detach())
    both = pkg.rms_norm(xs, w, 1e-5, xs)     # the rows are their own residual
    a, = torch.autograd.grad(both, xs, (dy, dh))
    b, = torch.autograd.grad((y, h), xs, (dy, dh))
    assert torch.allclose(a.float(), 2 * b.float(), rtol=2 ** -7)
    leaves = [t.clone().requires_grad_() for t in (x, residual)]   # each has a gradient of its own
    for used in ((0, 1), (1,)):
        for t in leaves:
            t.grad = None
        results = pkg.rms_norm(leaves[0], w, 1e-5, leaves[1])
        torch.autograd.backward([results[i] for i in used], [(dy, dh)[i] for i in used])
        kept = leaves[1].grad.clone()
        leaves[0].grad.zero_()
        assert torch.equal(leaves[1].grad, kept) and kept.any() and dh.any()
    one = pkg.rms_norm(x[0], w)              # a vector
    assert one.shape == (96,) and torch.equal(one, pkg.rms_norm(x[:1], w)[0])
    q, inv, _ = pkg.rms_norm_fp8(x[0], w)
    assert q.shape == (96,) and inv.shape == ()


def test_gradients_against_differences(dev):
    x, residual, w, dy, dh = (t.float() for t in inputs(dev, 6, 40, "fp32", "fp32", 9))
    leaves = [t.requires_grad_() for t in (x, residual, w)]
    y, h = pkg.rms_norm(leaves[0], leaves[2], 1e-5, leaves[1])
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))

    def value(a, r, b):
        a, r, b = a.double(), r.double(), b.double()
        s = a + r
        return ((s / (s.square().mean(1, keepdim=True) + 1e-5).sqrt() * b) * dy.double()).sum() + (s * dh.double()).sum()

    for i, t in enumerate(leaves):
        step = torch.randn(t.shape, generator=gen(20 + i)).to(dev) * 1e-4
        # in 64 bits of numbers that fp32 holds: the third derivative's share is below 1e-8 of the step's
        moved = [[s.detach().double() + (d * step.double() if s is t else 0) for s in leaves] for d in (1, -1)]
        slope = (value(*moved[0]) - value(*moved[1])) / 2
        assert abs(slope.item() - (grads[i].double() * step.double()).sum().item()) < 1e-5 * (grads[i].abs() * step.abs()).sum().item() + 1e-9


def test_past_32_bits(dev):
    rows, cols = (1 << 20) + 37, 2304   # 2.4e9 elements
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    x[:] = torch.randn(cols, generator=gen(3)).to(dev)
    x[-40:] = torch.randn(40, cols, generator=gen(5)).to(dev)
    w = torch.randn(cols, generator=gen(4)).to(dev).requires_grad_()
    last = x[-40:].clone()
    with torch.no_grad():
        assert torch.equal(pkg.rms_norm(x, w)[-40:], pkg.rms_norm(last, w))
        y, h = pkg.rms_norm(x, w, 1e-5, x)
        small = pkg.rms_norm(last, w, 1e-5, last)
        assert torch.equal(y[-40:], small[0]) and torch.equal(h[-40:], small[1])
        del y, h
        q, inv, _ = pkg.rms_norm_fp8(x, w)
        want = pkg.rms_norm_fp8(last, w)
        assert torch.equal(q[-40:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(inv[-40:], want[1])
        del q, inv
    xs = x.requires_grad_()
    dx, = torch.autograd.grad(pkg.rms_norm(xs, w.detach()), xs, x.detach())
    ls = last.requires_grad_()
    assert torch.equal(dx[-40:], torch.autograd.grad(pkg.rms_norm(ls, w.detach()), ls, last.detach())[0])


def test_refusals(dev):
    x, residual, w, dy, _ = inputs(dev, 4, 32, "bf16", "bf16", 1)
    one = torch.ones(1, device=dev)
    bad = [lambda: pkg.rms_norm(x, w[:31]), lambda: pkg.rms_norm(x, w.half()), lambda: pkg.rms_norm(x, w, -1.0),
           lambda: pkg.rms_norm(x, w, 1e-5, residual[:3]), lambda: pkg.rms_norm(x, w, 1e-5, residual.float()),
           lambda: pkg.rms_norm(x, w, 1e-5, residual.cpu()), lambda: pkg.rms_norm(x.double(), w), lambda: pkg.rms_norm(x, w, float("nan")),
           lambda: pkg.rms_norm_fp8(x, w, dtype=torch.float16), lambda: pkg.rms_norm_fp8(x, w, scale=one.double()),
           lambda: pkg.rms_norm_fp8(x, w, scale=torch.ones(2, device=dev)), lambda: pkg.rms_norm_fp8(x, w, amax=one),
           lambda: pkg.rms_norm_fp8(x, w, scale=one, amax=one), lambda: pkg.rms_norm_fp8(x, w, scale=one.cpu()),
           lambda: pkg.rms_norm_fp8(x.clone().requires_grad_(), w)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print(i)
    xs = x.clone().requires_grad_()
    y, h = pkg.rms_norm(xs, w, 1e-5, residual)
    g, = torch.autograd.grad((y, h), xs, (dy, dy), create_graph=True)
    leaf = x.float().requires_grad_()
    gg, = torch.autograd.grad(pkg.rms_norm(leaf, w.float()), leaf, dy.float().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        gg.sum().backward()
    y, h = pkg.rms_norm(xs, w, 1e-5, residual)
    h.add_(1)   # the backward pass needs it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    with pytest.raises(RuntimeError, match="transforms or tracing"):
        torch.func.vmap(lambda t: pkg.rms_norm(t, w))(x)


def test_other_streams_and_captured_passes(dev):
    x, residual, w, dy, dh = inputs(dev, 300, 1024, "bf16", "fp32", 11)
    want = check(x, residual, w, dy, dh)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = check(x, residual, w, dy, dh)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    scale, amax = torch.full((1,), 20.0, device=dev), torch.zeros(1, device=dev)
    xs, rs, ws = (t.clone().requires_grad_() for t in (x, residual, w))

    def step():
        y, h = pkg.rms_norm(xs, ws, 1e-5, rs)
        grads = torch.autograd.grad((y, h), (xs, ws), (dy, dh))
        with torch.no_grad():
            q, _, _ = pkg.rms_norm_fp8(xs, ws, 1e-5, rs, scale, amax)
        return (y.detach(), h.detach(), *grads, q.view(torch.uint8))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (21, 22, 23):
        fresh = inputs(dev, 300, 1024, "bf16", "fp32", seed)
        with torch.no_grad():
            xs.copy_(fresh[0])
            rs.copy_(fresh[1])
            ws.copy_(fresh[2])
            amax.zero_()
        graph.replay()
        torch.cuda.synchronize()
        copies, most = [t.clone() for t in held], amax.item()
        amax.zero_()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(copies, eager)) and amax.item() == most > 0
        del eager


def test_saved_tensors_are_looked_after(dev):
    """Hooks that move what is saved, a second pass over a freed graph, rows that were changed in place, checkpointing."""
    x, residual, w, dy, dh = inputs(dev, 30, 500, "bf16", "bf16", 21)
    want = check(x, residual, w, dy, dh)
    leaves = [t.detach().requires_grad_() for t in (x, residual, w)]

    def norm(a, r, b):
        return pkg.rms_norm(a, b, 1e-5, r)

    def check_grads(outs):
        got = torch.autograd.grad(outs, leaves, (dy, dh))
        assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])

    with torch.autograd.graph.save_on_cpu():
        outs = norm(*leaves)
    check_grads(outs)
    with pytest.raises(RuntimeError):
        check_grads(outs)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        outs = norm(*leaves)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        check_grads(outs)
    rows = leaves[0] * 1.0
    y = pkg.rms_norm(rows, leaves[2])
    rows.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves[2], dy)
    check_grads(torch.utils.checkpoint.checkpoint(norm, *leaves, use_reentrant=False))
    outs = norm(*leaves)
    check_outs = [o.clone() for o in outs]
    del outs   # (the sum is a result of the node that keeps it)
    assert torch.autograd.grad(check_outs, leaves, (dy, dh))[2].shape == (500,)


def test_gradients_with_tangents_are_refused(dev):
    x, w = (torch.randn(s, device=dev, requires_grad=True) for s in ((6, 32), (32,)))
    dy = torch.randn(6, 32, device=dev)
    for outs in (lambda: (pkg.rms_norm(x, w),), lambda: pkg.rms_norm(x, w, 1e-5, x.detach())):
        for i in range(len(outs())):
            with torch.autograd.forward_ad.dual_level():
                up = [torch.autograd.forward_ad.make_dual(dy, torch.ones_like(dy)) if j == i else dy for j in range(len(outs()))]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch.autograd.grad(outs(), x, up)


@pytest.mark.parametrize("rows, cols, t", [(20000, 4096, "bf16"), (9000, 4093, "fp32"), (9000, 4096, "fp32"), (70000, 512, "fp16")])
def test_results_that_outgrow_the_cache(dev, rows, cols, t):
    """Written with the streaming hint, by workgroups with several turns; row by row the bits of a few rows' call."""
    x, residual, w, dy, dh = inputs(dev, rows, cols, t, t, 3)
    with torch.no_grad():
        y, h = pkg.rms_norm(x, w, 1e-5, residual)
        q, inv, _ = pkg.rms_norm_fp8(x, w, 1e-5, residual)
        plain = pkg.rms_norm(x, w, 1e-5)
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(pkg.rms_norm(leaf, w, 1e-5, residual), leaf, (dy, dh))
    for part in (slice(0, 50), slice(rows // 2, rows // 2 + 50), slice(rows - 50, rows)):
        few = x[part].clone().requires_grad_()
        a, b = pkg.rms_norm(few, w, 1e-5, residual[part])
        assert torch.equal(a, y[part]) and torch.equal(b, h[part])
        assert torch.equal(torch.autograd.grad((a, b), few, (dy[part], dh[part]))[0], dx[part])
        with torch.no_grad():
            assert torch.equal(pkg.rms_norm(x[part], w, 1e-5), plain[part])
            c, d, _ = pkg.rms_norm_fp8(x[part], w, 1e-5, residual[part])
            assert torch.equal(c.view(torch.uint8), q[part].view(torch.uint8)) and torch.equal(d, inv[part])


def test_more_columns_than_a_grid_has_threads_for(dev):
    """Weights' gradients of rows of more than 2^28 columns.  Rows of 1 and -1: their squares and their sum are exact, the factor is 1 to
    a few 2^-24, and the gradients are dy and its negative, rounded to bfloat16."""
    cols = (1 << 28) + 70
    x = torch.ones(1, cols, dtype=torch.bfloat16, device=dev)
    x[:, 1::2] = -1
    dy = torch.randn(1, 1 << 20, generator=gen(1)).to(torch.bfloat16).to(dev).repeat(1, 257)[:, :cols].contiguous()
    w, b = (torch.ones(cols, dtype=torch.bfloat16, device=dev).requires_grad_() for _ in range(2))
    for norm, bias in ((pkg.rms_norm(x, w, 0.0), None), (pkg.layer_norm(x, w, b, 0.0), b)):
        grads = torch.autograd.grad(norm, (w,) if bias is None else (w, b), dy)
        assert torch.equal(grads[0], (dy * x)[0])
        assert bias is None or torch.equal(grads[1], dy[0])
        del norm, grads


@pytest.mark.parametrize("cols", [64, 1000, 16384, 100001, 1 << 20])
@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_codes_by_rows_follow_the_stated_operations(dev, cols, fmt):
    """Rows of 1 and -1 have a factor of 1, so y is the weight, in fp32: q = fp8(y (largest / most)), scale_inv = most / largest, bit by bit."""
    x = torch.ones(3, cols, device=dev)
    x[:, ::2] = -1
    largest = torch.finfo(fmt).max
    for seed in range(4):
        w = torch.randn(cols, generator=gen(seed)).to(dev)
        q, scale_inv, _ = pkg.rms_norm_fp8(x, w, 0.0, dtype=fmt)
        most = w.abs().max().cpu()
        by = torch.tensor(largest) / most   # (of the CPU, whose division is correctly rounded)
        want = ((x * w).cpu() * by).clamp(-largest, largest).to(fmt)
        assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))
        assert (scale_inv.cpu() == most / torch.tensor(largest)).all()
