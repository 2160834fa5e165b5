"""The global norm of many tensors and clipping by it, on the GPU, against 64 bits.

The squares are added up in fp64 and the norm is rounded to fp32 once: it is off by at most u = 2^-24 of itself.  The factor is
rounded to fp32 once, its product with a gradient once, and the result once more to its type: half a step of that and 2 u."""
import math

import pytest
import torch

import fp8_gmm_amd as pkg
from fp8_gmm_amd import backend

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def tensors_of(dev, sizes, types, seed=0, std=1e-2):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=dev) * std * (1 + i % 5)).to(types[i % len(types)]) for i, n in enumerate(sizes)]


def norm_of(tensors):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in tensors))


def check_scaled(got, grads, factor):
    for a, t in zip(got, grads):
        want = t.double() * factor
        h = torch.finfo(a.dtype).eps / 2
        tiny = torch.finfo(a.dtype).smallest_normal * h
        bad = ~((a.double() - want).abs() <= (h + 2.01 * U) * want.abs() + tiny)
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values are off"


def check_clip(grads, outs, max_norm):
    """Norm and results of one call; ``outs`` may be ``grads``."""
    before = [t.clone() for t in grads]
    norm = norm_of(before)
    got = backend.multi_clip(grads, outs, max_norm)
    assert got.dtype == FP32 and got.dim() == 0
    assert abs(got.item() - norm) <= 1.01 * U * norm
    alone = backend.multi_norm(before)
    assert torch.equal(alone, got)
    factor = min(1.0, max_norm / (norm + 1e-6))
    check_scaled(outs, before, factor)
    if factor == 1.0:
        for a, t in zip(outs, before):
            assert torch.equal(a, t.to(a.dtype))
    if outs is not grads:
        for t, c in zip(grads, before):
            assert torch.equal(t, c), "the tensors were written"
    return norm


SIZES = {
    "one": [1], "one value each": [1] * 7, "odd": [3, 1, 4097, 129, 65535, 17], "none among them": [0, 5, 0, 8192, 8193, 0],
    "chunks": [8192, 4096, 16384, 8191, 8193], "all empty": [0, 0], "more than a launch": [50 + 37 * i % 900 for i in range(300)],
    "many partial sums": [20000 + i for i in range(900)],
    **{f"{n} tensors": [1 + 41 * i % 300 for i in range(n)] for n in (64, 65, 112, 113, 200, 201, 400, 401)},
    "a long one among short ones": [10] * 150 + [3000001] + [20] * 150,
}


@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
@pytest.mark.parametrize("types", [[BF16], [FP16], [FP32], [FP32, BF16, FP16, BF16]], ids=["bf16", "fp16", "fp32", "mixed"])
def test_norm_and_clip(dev, sizes, types):
    grads = tensors_of(dev, sizes, types, seed=len(sizes))
    norm = norm_of(grads)
    check_clip(grads, [torch.empty_like(t) for t in grads], 0.25 * norm)
    check_clip(grads, [torch.empty(t.shape, device=dev) for t in grads], 0.3 * norm + 1e-3)
    check_clip(grads, [torch.empty(t.shape, dtype=t.dtype if i % 2 else FP32, device=dev) for i, t in enumerate(grads)], 1e-3)
    check_clip(grads, grads, 4 * norm + 1.0)     # within the bound, in place
    check_clip(grads, [torch.empty_like(t) for t in grads], math.inf)
    check_clip(grads, grads, 0.5 * norm)         # in place
    check_clip(grads, grads, 0.0)
    assert not any(t.any() for t in grads)


def test_packed_tensors_begin_at_any_element(dev):
    """Views of a bucket, one behind the other, and results in another: nothing between or beside them is written."""
    sizes = [7, 1, 8200, 33, 4095, 64, 16385, 2]
    for t, o in ((BF16, FP32), (FP16, FP16), (FP32, FP32)):
        flat = torch.randn(sum(sizes) + 9, device=dev).to(t)
        out = torch.full((sum(sizes) + 9 + len(sizes),), 7.0, dtype=o, device=dev)
        grads = list(flat[5:5 + sum(sizes)].split(sizes))
        outs, at = [], 3
        for n in sizes:
            outs.append(out[at: at + n])
            at += n + 1
        check_clip(grads, outs, 1.0)
        gaps = torch.ones_like(out, dtype=torch.bool)
        at = 3
        for n in sizes:
            gaps[at: at + n] = False
            at += n + 1
        assert (out[gaps] == 7.0).all()
        edge = flat.clone()
        check_clip(grads, grads, 1.0)
        assert torch.equal(flat[:5], edge[:5]) and torch.equal(flat[5 + sum(sizes):], edge[5 + sum(sizes):])


def test_shapes_and_strides(dev):
    g = torch.Generator(device=dev).manual_seed(2)
    base = torch.randn(24, 36, generator=g, device=dev)
    grads = [base.t(), torch.randn(4, 5, 6, 7, generator=g, device=dev).permute(2, 0, 3, 1), torch.randn(40, 30, generator=g, device=dev)[::2, 3:17],
             torch.randn((), generator=g, device=dev), torch.randn(0, 4, device=dev), torch.randn(10, 1, generator=g, device=dev).expand(10, 8)]
    check_clip(grads, [torch.empty(t.shape, device=dev) for t in grads], 0.5)
    outs = [torch.zeros(t.shape[::-1], device=dev).permute(list(range(t.dim() - 1, -1, -1))) for t in grads]   # other orders than their tensors
    check_clip(grads, outs, 0.5)
    room = [torch.full((2 * t.shape[0], 30), 7.0, device=dev) for t in grads[2:3]]
    check_clip(grads[2:3], [room[0][::2, 5:19]], 0.5)   # a result with gaps
    assert (room[0][1::2] == 7.0).all() and (room[0][:, :5] == 7.0).all() and (room[0][:, 19:] == 7.0).all()
    first = grads[:4]
    check_clip(first, first, 0.5)   # in place, one of them with gaps


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42, 3e38])
def test_norms_of_any_magnitude(dev, scale):
    """Squares that fp32 does not hold; 3e38: the norm itself lies past fp32 and is infinite there."""
    t = torch.randn(5000, device=dev).clamp(-1, 1) * scale if scale < 1e38 else torch.full((5000,), scale, device=dev)
    norm = norm_of([t])
    got = backend.multi_norm([t]).item()
    if norm > torch.finfo(FP32).max:
        assert got == math.inf
        return
    # subnormal norms: half a step of those
    assert abs(got - norm) <= 1.01 * U * norm + 2.0 ** -150
    out = torch.empty_like(t)
    backend.multi_clip([t], [out], norm / 2)
    check_scaled([out], [t], min(1.0, norm / 2 / (norm + 1e-6)))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_no_number(dev, value):
    """As torch's call: an infinite norm leaves zeros and NaN, a NaN leaves NaN."""
    for t in (BF16, FP16, FP32):
        grads = [torch.randn(3000, device=dev).to(t), torch.randn(77, device=dev)]
        grads[0][2999] = value
        theirs = [torch.nn.Parameter(torch.empty_like(x)) for x in grads]
        for p, x in zip(theirs, grads):
            p.grad = x.clone()
        want = torch.nn.utils.clip_grad_norm_(theirs, 1.0, foreach=False)
        got = backend.multi_clip(grads, grads, 1.0)
        assert torch.equal(got, want.float()) or (torch.isnan(got) and torch.isnan(want))
        for a, p in zip(grads, theirs):
            assert torch.equal(a.isnan(), p.grad.isnan()) and torch.equal(a.nan_to_num(), p.grad.nan_to_num())


def test_past_32_bits(dev):
    """One tensor of more than 2^31 elements beside a short one, in place."""
    n = (1 << 31) + 12345
    big = torch.empty(n, dtype=BF16, device=dev).fill_(2.0 ** -10)
    big[-1] = 3.0
    small = torch.full((5,), 2.0, device=dev)
    norm = math.sqrt((n - 1) * 2.0 ** -20 + 9.0 + 20.0)
    got = pkg.backend.multi_clip([big, small], [big, small], norm / 4).item()
    assert abs(got - norm) <= 1.01 * U * norm
    factor = norm / 4 / (norm + 1e-6)
    piece = torch.tensor([2.0 ** -10, 3.0], dtype=torch.float64) * factor
    assert abs(big[-1].item() - piece[1].item()) <= (2.0 ** -8 + 3 * U) * 3.0
    part = big[:-1].view(torch.int16)
    first = int(part[0])
    assert all(bool((p == first).all()) for p in part.split(1 << 28))
    assert abs(big[0].item() - piece[0].item()) <= (2.0 ** -8 + 3 * U) * piece[0].item()
    check_scaled([small], [torch.full((5,), 2.0, device=dev)], factor)


def test_results_are_the_same_from_call_to_call_and_side_by_side(dev):
    grads = tensors_of(dev, [20000 + 7 * i for i in range(200)], [BF16, FP32])
    first = [torch.empty_like(t) for t in grads]
    norm = backend.multi_clip(grads, first, 0.7)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs = [torch.empty_like(t) for t in grads]
            got.append((backend.multi_clip(grads, outs, 0.7), outs))
    torch.cuda.synchronize()
    for n, outs in got:
        assert torch.equal(n, norm) and all(torch.equal(a, c) for a, c in zip(outs, first))


def test_captured_clipping_replays(dev):
    """The table of the tensors is part of the graph: the lists that it was made from are gone."""
    grads = tensors_of(dev, [100 + 61 * i for i in range(150)], [BF16, FP32])
    outs = [torch.empty_like(t) for t in grads]
    backend.multi_clip(grads, outs, 0.7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = backend.multi_clip(list(grads), list(outs), 0.7)
    for k in range(4):
        for i, t in enumerate(tensors_of(dev, [t.numel() for t in grads], [BF16, FP32], seed=50 + k, std=10.0 ** -k)):
            grads[i].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = [torch.empty_like(t) for t in grads]
        assert torch.equal(backend.multi_clip(grads, want, 0.7), norm)
        assert all(torch.equal(a, c) for a, c in zip(outs, want))
        torch.randn(1 << 20, device=dev).sum().item()


def test_clip_grad_norm(dev):
    params = [torch.nn.Parameter(torch.zeros(s, device=dev, dtype=t)) for s, t in (((8, 64, 32), BF16), ((5,), FP32), ((3, 3), FP16))]
    params.append(torch.nn.Parameter(torch.zeros(4, device=dev)))   # without a gradient
    assert pkg.clip_grad_norm_(params, 1.0).item() == 0.0 and pkg.clip_grad_norm_([], 1.0).item() == 0.0
    for p in params[:3]:
        p.grad = torch.randn_like(p) * 0.1
    before = [p.grad.clone() for p in params[:3]]
    norm = norm_of(before)
    versions = [p.grad._version for p in params[:3]]
    got = pkg.clip_grad_norm_(iter(params), 0.3 * norm, foreach=True)   # a generator is walked through once
    assert abs(got.item() - norm) <= 1.01 * U * norm and not got.requires_grad
    check_scaled([p.grad for p in params[:3]], before, 0.3 * norm / (norm + 1e-6))
    assert all(p.grad._version > v for p, v in zip(params, versions)), "autograd does not see the change"
    single = params[1]
    single.grad = torch.full((5,), 3.0, device=dev)
    assert abs(pkg.clip_grad_norm_(single, 1.0).item() - math.sqrt(45.0)) <= 1.01 * U * math.sqrt(45.0)
    single.grad[2] = math.inf
    kept = single.grad.clone()
    with pytest.raises(RuntimeError, match="inf"):
        pkg.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert torch.equal(single.grad, kept)
    with pytest.raises(RuntimeError, match="2-norm"):
        pkg.clip_grad_norm_(params, 1.0, norm_type=1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        pkg.clip_grad_norm_([single, single], 1.0)
    single.grad = torch.zeros(1, device=dev).expand(5)
    with pytest.raises(RuntimeError):
        pkg.clip_grad_norm_(params, 1.0)


@pytest.mark.parametrize("slices", [lambda g: (g[:, :37], g[:, 37:100]), lambda g: (g[:, ::2], g[:, 1::2]), lambda g: (g[0::2], g[1::2], g[:0]),
                                    lambda g: (g.view(5, 10, 10, 10)[:, :, :3], g.view(5, 10, 10, 10)[:, :, 3:]), lambda g: (g[7:8, 3:], g[7, :3])],
                         ids=["columns", "every other column", "every other row", "inner", "a row"])
def test_slices_of_one_buffer_are_clipped_in_place(dev, slices):
    g = torch.Generator(device=dev).manual_seed(11)
    buffer = torch.randn(50, 100, generator=g, device=dev)
    parts, before = slices(buffer), buffer.clone()
    copies = [p.clone() for p in slices(before)]
    norm = norm_of(copies)
    got = backend.multi_clip(parts, parts, 0.5 * norm)
    assert abs(got.item() - norm) <= 1.01 * U * norm
    check_scaled(parts, copies, 0.5 * norm / (norm + 1e-6))
    assert sum(p.numel() for p in parts) == (buffer != before).sum().item()   # (half of no value is the value)


def test_strides_of_a_single_element_say_nothing(dev):
    flat = torch.ones(5, device=dev)
    norm = backend.multi_clip([flat.as_strided((1, 5), (7, 1))], [flat.as_strided((1, 5), (1, 1))], 1.0)
    assert abs(norm.item() - math.sqrt(5)) <= 1.01 * U * math.sqrt(5) and abs(flat[0].item() - 1 / math.sqrt(5)) < 1e-6


def test_refusals(dev):
    a, b = torch.ones(16, device=dev), torch.ones(16, device=dev)
    flat = torch.ones(40, device=dev)
    grid = torch.ones(6, 10, device=dev)
    wide = torch.ones(1, 4, 4, device=dev).expand(2, 4, 4)
    square = wide[1]
    leaf = torch.ones(16, device=dev, requires_grad=True)
    for ins, outs, what in (([a], [], "a result for every"), ([], [], "at least one"), ([a, b], [a, a], "overlaps"), ([a, b], [b, a], "overlaps"),
                            ([flat[:20], a], [flat[5:25], a], "overlaps"), ([flat[:20], flat[30:]], [b.new_empty(20), flat[10:20]], "overlaps"),
                            ([a], [a.half()], "shapes"), ([a], [torch.ones(4, 4, device=dev)], "shapes"), ([a.double()], [a], "bfloat16, float16 or float32"),
                            ([a], [a.cpu()], "GPU tensors"), ([a.cpu()], [a.cpu()], "GPU tensors"), ([a], [leaf], "requires a gradient"),
                            ([grid[:, :6], grid[:, 5:]], [grid[:, :6], grid[:, 5:]], "overlaps"),
                            ([grid[:4, :4]], [grid[:4, :4].t()], "overlaps"), ([grid[:4, :4], a], [grid[2:, 2:6], b], "overlaps"),
                            ([square.t(), a], [square, b], "overlaps"), ([a.view(4, 4).t(), b], [square, a], "overlaps"),
                            ([square, square], [square.new_empty(4, 4).t(), wide[0]], "overlaps"),
                            ([a.to_sparse()], [a], "dense")):
        with pytest.raises(RuntimeError, match=what):
            backend.multi_clip(ins, outs, 1.0)
    with torch.inference_mode():
        frozen = torch.ones(16, device=dev)
        backend.multi_clip([frozen], [frozen], 2.0)
    before = frozen.clone()
    with pytest.raises(RuntimeError, match="inference"):
        backend.multi_clip([frozen], [frozen], 1.0)
    with pytest.raises(RuntimeError, match="dense"):
        backend.multi_norm([torch._neg_view(a)])
    assert torch.equal(frozen, before) and (before == torch.tensor(2 / (4 + 1e-6), device=dev)).all()   # 16 ones have norm 4
    for bad in (-1.0, math.nan):
        with pytest.raises(RuntimeError, match="max_norm"):
            backend.multi_clip([a], [a], bad)
    with pytest.raises(RuntimeError):
        backend.multi_clip([a], [torch.ones(1, device=dev).expand(16)], 1.0)
    with pytest.raises(RuntimeError, match="at least one"):
        backend.multi_norm([])
    assert (a == 1).all() and (b == 1).all() and (flat == 1).all()


def test_transforms_tangents_and_tracing_are_refused(dev):
    """A result without its derivative would be a wrong one."""
    t, out = torch.ones(16, device=dev), torch.empty(16, device=dev)
    calls = {"multi_norm": lambda v: backend.multi_norm([out, v]), "multi_clip": lambda v: backend.multi_clip([out, v], [out, v], 1.0),
             "into another": lambda v: backend.multi_clip([out, v], [out, t], 1.0)}
    for name, call in calls.items():
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.vmap(call)(torch.ones(3, 16, device=dev))
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.grad(lambda v: call(v).sum())(t)
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.jit.trace(call, (t,), check_trace=False)
        for mode in (torch.enable_grad, torch.no_grad):
            with torch.autograd.forward_ad.dual_level(), mode():
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t)))
    leaf = torch.nn.Parameter(torch.ones(16, device=dev))
    with torch.autograd.forward_ad.dual_level():
        leaf.grad = torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t))
        with pytest.raises(RuntimeError, match="forward-mode"):
            pkg.clip_grad_norm_([leaf], 1.0)
    assert (t == 1).all()


@pytest.mark.parametrize("wider", [False, True], ids=["in place", "into fp32"])
def test_workgroups_with_several_chunks_cross_the_tensors_borders(dev, wider):
    """More chunks of 16 KB than the scaling has workgroups (2^20, or 2^19 by halves into fp32): some walk back over several, and over
    short tensors between long ones.  Every tensor holds one value, so its results are all the same bits."""
    long = 8192 * (((1 << 20) + (1 << 18)) // (16 if wider else 8)) + 4321
    sizes = [n for k in range(8) for n in [long + k] + [1 + (977 * (11 * k + j)) % 20000 for j in range(11)]]
    flat = torch.empty(sum(sizes), dtype=BF16, device=dev)
    grads = list(flat.split(sizes))
    values = [2.0 ** -12 * (1 + i % 7) for i in range(len(sizes))]
    for t, v in zip(grads, values):
        t.fill_(v)
    assert sum((2 * n + 16383) // 16384 for n in sizes) > ((1 << 20) if not wider else 1 << 19)
    outs = list(torch.full((sum(sizes),), 7.0, device=dev).split(sizes)) if wider else grads
    norm = math.sqrt(math.fsum(n * v * v for n, v in zip(sizes, values)))
    got = backend.multi_clip(grads, outs, 0.3 * norm)
    assert abs(got.item() - norm) <= 1.01 * U * norm
    factor = 0.3 * norm / (norm + 1e-6)
    for t, v in zip(outs, values):
        check_scaled([t[:1]], [torch.tensor([v], device=dev)], factor)
        bits = t.view(torch.int32 if wider else torch.int16)
        first = bits[0].item()
        assert all(bool((p == first).all()) for p in bits.split(1 << 28))
    if wider:
        assert all(bool((p == v).all()) for t, v in zip(grads, values) for p in t.split(1 << 28)), "the tensors were written"
