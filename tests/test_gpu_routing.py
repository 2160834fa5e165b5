"""The choice of experts and the gradient of its weights on the GPU, against a plain implementation in 64 bits.

The choice has to be equal: what 64 bits tell apart, the kernel does.  Tolerances of the weights: u = 2^-24.  A probability takes an
exponential (a unit in the last place, 2 u), a sum of at most 64 + 6 numbers that are not negative, and a division; the difference from
the row's largest score is rounded by u times its magnitude, which the exponential turns into a relative error: k = (80 + 2 max |s|) u.
Renormalizing divides two such: 2 k and 20 u of its sum."""
import pytest
import torch
import torch.utils.checkpoint

import fp8_gmm_amd as pkg
from fp8_gmm_amd import moe, moe_ops

from helpers import gen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(scores, top_k, scoring, bias, groups, top_groups, renormalize, scale, group_best):
    """(weights, selected) in 64 bits, on the CPU."""
    s = scores.detach().double().cpu()
    tokens, experts = s.shape
    p = torch.sigmoid(s) if scoring == "sigmoid" else torch.softmax(s, 1)
    plain = bias is None and (groups == 1 or group_best == 1)   # the scores decide
    c = s.clone() if plain else p if bias is None else p + bias.double().cpu()
    order = c.sort(dim=1, descending=True, stable=True).indices
    if groups > 1:
        parts = c.view(tokens, groups, -1)
        value = parts.sort(dim=2, descending=True).values[:, :, :group_best].sum(2)
        kept = value.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        stays = torch.zeros(tokens, groups, dtype=torch.long).scatter_(1, kept, 1).repeat_interleave(experts // groups, 1)
        order = order.gather(1, stays.gather(1, order).sort(dim=1, descending=True, stable=True).indices)
    selected = order[:, :top_k]
    w = p.gather(1, selected)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    return w * scale, selected


def check(scores, top_k, scoring="softmax", bias=None, groups=1, top_groups=1, renormalize=False, scale=1.0, group_best=2):
    s = scores.detach().requires_grad_()
    got_w, got_i = moe_ops.select_experts(s, top_k, scoring, bias, groups, top_groups, renormalize, scale, group_best)
    with torch.no_grad():
        again = moe_ops.select_experts(scores, top_k, scoring, bias, groups, top_groups, renormalize, scale, group_best)
        assert torch.equal(again[0], got_w) and torch.equal(again[1], got_i)
    assert got_w.dtype == torch.float32 and got_i.dtype == torch.int64 and got_w.shape == got_i.shape == (scores.shape[0], top_k)
    want_w, want_i = reference(scores, top_k, scoring, bias, groups, top_groups, renormalize, scale, group_best)
    assert torch.equal(got_i.cpu(), want_i), f"{int((got_i.cpu() != want_i).sum())} choices differ"
    k = (80 + 2 * scores.detach().float().abs().max().item()) * U * (2 if renormalize else 1) + (20 * U if renormalize else 0)
    off = (got_w.double().cpu() - want_w).abs()
    assert (off <= k * want_w.abs() + 1e-38).all(), (off / want_w.abs()).max().item() / k
    # the gradient
    dw = torch.randn(got_w.shape, generator=gen(5)).to(scores.device)
    ds, = torch.autograd.grad(got_w, s, dw)
    assert ds.dtype == scores.dtype and ds.shape == scores.shape
    x = scores.detach().double().cpu()
    p = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, 1)
    v = p.gather(1, want_i)
    total = v.sum(1, keepdim=True)
    g = dw.double().cpu() * scale
    part = g.abs()
    if renormalize:
        dot = (g * v).sum(1, keepdim=True)
        part = (g.abs() + (g * v).abs().sum(1, keepdim=True) / total) / total
        g = (g - dot / total) / total
    if scoring == "sigmoid":
        rest = torch.sigmoid(-x).gather(1, want_i)
        want = torch.zeros_like(p).scatter_(1, want_i, g * v * rest)
        bound = torch.zeros_like(p).scatter_(1, want_i, part * v * rest)
    else:
        want = p * (torch.zeros_like(p).scatter_(1, want_i, g) - (g * v).sum(1, keepdim=True))
        bound = p * (torch.zeros_like(p).scatter_(1, want_i, part) + (part * v).sum(1, keepdim=True))
    h = torch.finfo(scores.dtype).eps / 2
    tiny = torch.finfo(scores.dtype).smallest_normal * h * 2
    off = (ds.double().cpu() - want).abs()
    tol = 4 * k * bound
    assert (off <= tol + h * (want.abs() + tol) + tiny).all(), (off / (tol + h * (want.abs() + tol) + tiny)).max().item()
    return got_w.detach(), got_i, ds


def scores_of(dev, tokens, experts, t, seed, std=1.5):
    return (torch.randn(tokens, experts, generator=gen(seed)) * std).to(TYPES[t]).to(dev)


SIZES = [(1, 1, 1), (1, 8, 2), (5, 2, 2), (7, 16, 8), (33, 17, 3), (64, 31, 16), (100, 33, 4), (257, 64, 6), (130, 65, 8), (1000, 100, 8),
         (17, 128, 16), (301, 129, 8), (515, 256, 8), (9, 257, 5), (40, 511, 16), (21, 512, 8), (13, 513, 8), (6, 1024, 16), (5, 1025, 2),
         (3, 4096, 16)]


@pytest.mark.parametrize("tokens, experts, top_k", SIZES)
@pytest.mark.parametrize("t", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_against_64_bits(dev, tokens, experts, top_k, t, scoring):
    seed = tokens + experts
    scores = scores_of(dev, tokens, experts, t, seed)
    bias = (torch.randn(experts, generator=gen(seed + 1)) * (0.1 if scoring == "sigmoid" else 0.5 / experts)).to(dev)
    for b in (None, bias, torch.zeros_like(bias)):
        check(scores, top_k, scoring, b, renormalize=seed % 2 == 0, scale=2.5)


GROUPS = [(33, 16, 2, 1, 4), (65, 64, 8, 4, 8), (300, 256, 8, 4, 8), (300, 256, 8, 8, 8), (41, 160, 8, 3, 6), (41, 160, 16, 3, 16), (20, 60, 5, 2, 7),
          (9, 512, 16, 4, 8), (9, 384, 2, 1, 8), (5, 1024, 8, 2, 8), (3, 4096, 16, 16, 16), (50, 12, 12, 5, 5), (7, 9, 3, 1, 3), (64, 128, 4, 2, 1),
          (30, 48, 3, 2, 8), (30, 96, 6, 5, 8)]


@pytest.mark.parametrize("tokens, experts, groups, top_groups, top_k", GROUPS)
@pytest.mark.parametrize("t", ["bf16", "fp32"])
@pytest.mark.parametrize("scoring, best", [("softmax", 1), ("softmax", 2), ("sigmoid", 1), ("sigmoid", 2)])
def test_groups_against_64_bits(dev, tokens, experts, groups, top_groups, top_k, t, scoring, best):
    scores = scores_of(dev, tokens, experts, t, experts + groups, 1.0)
    bias = (torch.randn(experts, generator=gen(3)) * (0.1 if scoring == "sigmoid" else 0.5 / experts)).to(dev)
    for b in (None, bias):
        check(scores, top_k, scoring, b, groups, top_groups, True, 1.0, best)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, top_groups", [(1, 1), (8, 3)])
def test_equal_values_take_the_lower_number(dev, scoring, groups, top_groups):
    scores = torch.randint(-2, 3, (400, 128), generator=gen(1)).to(torch.bfloat16).to(dev)
    for b in (None, torch.zeros(128, device=dev), torch.randint(0, 2, (128,), generator=gen(2)).float().mul(0.25).to(dev)):
        check(scores, 8, scoring, b, groups, top_groups)
    same = torch.full((3, 128), 0.5, device=dev)
    _, selected, _ = check(same, 6, scoring, None, groups, top_groups)
    assert selected.tolist() == [[0, 1, 2, 3, 4, 5]] * 3
    signed = torch.zeros(2, 16, device=dev)
    signed[0, :8] = -0.0
    assert moe_ops.select_experts(signed, 3, scoring)[1].tolist() == [[0, 1, 2]] * 2


def test_values_that_32_bits_do_not_tell_apart(dev):
    """Sums with the bias that differ by 2^-30 of themselves have an order."""
    experts = 64
    scores = torch.zeros(1, experts, device=dev)
    scores[0] += torch.arange(experts, device=dev) * 2.0 ** -26   # p grows by 2^-28 from one to the next
    bias = torch.full((experts,), 0.25, device=dev)
    check(scores, 8, "sigmoid", bias)
    assert moe_ops.select_experts(scores, 8, "sigmoid", bias)[1][0].tolist() == list(range(63, 55, -1))


def test_masked_scores(dev):
    """Experts that are switched off: minus infinity, or the type's lowest value."""
    for t in (torch.bfloat16, torch.float32):
        scores = scores_of(dev, 200, 64, "fp32", 3).to(t)
        scores[:, 5:50] = -float("inf")
        scores[::2, 5:50] = torch.finfo(t).min
        for scoring in ("softmax", "sigmoid"):
            w, i = moe_ops.select_experts(scores, 8, scoring)
            assert ((i < 5) | (i >= 50)).all() and torch.isfinite(w).all() and (w > 0).all()
            s = scores.clone().requires_grad_()
            w, i = moe_ops.select_experts(s, 8, scoring, None, 8, 2, True)
            ds, = torch.autograd.grad(w, s, torch.randn(w.shape, generator=gen(1)).to(dev))
            assert ((i < 8) | (i >= 48)).all() and torch.isfinite(ds).all() and not ds[:, 5:50].any()


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts, times", [(64, 1), (64, 20), (256, 1), (256, 20)])
def test_every_score_of_16_bits(dev, t, experts, times):
    """All bit patterns in any company: zeros are equal, NaN and minus infinity are equal and last."""
    g = gen(7)
    bits = torch.cat([torch.randperm(1 << 16, generator=g) for _ in range(times)])
    bits[::97] = torch.tensor([0, 0x8000, 0x7f80, 0xff80, 0x7c00, 0xfc00, 0x7fff, 0xffff])[torch.randint(0, 8, bits[::97].shape, generator=g)]
    scores = (bits - (bits >> 15 << 16)).to(torch.int16).view(t).view(-1, experts).to(dev)
    _, selected = moe_ops.select_experts(scores, 8)
    order = scores.double().nan_to_num(nan=-float("inf"), posinf=float("inf"), neginf=-float("inf"))
    want = order.sort(dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(selected, want)


@pytest.mark.parametrize("tokens", [40, 5000, 20000])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
def test_tokens_with_few_experts_left(dev, tokens, t):
    scores = scores_of(dev, tokens, 32, "fp32", 5).to(t)
    scores[1::4, :29] = -float("inf")   # three are left
    scores[2::4] = -float("inf")        # none
    for kind in (dict(), dict(bias=torch.zeros(32, device=dev)), dict(groups=4, top_groups=3)):
        for scoring in ("softmax", "sigmoid"):
            s = scores.clone().requires_grad_()
            w, i = moe_ops.select_experts(s, 8, scoring, **kind)
            ds, = torch.autograd.grad(w, s, torch.ones_like(w))
            assert (i[1::4, :3] >= 29).all() and i[2::4].tolist() == [list(range(8))] * len(i[2::4])
            assert i[1::4, 3:].tolist() == [[0, 1, 2, 3, 4]] * len(i[1::4])
            assert (w[1::4, :3] > 0).all() and not w[1::4, 3:].any() and not ds[1::4, :29].any()
            assert w[2::4].isnan().all() if scoring == "softmax" else not w[2::4].any()
            for kept in (w, ds):
                assert torch.isfinite(kept[0::4]).all() and torch.isfinite(kept[1::4]).all() and torch.isfinite(kept[3::4]).all()
    bias = torch.zeros(32, device=dev)
    bias[4:20] = -float("inf")
    for scoring in ("softmax", "sigmoid"):
        w, i = moe_ops.select_experts(scores[0::4].contiguous(), 8, scoring, bias)
        assert ((i < 4) | (i >= 20)).all() and torch.isfinite(w).all()


def test_what_is_no_number(dev):
    scores = scores_of(dev, 4, 32, "fp32", 3)
    scores[0, 3] = float("nan")
    scores[1, 3] = float("inf")
    scores[2] = float("nan")
    for kind in (dict(), dict(bias=torch.zeros(32, device=dev)), dict(groups=4, top_groups=2)):
        w, i = moe_ops.select_experts(scores, 8, "sigmoid", **kind)
        assert (i >= 0).all() and (i < 32).all() and all(len(set(r)) == 8 for r in i.tolist())
        assert 3 not in i[0].tolist() and torch.isfinite(w[[0, 1, 3]]).all() and w[2].isnan().all()
        assert i[1, 0] == 3 or 3 not in i[1].tolist() and "groups" in kind   # (a group stays by its two largest)
        w, i = moe_ops.select_experts(scores, 8, "softmax", **kind)
        assert (i >= 0).all() and (i < 32).all() and all(len(set(r)) == 8 for r in i.tolist())
        assert w[:3].isnan().all() and torch.isfinite(w[3]).all()


def test_views_types_of_gradients_and_empty_batches(dev):
    scores = scores_of(dev, 50, 40, "bf16", 4)
    want = check(scores, 4, "sigmoid", None, 4, 2, True)
    wide = torch.zeros(50, 77, dtype=scores.dtype, device=dev)
    wide[:, 5:45] = scores
    turned = scores.t().contiguous().t()
    for s in (wide[:, 5:45], turned):
        got = check(s, 4, "sigmoid", None, 4, 2, True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    spread = torch.zeros(80, device=dev)
    spread[::2] = torch.randn(40, generator=gen(1)).to(dev) * 0.1
    a = moe_ops.select_experts(scores, 4, "sigmoid", spread[::2])
    b = moe_ops.select_experts(scores, 4, "sigmoid", spread[::2].contiguous())
    assert torch.equal(a[1], b[1])
    s = scores.clone().requires_grad_()
    w, _ = moe_ops.select_experts(s, 4, "sigmoid", None, 4, 2, True)
    dw = torch.randn(50, 4, generator=gen(5)).to(dev)
    one = torch.autograd.grad(w, s, torch._neg_view(-dw), retain_graph=True)[0]
    assert torch.equal(one, want[2])
    w.sum().backward()   # an expanded gradient
    empty = scores[:0].requires_grad_()
    w, i = moe_ops.select_experts(empty, 4, "softmax")
    assert w.shape == i.shape == (0, 4) and torch.autograd.grad(w.sum(), empty)[0].shape == (0, 40)


def test_past_32_bits(dev):
    tokens, experts = (1 << 22) + 5, 520   # 2.2e9 scores
    scores = torch.empty(tokens, experts, dtype=torch.bfloat16, device=dev)
    scores[:] = torch.randn(experts, generator=gen(3)).to(dev)
    scores[-60:] = scores_of(dev, 60, experts, "bf16", 4)
    last = scores[-50:].clone()
    w, i = moe_ops.select_experts(scores, 8, "softmax")
    a, b = moe_ops.select_experts(last, 8, "softmax")
    assert torch.equal(w[-50:], a) and torch.equal(i[-50:], b)
    del w, i
    s, ls = scores.requires_grad_(), last.requires_grad_()
    w, _ = moe_ops.select_experts(s, 2, "sigmoid")
    ds, = torch.autograd.grad(w, s, torch.ones_like(w))
    w, _ = moe_ops.select_experts(ls, 2, "sigmoid")
    assert torch.equal(ds[-50:], torch.autograd.grad(w, ls, torch.ones_like(w))[0])


def test_gradients_against_differences(dev):
    for scoring, renormalize in (("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)):
        scores = scores_of(dev, 20, 24, "fp32", 8)
        s = scores.clone().requires_grad_()
        w, chosen = moe_ops.select_experts(s, 4, scoring, None, 4, 2, renormalize, 2.5)
        dw = torch.randn(w.shape, generator=gen(5)).to(dev)
        ds, = torch.autograd.grad(w, s, dw)
        step = torch.randn(scores.shape, generator=gen(6)).to(dev).double() * 1e-5

        def value(x):
            p = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, 1)
            v = p.gather(1, chosen)
            return (2.5 * (v / v.sum(1, keepdim=True) if renormalize else v) * dw.double()).sum()

        slope = (value(scores.double() + step) - value(scores.double() - step)) / 2
        assert abs(slope.item() - (ds.double() * step).sum().item()) < 1e-5 * (ds.double() * step).abs().sum().item()


def test_refusals(dev):
    s = scores_of(dev, 4, 32, "fp32", 1)
    bias = torch.zeros(32, device=dev)
    bad = [dict(top_k=0), dict(top_k=17), dict(top_k=33), dict(top_k=9, groups=4, top_groups=1), dict(groups=5), dict(groups=32), dict(groups=0),
           dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(group_best=3), dict(scoring="max"), dict(bias=bias[:31]),
           dict(bias=bias.half()), dict(bias=bias.cpu()), dict(scale=float("inf"))]
    for kind in bad:
        with pytest.raises(RuntimeError, match="fp8_gmm_amd"):
            moe_ops.select_experts(s, **{"top_k": 2, **kind})
    for t in (s.double(), s[0], s.cpu(), torch.zeros(2, 4097, device=dev), torch.zeros(2, 0, device=dev)):
        with pytest.raises(RuntimeError, match="fp8_gmm_amd"):
            moe_ops.select_experts(t, 1)
    leaf = s.clone().requires_grad_()
    w, _ = moe_ops.select_experts(leaf, 2)
    g, = torch.autograd.grad(w, leaf, torch.ones_like(w).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        g.sum().backward()
    w, _ = moe_ops.select_experts(leaf * 1.0, 2)
    with pytest.raises(RuntimeError, match="transforms or tracing"):
        torch.func.vmap(lambda t: moe_ops.select_experts(t, 2)[0])(s[None])


def test_other_streams_and_captured_passes(dev):
    scores = scores_of(dev, 300, 256, "bf16", 2)
    bias = (torch.randn(256, generator=gen(3)) * 0.1).to(dev)
    options = ("sigmoid", bias, 8, 4, True, 2.5)
    want = check(scores, 8, *options)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = check(scores, 8, *options)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    s = scores.clone().requires_grad_()
    dw = torch.randn(300, 8, generator=gen(5)).to(dev)

    def step():
        w, i = moe_ops.select_experts(s, 8, *options)
        return (w.detach(), i, *torch.autograd.grad(w, s, dw))

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
    for seed in (31, 32, 33):
        with torch.no_grad():
            s.copy_(scores_of(dev, 300, 256, "bf16", seed))
            bias.copy_(torch.randn(256, generator=gen(seed)).to(dev) * 0.1)
        graph.replay()
        torch.cuda.synchronize()
        copies = [t.clone() for t in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(copies, eager))
        del eager


@pytest.mark.parametrize("kind", ["linear", "mlp"])
def test_a_routed_layer_chooses_so(dev, kind):
    """The layer with the options, step by step by the public calls: the same bits."""
    torch.manual_seed(0)
    cls = {"linear": moe.Fp8LinearModule, "mlp": moe.Fp8MlpModule}[kind]
    routing = moe_ops.Routing("sigmoid", bias=True, groups=4, top_groups=2, renormalize=True, scale=2.5)
    layer = cls(64, 128, 16, 4, device=dev, rms_norm=True, routing=routing)
    layer.expert_bias.copy_(torch.randn(16, generator=gen(1)) * 0.1)
    twin = cls(64, 128, 16, 4, device=dev)
    twin.load_state_dict({k: v for k, v in layer.state_dict().items() if "extra" not in k and k not in ("expert_bias", "row_norm.weight")},
                         strict=False)
    x = torch.randn(200, 64, generator=gen(2)).to(torch.bfloat16).to(dev)
    xa, xb = x.clone().requires_grad_(), x.clone().requires_grad_()
    out = layer(xa)
    rows = pkg.rms_norm(xb, layer.row_norm.weight)
    w, chosen = moe_ops.select_experts(twin.gating_network(rows), 4, "sigmoid", layer.expert_bias, 4, 2, True, 2.5)
    indices, bin_ids, bins, counts, inverse = moe_ops.indices_bins_and_inverse(chosen.flatten(), 16)
    want = twin.compute(rows, counts, indices, bin_ids, w.flatten(), bins, 4, inverse)
    assert torch.equal(out, want) and torch.equal(layer.tokens_per_expert, counts)
    dy = (torch.randn(200, 64, generator=gen(3)) * 0.1).to(torch.bfloat16).to(dev)
    out.backward(dy)
    want.backward(dy)
    assert torch.equal(layer.gating_network.weight.grad, twin.gating_network.weight.grad) or torch.allclose(
        layer.gating_network.weight.grad.float(), twin.gating_network.weight.grad.float(), rtol=0.02, atol=1e-4)
    assert torch.allclose(xa.grad.float(), xb.grad.float(), rtol=0.02, atol=2e-3) and layer.row_norm.weight.grad is not None
    layer.bfloat16()   # the bias is cast with the rest
    assert layer.expert_bias.dtype == torch.bfloat16 and torch.isfinite(layer(x)).all()


def test_saved_tensors_are_looked_after(dev):
    scores = scores_of(dev, 50, 64, "bf16", 4)
    want = check(scores, 6, "sigmoid", None, 8, 4, True)
    leaf = scores.clone().requires_grad_()
    dw = torch.randn(50, 6, generator=gen(5)).to(dev)

    def choose(t):
        return moe_ops.select_experts(t, 6, "sigmoid", None, 8, 4, True)[0]

    with torch.autograd.graph.save_on_cpu():
        w = choose(leaf)
    assert torch.equal(torch.autograd.grad(w, leaf, dw)[0], want[2])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(w, leaf, dw)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        w = choose(leaf)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(w, leaf, dw)
    logits = leaf * 1.0
    w = choose(logits)
    logits.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(w, leaf, dw)
    again = torch.utils.checkpoint.checkpoint(choose, leaf, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, leaf, dw)[0], want[2])
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(choose(leaf), leaf, torch.autograd.forward_ad.make_dual(dw, torch.ones_like(dw)))


@pytest.mark.parametrize("experts, top_k, groups", [(16, 2, 1), (60, 8, 4), (64, 6, 8), (40, 9, 1), (128, 8, 8), (256, 8, 8), (512, 4, 1)])
def test_many_tokens_and_few_choose_alike(dev, experts, top_k, groups):
    """Each number of tokens shares out the lanes in its own way."""
    for t in ("bf16", "fp32"):
        scores = scores_of(dev, 10000, experts, t, experts)
        bias = (torch.randn(experts, generator=gen(3)) * 0.1).to(dev)
        for b in (None, bias):
            w, i, ds = check(scores, top_k, "sigmoid", b, groups, (groups + 1) // 2, False)
            for n in (1, 2000, 5000):
                part = scores[:n].clone().requires_grad_()
                pw, pi = moe_ops.select_experts(part, top_k, "sigmoid", b, groups, (groups + 1) // 2)
                assert torch.equal(pw, w[:n]) and torch.equal(pi, i[:n])
                dw = torch.randn(w.shape, generator=gen(5)).to(dev)[:n]
                assert torch.equal(torch.autograd.grad(pw, part, dw)[0], ds[:n])
