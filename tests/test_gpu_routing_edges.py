"""The choice of experts where scores, biases or groups leave few experts or small probabilities, on the GPU."""
import pytest
import torch

from fp8_gmm_amd import moe_ops

from helpers import gen
from test_gpu_routing import TYPES, U, reference, scores_of

pytestmark = pytest.mark.gpu

INF = float("inf")


def check_shares(scores, top_k, scoring, bias, groups=1, top_groups=1, scale=1.0):
    """Renormalized weights and their gradient, against shares that are formed from logarithms in 64 bits: the probabilities themselves
    are too small for those as well.  Tolerances are those of test_gpu_routing.check: k of the weights and 4 k of what a gradient is the
    difference of."""
    s = scores.clone().requires_grad_()
    w, chosen = moe_ops.select_experts(s, top_k, scoring, bias, groups, top_groups, True, scale)
    _, want = reference(scores, top_k, scoring, bias, groups, top_groups, False, scale, 2)
    assert torch.equal(chosen.cpu(), want)
    x = scores.double().cpu().gather(1, want)
    share = torch.softmax(torch.nn.functional.logsigmoid(x) if scoring == "sigmoid" else x, 1)
    k = 2 * (80 + 2 * scores.float().abs().max().item()) * U + 20 * U
    off = (w.detach().double().cpu() - share * scale).abs()
    assert (off <= k * share * scale + 1e-38).all(), (off / share).max().item() / k
    dw = torch.randn(w.shape, generator=gen(5)).to(scores.device)
    ds, = torch.autograd.grad(w, s, dw)
    rest = torch.sigmoid(-x) if scoring == "sigmoid" else torch.ones_like(x)
    g = dw.double().cpu() * scale
    zeros = torch.zeros(scores.shape, dtype=torch.float64)
    wanted = zeros.scatter(1, want, rest * share * (g - (g * share).sum(1, keepdim=True)))
    bound = zeros.scatter(1, want, rest * share * (g.abs() + (g * share).abs().sum(1, keepdim=True)))
    h, tiny = torch.finfo(scores.dtype).eps / 2, torch.finfo(scores.dtype).smallest_normal
    off = (ds.double().cpu() - wanted).abs()
    assert (off <= 4 * k * bound + h * (wanted.abs() + 4 * k * bound) + tiny).all()
    return w.detach(), chosen, ds


@pytest.mark.parametrize("tokens, experts", [(9, 16), (40, 64), (20000, 64), (40, 256), (5000, 256), (300, 600), (30, 1500)])
@pytest.mark.parametrize("t", ["bf16", "fp32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_renormalized_weights_of_small_probabilities(dev, tokens, experts, t, scoring):
    """The chosen weights are shares of one another, however small their probabilities: 100 and 600 below the row's largest score,
    which a bias of minus infinity or the choice of groups removes, or far below zero."""
    for far in (100.0, 600.0):
        scores = scores_of(dev, tokens, experts, "fp32", experts)
        scores[:, 5:] -= far
        scores[1::2] -= far if scoring == "sigmoid" else 0.0
        scores = scores.to(TYPES[t])
        bias = torch.zeros(experts, device=dev)
        bias[:5] = -INF
        w, chosen, ds = check_shares(scores, 8, scoring, bias, scale=2.5)
        assert (chosen >= 5).all() and torch.isfinite(w).all() and torch.isfinite(ds).all() and ds[:, 5:].any()
    scores = scores_of(dev, tokens, experts, "fp32", experts) - 100.0   # by sigmoid all far below zero
    check_shares(scores.to(TYPES[t]), 6, scoring, None, 2, 1)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
def test_renormalized_weights_behind_a_bias(dev, t):
    """The row's largest score goes by a bias against it, and groups stay by the others, whose probabilities are all but nothing."""
    scores = scores_of(dev, 50, 64, "fp32", 4).to(t)
    scores[:, 3] = 120.0
    bias = torch.zeros(64, device=dev)
    bias[3] = -2.0
    w, chosen, ds = check_shares(scores, 4, "softmax", bias, 8, 2)
    assert (chosen != 3).all() and torch.isfinite(w).all() and torch.isfinite(ds).all()
    total = w.double().sum(1)
    assert ((total - 1).abs() <= 8 * 2.0 ** -24).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_renormalized_weights_of_what_is_no_number(dev, scoring):
    """A NaN makes all of its token's softmax one, of a sigmoid only what is chosen; chosen weights that are all zeros are no numbers."""
    scores = scores_of(dev, 4, 32, "fp32", 3)
    scores[0, 3] = float("nan")
    scores[1, 3] = INF
    scores[2] = -INF
    for bias in (None, torch.zeros(32, device=dev)):
        w, chosen = moe_ops.select_experts(scores, 8, scoring, bias, renormalize=True)
        assert (w[:2].isnan().all() if scoring == "softmax" else torch.isfinite(w[:2]).all())
        assert w[2].isnan().all() and torch.isfinite(w[3]).all()
        assert ((chosen >= 0) & (chosen < 32)).all()


def chosen_of(scores, top_k, scoring, bias, groups, top_groups, best):
    """The choice in 64 bits, on the CPU.  Off is an expert whose score is a NaN or minus infinity, or whose bias is one: it goes last
    and adds nothing to its group."""
    s = scores.double().cpu()
    tokens, experts = s.shape
    far = s.masked_fill(s.isnan(), -INF)
    p = torch.sigmoid(s) if scoring == "sigmoid" else torch.softmax(far, 1).nan_to_num(0.0).masked_fill(far == INF, INF)
    c = far if bias is None and (groups == 1 or best == 1) else p if bias is None else p + bias.double().cpu()
    off = (far == -INF) | c.isnan() | (c == -INF)
    c = c.masked_fill(off, -INF)
    order = c.sort(dim=1, descending=True, stable=True).indices
    if groups > 1:
        two = c.view(tokens, groups, -1).sort(dim=2, descending=True).values[:, :, :best]
        value = two.masked_fill(two == -INF, 0.0).sum(2).masked_fill((two == -INF).all(2), -INF)
        kept = value.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        stays = torch.zeros(tokens, groups, dtype=torch.long).scatter_(1, kept, 1).repeat_interleave(experts // groups, 1)
        order = order.gather(1, stays.gather(1, order).sort(dim=1, descending=True, stable=True).indices)
    return order[:, :top_k]


LAYOUTS = [(40, 16, 1, 1), (40, 64, 8, 3), (20000, 64, 8, 3), (20000, 30, 5, 2), (40, 256, 8, 4), (5000, 256, 8, 4), (5000, 240, 6, 3),
           (300, 600, 4, 2), (30, 1500, 3, 2)]


@pytest.mark.parametrize("tokens, experts, groups, top_groups", LAYOUTS)
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_experts_that_are_switched_off_stay_off(dev, tokens, experts, groups, top_groups, t, scoring):
    """By a score of minus infinity whatever their bias is, which balancing raises for an expert without load."""
    scores = scores_of(dev, tokens, experts, "fp32", experts).to(t)
    off = torch.rand(tokens, experts, generator=gen(1)) < torch.tensor([0.0, 0.3, 0.8, 0.97])[torch.arange(tokens) % 4, None]
    scores[off.to(dev)] = -INF
    bias = (torch.randn(experts, generator=gen(2)) * 0.1).to(dev)
    bias[::3] += 0.9
    for best in (1, 2):
        for kind in ((1, 1), (groups, top_groups)):
            _, got = moe_ops.select_experts(scores, 6, scoring, bias, *kind, group_best=best)
            assert torch.equal(got.cpu(), chosen_of(scores, 6, scoring, bias, *kind, best)), (best, kind)
    bias[1::5] = -INF   # and by a bias of minus infinity
    for best in (1, 2):
        for kind in ((1, 1), (groups, top_groups)):
            _, got = moe_ops.select_experts(scores, 6, scoring, bias, *kind, group_best=best)
            assert torch.equal(got.cpu(), chosen_of(scores, 6, scoring, bias, *kind, best)), (best, kind)


def test_a_group_of_one_that_is_left_stays(dev):
    """A group with one expert that is not off is ahead of a group without any, and counts that one."""
    for scoring in ("softmax", "sigmoid"):
        for by_bias in (True, False):
            scores = torch.zeros(3, 32, device=dev)
            scores[:, 21] = 1.0
            bias = torch.zeros(32, device=dev)
            if by_bias:
                bias[:21] = -INF
                bias[22:] = -INF
            else:
                scores[:, :21] = -INF
                scores[:, 22:] = -INF
            w, chosen = moe_ops.select_experts(scores, 2, scoring, bias, 4, 1)
            assert chosen.tolist() == [[21, 16]] * 3 and (w[:, 0] > 0).all()


@pytest.mark.parametrize("tokens, experts, groups", [(2000, 8, 4), (2000, 32, 16), (20000, 32, 8), (2000, 64, 8), (20000, 64, 8), (1500, 256, 8),
                                                     (5000, 256, 8), (5000, 240, 6), (1000, 1024, 16), (500, 3000, 12)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
def test_groups_of_equal_sums_stay_in_their_order(dev, tokens, experts, groups, t):
    """The sigmoids of x and -x add up to 1, whatever x is, and with a bias of -1/4 each to 1/2: the first groups stay.  2^-30 more of one
    of them decides."""
    size = experts // groups
    x = (torch.rand(tokens, groups, generator=gen(experts)) * 8).to(t).float()
    scores = torch.full((tokens, groups, size), -30.0)
    scores[:, :, 0], scores[:, :, size - 1] = x, -x
    turned = torch.rand(tokens, groups, generator=gen(1)) < 0.5
    scores[turned] = scores[turned].flip(1)
    scores = scores.view(tokens, experts).to(t).to(dev)
    zeros, less = torch.zeros(experts, device=dev), torch.full((experts,), -0.25, device=dev)
    for bias in (None, zeros, less):
        for kept in (1, 2, min(groups - 1, 8)):
            _, chosen = moe_ops.select_experts(scores, 2 * kept, "sigmoid", bias, groups, kept)
            stays = torch.zeros(tokens, groups, dtype=torch.bool, device=dev).scatter_(1, chosen // size, True)
            assert stays[:, :kept].all() and not stays[:, kept:].any(), (kept, int(stays[:, kept:].any(1).sum()))
    last = zeros.clone()
    last[-size] = last[-1] = 2.0 ** -30
    _, chosen = moe_ops.select_experts(scores, 2, "sigmoid", last, groups, 1)
    assert (chosen // size == groups - 1).all()


@pytest.mark.parametrize("tokens, experts, groups, top_groups", LAYOUTS)
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_that_are_no_numbers_go_last(dev, tokens, experts, groups, top_groups, t, scoring):
    """And leave the others' order as it is, by the scores alone as with a bias; beside plus infinity, which goes first, all other
    probabilities are zero."""
    scores = scores_of(dev, tokens, experts, "fp32", experts).to(t)
    r = torch.rand(tokens, experts, generator=gen(1)).to(dev)
    share = torch.tensor([0.0, 1 / experts, 0.5, 1.0], device=dev)[torch.arange(tokens, device=dev) % 4, None]
    scores[r < share] = float("nan")
    scores[(r > 1 - 1 / experts) & (torch.arange(tokens, device=dev) % 3 == 0)[:, None]] = INF
    zeros = torch.zeros(experts, device=dev)
    bias = (torch.randn(experts, generator=gen(2)) * 0.1).to(dev)
    for best in (1, 2):
        for kind in ((1, 1), (groups, top_groups)):
            for b in (None, zeros, bias):
                w, got = moe_ops.select_experts(scores, 6, scoring, b, *kind, group_best=best)
                assert torch.equal(got.cpu(), chosen_of(scores, 6, scoring, b, *kind, best)), (best, kind)
                if scoring == "softmax":
                    assert torch.equal(w.isnan().any(1), ~torch.isfinite(scores).all(1))


@pytest.mark.parametrize("tokens, experts, top_k", [((1 << 29) + 5, 2, 1), ((1 << 28) + 5, 9, 9)])
def test_more_tokens_than_a_grid_has_threads_for(dev, tokens, experts, top_k):
    """By 8 lanes to a token and by 16: the same rows again and again have the same results."""
    block = 1 << 20
    rows = torch.randn(block, experts, generator=gen(1)).to(torch.bfloat16).to(dev)
    dw = torch.randn(block, top_k, generator=gen(2)).to(dev)
    scores = torch.empty(tokens, experts, dtype=rows.dtype, device=dev)
    grads = torch.empty(tokens, top_k, device=dev)
    for at in range(0, tokens, block):
        n = min(block, tokens - at)
        scores[at: at + n], grads[at: at + n] = rows[:n], dw[:n]
    part = rows.requires_grad_()
    want = moe_ops.select_experts(part, top_k, "softmax", renormalize=top_k > 1)
    scores.requires_grad_()
    w, chosen = moe_ops.select_experts(scores, top_k, "softmax", renormalize=top_k > 1)
    ds, = torch.autograd.grad(w, scores, grads)
    wanted = (*(t.detach() for t in want), *torch.autograd.grad(want[0], part, dw))
    del grads, scores
    for at in range(0, tokens, block):
        n = min(block, tokens - at)
        for got, one in zip((w.detach(), chosen, ds), wanted):
            assert torch.equal(got[at: at + n], one[:n]), at


@pytest.mark.parametrize("tokens, experts", [(5, 16), (10000, 64), (300, 256), (9000, 256), (40, 1500)])
def test_small_softmax_weights_have_their_values(dev, tokens, experts):
    """Down to fp32's subnormal numbers: e^-88 to e^-100 of the row's largest score, which is alone above them.  Tolerance: the sum of
    expf's unit, the division's and the last rounding (2 + 1 + 1 units of 2^-24, and of the difference, up to 100, 100 units), and
    half of 2^-149 for each of the three that may be subnormal."""
    scores = -88.0 - 12.0 * torch.rand(tokens, experts, generator=gen(experts))
    scores[:, 0] = 0.0
    w, chosen = moe_ops.select_experts(scores.to(dev), 6)
    want = torch.softmax(scores.double(), 1).gather(1, chosen.cpu())
    off = (w.double().cpu() - want).abs()
    assert (off <= 104 * U * want + 1.5 * 2.0 ** -149).all() and (w > 0).all()
