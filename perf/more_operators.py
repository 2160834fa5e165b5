"""The operators of a block with routed experts and of the optimizer's step, as cases that can be prepared, run and timed one by
one.

``listed()`` are the representative calls, from the smallest to the largest; ``draw(rng)`` gives more of the same ranges.
A case names what is called (``kind``) and its sizes:

* ``rms``    root-mean-square norm of the rows in front of a layer, with the residual's addition in front where there is one:
             forward alone (``train`` false), or forward and the gradients of the rows, the residual and the weight
* ``rms8``   the same norm with its result in 8 bits: by the tensor's own scale, whose largest magnitude is recorded for the next
             step (``scaled`` "tensor"), or by a scale for every row (``scaled`` "rows")
* ``route``  the choice of a token's experts from its scores and their weights: forward alone, or with the scores' gradient
* ``adamw``  a step over a list of tensors, with moments in 32 bits or in 8 with a scale for every 128 of them

With ``own`` false ``run`` computes them by elementary torch operations in 32 bits, rounded once at the end; with ``own``
true it makes the calls of this package.
"""
import math

import torch

own = False

EPS = 1e-6
ADAM = {"lr": 1e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
BLOCK = 128   # moments to a scale
# thresholds of the moments' rounding in units of 2^-32: a step's share and an element's, each spread evenly by its multiples
STEP, ELEMENT = 0x9E3779B9, 0x6A09E667


def listed():
    return [
        # decoding one token: the residual's addition and the norm of a single row, nothing but latency
        {"name": "rms_token", "kind": "rms", "rows": 1, "hidden": 4096, "type": "bf16", "weights": "bf16", "residual": True,
         "train": False},
        # the batch of the headline workload in front of its routed layer, the residual stream added on the way
        {"name": "rms_batch", "kind": "rms", "rows": 16384, "hidden": 4096, "type": "bf16", "weights": "bf16", "residual": True,
         "train": True},
        # rows whose bytes are no multiple of anything, fp16, the weight kept in fp32, the first norm of a model
        {"name": "rms_odd", "kind": "rms", "rows": 4001, "hidden": 1411, "type": "fp16", "weights": "fp32", "residual": False,
         "train": True},
        # decoding 64 sequences in front of a product in 8 bits, every row with its own scale
        {"name": "rms8_decode", "kind": "rms8", "rows": 64, "hidden": 4096, "type": "bf16", "weights": "bf16", "residual": True,
         "scaled": "rows", "format": "e4m3"},
        # the same batch as above by delayed scaling
        {"name": "rms8_batch", "kind": "rms8", "rows": 16384, "hidden": 4096, "type": "bf16", "weights": "bf16", "residual": True,
         "scaled": "tensor", "format": "e4m3"},
        # decoding one token over many experts in groups
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5, "type": "fp32", "train": False},
        # a training batch over the same experts, scores as a bf16 gate gives them
        {"name": "route_groups", "kind": "route", "tokens": 16384, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5, "type": "bf16", "train": True},
        # a long batch over fewer experts by softmax alone
        {"name": "route_softmax", "kind": "route", "tokens": 131072, "experts": 64, "top_k": 6, "scoring": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "renormalize": False, "scale": 1.0, "type": "bf16", "train": True},
        # norms, gates and biases alone: a few short tensors in fp32
        {"name": "adamw_small", "kind": "adamw", "tensors": 24, "least": 16, "most": 8192, "type": "fp32", "grads": "fp32",
         "masters": False, "bits": 32, "clipped": False},
        # the two weight stacks of the headline workload's experts: bf16 weights, fp32 masters and moments, clipped on the way
        {"name": "adamw_experts", "kind": "adamw", "tensors": 2, "least": 8 * 14336 * 4096, "most": 8 * 14336 * 4096,
         "type": "bf16", "grads": "bf16", "masters": True, "bits": 32, "clipped": True},
        # a model of many layers: hundreds of tensors of every size, gradients in a bucket of fp32
        {"name": "adamw_many", "kind": "adamw", "tensors": 400, "least": 64, "most": 4 << 20, "type": "bf16", "grads": "fp32",
         "masters": False, "bits": 32, "clipped": True},
        # a model whose moments are kept in 8 bits to leave the memory to its weights
        {"name": "adamw_8bit", "kind": "adamw", "tensors": 96, "least": 1024, "most": 16 << 20, "type": "bf16", "grads": "bf16",
         "masters": False, "bits": 8, "clipped": True},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["rms", "rms8", "route", "adamw"])
    while True:
        case = {"kind": kind, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if kind in ("rms", "rms8"):
            case.update(rows=_log_int(rng, 1, 65536), hidden=_log_int(rng, 64, 16384), weights=rng.choice([case["type"], "fp32"]),
                        residual=rng.random() < 0.6)
            if kind == "rms":
                case["train"] = rng.random() < 0.7
            else:
                case.update(scaled=rng.choice(["tensor", "rows"]), format=rng.choice(["e4m3", "e4m3", "e5m2"]))
            if case["rows"] * case["hidden"] <= 16384 * 4096:
                return case
        elif kind == "route":
            groups = rng.choice([1, 1, 2, 4, 8])
            case.update(tokens=_log_int(rng, 1, 131072), experts=groups * _log_int(rng, 2, 384 // groups), groups=groups,
                        top_groups=rng.randint(1, groups), scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                        scale=rng.choice([1.0, 2.5]), train=rng.random() < 0.7)
            case["top_k"] = rng.randint(1, min(8, case["experts"] // groups * case["top_groups"]))
            case["renormalize"] = case["top_k"] > 1 and rng.random() < 0.5   # (a single weight would be a constant)
            if case["type"] != "fp16" and case["tokens"] * case["experts"] <= 131072 * 64:
                return case
        else:
            case.update(tensors=_log_int(rng, 1, 400), least=_log_int(rng, 1, 4096), most=_log_int(rng, 4096, 16 << 20),
                        grads=rng.choice([case["type"], "fp32"]), masters=case["type"] != "fp32" and rng.random() < 0.4,
                        bits=rng.choice([32, 8]), clipped=rng.random() < 0.5)
            if sum(_sizes(case)) <= 256 << 20:
                return case


def _sizes(case):
    """The tensors' numbers of elements: spread evenly over their logarithm, in an order of no meaning."""
    ratio = case["most"] / case["least"]
    return [int(round(case["least"] * ratio ** (0.6180339887498949 * (i + 1) % 1.0))) for i in range(case["tensors"])]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return torch.randn(*shape, generator=g, device=dev).mul_(std).add_(mean).to(to)

    state = {"case": case, "kind": case["kind"], "train": case.get("train", False), "type": dtype}
    if case["kind"] in ("rms", "rms8"):
        rows, hidden, params = case["rows"], case["hidden"], TYPES[case["weights"]]
        # a residual stream: rows of different magnitude, some columns much larger than the others
        stream = normal(rows, hidden, to=torch.float32) * (0.5 + 2.0 * torch.rand(rows, 1, generator=g, device=dev))
        stream = (stream + normal(1, hidden, std=0.5, to=torch.float32)).to(dtype)
        x = normal(rows, hidden, std=0.5) if case["residual"] else stream
        state.update(x=x.requires_grad_(state["train"]), weight=normal(hidden, std=0.1, mean=1.0, to=params).requires_grad_(state["train"]),
                     residual=stream.requires_grad_(state["train"]) if case["residual"] else None)
        if state["train"]:
            state["dy"] = normal(rows, hidden, std=1e-2)
            state["dh"] = normal(rows, hidden, std=1e-2) if case["residual"] else None
        if case["kind"] == "rms8":
            by_tensor = case["scaled"] == "tensor"
            # the scale that the last steps' largest magnitude gave, with some room
            state.update(format=TYPES[case["format"]], largest=LARGEST[case["format"]],
                         scale=torch.full((1,), LARGEST[case["format"]] / 8.0, device=dev) if by_tensor else None,
                         amax=torch.zeros(1, device=dev) if by_tensor else None)
    elif case["kind"] == "route":
        tokens, experts = case["tokens"], case["experts"]
        # scores of which some experts get more than others, and the bias that training has found against that
        lean = torch.randn(experts, generator=g, device=dev) * 0.3
        scores = (torch.randn(tokens, experts, generator=g, device=dev) + lean).to(dtype)
        state.update(scores=scores.requires_grad_(state["train"]),
                     bias=-lean * (0.2 if case["scoring"] == "sigmoid" else 0.5 / experts) if case["bias"] else None)
        if state["train"]:
            state["dw"] = normal(tokens, case["top_k"], std=1e-2, to=torch.float32)
    else:
        sizes = _sizes(case)
        # an optimizer's own memory, a tensor's part beginning on a block; the gradients one behind the other in a bucket
        flat = {"grads": torch.empty(sum(sizes), dtype=TYPES[case["grads"]], device=dev)}
        total = sum(-(-n // BLOCK) for n in sizes) * BLOCK
        flat["params"] = torch.zeros(total, dtype=dtype, device=dev)
        flat["masters"] = torch.zeros(total, device=dev) if case["masters"] else None
        for moment in ("exp_avgs", "exp_avg_sqs"):
            flat[moment] = torch.zeros(total, dtype=torch.float8_e4m3fn if case["bits"] == 8 else torch.float32, device=dev)
        flat["scales"] = [torch.zeros(total // BLOCK, device=dev) for _ in range(2)] if case["bits"] == 8 else []
        state.update(flat=flat, grads=list(flat["grads"].split(sizes)), params=[], exp_avgs=[], exp_avg_sqs=[], step=40,
                     masters=[] if case["masters"] else None, scales=([], []) if case["bits"] == 8 else None,
                     norm=torch.full((), 2.0, device=dev) if case["clipped"] else None)
        at = 0
        for i, (n, grad) in enumerate(zip(sizes, state["grads"])):   # tensors of different magnitude, moments as training leaves them
            std = 1e-3 * (1 + i % 7)
            for name in ("params", "exp_avgs", "exp_avg_sqs") + (("masters",) if case["masters"] else ()):
                state[name].append(flat[name][at: at + n])
            weight = torch.randn(n, generator=g, device=dev).mul_(0.02)
            state["params"][i].copy_(weight)
            if case["masters"]:
                state["masters"][i].copy_(weight)
            del weight
            grad.copy_(torch.randn(n, generator=g, device=dev).mul_(std))
            m = torch.randn(n, generator=g, device=dev).mul_(0.2 * std)
            v = torch.rand(n, generator=g, device=dev).add_(0.05).mul_(std * std)
            if case["bits"] == 8:
                v.sqrt_()
                for values, moment, k in ((m, "exp_avgs", 0), (v, "exp_avg_sqs", 1)):
                    scale = flat["scales"][k][at // BLOCK: at // BLOCK + -(-n // BLOCK)]
                    scale.copy_(_block_max(values) / 448.0)
                    state[moment][i].copy_((values / _spread(scale, n)).clamp_(-448, 448))
                    state["scales"][k].append(scale)
            else:
                state["exp_avgs"][i].copy_(m)
                state["exp_avg_sqs"][i].copy_(v)
            del m, v
            at += -(-n // BLOCK) * BLOCK
    return state


def _block_max(t):
    """The largest magnitude of every block of a moment; the last one may be short."""
    return torch.nn.functional.pad(t.abs(), (0, -t.numel() % BLOCK)).view(-1, BLOCK).amax(1)


def _spread(scales, n):
    return scales.repeat_interleave(BLOCK)[:n]


def _plain_norm(s):
    """The rows that are normed, in 32 bits, their factors and the normed rows."""
    h = s["x"].detach()
    if s["residual"] is not None:
        h = (h.float() + s["residual"].detach().float()).to(s["type"])
    rows = h.float()
    r = (rows.square().mean(1, keepdim=True) + EPS).rsqrt()
    return h, rows, r, rows * r * s["weight"].detach().float()


def _plain_rms(s):
    h, rows, r, y = _plain_norm(s)
    out = [y.to(s["type"])] + ([h] if s["residual"] is not None else [])
    if s["train"]:
        dy = s["dy"].float()
        g = dy * s["weight"].detach().float()
        hat = rows * r
        dx = r * (g - hat * (g * hat).mean(1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["dh"].float()
        out += [dx.to(s["type"]), (dy * hat).sum(0).to(s["weight"].dtype)]
    return out


def _plain_rms8(s):
    h, _, _, y = _plain_norm(s)
    largest = s["largest"]
    if s["scale"] is not None:
        s["amax"].copy_(torch.maximum(s["amax"], y.abs().max()))
        q, told = y * s["scale"], s["amax"]
    else:
        told = y.abs().amax(1).clamp(min=2.0 ** -100) / largest
        q = y / told[:, None]
    return [q.clamp(-largest, largest).to(s["format"]), told] + ([h] if s["residual"] is not None else [])


def _plain_route(s):
    c = s["case"]
    scores = s["scores"].detach()
    tokens, experts = scores.shape

    def score(t):
        if c["scoring"] == "sigmoid":
            return 1 / (1 + torch.exp(-t))
        e = torch.exp(t - t.amax(1, keepdim=True))
        return e / e.sum(1, keepdim=True)

    # which experts: in 64 bits, where neighbours that 32 bits cannot tell apart have an order too
    choice = score(scores.double())
    if s["bias"] is not None:
        choice = choice + s["bias"].double()
    if c["groups"] > 1:
        parts = choice.view(tokens, c["groups"], -1)
        best = parts.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.zeros(tokens, c["groups"], dtype=torch.bool, device=scores.device)
        kept.scatter_(1, best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]], True)
        choice = parts.masked_fill(~kept[:, :, None], -math.inf).view(tokens, experts)
    selected = choice.sort(dim=1, descending=True, stable=True).indices[:, :c["top_k"]].contiguous()
    p = score(scores.float())
    chosen = p.gather(1, selected)
    total = chosen.sum(1, keepdim=True)
    out = [chosen / total * c["scale"] if c["renormalize"] else chosen * c["scale"], selected]
    if s["train"]:
        dw = s["dw"] * c["scale"]
        if c["renormalize"]:
            dw = (dw - (dw * chosen).sum(1, keepdim=True) / total) / total
        if c["scoring"] == "sigmoid":
            x = scores.float().gather(1, selected)
            ds = torch.zeros_like(p).scatter_(1, selected, dw * chosen / (1 + torch.exp(x)))
        else:
            ds = p * (torch.zeros_like(p).scatter_(1, selected, dw) - (dw * chosen).sum(1, keepdim=True))
        out.append(ds.to(scores.dtype))
    return out


def _grid(y):
    """The numbers of 8 bits around a magnitude: the one that is not above it, and the next."""
    off = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)
    low = (y + off).view(torch.int32) & -(1 << 20)
    return low.view(torch.float32) - off, (low + (1 << 20)).view(torch.float32) - off


def _threshold(n, step, device):
    """A threshold in units of 2^-32 for every element of a tensor."""
    return (torch.arange(n, device=device) * ELEMENT + step * STEP) & 0xFFFFFFFF


def _plain_adamw(s):
    (b1, b2), lr, step = ADAM["betas"], ADAM["lr"], s["step"]
    factor = 1.0 if s["norm"] is None else (1.0 / (s["norm"] + 1e-6)).clamp(max=1.0)
    bits8 = s["scales"] is not None
    for i, (param, grad) in enumerate(zip(s["params"], s["grads"])):
        n = param.numel()
        g = grad.float() * factor
        m, v = s["exp_avgs"][i], s["exp_avg_sqs"][i]
        if bits8:
            m = m.float() * _spread(s["scales"][0][i], n)
            v = (v.float() * _spread(s["scales"][1][i], n)).square()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        root = v.sqrt()
        master = param.float() if s["masters"] is None else s["masters"][i]
        moved = master - (lr * ADAM["weight_decay"]) * master \
            - (lr / (1 - b1 ** step)) * m / (root / math.sqrt(1 - b2 ** step) + ADAM["eps"])
        if s["masters"] is not None:
            master.copy_(moved)
        param.copy_(moved)
        if not bits8:
            s["exp_avgs"][i].copy_(m)
            s["exp_avg_sqs"][i].copy_(v)
            continue
        h = _threshold(n, step, param.device)
        largest = _block_max(m)
        s["scales"][0][i].copy_(largest / 448.0)
        y = (m * _spread(448.0 / largest, n)).nan_to_num(0.0)
        low, high = _grid(y.abs())
        up = (y.abs() - low) / (high - low) + (h >> 12) * 2.0 ** -20 >= 1
        s["exp_avgs"][i].copy_(torch.where(up, high, low).clamp(max=448.0).copysign(y))
        largest = _block_max(root)
        s["scales"][1][i].copy_(largest / 448.0)
        y = (root * _spread(448.0 / largest, n)).nan_to_num(0.0)
        low, high = _grid(y)
        up = (y - low) * (y + low) > ((h ^ 0x80000000) >> 8) * 2.0 ** -24 * ((high - low) * (high + low))
        q = torch.where(up, high, low).clamp(max=448.0)
        s["exp_avg_sqs"][i].copy_(torch.where((y > 0) & (q == 0), high, q))
    return _adamw_outputs(s)


def _adamw_outputs(s):
    flat = s["flat"]
    return [flat["params"], flat["exp_avgs"], flat["exp_avg_sqs"], flat["masters"], *flat["scales"]]


def run(state):
    if state["kind"] == "adamw":
        state["step"] += 1
    if not own:
        return {"rms": _plain_rms, "rms8": _plain_rms8, "route": _plain_route, "adamw": _plain_adamw}[state["kind"]](state)
    import fp8_gmm_amd as fp8

    s = state
    if s["kind"] == "rms":
        out = fp8.rms_norm(s["x"], s["weight"], EPS, s["residual"])
        if s["residual"] is None:
            return [out.detach(), *torch.autograd.grad(out, (s["x"], s["weight"]), s["dy"])] if s["train"] else [out]
        if not s["train"]:
            return list(out)
        y, h = out
        dx, _, dw = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
        return [y.detach(), h.detach(), dx, dw]
    if s["kind"] == "rms8":
        q, scale_inv, h = fp8.rms_norm_fp8(s["x"], s["weight"], EPS, s["residual"], s["scale"], s["amax"], s["format"])
        return [q, s["amax"] if scale_inv is None else scale_inv] + ([] if h is None else [h])
    if s["kind"] == "route":
        c = s["case"]
        weights, selected = fp8.moe_ops.select_experts(s["scores"], c["top_k"], c["scoring"], s["bias"], c["groups"], c["top_groups"],
                                                       c["renormalize"], c["scale"])
        if not s["train"]:
            return [weights, selected]
        return [weights.detach(), selected, *torch.autograd.grad(weights, s["scores"], s["dw"])]
    fp8.backend.multi_adamw(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["step"], **ADAM, scales=s["scales"],
                            masters=s["masters"], norm=s["norm"], max_norm=None if s["norm"] is None else 1.0)
    return _adamw_outputs(s)


def work(case):
    size = BYTES[case["type"]]
    if case["kind"] in ("rms", "rms8"):
        values, params = case["rows"] * case["hidden"], case["hidden"] * BYTES[case["weights"]]
        streams = 2 if case["residual"] else 0   # the residual and the sum
        if case["kind"] == "rms8":
            return {"bytes": values * (size * (1 + streams) + 1) + params + (4 * case["rows"] if case["scaled"] == "rows" else 8),
                    "flops": values * 7}
        # x and y, residual and sum; with the gradients dy, that of the sum, and dx
        train = case["train"]
        return {"bytes": values * size * (2 + streams + (2 + (1 if case["residual"] else 0) if train else 0)) + params * (2 if train else 1),
                "flops": values * (17 if train else 5)}
    if case["kind"] == "route":
        scores, chosen = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        return {"bytes": scores * size * (2 if case["train"] else 1) + chosen * (12 + (4 if case["train"] else 0))
                + (4 * case["experts"] if case["bias"] else 0),
                "flops": scores * (20 if case["train"] else 10)}
    sizes = _sizes(case)
    values, blocks = sum(sizes), sum(-(-n // BLOCK) for n in sizes)
    weights = 8 + size if case["masters"] else 2 * size
    moments = values * 16 if case["bits"] == 32 else values * 4 + blocks * 16
    return {"bytes": values * (weights + BYTES[case["grads"]]) + moments, "flops": values * 16}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("rms", "rms8"):
        x, w = s["x"].detach(), s["weight"].detach().double()
        n = x.shape[1]
        h = x.double()
        if s["residual"] is not None:   # rounded once: what the norm is of
            h = (h + s["residual"].detach().double()).to(s["type"]).double()
        norm = (torch.einsum("ij,ij->i", h, h) / n + EPS).sqrt()[:, None]
        y = h / norm * w
        added = [h] if s["residual"] is not None else []
        if case["kind"] == "rms8":
            if case["scaled"] == "tensor":
                return [(y * s["scale"].double()).clamp(-s["largest"], s["largest"]), y.abs().max().reshape(1)] + added
            scale = y.abs().max(1).values.clamp(min=2.0 ** -100) / s["largest"]
            return [y / scale[:, None], scale] + added
        if not s["train"]:
            return [y] + added
        dy = s["dy"].double()
        g = dy * w
        dx = g / norm - h * (torch.einsum("ij,ij->i", g, h)[:, None] / (n * norm ** 3))
        if s["dh"] is not None:
            dx = dx + s["dh"].double()
        return [y] + added + [dx, torch.einsum("ij,ij->j", dy, h / norm)]
    if case["kind"] == "route":
        scores = s["scores"].detach().double()
        p = torch.sigmoid(scores) if case["scoring"] == "sigmoid" else torch.softmax(scores, 1)
        left = p.clone() if s["bias"] is None else p + s["bias"].double()
        tokens, experts = scores.shape
        size = experts // case["groups"]
        places = torch.arange(experts, device=scores.device)

        def take(values, n):
            """The places of the n largest values of every row, the first of equal ones first."""
            found = []
            for _ in range(n):
                top = values.max(1, keepdim=True).values
                found.append(torch.where(values == top, places[:values.shape[1]], experts).min(1).values)
                values = values.scatter(1, found[-1][:, None], -math.inf)
            return torch.stack(found, 1)

        if case["groups"] > 1:
            groups = left.view(-1, size)
            two = groups.gather(1, take(groups, min(2, size))).sum(1).view(tokens, -1)
            kept = torch.ones_like(two, dtype=torch.bool).scatter(1, take(two, case["top_groups"]), False)
            left = left.masked_fill(kept.repeat_interleave(size, 1), -math.inf)
        selected = take(left, case["top_k"])
        if not s["train"]:
            w = p.gather(1, selected)
            return [(w / w.sum(1, keepdim=True) if case["renormalize"] else w) * case["scale"], selected]
        with torch.enable_grad():
            scores.requires_grad_()
            w = (torch.sigmoid(scores) if case["scoring"] == "sigmoid" else torch.softmax(scores, 1)).gather(1, selected)
            w = (w / w.sum(1, keepdim=True) if case["renormalize"] else w) * case["scale"]
            return [w.detach(), selected, *torch.autograd.grad(w, scores, s["dw"].double())]
    (b1, b2), lr, step = ADAM["betas"], ADAM["lr"], s["step"] + 1
    factor = 1.0 if s["norm"] is None else min(1.0, 1.0 / (float(s["norm"]) + 1e-6))
    total = s["flat"]["params"].numel()
    params, avgs, roots = (torch.zeros(total, dtype=torch.float64, device=s["flat"]["params"].device) for _ in range(3))
    scales = [torch.zeros(total // BLOCK, dtype=torch.float64, device=params.device) for _ in s["flat"]["scales"]]
    at = 0
    for i, grad in enumerate(s["grads"]):
        n = grad.numel()
        g = grad.double().mul_(factor)
        m, v = s["exp_avgs"][i].double(), s["exp_avg_sqs"][i].double()
        if scales:
            m *= _spread(s["scales"][0][i].double(), n)
            v = v.mul_(_spread(s["scales"][1][i].double(), n)).square_()
        m += (1 - b1) * (g - m)
        v += (1 - b2) * (g.square_() - v)
        p = (s["params"] if s["masters"] is None else s["masters"])[i].double()
        params[at: at + n] = p.mul_(1 - lr * ADAM["weight_decay"]).addcdiv_(
            m / (1 - b1 ** step), (v / (1 - b2 ** step)).sqrt_().add_(ADAM["eps"]), value=-lr)
        for t, k, to in ((m, 0, avgs), (v.sqrt_() if scales else v, 1, roots)):
            if scales:   # ahead of the rounding to 8 bits
                scale = _block_max(t) / 448.0
                scales[k][at // BLOCK: at // BLOCK + scale.numel()] = scale
                t = (t / _spread(scale, n)).nan_to_num_(0.0)
            to[at: at + n] = t
        at += -(-n // BLOCK) * BLOCK
    return [params, avgs, roots, params if case["masters"] else None, *scales]
