"""The operators around the routed layers of a training step, as cases that can be prepared, run and timed one by one.

``listed()`` are the representative calls, from the smallest to the largest; ``draw(rng)`` gives more of the same ranges.
A case names what is called (``kind``) and its sizes:

* ``norm``       layer norm of the rows in front of a routed layer: forward alone (``train`` false), or forward and the
                 gradients of the rows, the weight and the bias
* ``clip``       the global norm of a list of gradients and their scaling by it: into tensors of the optimizer's own, or
                 in place where the norm is within its bound
* ``embedding``  rows of a table by token id, scaled: the lookup alone (``train`` false), or with the table's gradient

With ``own`` false ``run`` computes them by elementary torch operations in 32 bits, rounded once at the end; with ``own``
true it makes the calls of this package.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # decoding one token: the norm of a single row, nothing but latency
        {"name": "norm_token", "kind": "norm", "rows": 1, "hidden": 4096, "type": "bf16", "weights": "bf16", "bias": True,
         "train": False},
        # a short odd batch in training, the parameters kept in fp32
        {"name": "norm_short", "kind": "norm", "rows": 1531, "hidden": 1024, "type": "bf16", "weights": "fp32", "bias": True,
         "train": True},
        # the batch of the headline workload in front of its routed layer
        {"name": "norm_batch", "kind": "norm", "rows": 16384, "hidden": 4096, "type": "bf16", "weights": "bf16", "bias": True,
         "train": True},
        # rows whose bytes are no multiple of anything, fp16, without a bias
        {"name": "norm_odd", "kind": "norm", "rows": 4001, "hidden": 1411, "type": "fp16", "weights": "fp16", "bias": False,
         "train": True},
        # many rows of a residual stream kept in fp32
        {"name": "norm_fp32", "kind": "norm", "rows": 65536, "hidden": 2048, "type": "fp32", "weights": "fp32", "bias": True,
         "train": True},
        # the gradients of norms, gates and biases alone: a few short tensors
        {"name": "clip_small", "kind": "clip", "tensors": 24, "least": 16, "most": 8192, "type": "fp32", "outs": "fp32",
         "clipped": True},
        # the two weight stacks of the headline workload's experts, into the fp32 gradients that the optimizer steps on
        {"name": "clip_experts", "kind": "clip", "tensors": 2, "least": 8 * 14336 * 4096, "most": 8 * 14336 * 4096,
         "type": "bf16", "outs": "fp32", "clipped": True},
        # a model of many layers: hundreds of tensors of every size, packed one behind the other in a bucket
        {"name": "clip_many", "kind": "clip", "tensors": 400, "least": 64, "most": 4 << 20, "type": "bf16", "outs": "bf16",
         "clipped": True},
        # most steps of a training run: the norm is within its bound and the gradients stay as they are
        {"name": "clip_within", "kind": "clip", "tensors": 96, "least": 1024, "most": 16 << 20, "type": "bf16", "outs": "",
         "clipped": False},
        # decoding: the rows of 64 sequences' tokens
        {"name": "embedding_decode", "kind": "embedding", "tokens": 64, "table": 32000, "hidden": 4096, "type": "bf16",
         "ids": "uniform", "scaled": True, "padding": False, "train": False},
        # a short batch over a small table in fp32
        {"name": "embedding_short", "kind": "embedding", "tokens": 1000, "table": 4001, "hidden": 256, "type": "fp32",
         "ids": "zipf", "scaled": True, "padding": True, "train": True},
        # the batch of the headline workload: a few tokens make up much of a text, and some positions are padding
        {"name": "embedding_batch", "kind": "embedding", "tokens": 16384, "table": 32000, "hidden": 4096, "type": "bf16",
         "ids": "zipf", "scaled": True, "padding": True, "train": True},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "clip", "embedding"])
    while True:
        case = {"kind": kind, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if kind == "norm":
            case.update(rows=_log_int(rng, 1, 65536), hidden=_log_int(rng, 64, 16384), bias=rng.random() < 0.7,
                        weights=rng.choice([case["type"], "fp32"]), train=rng.random() < 0.7)
            if case["rows"] * case["hidden"] <= 65536 * 2048:
                return case
        elif kind == "clip":
            case.update(tensors=_log_int(rng, 1, 400), least=_log_int(rng, 1, 4096), most=_log_int(rng, 4096, 16 << 20),
                        clipped=rng.random() < 0.7)
            case["outs"] = rng.choice([case["type"], "fp32"]) if case["clipped"] else ""
            if sum(_sizes(case)) <= 256 << 20:
                return case
        else:
            case.update(tokens=_log_int(rng, 1, 65536), table=_log_int(rng, 64, 131072), hidden=_log_int(rng, 64, 8192),
                        ids=rng.choice(["zipf", "uniform"]), scaled=rng.random() < 0.7, padding=rng.random() < 0.5,
                        train=rng.random() < 0.7)
            if case["tokens"] * case["hidden"] <= 16384 * 4096 and case["table"] * case["hidden"] <= 32000 * 4096:
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

    state = {"kind": case["kind"], "train": case.get("train", True), "type": dtype}
    if case["kind"] == "norm":
        rows, hidden, params = case["rows"], case["hidden"], TYPES[case["weights"]]
        # a residual stream: rows of different magnitude, off zero, some columns much larger than the others
        x = normal(rows, hidden, to=torch.float32) * (0.5 + 2.0 * torch.rand(rows, 1, generator=g, device=dev))
        x += normal(1, hidden, std=0.5, to=torch.float32) + normal(rows, 1, std=0.2, to=torch.float32)
        state.update(x=x.to(dtype).requires_grad_(state["train"]),
                     weight=normal(hidden, std=0.1, mean=1.0, to=params).requires_grad_(state["train"]),
                     bias=normal(hidden, std=0.1, to=params).requires_grad_(state["train"]) if case["bias"] else None)
        if state["train"]:
            state["dy"] = normal(rows, hidden, std=1e-2)
    elif case["kind"] == "clip":
        sizes = _sizes(case)
        total = sum(sizes)
        # a bucket, and its tensors as the views of it that a data-parallel program's parameters have for gradients
        flat = torch.empty(total, dtype=dtype, device=dev)
        at = 0
        for i, n in enumerate(sizes):   # tensors of different magnitude
            flat[at: at + n] = torch.randn(n, generator=g, device=dev).mul_(1e-3 * (1 + i % 7))
            at += n
        root = math.sqrt(total)
        state.update(flat=flat, grads=list(flat.split(sizes)), max_norm=1e-4 * root if case["clipped"] else 10.0 * root)
        if case["outs"]:
            state["flat_out"] = torch.empty(total, dtype=TYPES[case["outs"]], device=dev)
            state["outs"] = list(state["flat_out"].split(sizes))
        else:
            state["flat_out"], state["outs"] = flat, state["grads"]
    else:
        tokens, table, hidden = case["tokens"], case["table"], case["hidden"]
        u = torch.rand(tokens, generator=g, device=dev, dtype=torch.float64)
        # uniform over the logarithm: the frequencies of words; which rows the frequent ones have is left to chance
        rank = (table ** u - 1).long().clamp_(0, table - 1) if case["ids"] == "zipf" else (u * table).long()
        ids = torch.randperm(table, generator=g, device=dev)[rank]
        padding = 0 if case["padding"] else None
        if case["padding"]:
            ids[tokens - tokens // 8:] = 0   # the end of a padded batch
        state.update(ids=ids, weight=normal(table, hidden, std=0.02).requires_grad_(state["train"]), padding=padding,
                     scale=math.sqrt(hidden) if case["scaled"] else 1.0)
        if state["train"]:
            state["dy"] = normal(tokens, hidden, std=1e-2)
    return state


def _plain_norm(s):
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    centred = x - x.mean(1, keepdim=True)
    rstd = (centred.square().mean(1, keepdim=True) + EPS).rsqrt()
    hat = centred * rstd
    y = hat * w
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    out = [y.to(s["type"])]
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        out += [dx.to(s["type"]), (dy * hat).sum(0).to(s["weight"].dtype)]
        if s["bias"] is not None:
            out.append(dy.sum(0).to(s["bias"].dtype))
    return out


def _plain_clip(s):
    squares = [t.float().square().sum() for t in s["grads"]]
    norm = torch.stack(squares).double().sum().sqrt().float()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    done = [out.copy_(t.float() * factor) for t, out in zip(s["grads"], s["outs"])]
    return [norm, s["flat_out"]] if done else [norm]


def _plain_embedding(s):
    ids, w = s["ids"], s["weight"].detach()
    out = [(w[ids].float() * s["scale"]).to(s["type"])]
    if s["train"]:
        grad = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids, s["dy"].float())
        if s["padding"] is not None:
            grad[s["padding"]] = 0
        out.append((grad * s["scale"]).to(s["type"]))
    return out


def run(state):
    if not own:
        return {"norm": _plain_norm, "clip": _plain_clip, "embedding": _plain_embedding}[state["kind"]](state)
    import fp8_gmm_amd as fp8

    s = state
    if s["kind"] == "norm":
        y = fp8.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        if not s["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [t for t in (s["x"], s["weight"], s["bias"]) if t is not None], s["dy"])]
    if s["kind"] == "clip":
        return [fp8.backend.multi_clip(s["grads"], s["outs"], s["max_norm"]), s["flat_out"]]
    y = fp8.embedding(s["ids"], s["weight"], s["scale"], s["padding"])
    return [y.detach(), *torch.autograd.grad(y, s["weight"], s["dy"])] if s["train"] else [y]


def work(case):
    size = BYTES[case["type"]]
    if case["kind"] == "norm":
        values, params = case["rows"] * case["hidden"], case["hidden"] * BYTES[case["weights"]] * (2 if case["bias"] else 1)
        # x and y; with the gradients dy and dx as well, and the parameters' own
        return {"bytes": values * size * (4 if case["train"] else 2) + params * (2 if case["train"] else 1),
                "flops": values * (20 if case["train"] else 8)}
    if case["kind"] == "clip":
        values = sum(_sizes(case))
        return {"bytes": values * (size + (BYTES[case["outs"]] if case["outs"] else 0)), "flops": values * 3}
    values = case["tokens"] * case["hidden"]
    read = min(case["tokens"], case["table"]) * case["hidden"]   # no row of the table has to come twice
    return {"bytes": (values + read) * size + case["tokens"] * 8
            + ((values + case["table"] * case["hidden"]) * size if case["train"] else 0),
            "flops": values * (2 if case["train"] else 1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        x, w = s["x"].detach().double(), s["weight"].detach().double()
        n = x.shape[1]
        mean = x.sum(1, keepdim=True) / n
        std = (((x - mean) ** 2).sum(1, keepdim=True) / n + EPS).sqrt()
        z = (x - mean) / std
        out = [z * w if s["bias"] is None else torch.addcmul(s["bias"].detach().double(), z, w)]
        if s["train"]:
            dy = s["dy"].double()
            dz = dy * w
            # the projection of dz onto what is orthogonal to the ones and to z
            dz -= dz.sum(1, keepdim=True) / n + z * ((dz * z).sum(1, keepdim=True) / n)
            out += [dz / std, torch.einsum("ij,ij->j", dy, z)]
            if s["bias"] is not None:
                out.append(torch.ones(1, x.shape[0], dtype=torch.float64, device=x.device).mm(dy)[0])
        return out
    if case["kind"] == "clip":
        flat = s["flat"]
        parts = flat.split(1 << 26)
        norm = math.sqrt(math.fsum(float(p.double().dot(p.double())) for p in parts))
        factor = min(1.0, s["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64), flat.double().mul_(factor)]
    ids, w = s["ids"], s["weight"].detach()
    out = [w.index_select(0, ids).double() * s["scale"]]
    if s["train"]:
        counted = torch.ones_like(ids, dtype=torch.bool) if s["padding"] is None else ids != s["padding"]
        grad = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        grad.index_put_((ids[counted],), s["dy"][counted].double() * s["scale"], accumulate=True)
        out.append(grad)
    return out
