"""Root-mean-square norm, the choice of experts and the optimizer's step without a GPU: what the entry points refuse, and the sizes of
workspaces.  No kernel is launched: every refusal is the host's, ahead of any launch."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses import FakeTensorMode

import fp8_gmm_amd as pkg
from fp8_gmm_amd import _lib, backend, moe, moe_ops

OK, NULL, SHAPE, FORMAT, ALIGN, ARGUMENT, WORKSPACE = 0, -1, -2, -3, -4, -6, -9
P = 0x10000   # an address that nothing follows


def test_cpu_tensors_are_refused():
    x, w = torch.ones(2, 8), torch.ones(8)
    for call in (lambda: pkg.rms_norm(x, w), lambda: pkg.rms_norm(x, w, 1e-5, x), lambda: pkg.rms_norm_fp8(x, w),
                 lambda: pkg.RMSNorm(8, device="cpu")(x), lambda: moe_ops.select_experts(x, 2),
                 lambda: backend.multi_adamw([x], [x], [x], [x], 1, 1e-3)):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


def test_lists_of_what_is_no_tensor_are_refused():
    x = torch.ones(8)
    for bad in (5, None, [x, None], [x, 1.0], ["x"], [[x]]):
        for i in range(4):
            with pytest.raises(TypeError):
                backend.multi_adamw(*[bad if j == i else [x] for j in range(4)], 1, 1e-3)
        with pytest.raises(TypeError):
            backend.multi_adamw([x], [x], [x], [x], 1, 1e-3, scales=([x], bad))
        with pytest.raises(RuntimeError if bad is None else TypeError):   # None: without masters
            backend.multi_adamw([x], [x], [x], [x], 1, 1e-3, masters=bad)
    for given in ((x,), iter([x]), (t for t in [x])):   # anything that iterates over tensors
        with pytest.raises(RuntimeError, match="GPU tensors"):
            backend.multi_adamw(given, [x], [x], [x], 1, 1e-3)


def test_modules_hold_their_parameters():
    norm = pkg.RMSNorm(16, eps=1e-6, dtype=torch.float32, device="cpu")
    assert list(norm.state_dict()) == ["weight"] and (norm.weight == 1).all() and "1e-06" in repr(norm)
    plain = moe.Fp8MlpModule(32, 64, 4, 1, device="cpu")
    assert not any("norm" in k or "bias" in k for k in plain.state_dict()) and plain.row_norm is None
    assert not hasattr(plain, "expert_bias") and not hasattr(plain, "tokens_per_expert")
    normed = moe.Fp8LinearModule(32, 64, 4, 1, device="cpu", rms_norm=True, routing=moe_ops.Routing("sigmoid", bias=True))
    assert {"row_norm.weight", "expert_bias"} <= set(normed.state_dict()) and "row_norm.bias" not in normed.state_dict()
    assert normed.expert_bias.dtype == torch.float32 and not normed.expert_bias.any()
    unbiased = moe.Fp8MlpModule(32, 64, 4, 1, device="cpu", routing=moe_ops.Routing())
    assert unbiased.expert_bias is None and "expert_bias" not in unbiased.state_dict()
    with pytest.raises(ValueError, match="one norm"):
        moe.Fp8MlpModule(32, 64, 4, 1, device="cpu", layer_norm=True, rms_norm=True)
    with pytest.raises(ValueError, match="scoring"):
        moe_ops.Routing("max")


def test_optimizer_options():
    p = [torch.nn.Parameter(torch.ones(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.5)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16),
                dict(max_norm=-1.0), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            pkg.AdamW(p, **bad)
    opt = pkg.AdamW(p, lr=1e-2, state_bits=8)
    opt.step()   # nothing to do without gradients
    assert opt.state_dict()["param_groups"][0]["lr"] == 1e-2 and not opt.state
    opt.step(lambda: None)
    assert opt.step(lambda: torch.tensor(2.0)) == 2.0
    p[0].grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        opt.step()


def test_optimizer_state_keeps_its_types_in_a_checkpoint():
    p = [torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16)), torch.nn.Parameter(torch.ones(2, dtype=torch.bfloat16))]
    opt = pkg.AdamW(p, state_bits=8, master_weights=True)
    for q in p:
        q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="GPU tensors"):   # the states are there, the step is not
        opt.step()
    state = opt.state[p[0]]
    state["exp_avg_scale"].fill_(1 / 3)
    state["master"].fill_(1 / 3)
    other = pkg.AdamW([torch.nn.Parameter(q.detach().clone()) for q in p], state_bits=8, master_weights=True)
    other.load_state_dict(opt.state_dict())
    got = other.state[other.param_groups[0]["params"][0]]
    assert got["exp_avg"].dtype == torch.float8_e4m3fn and got["exp_avg_scale"].dtype == got["master"].dtype == torch.float32
    assert torch.equal(got["master"], state["master"]) and got["master"] is not state["master"] and got["exp_avg_scale"].shape == (3,)


def test_optimizer_takes_a_checkpoint_of_other_options():
    def make(**options):
        return pkg.AdamW([torch.nn.Parameter(torch.full((3,), i + 1.0, dtype=torch.bfloat16)) for i in range(2)], **options)

    def stepped(*steps, **options):
        opt = make(**options)
        for p, step in zip(opt.param_groups[0]["params"], steps):
            opt._init_state(p, opt.state[p])
            if not opt.capturable:
                opt.state[p]["step"] = step
        if opt.capturable:
            opt.param_groups[0]["steps"] = torch.tensor(steps[0])
        return opt

    counted = make()
    counted.load_state_dict(stepped(7, 7, capturable=True, lr=torch.tensor(0.5)).state_dict())
    assert all(counted.state[p]["step"] == 7 for p in counted.param_groups[0]["params"])
    assert counted.param_groups[0]["steps"] is None and counted.param_groups[0]["lr"] == 0.5
    on_device = make(capturable=True)
    on_device.load_state_dict(stepped(4, 4).state_dict())
    assert on_device.param_groups[0]["steps"].dtype == torch.int64 and on_device.param_groups[0]["steps"].item() == 4
    assert not any("step" in on_device.state[p] for p in on_device.param_groups[0]["params"])
    fresh = make(capturable=True)
    fresh.load_state_dict(make().state_dict())
    assert fresh.param_groups[0]["steps"] is None and not fresh.state
    with pytest.raises(ValueError, match="different"):
        make(capturable=True).load_state_dict(stepped(4, 5).state_dict())
    masters = make(master_weights=True)
    masters.load_state_dict(stepped(4, 4).state_dict())
    assert all(torch.equal(masters.state[p]["master"], p.detach().float()) for p in masters.param_groups[0]["params"])
    without = make()
    without.load_state_dict(masters.state_dict())
    assert not any("master" in without.state[p] for p in without.param_groups[0]["params"])
    plain = torch.optim.AdamW([torch.nn.Parameter(torch.ones(3)) for _ in range(2)])
    for opt, other in ((make(), stepped(1, 1, state_bits=8)), (make(state_bits=8), stepped(1, 1)), (make(), plain)):
        with pytest.raises(ValueError, match="not a checkpoint"):
            opt.load_state_dict(other.state_dict())
        assert not opt.state


def test_rms_norm_status():
    L = _lib.load()

    def forward(x=P, ldx=64, res=None, ldr=64, w=P, y=P, h=None, rstd=None, rows=4, cols=64, eps=1e-5, t=0, p=0):
        return L.fp8gmm_rms_norm(x, ldx, res, ldr, w, y, h, rstd, rows, cols, eps, t, p, None)

    def fp8(x=P, ldx=64, res=None, ldr=64, w=P, q=P, h=None, scale=P, amax=None, inv=None, rows=4, cols=64, eps=1e-5, t=0, p=0, fmt=0):
        return L.fp8gmm_rms_norm_fp8(x, ldx, res, ldr, w, q, h, scale, amax, inv, rows, cols, eps, t, p, fmt, None)

    def backward(dy=P, ldy=64, dh=None, ldd=64, h=P, ldh=64, w=P, rstd=P, dx=P, dw=P, rows=4, cols=64, t=0, p=0, work=P, size=1 << 20):
        return L.fp8gmm_rms_norm_backward(dy, ldy, dh, ldd, h, ldh, w, rstd, dx, dw, rows, cols, t, p, work, size, None)

    for call in (forward, fp8, backward):
        for bad, status in ((dict(t=3), FORMAT), (dict(t=-1), FORMAT), (dict(t=2, p=0), FORMAT), (dict(t=0, p=1), FORMAT),
                            (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(cols=0), SHAPE), (dict(cols=(1 << 30) + 1), SHAPE),
                            (dict(w=None), NULL)):
            assert call(**bad) == status, bad
    for call in (forward, fp8):
        assert call(x=None) == NULL and call(ldx=63) == SHAPE and call(res=P, ldr=63, h=P) == SHAPE and call(res=P) == NULL
        assert call(eps=-1.0) == ARGUMENT and call(eps=float("nan")) == ARGUMENT and call(rows=0, x=None) == OK
    assert forward(y=None) == NULL and fp8(q=None) == NULL and fp8(fmt=2) == FORMAT
    assert fp8(scale=None) == ARGUMENT and fp8(inv=P) == ARGUMENT and fp8(scale=None, inv=P, amax=P) == ARGUMENT
    assert backward(ldy=63) == SHAPE and backward(ldh=63) == SHAPE and backward(dh=P, ldd=63) == SHAPE
    assert backward(dy=None) == NULL and backward(h=None) == NULL and backward(rstd=None) == NULL and backward(work=None) == NULL
    assert backward(work=P + 8) == ALIGN
    need = L.fp8gmm_rms_norm_workspace_bytes(4, 64, 0)
    assert need > 0 and backward(size=need - 1) == WORKSPACE
    assert backward(dx=None, dw=None) == OK and backward(rows=0, dw=None) == OK
    for rows, cols, t in ((1, 1, 0), (1, 4096, 0), (100, 4097, 2), (16384, 4096, 0), (65536, 2048, 2), (10, 100000, 1)):
        size = L.fp8gmm_rms_norm_workspace_bytes(rows, cols, t)
        assert size % (4 * cols) == 0 and 1 <= size // (4 * cols) <= min(rows, 512)
    assert L.fp8gmm_rms_norm_workspace_bytes(0, 64, 0) == 0 and L.fp8gmm_rms_norm_workspace_bytes(4, 0, 0) == 0


class Choice(ctypes.Structure):
    _fields_ = [("bias", ctypes.c_void_p)] + [(n, ctypes.c_int32) for n in (
        "experts", "top_k", "scoring", "groups", "top_groups", "group_best", "renormalize")] + [("scale", ctypes.c_float)]


def test_choice_status():
    L = _lib.load()
    assert ctypes.sizeof(Choice) == 40

    def choice(**kw):
        return ctypes.byref(Choice(**{**dict(bias=None, experts=64, top_k=8, scoring=1, groups=8, top_groups=4, group_best=2, renormalize=1,
                                             scale=1.0), **kw}))

    def forward(c, scores=P, t=0, tokens=4, w=P, s=P):
        return L.fp8gmm_select_experts(scores, t, tokens, c, w, s, None)

    def backward(c, scores=P, t=0, tokens=4, s=P, dw=P, ds=P):
        return L.fp8gmm_select_experts_backward(scores, t, tokens, c, s, dw, ds, None)

    for call in (forward, backward):
        for bad in (dict(top_k=0), dict(top_k=17), dict(top_groups=1, top_k=9), dict(groups=0), dict(groups=5), dict(groups=32), dict(top_groups=0),
                    dict(top_groups=9), dict(group_best=0), dict(group_best=3), dict(scoring=2), dict(scoring=-1)):
            assert call(choice(**bad)) == ARGUMENT, bad
        for bad in (dict(experts=0), dict(experts=4097), dict(experts=-1)):
            assert call(choice(**bad)) == SHAPE
        assert call(None) == NULL and call(choice(), t=3) == FORMAT and call(choice(), tokens=-1) == SHAPE and call(choice(), tokens=1 << 31) == SHAPE
        assert call(choice(), scores=None) == NULL and call(choice(), s=None) == NULL and call(choice(), tokens=0, scores=None) == OK
    assert forward(choice(), w=None) == NULL and backward(choice(), dw=None) == NULL and backward(choice(), ds=None) == NULL


class AdamwTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")] + [
        ("count", ctypes.c_int64), ("type", ctypes.c_int32), ("grad_type", ctypes.c_int32)]


class AdamwStep(ctypes.Structure):
    _fields_ = [(n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "max_norm")] + [
        (n, ctypes.c_void_p) for n in ("norm", "step_dev", "lr_dev")] + [("step", ctypes.c_int64), ("bits", ctypes.c_int32),
                                                                         ("reserved", ctypes.c_int32)]


def test_adamw_status():
    L = _lib.load()
    assert ctypes.sizeof(AdamwTensor) == 72 and ctypes.sizeof(AdamwStep) == 88
    step = 0x100000

    def tensor(at=0, **kw):
        place = P + at * 8 * step
        names = ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
        return AdamwTensor(**{**{n: place + i * step for i, n in enumerate(names)}, "master": None, "count": 1000, "type": 0, "grad_type": 0, **kw})

    def call(*tensors, **kw):
        table = (AdamwTensor * max(1, len(tensors)))(*tensors)
        a = AdamwStep(**{**dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, step=1, bits=32), **kw})
        return L.fp8gmm_multi_adamw(table, len(tensors), ctypes.byref(a), None)

    assert call() == OK and call(tensor(count=0, param=None)) == OK
    for bad in (dict(bits=16), dict(step=0), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(eps=-1.0), dict(weight_decay=-1.0),
                dict(lr=-1.0), dict(lr=float("nan")), dict(norm=P, max_norm=-1.0)):
        assert call(tensor(), **bad) == ARGUMENT, bad
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert call(tensor(**{name: None})) == NULL
        assert call(tensor(**{name: P + 1})) == ALIGN
    for name in ("exp_avg_scale", "exp_avg_sq_scale"):
        assert call(tensor(**{name: None}), bits=8) == NULL and call(tensor(**{name: P + 2}), bits=8) == ALIGN
    assert call(tensor(exp_avg=P + 4 * step + 4), bits=8) == ALIGN
    for bad in (dict(type=3), dict(type=-1), dict(type=2, grad_type=0), dict(type=0, grad_type=1)):
        assert call(tensor(**bad)) == FORMAT
    for count in (-1, (1 << 32) + 1):
        assert call(tensor(count=count)) == SHAPE
    assert call(tensor(type=2, grad_type=2, master=P + 7 * step)) == ARGUMENT               # its own master
    assert call(tensor(), tensor(1, master=P + 7 * step)) == ARGUMENT                       # masters of some
    assert call(tensor(), tensor()) == ARGUMENT and call(tensor(grad=P)) == ARGUMENT        # shared memory
    assert call(tensor(exp_avg=P + 1998)) == ALIGN and call(tensor(exp_avg=P + 1996)) == ARGUMENT
    assert call(tensor(exp_avg_scale=P + 5 * step), bits=8) == ARGUMENT
    for name in ("norm", "step_dev", "lr_dev"):
        assert call(tensor(), **{name: P + 1800}) == ARGUMENT and call(tensor(), **{name: P + 2 * step + 16}) == ARGUMENT
        assert call(tensor(), **{name: P - 2}) == ALIGN
    # in any order of the tensors' addresses
    assert call(tensor(3), tensor(1), tensor(2, param=P + (8 + 2) * step + 400)) == ARGUMENT
    assert call(tensor(1), tensor(3), tensor(2), tensor(0), tensor(2)) == ARGUMENT
    assert L.fp8gmm_multi_adamw(None, 1, ctypes.byref(AdamwStep(bits=32, step=1)), None) == NULL
    assert L.fp8gmm_multi_adamw(None, 0, None, None) == NULL and L.fp8gmm_multi_adamw(None, -1, None, None) == ARGUMENT


def fake_gpu(*shape, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype)


@pytest.mark.parametrize("rows, cols", [(1, (1 << 30) + 1), (1, (1 << 32) + 64), (3, 1 << 32), (1 << 31, 8), ((1 << 32) + 1, 8)])
def test_sizes_are_refused_before_they_are_cut_to_32_bits(rows, cols):
    with FakeTensorMode():
        x, w = fake_gpu(rows, cols), fake_gpu(cols)
        for call in (lambda: pkg.rms_norm(x, w), lambda: pkg.rms_norm(x, w, 1e-5, x), lambda: pkg.rms_norm_fp8(x, w)):
            with pytest.raises(RuntimeError, match=r"2\^30 columns"):
                call()
        with pytest.raises(RuntimeError, match="experts are supported"):
            moe_ops.select_experts(x, 1)
        if rows * cols > 1 << 32:
            with pytest.raises(RuntimeError, match=r"2\^32 elements"):
                backend.multi_adamw([x], [x], [x], [x], 1, 1e-3)
    with FakeTensorMode():
        with pytest.raises(RuntimeError, match="top_k"):
            moe_ops.select_experts(fake_gpu(4, 64), (1 << 32) + 1)
        with pytest.raises(RuntimeError, match="groups"):
            moe_ops.select_experts(fake_gpu(4, 64), 1, groups=(1 << 32) + 1)


@pytest.mark.parametrize("grad", [True, False], ids=["with gradients", "without"])
def test_tangents_are_refused_whatever_the_gradient_mode(grad):
    with FakeTensorMode(), fw.dual_level():
        x, w, one = fake_gpu(3, 16), fake_gpu(16), fake_gpu(1)
        dx, dw, d1 = (fw.make_dual(t, torch.empty_like(t)) for t in (x, w, one))
        calls = [lambda: pkg.rms_norm(dx, w), lambda: pkg.rms_norm(x, dw), lambda: pkg.rms_norm(x, w, 1e-5, dx),
                 lambda: pkg.rms_norm_fp8(dx, w), lambda: pkg.rms_norm_fp8(x, w, 1e-5, dx), lambda: moe_ops.select_experts(dx, 2),
                 lambda: moe_ops.select_experts(x, 2, bias=dw)]
        calls += [lambda i=i: backend.multi_adamw(*[[dx if j == i else x] for j in range(4)], 1, 1e-3) for i in range(4)]
        calls += [lambda: backend.multi_adamw([x], [x], [x], [x], 1, 1e-3, norm=d1, max_norm=1.0),
                  lambda: backend.multi_adamw([x], [x], [x], [x], 1, d1)]
        for call in calls:
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_transforms_and_tracing_are_refused():
    x, w = torch.ones(3, 8), torch.ones(8)
    for name, call in (("rms_norm", lambda t: pkg.rms_norm(t, w)), ("rms_norm_fp8", lambda t: pkg.rms_norm_fp8(t, w)[0].float()),
                       ("select_experts", lambda t: moe_ops.select_experts(t[None], 2)[0]),
                       ("multi_adamw", lambda t: backend.multi_adamw([t], [t], [t], [t], 1, 1e-3))):
        for transformed in (lambda: torch.func.vmap(call)(x), lambda: torch.func.grad(lambda t: call(t).sum())(w),
                            lambda: torch.func.jvp(call, (w,), (w,)), lambda: torch.jit.trace(call, (w,), check_trace=False)):
            with pytest.raises(RuntimeError, match=f"{name} does not run under torch.func transforms or tracing"):
                transformed()
        with pytest.raises(RuntimeError, match="GPU tensors"):   # and not afterwards
            call(w)
