"""Layer norm, embedding and the norm of many tensors without a GPU: what the entry points refuse, and the sizes of workspaces.
No kernel is launched: every refusal is the host's, ahead of any launch."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses import FakeTensorMode

import fp8_gmm_amd as pkg
from fp8_gmm_amd import _lib, backend, moe, native

OK, NULL, SHAPE, FORMAT, ALIGN, ARGUMENT, WORKSPACE = 0, -1, -2, -3, -4, -6, -9
P = 0x10000   # an address that nothing follows


def test_cpu_tensors_are_refused():
    x, w = torch.ones(2, 8), torch.ones(8)
    for call in (lambda: pkg.layer_norm(x, w), lambda: pkg.embedding(torch.tensor([0]), x), lambda: backend.multi_norm([x]),
                 lambda: backend.multi_clip([x], [x], 1.0), lambda: pkg.LayerNorm(8, device="cpu")(x),
                 lambda: pkg.Embedding(4, 8, device="cpu")(torch.tensor([1]))):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


def test_modules_hold_their_parameters():
    norm = pkg.LayerNorm(16, eps=1e-6, bias=False, dtype=torch.float32, device="cpu")
    assert norm.bias is None and list(norm.state_dict()) == ["weight"] and (norm.weight == 1).all() and "1e-06" in repr(norm)
    table = pkg.Embedding(10, 4, scale=2.0, padding_idx=-1, device="cpu")
    assert table.weight.shape == (10, 4) and not table.weight[9].any() and table.weight[8].any() and "scale=2.0" in repr(table)
    plain = moe.Fp8MlpModule(32, 64, 2, 1, device="cpu")
    normed = moe.Fp8LinearModule(32, 64, 2, 1, device="cpu", layer_norm=True)
    assert plain.row_norm is None and not any("norm" in k for k in plain.state_dict())
    assert {"row_norm.weight", "row_norm.bias"} <= set(normed.state_dict())


def test_clipping_without_gradients():
    p = torch.nn.Parameter(torch.ones(3))
    assert pkg.clip_grad_norm_([p], 1.0) == 0.0 and pkg.clip_grad_norm_(p, 1.0) == 0.0
    with pytest.raises(RuntimeError, match="2-norm"):
        pkg.clip_grad_norm_([p], 1.0, norm_type=float("inf"))


def test_layer_norm_status():
    L = _lib.load()

    def forward(x=P, ldx=64, w=P, b=None, y=P, mean=None, rstd=None, rows=4, cols=64, eps=1e-5, t=0, p=0):
        return L.fp8gmm_layer_norm(x, ldx, w, b, y, mean, rstd, rows, cols, eps, t, p, None)

    def backward(dy=P, ldy=64, x=P, ldx=64, w=P, mean=P, rstd=P, dx=P, dw=P, db=P, rows=4, cols=64, t=0, p=0, work=P, size=1 << 20):
        return L.fp8gmm_layer_norm_backward(dy, ldy, x, ldx, w, mean, rstd, dx, dw, db, rows, cols, t, p, work, size, None)

    for call in (forward, backward):
        for bad, status in ((dict(t=3), FORMAT), (dict(t=-1), FORMAT), (dict(t=2, p=0), FORMAT), (dict(t=0, p=1), FORMAT),
                            (dict(rows=-1), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(cols=0), SHAPE), (dict(cols=(1 << 30) + 1), SHAPE),
                            (dict(ldx=63), SHAPE), (dict(x=None), NULL), (dict(w=None), NULL)):
            assert call(**bad) == status, bad
    assert forward(y=None) == NULL and forward(mean=P) == NULL and forward(rstd=P) == NULL
    assert forward(eps=-1.0) == ARGUMENT and forward(eps=float("nan")) == ARGUMENT
    assert forward(rows=0, x=None, y=None) == OK
    assert backward(ldy=63) == SHAPE and backward(mean=None) == NULL and backward(dy=None) == NULL and backward(work=None) == NULL
    assert backward(work=P + 8) == ALIGN
    need = L.fp8gmm_layer_norm_workspace_bytes(4, 64, 0)
    assert need > 0 and backward(size=need - 1) == WORKSPACE
    assert backward(dx=None, dw=None, db=None) == OK and backward(rows=0, dw=None, db=None) == OK


def test_layer_norm_workspace_holds_a_partial_sum_of_both_gradients_per_workgroup():
    L = _lib.load()
    for rows, cols, t in ((1, 1, 0), (1, 4096, 0), (100, 4097, 2), (16384, 4096, 0), (65536, 2048, 2), (10, 100000, 1)):
        size = L.fp8gmm_layer_norm_workspace_bytes(rows, cols, t)
        assert size % (8 * cols) == 0 and 1 <= size // (8 * cols) <= min(rows, 512)
    assert L.fp8gmm_layer_norm_workspace_bytes(0, 64, 0) == 0 and L.fp8gmm_layer_norm_workspace_bytes(4, 0, 0) == 0


def test_embedding_status():
    L = _lib.load()

    def lookup(ids=P, ids64=1, n=4, w=P, table=10, cols=8, scale=1.0, t=0, y=P):
        return L.fp8gmm_embedding(ids, ids64, n, w, table, cols, scale, t, y, None)

    def backward(ids=P, ids64=1, n=4000, dy=P, dw=P, table=10, cols=8, scale=1.0, padding=-1, t=0, work=P, size=1 << 30):
        return L.fp8gmm_embedding_backward(ids, ids64, n, dy, dw, table, cols, scale, padding, t, work, size, None)

    for call in (lookup, backward):
        for bad, status in ((dict(t=3), FORMAT), (dict(n=-1), SHAPE), (dict(n=(1 << 28) + 1), SHAPE), (dict(table=-1), SHAPE),
                            (dict(table=(1 << 31) - 1), SHAPE), (dict(cols=-1), SHAPE), (dict(cols=(1 << 23) + 1), SHAPE), (dict(ids=None), NULL)):
            assert call(**bad) == status, bad
    assert lookup(w=None) == NULL and lookup(y=None) == NULL and lookup(n=0, ids=None, w=None, y=None) == OK and lookup(cols=0) == OK
    assert backward(dw=None) == NULL and backward(dy=None) == NULL and backward(work=None) == NULL
    assert backward(dw=P + 8) == ALIGN and backward(work=P + 4) == ALIGN
    assert backward(table=0) == OK and backward(cols=0) == OK
    need = L.fp8gmm_embedding_workspace_bytes(4000, 10, 8, 0)
    assert L.fp8gmm_embedding_workspace_bytes(4, 10, 8, 0) == 0 and need > 0 and backward(size=need - 1) == WORKSPACE
    assert L.fp8gmm_embedding_workspace_bytes(0, 10, 8, 0) == 0 and L.fp8gmm_embedding_workspace_bytes(4, 0, 8, 0) == 0


def test_multi_norm_status():
    L = _lib.load()
    assert ctypes.sizeof(_lib.NormTensor) == 32

    def call(tensors, clip, n=None, norm=P, work=P, size=1 << 20, max_norm=1.0):
        table = (_lib.NormTensor * max(1, len(tensors)))(*[_lib.NormTensor(*t) for t in tensors])
        n = len(tensors) if n is None else n
        if clip:
            return L.fp8gmm_multi_clip(table, n, max_norm, norm, work, size, None)
        return L.fp8gmm_multi_norm(table, n, norm, work, size, None)

    good = (P, P, 10, 0, 0)
    for clip in (False, True):
        assert call([good], clip, n=-1) == ARGUMENT and call([good], clip, norm=None) == NULL and call([good], clip, work=None) == NULL
        assert call([good], clip, work=P + 8) == ALIGN and call([good], clip, size=L.fp8gmm_multi_norm_workspace_bytes(1) - 1) == WORKSPACE
        for bad, status in (((P, P, 10, 3, 0), FORMAT), ((P, P, -1, 0, 0), SHAPE), ((P, P, 1 << 40, 0, 0), SHAPE), (((1 << 48) + P, P, 10, 0, 0), ARGUMENT), ((None, P, 10, 0, 0), NULL),
                            ((P + 1, P, 10, 0, 0), ALIGN), ((P + 2, P, 10, 2, 2), ALIGN)):
            assert call([good, bad], clip) == status, bad
        assert call([(P, P, 1 << 39, 0, 0), (P, P, 1 << 39, 0, 0)], clip) == SHAPE
    assert L.fp8gmm_multi_norm(None, 1, P, P, 1 << 20, None) == NULL
    for bad, status in (((P, None, 10, 0, 0), NULL), ((P, P, 10, 0, 1), FORMAT), ((P, P, 10, 2, 0), FORMAT), ((P, P + 2, 10, 0, 2), ALIGN), ((P, (1 << 48) + P, 10, 0, 0), ARGUMENT),
                        ((P, P, 10, 0, 2), ARGUMENT), ((P, P + 18, 10, 0, 0), ARGUMENT), ((P + 18, P, 10, 0, 0), ARGUMENT)):
        assert call([bad], True) == status, bad
    assert call([good, good], True) == ARGUMENT                                         # the same one twice
    assert call([good, (P + 4, P + 4096, 10, 0, 0)], True) == ARGUMENT                  # what one writes another reads
    assert call([(P, P + 4096, 10, 0, 0), (P + 64, P + 4100, 10, 0, 0)], True) == ARGUMENT
    assert call([good], True, max_norm=-1.0) == ARGUMENT and call([good], True, max_norm=float("nan")) == ARGUMENT
    assert L.fp8gmm_multi_norm_workspace_bytes(-1) == 0 and L.fp8gmm_multi_norm_workspace_bytes(0) > 0


# Tensors without memory that say they are on a GPU: a refusal ahead of any launch needs no more.
def fake_gpu(*shape, dtype=torch.bfloat16):
    return torch.empty(1, dtype=dtype, device="cuda").expand(*shape)


@pytest.mark.parametrize("rows, cols", [(1, (1 << 30) + 1), (1, (1 << 32) + 64), (3, 1 << 32), (1 << 31, 8), ((1 << 32) + 1, 8)])
def test_layer_norm_refuses_sizes_before_they_are_cut_to_32_bits(rows, cols):
    with FakeTensorMode():
        x, w = fake_gpu(rows, cols), fake_gpu(cols)
        with pytest.raises(RuntimeError, match=r"2\^30 columns"):
            pkg.layer_norm(x, w)


@pytest.mark.parametrize("grad", [True, False], ids=["with gradients", "without"])
def test_tangents_are_refused_whatever_the_gradient_mode(grad):
    """torch keeps tangents under ``no_grad``, so a result without one would be a wrong derivative; it drops them in inference mode."""
    with FakeTensorMode(), fw.dual_level():
        x, table, ids = torch.empty(3, 16, device="cuda"), torch.empty(5, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
        w = torch.empty(16, device="cuda")
        dx, dw, dt = (fw.make_dual(t, torch.empty_like(t)) for t in (x, w, table))
        calls = [lambda: pkg.layer_norm(dx, w), lambda: pkg.layer_norm(x, dw), lambda: pkg.layer_norm(x, w, dw), lambda: pkg.embedding(ids, dt)]
        for call in calls:
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.inference_mode(), pytest.raises(Exception) as e:   # goes on as far as the missing GPU
                call()
            assert "forward-mode" not in str(e.value)


@pytest.mark.parametrize("grad", [True, False], ids=["with gradients", "without"])
def test_grouped_modules_refuse_tangents_whatever_the_gradient_mode(grad):
    with FakeTensorMode(), fw.dual_level():
        scores = fw.make_dual(torch.empty(3, 8, device="cuda"), torch.empty(3, 8, device="cuda"))
        with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
            native.route(scores, 2)


def test_transforms_and_tracing_are_refused():
    x, w, ids = torch.ones(3, 8), torch.ones(8), torch.zeros(2, dtype=torch.int64)
    for name, call in (("layer_norm", lambda t: pkg.layer_norm(t, w)), ("embedding", lambda t: pkg.embedding(ids, t[None])),
                       ("multi_norm", lambda t: backend.multi_norm([t])), ("multi_clip", lambda t: backend.multi_clip([t], [t], 1.0))):
        for transformed in (lambda: torch.func.vmap(call)(x), lambda: torch.func.grad(lambda t: call(t).sum())(w),
                            lambda: torch.func.jvp(call, (w,), (w,)), lambda: torch.jit.trace(call, (w,), check_trace=False)):
            with pytest.raises(RuntimeError, match=f"{name} does not run under torch.func transforms or tracing"):
                transformed()
        with pytest.raises(RuntimeError, match="GPU tensors"):   # and not afterwards
            call(w)
