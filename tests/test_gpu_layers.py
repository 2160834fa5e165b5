"""Layer norm and embedding with their gradients on the GPU, against plain implementations in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, h half a step of the result's type (``finfo.eps / 2``).  A sum of
a row is taken by at most 1024 threads, each over cols / threads elements (at most 32 of them where a row fits the registers),
then by halving and over at most 16 wavefronts: K(cols) = 64 + cols / 1024 additions bound its error by K u times the sum of the
magnitudes, and a factor of 2 covers the few products around it."""
import math

import pytest
import torch
import torch.utils.checkpoint

import fp8_gmm_amd as pkg
from fp8_gmm_amd import moe

from helpers import gen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PAIRS = [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")]


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    """Half a step of the type's subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def assert_within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} are off, by up to {(off / tol)[bad].max().item():.3g} of what is allowed"


def norm_reference(x, w, b, dy, eps):
    """(y, dx, dw, db) in 64 bits, and the bound of each one's error in 32 bits (without the final rounding)."""
    x, w, dy = x.double(), w.double(), dy.double()
    cols, rows = x.shape[1], x.shape[0]
    k = 2 * (64 + cols / 1024) * U
    mean = x.mean(1, keepdim=True)
    r = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    z = (x - mean) * r
    y = z * w + (b.double() if b is not None else 0.0)
    dz = k * (r * x.abs().mean(1, keepdim=True) + z.abs())   # error of z: of the mean, and of r and the products
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * z).mean(1, keepdim=True)
    dx = r * (g - m1 - z * m2)
    tol_y = dz * w.abs() + 2 * U * (y.abs() + (b.double().abs() if b is not None else 0.0))
    tol_x = r * (k * (g.abs() + g.abs().mean(1, keepdim=True) + z.abs() * (g * z).abs().mean(1, keepdim=True))
                 + m2.abs() * dz + z.abs() * (g.abs() * dz).mean(1, keepdim=True))
    # rows: some per thread, then per workgroup, then over the workgroups, a sixteenth at a time
    kr = (64 + rows / 256) * U
    tol_w = kr * (dy * z).abs().sum(0) + (dy.abs() * dz).sum(0)
    tol_b = kr * dy.abs().sum(0)
    return (y, dx, (dy * z).sum(0), dy.sum(0)), (tol_y, tol_x, tol_w, tol_b)


def norm_inputs(dev, rows, cols, t, p, bias, seed, offset=0.0):
    g = gen(seed)
    x = (torch.randn(rows, cols, generator=g) * 2 + torch.randn(1, cols, generator=g) + offset).to(TYPES[t]).to(dev)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(TYPES[p]).to(dev)
    b = (0.3 * torch.randn(cols, generator=g)).to(TYPES[p]).to(dev) if bias else None
    dy = (0.1 * torch.randn(rows, cols, generator=g)).to(TYPES[t]).to(dev)
    return x, w, b, dy


def check_norm(x, w, b, dy, eps=1e-5, what=""):
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    bs = b.detach().requires_grad_() if b is not None else None
    y = pkg.layer_norm(xs, ws, bs, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(pkg.layer_norm(x, w, b, eps), y), "inference differs from training"
    got = (y,) + torch.autograd.grad(y, [t for t in (xs, ws, bs) if t is not None], dy)
    flat = [t.reshape(-1, x.shape[-1]) for t in (x, dy)]
    want, tol = norm_reference(flat[0], w, b, flat[1], eps)
    for a, v, e, name in zip(got, want, tol, ("y", "dx", "dw", "db")):
        assert_within(a.detach().reshape(v.shape), v, e + half_step(a.dtype) * (v.abs() + e) + smallest(a.dtype), f"{what} {name}")
    return got


SHAPES = [(1, 1), (3, 7), (5, 64), (40, 127), (17, 129), (33, 512), (7, 1000), (129, 1411), (65, 2048), (1531, 1024), (9, 4097),
          (300, 4096), (3, 8191), (5, 16384), (700, 768), (5000, 24)]
# columns on both sides of where a row takes another number of threads, of pieces per thread, or another kernel
SHAPES += [(37, c + d) for c in (4, 8, 64, 128, 256, 512, 768, 1024, 1536, 2048, 6144, 8192, 16384) for d in (-1, 0, 1, 8)]
SHAPES += [(1001, c) for c in (192, 193, 384, 385)] + [(70000, 129)]


@pytest.mark.parametrize("rows, cols", SHAPES)
@pytest.mark.parametrize("t, p", PAIRS)
def test_layer_norm_against_64_bits(dev, rows, cols, t, p):
    check_norm(*norm_inputs(dev, rows, cols, t, p, (rows + cols) % 3 != 0, 1000 + rows + cols), what=f"{rows} x {cols}")


@pytest.mark.parametrize("t, p, cols", [("bf16", "fp32", 32768), ("fp16", "fp16", 32769), ("fp32", "fp32", 16384), ("fp32", "fp32", 20001),
                                        ("bf16", "bf16", 70003)])
def test_layer_norm_of_long_rows(dev, t, p, cols):
    """The widest rows that stay in registers, and those that do not."""
    check_norm(*norm_inputs(dev, 70, cols, t, p, True, cols), what=f"{cols} columns")


@pytest.mark.parametrize("t, offset", [("fp32", 1000.0), ("fp32", -3e4), ("bf16", 200.0)])
def test_layer_norm_of_rows_far_off_zero(dev, t, offset):
    check_norm(*norm_inputs(dev, 37, 1030, t, "fp32", True, 5, offset), what=f"offset {offset}")


@pytest.mark.parametrize("t, cols", [("fp32", 512), ("fp32", 768), ("fp32", 2048), ("fp32", 4096), ("bf16", 2048)])
def test_layer_norm_of_whole_pieces_off_their_alignment(dev, t, cols):
    """Rows that share their threads another way when they, or their gradients, begin between two pieces."""
    x, w, b, dy = norm_inputs(dev, 130, cols, t, t, True, cols)
    off = torch.empty(130 * cols + 1, dtype=x.dtype, device=dev)
    for xv, dv in ((x, dy), (off[1:].view(130, cols).copy_(x), dy), (x, off[1:].view(130, cols).copy_(dy))):
        check_norm(xv, w, b, dv, what=f"{xv.data_ptr() % 16} {dv.data_ptr() % 16}")


def test_layer_norm_takes_views(dev):
    """Rows with a pitch, at any element, of more dimensions; columns that are no neighbours; gradients that are expanded."""
    x, w, b, dy = norm_inputs(dev, 24, 650, "bf16", "bf16", True, 7)
    want = check_norm(x, w, b, dy)
    wide = torch.empty(24, 1301, dtype=x.dtype, device=dev)
    wide[:, 3:653] = x
    dwide = torch.empty(24, 900, dtype=x.dtype, device=dev)
    dwide[:, 1:651] = dy
    flat = torch.empty(24 * 650 + 1, dtype=x.dtype, device=dev)
    flat[1:] = x.reshape(-1)
    for name, xv, dv in (("pitch", wide[:, 3:653], dwide[:, 1:651]), ("at an odd element", flat[1:].view(24, 650), dy),
                         ("three dimensions", x.view(2, 12, 650), dy.view(2, 12, 650)),
                         ("transposed", x.t().contiguous().t(), dy.t().contiguous().t()),
                         ("dimensions exchanged", x.view(2, 12, 650).transpose(0, 1).contiguous().transpose(0, 1), dy.view(2, 12, 650))):
        got = check_norm(xv, w, b, dv, what=name)
        for a, c in zip(got, want):
            assert torch.equal(a.reshape(c.shape), c), name
    check_norm(x, w, b, dy[:1].expand(24, 650), what="one gradient for all rows")
    check_norm(x, w, b, torch.full((1, 1), 0.5, dtype=x.dtype, device=dev).expand(24, 650), what="one number for a gradient")
    check_norm(x[:1], w, b, dy[:1], what="one row")
    strided = torch.empty(650, 2, dtype=w.dtype, device=dev)
    strided[:, 0] = w
    check_norm(x, strided[:, 0], b, dy, what="strided weight")


def test_layer_norm_without_rows_and_with_some_gradients(dev):
    w = torch.ones(33, device=dev, requires_grad=True)
    b = torch.zeros(33, device=dev, requires_grad=True)
    x = torch.empty(0, 33, dtype=torch.bfloat16, device=dev, requires_grad=True)
    y = pkg.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert gx.shape == x.shape and not gw.any() and not gb.any()
    x, w, b, dy = norm_inputs(dev, 50, 200, "bf16", "bf16", True, 3)
    every = check_norm(x, w, b, dy)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1), (1, 1, 0)):
        leaves = [t.detach().requires_grad_(bool(f)) for t, f in zip((x, w, b), which)]
        y = pkg.layer_norm(*leaves)
        got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
        for a, c in zip(got, [c for c, f in zip(every[1:], which) if f]):
            assert torch.equal(a, c), which
    with torch.no_grad():
        assert not pkg.layer_norm(x, w.requires_grad_(), b).requires_grad


def test_layer_norm_keeps_what_is_no_number_in_its_row(dev):
    x, w, b, dy = norm_inputs(dev, 40, 1024, "bf16", "bf16", True, 11)
    clean = check_norm(x, w, b, dy)
    dirty = x.clone()
    dirty[3, 5], dirty[17, 1023], dirty[18, 0] = math.nan, math.inf, -math.inf
    xs = dirty.requires_grad_()
    y = pkg.layer_norm(xs, w, b)
    (dx,) = torch.autograd.grad(y, xs, dy)
    other = [i for i in range(40) if i not in (3, 17, 18)]
    assert torch.equal(y[other], clean[0][other]) and torch.equal(dx[other], clean[1][other])
    for i in (3, 17, 18):
        assert torch.isnan(y[i]).any() and torch.isnan(dx[i]).any()
    # a row of one value has a variance of zero: z is 0, and y the bias; with eps of zero it is no number
    flat = torch.full((2, 1024), 0.75, dtype=torch.bfloat16, device=dev)
    assert torch.equal(pkg.layer_norm(flat, w, b), b.expand(2, -1))
    assert torch.isnan(pkg.layer_norm(flat, w, b, 0.0)).all()


@pytest.mark.parametrize("t, cols", [("fp32", 128), ("fp32", 4), ("fp32", 2), ("bf16", 64), ("bf16", 256), ("bf16", 4)])
def test_layer_norm_of_equal_values_next_to_infinity(dev, t, cols):
    """The mean of rows of one value is that value, and z is 0 although the mean times rstd is infinite: threads without columns
    and rows that are none leave nothing behind."""
    x = torch.full((5, cols), 2.0 ** 120, dtype=TYPES[t], device=dev)
    g = gen(cols)
    w, b = (torch.randn(cols, generator=g).to(TYPES[t]).to(dev) for _ in range(2))
    dy = torch.randn(5, cols, generator=g).to(TYPES[t]).to(dev)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    y = pkg.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    if cols * 2.0 ** 120 > torch.finfo(torch.float32).max:   # 256 * 2^120 = 2^128: the sum of a row is kept in fp32
        assert y.isnan().all() and dx.isnan().all()
        return
    assert torch.equal(y, b.expand(5, -1)) and not dw.any()
    h = dy.double() * w.double()
    want = (h - h.mean(1, keepdim=True)) / math.sqrt(1e-5)
    assert_within(dx, want, half_step(dx.dtype) * want.abs() + 70 * U * (h.abs() + h.abs().mean(1, keepdim=True)) / math.sqrt(1e-5), "dx")
    assert_within(db, dy.double().sum(0), half_step(db.dtype) * dy.double().sum(0).abs() + 8 * U * dy.double().abs().sum(0), "db")


def test_layer_norm_past_32_bits(dev):
    """More rows than one launch takes, and more elements than 32 bits count."""
    rows, cols = (1 << 21) + 37, 1040
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev).normal_()
    dy = torch.empty_like(x).normal_()
    w = torch.rand(cols, device=dev) + 0.5
    xs, ws = x.requires_grad_(), w.requires_grad_()
    y = pkg.layer_norm(xs, ws)
    dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    for part in (slice(0, 5), slice((1 << 21) - 3, (1 << 21) + 3), slice(rows - 5, rows)):
        want, tol = norm_reference(x.detach()[part], w.detach(), None, dy[part], 1e-5)
        for a, v, e in ((y[part], want[0], tol[0]), (dx[part], want[1], tol[1])):
            assert_within(a.detach(), v, e + half_step(a.dtype) * (v.abs() + e) + smallest(a.dtype), str(part))
    total, bound, size = (torch.zeros(cols, dtype=torch.float64, device=dev) for _ in range(3))
    for xp, dp in zip(x.detach().split(1 << 18), dy.split(1 << 18)):
        want, tol = norm_reference(xp, w.detach(), None, dp, 1e-5)
        total += want[2]
        bound += tol[2]
        size += tol[2] / (64 * U)   # at least the magnitudes that were added
    # a thread adds up the rows of its workgroup's turn: at most 1 / 1024 of all of them
    assert_within(dw, total, bound + rows / 1024 * U * size + half_step(dw.dtype) * total.abs(), "dw")


# ---- embedding -------------------------------------------------------------------------------------------------------
def check_embedding(dev, ids, table, cols, t, scale=1.0, padding=None, seed=0, id_type=torch.int64):
    g = gen(seed)
    w = torch.randn(table, cols, generator=g).to(TYPES[t]).to(dev).requires_grad_()
    ids = ids.to(id_type).to(dev)
    dy = torch.randn(*ids.shape, cols, generator=g).to(TYPES[t]).to(dev)
    y = pkg.embedding(ids, w, scale, padding)
    assert y.shape == (*ids.shape, cols) and y.dtype == w.dtype
    inside = (ids >= 0) & (ids < table)
    rows = torch.where(inside, ids, 0).long()
    want = w.detach().double()[rows] * scale * inside[..., None] if table else torch.zeros(y.shape, dtype=torch.float64, device=dev)
    if scale == 1.0:
        assert torch.equal(y.double(), want)
    else:
        assert_within(y.detach(), want, (half_step(w.dtype) + 2 * U) * want.abs() + smallest(w.dtype), "y")
    (dw,) = torch.autograd.grad(y, w, dy)
    assert dw.shape == w.shape and dw.dtype == w.dtype
    pad = None if padding is None else padding % table
    counted = (inside if pad is None else inside & (ids != pad)).reshape(-1)
    flat, grads = rows.reshape(-1)[counted], dy.reshape(-1, cols)[counted].double() * scale
    total = torch.zeros(table, cols, dtype=torch.float64, device=dev).index_add_(0, flat, grads)
    size = torch.zeros_like(total).index_add_(0, flat, grads.abs())
    count = torch.bincount(flat, minlength=table)[:, None]
    # a row's tokens one after the other, and the product with the scale
    assert_within(dw, total, half_step(w.dtype) * total.abs() + (count + 4) * 2 * U * size + smallest(w.dtype) * (count > 0), "dw")
    assert not dw[(count == 0).reshape(-1)].any(), "a row without tokens has a gradient"
    (again,) = torch.autograd.grad(pkg.embedding(ids, w, scale, padding), w, dy)
    assert torch.equal(again, dw), "the gradient is not the same from call to call"
    return y.detach(), dw


@pytest.mark.parametrize("tokens, table, cols", [(1, 1, 1), (1, 5, 64), (7, 300, 33), (64, 4001, 256), (513, 17, 100), (1000, 4001, 250),
                                                 (1024, 1024, 512), (4096, 100, 1030), (5000, 70000, 24), (16384, 2000, 64),
                                                 (16385, 2000, 64), (20000, 3, 40), (3000, 262143, 8), (3000, 262144, 8), (40000, 300000, 16),
                                                 (131072, 600, 8), (131073, 60000, 9),
                                                 (768 * 2048, 900, 8), (768 * 2048 + 1, 60000, 9)])
@pytest.mark.parametrize("t", ["bf16", "fp16", "fp32"])
def test_embedding_against_64_bits(dev, tokens, table, cols, t):
    """The sort in one workgroup and in many, of one to three digits; runs that end inside, at and beyond a chunk's end."""
    g = gen(tokens + table)
    ids = (torch.rand(tokens, generator=g, dtype=torch.float64) ** 3 * table).long().clamp_(max=table - 1)
    check_embedding(dev, ids, table, cols, t, scale=(1.0, math.sqrt(cols))[tokens % 2], padding=(None, 0, -1)[tokens % 3], seed=tokens)


@pytest.mark.parametrize("tokens, rows", [(9001, 131072), (16383, 200000), (16384, 262143), (16385, 131072)])
def test_embedding_gradient_of_a_large_table(dev, tokens, rows):
    """Zeros that outlast the sort beside them."""
    ids = (torch.rand(tokens, generator=gen(tokens), dtype=torch.float64) ** 2 * rows).long().clamp_(max=rows - 1)
    check_embedding(dev, ids, rows, 520, "bf16", seed=tokens)


@pytest.mark.parametrize("tokens, cols", [(300, 65), (1024, 515), (9000, 700), (30000, 130)])
def test_embedding_of_one_id_and_of_runs(dev, tokens, cols):
    """All tokens the same, as many runs as tokens, runs of 8, 31, 32 and 33, and ids in falling order."""
    one = torch.full((tokens,), 5)
    check_embedding(dev, one, 9, cols, "fp32", 0.5)
    check_embedding(dev, one, 9, cols, "bf16", padding=5)
    check_embedding(dev, torch.arange(tokens).flip(0), tokens, cols, "bf16", 2.0)
    for run in (8, 31, 32, 33, 64, 65, 127, 129, 300):
        check_embedding(dev, torch.arange(tokens) // run, tokens, cols, "fp16", seed=run)


def test_embedding_of_ids_outside_the_table(dev):
    ids = torch.tensor([[0, 3, -1, 9], [10, 2 ** 40, -2 ** 62, 3]])
    y, dw = check_embedding(dev, ids, 10, 48, "bf16", 1.5, padding=3)
    assert not y[0, 2].any() and not y[1, :3].any() and not dw[3].any() and dw[9].any()
    check_embedding(dev, torch.tensor([2147483647, -2147483648, 1]), 4, 10, "fp32", id_type=torch.int32)
    # a table sharded by rows: the shards' results add up to the whole one's
    w = torch.randn(100, 24, device=dev)
    ids = torch.randint(0, 100, (50,), device=dev)
    assert torch.equal(pkg.embedding(ids, w[:60]) + pkg.embedding(ids - 60, w[60:]), pkg.embedding(ids, w))


def test_embedding_shapes_and_views(dev):
    check_embedding(dev, torch.tensor(3), 5, 16, "bf16")
    check_embedding(dev, torch.empty(0, dtype=torch.long), 5, 16, "bf16")
    check_embedding(dev, torch.empty(3, 0, dtype=torch.long), 7, 3, "fp32")
    check_embedding(dev, torch.randint(0, 9, (4, 3, 5)), 9, 12, "fp32", id_type=torch.int32)
    check_embedding(dev, torch.randint(0, 9, (6, 8)).t()[::2], 9, 12, "fp16")
    w = torch.randn(5, 0, device=dev, requires_grad=True)
    y = pkg.embedding(torch.tensor([1, 2], device=dev), w)
    assert y.shape == (2, 0) and torch.autograd.grad(y.sum(), w)[0].shape == (5, 0)
    none = torch.empty(0, 6, device=dev, requires_grad=True)
    y = pkg.embedding(torch.tensor([0, 1], device=dev), none)
    assert not y.any() and torch.autograd.grad(y.sum(), none)[0].shape == (0, 6)
    # a table and a gradient at any element
    flat = torch.randn(1 + 20 * 31, device=dev).to(torch.bfloat16)
    odd = flat[1:].view(20, 31).requires_grad_()
    ids = torch.randint(0, 20, (70,), device=dev)
    y = pkg.embedding(ids, odd)
    assert torch.equal(y, odd.detach().clone()[ids])
    up = torch.randn(1, 1, device=dev).to(torch.bfloat16).expand(70, 31)
    want = torch.zeros(20, 31, dtype=torch.float64, device=dev).index_add_(0, ids, up.double())
    (got,) = torch.autograd.grad(y, odd, up)
    assert_within(got, want, (half_step(got.dtype) + 200 * U) * want.abs(), "expanded gradient")


def test_embedding_past_32_bits(dev):
    table, cols = (1 << 19) + 3, 4104   # 2.15e9 elements
    w = torch.empty(table, cols, dtype=torch.bfloat16, device=dev).normal_().requires_grad_()
    ids = torch.tensor([table - 1, 7, table - 1, 1 << 18, (1 << 19) - 1, table], device=dev)
    dy = torch.randn(6, cols, device=dev).to(torch.bfloat16)
    y = pkg.embedding(ids, w)
    assert torch.equal(y[:5], w.detach()[ids[:5]]) and not y[5].any()
    (dw,) = torch.autograd.grad(y, w, dy)
    assert torch.equal(dw[7], dy[1]) and torch.equal(dw[1 << 18], dy[3]) and torch.equal(dw[(1 << 19) - 1], dy[4])
    assert_within(dw[-1], dy[0].double() + dy[2].double(), half_step(dw.dtype) * 1.001 * (dy[0].double() + dy[2].double()).abs(), "last row")
    assert sum(int(p.any(1).sum()) for p in dw.split(1 << 16)) == 4


# ---- how they are called ---------------------------------------------------------------------------------------------
def test_gradients_against_differences(dev):
    """A loss in fp32 along random directions: central differences in the plain form in 64 bits."""
    g = gen(77)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6, 40), (40,), (40,)))
    dy = torch.randn(6, 40, generator=g, dtype=torch.float64)

    def loss(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return ((c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b) * dy).sum().item()

    leaves = [t.float().to(dev).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(pkg.layer_norm(*leaves), leaves, dy.float().to(dev))
    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=g, dtype=torch.float64)
        at = [t.detach().double().cpu() for t in leaves]
        step = 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + step * v, at[i] - step * v
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # third derivatives of order one over steps of 1e-5, and fp32 sums of 240 products
        assert abs((grads[i].double().cpu() * v).sum().item() - slope) <= 1e-4 * max(1.0, abs(slope))


def test_second_derivatives_and_transforms_are_refused(dev):
    x = torch.randn(4, 8, device=dev, requires_grad=True)
    w = torch.ones(8, device=dev, requires_grad=True)
    (gx,) = torch.autograd.grad(pkg.layer_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        gx.sum().backward()
    ids = torch.tensor([1, 2], device=dev)
    up = torch.randn(2, 8, device=dev, requires_grad=True)
    (gx,) = torch.autograd.grad(pkg.embedding(ids, x), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        gx.square().sum().backward()
    for call in (lambda t: pkg.layer_norm(t, w), lambda t: pkg.embedding(ids, t)):
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.vmap(call)(x.expand(2, 4, 8))
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)))


def test_saved_tensors_are_looked_after(dev):
    """Hooks that move what is saved, a second pass over a freed graph, rows and ids that were changed in place."""
    x, w, b, dy = norm_inputs(dev, 30, 500, "bf16", "bf16", True, 21)
    want = check_norm(x, w, b, dy)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    with torch.autograd.graph.save_on_cpu():
        y = pkg.layer_norm(*leaves)
    for a, c in zip(torch.autograd.grad(y, leaves, dy), want[1:]):
        assert torch.equal(a, c)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        y = pkg.layer_norm(*leaves)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(y, leaves, dy)
    rows = (leaves[0] * 1.0)
    y = pkg.layer_norm(rows, *leaves[1:])
    rows.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)
    again = torch.utils.checkpoint.checkpoint(pkg.layer_norm, *leaves, use_reentrant=False)
    for a, c in zip(torch.autograd.grad(again, leaves, dy), want[1:]):
        assert torch.equal(a, c)
    ids = torch.tensor([1, 2, 3], device=dev)
    table = torch.randn(9, 16, device=dev, requires_grad=True)
    y = pkg.embedding(ids, table)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), table)


def test_other_streams(dev):
    x, w, b, dy = norm_inputs(dev, 200, 1000, "bf16", "bf16", True, 31)
    want = check_norm(x, w, b, dy)
    table = torch.randn(50, 64, device=dev, requires_grad=True)
    ids = torch.randint(0, 50, (300,), device=dev)
    up = torch.randn(300, 64, device=dev)
    (gt,) = torch.autograd.grad(pkg.embedding(ids, table), table, up)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:   # side by side, each with its own workspace
        with torch.cuda.stream(s):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            results.append(torch.autograd.grad(pkg.layer_norm(*leaves), leaves, dy)
                           + torch.autograd.grad(pkg.embedding(ids, table), table, up))
    torch.cuda.synchronize()
    for r in results:
        for a, c in zip(r, (*want[1:], gt)):
            assert torch.equal(a, c)


@pytest.mark.parametrize("tokens, rows", [(700, 500), (3000, 70000), (20000, 500)])
def test_captured_passes_replay(dev, tokens, rows):
    """Both operators, forward and backward, in one graph: four replays with new inputs and eager work in between."""
    g = torch.Generator(device=dev).manual_seed(3)

    def inputs():
        return (torch.randint(0, rows, (tokens,), generator=g, device=dev),
                torch.randn(tokens, 264, generator=g, device=dev).to(torch.bfloat16))

    table = torch.randn(rows, 264, generator=g, device=dev).to(torch.bfloat16).requires_grad_()
    w, b = torch.rand(264, device=dev).requires_grad_(), torch.rand(264, device=dev).requires_grad_()

    def step(ids, dy):
        y = pkg.layer_norm(pkg.embedding(ids, table, 3.0, 0), w, b)
        return (y.detach(), *torch.autograd.grad(y, (table, w, b), dy))

    ids, dy = inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ids, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ids, dy)
    for _ in range(4):
        new = inputs()
        ids.copy_(new[0])
        dy.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, c in zip(got, step(*new)):
            assert torch.equal(a, c)
        torch.randn(1 << 20, device=dev).sum().item()


# ---- in the layers ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["linear", "mlp"])
def test_routed_layer_norms_its_rows(dev, kind):
    """``layer_norm=True`` is the layer on normed rows, bit for bit, and its gradients go back through the norm."""
    make = moe.Fp8LinearModule if kind == "linear" else moe.Fp8MlpModule
    with_norm, without = (make(256, 512, 4, 2, device=dev, layer_norm=f) for f in (True, False))
    assert "row_norm.weight" in with_norm.state_dict() and without.row_norm is None
    with torch.no_grad():
        with_norm.row_norm.weight.normal_(1, 0.1)
        with_norm.row_norm.bias.normal_(0, 0.1)
    without.load_state_dict({k: v for k, v in with_norm.state_dict().items() if not k.startswith("row_norm")})
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(300, 256, generator=g, device=dev).to(torch.bfloat16)
    dy = (torch.randn(300, 256, generator=g, device=dev) * 1e-2).to(torch.bfloat16)
    grads = []
    for module in (with_norm, without):
        xs = x.clone().requires_grad_()
        norm = with_norm.row_norm
        norm.zero_grad()
        with pkg.fp8_autocast(fp8_recipe=pkg.DelayedScaling(amax_history_len=1)):
            out = module(xs) if module is with_norm else module(pkg.layer_norm(xs, norm.weight, norm.bias, norm.eps))
        out.backward(dy)
        grads.append([out.detach(), xs.grad, norm.weight.grad.clone(), norm.bias.grad.clone(), module.gating_network.weight.grad])
    for a, c in zip(*grads):
        assert torch.equal(a, c) and torch.isfinite(a.float()).all() and a.any()


def test_routed_layers_of_before_run_as_they_did(dev):
    """A layer without the option's attribute (pickled ahead of it), and a subclass that has a norm of its own by the usual name."""
    class Own(moe.Fp8MlpModule):
        def __init__(self, *args, **kwargs):
            super().__init__(*args, **kwargs)
            self.layer_norm = torch.nn.LayerNorm(256, dtype=torch.bfloat16, device=dev)

    plain, own = moe.Fp8MlpModule(256, 512, 4, 2, device=dev), Own(256, 512, 4, 2, device=dev)
    own.load_state_dict(plain.state_dict(), strict=False)
    old = moe.Fp8MlpModule(256, 512, 4, 2, device=dev)
    old.load_state_dict(plain.state_dict())
    del old.row_norm
    x = torch.randn(300, 256, generator=torch.Generator(device=dev).manual_seed(6), device=dev).to(torch.bfloat16)
    with torch.no_grad(), pkg.fp8_autocast(fp8_recipe=pkg.DelayedScaling(amax_history_len=1)):
        want, *got = [module(x) for module in (plain, own, old)]
    assert all(torch.equal(g, want) for g in got)


def test_a_training_step_of_a_small_model(dev):
    """Embedding, two routed layers with their norms on a residual stream, a loss; the gradients of the embedding and of the last
    norm against 64 bits from what reached them, then clipping: every gradient is scaled by the same factor."""
    hidden, vocabulary, tokens = 256, 1000, 700
    g = torch.Generator(device=dev).manual_seed(9)
    emb = pkg.Embedding(vocabulary, hidden, scale=2.0, padding_idx=0, device=dev)
    assert not emb.weight[0].any()
    layers = torch.nn.ModuleList([moe.Fp8MlpModule(hidden, 512, 4, 2, device=dev, layer_norm=True) for _ in range(2)])
    last = pkg.LayerNorm(hidden, device=dev)
    params = [*emb.parameters(), *layers.parameters(), *last.parameters()]
    ids = torch.randint(0, vocabulary, (tokens,), generator=g, device=dev)
    ids[-50:] = 0
    dy = torch.randn(tokens, hidden, generator=g, device=dev).to(torch.bfloat16)
    with pkg.fp8_autocast(fp8_recipe=pkg.DelayedScaling(amax_history_len=1)):
        rows = h = emb(ids)
        rows.retain_grad()
        for layer in layers:
            h = h + layer(h)
        h.retain_grad()
        out = last(h)
    out.backward(dy)
    want, tol = norm_reference(h.detach(), last.weight.detach(), last.bias.detach(), dy, last.eps)
    for a, v, e in zip((out.detach(), h.grad, last.weight.grad, last.bias.grad), want, tol):
        assert_within(a, v, e + half_step(a.dtype) * (v.abs() + e) + smallest(a.dtype), "last norm")
    counted = ids != 0
    total = torch.zeros(vocabulary, hidden, dtype=torch.float64, device=dev)
    total.index_add_(0, ids[counted], rows.grad[counted].double() * 2.0)
    size = torch.zeros_like(total).index_add_(0, ids[counted], rows.grad[counted].double().abs() * 2.0)
    assert_within(emb.weight.grad, total, half_step(torch.bfloat16) * total.abs() + 100 * U * size, "embedding")
    before = [p.grad.clone() for p in params]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in before))
    got = pkg.clip_grad_norm_(params, 0.5 * norm)
    assert abs(got.item() - norm) <= 2 * U * norm
    factor = 0.5 * norm / (norm + 1e-6)
    for p, t in zip(params, before):
        want = t.double() * factor
        assert_within(p.grad, want, (half_step(t.dtype) + 4 * U) * want.abs() + smallest(t.dtype), "clipped")


def test_kernel_timing_sees_the_calls(dev):
    from fp8_gmm_amd import backend

    x = torch.randn(8, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    with backend.kernel_timing() as timing:
        y = pkg.layer_norm(x, w)
        y.sum().backward()
        pkg.embedding(torch.tensor([1], device=dev), x).sum().backward()
        backend.multi_clip([x.grad], [x.grad], 1.0)
        backend.multi_norm([x.grad])
    names = {"layer_norm", "layer_norm_backward", "embedding", "embedding_backward", "multi_clip", "multi_norm"}
    assert names <= set(timing.summary())


# ---- gradients and rows of other kinds -------------------------------------------------------------------------------
@pytest.mark.parametrize("rows, cols, t", [(40, 127, "bf16"), (24, 640, "fp32"), (6, 1, "fp32"), (3, 20001, "bf16")])
def test_layer_norm_of_negated_gradients(dev, rows, cols, t):
    """torch hands a gradient on with its sign in a bit beside it (``torch.complex(a, y).conj()`` sends such ones to y): contiguous, strided
    in a single column, and what a saved-tensor hook returns."""
    x, w, b, dy = norm_inputs(dev, rows, cols, t, t, True, rows + cols)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(pkg.layer_norm(*leaves), leaves, -dy)
    wide = torch.empty(rows, 2 * cols, dtype=dy.dtype, device=dev)
    wide[:, ::2] = dy
    for up in (torch._neg_view(dy), torch._neg_view(wide)[:, ::2]):
        assert up.is_neg()
        for a, c in zip(torch.autograd.grad(pkg.layer_norm(*leaves), leaves, up), want):
            assert torch.equal(a, c)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: -v, torch._neg_view):
        y = pkg.layer_norm(*leaves)
    for a, c in zip(torch.autograd.grad(y, leaves, -dy), want):
        assert torch.equal(a, c)


@pytest.mark.parametrize("tokens", [1, 50, 3000])
def test_embedding_of_negated_gradients(dev, tokens):
    table = torch.randn(60, 24, device=dev, requires_grad=True)
    ids = torch.randint(0, 60, (tokens,), generator=gen(tokens)).to(dev)
    dy = torch.randn(tokens, 24, generator=gen(tokens)).to(dev)
    (want,) = torch.autograd.grad(pkg.embedding(ids, table, 3.0), table, -dy)
    (got,) = torch.autograd.grad(pkg.embedding(ids, table, 3.0), table, torch._neg_view(dy))
    assert torch.equal(got, want)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: -v, torch._neg_view):
        y = pkg.embedding(ids, table, 3.0)
    (got,) = torch.autograd.grad(y, table, -dy)
    assert torch.equal(got, want)
    single = torch.randn(60, 1, device=dev, requires_grad=True)
    up = torch.complex(torch.randn(tokens, 1, device=dev), torch.randn(tokens, 1, device=dev))
    (got,) = torch.autograd.grad(torch.complex(torch.zeros(tokens, 1, device=dev), pkg.embedding(ids, single)).conj(), single, up)
    (want,) = torch.autograd.grad(pkg.embedding(ids, single), single, (-up.imag).clone())
    assert torch.equal(got, want)


@pytest.mark.parametrize("t, cols", [("bf16", 20001), ("fp32", 20001), ("fp32", 20000)])
def test_layer_norm_of_long_rows_of_equal_values(dev, t, cols):
    """z is 0 although the mean times rstd is infinite, behind a row's end too.  Powers of two: the sum of a row is exact."""
    x = torch.full((3, cols), 2.0 ** 112, dtype=TYPES[t], device=dev)
    eps = 1e-12
    g = gen(cols)
    w, b = (torch.randn(cols, generator=g).to(TYPES[t]).to(dev) for _ in range(2))
    dy = torch.randn(3, cols, generator=g).to(TYPES[t]).to(dev)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    y = pkg.layer_norm(*leaves, eps)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y, b.expand(3, -1)) and not dw.any()
    h = dy.double() * w.double()
    want = (h - h.mean(1, keepdim=True)) / math.sqrt(eps)
    bound = 2 * (64 + cols / 1024) * U * (h.abs() + h.abs().mean(1, keepdim=True)) / math.sqrt(eps)
    assert_within(dx, want, half_step(dx.dtype) * (want.abs() + bound) + bound, "dx")
    assert_within(db, dy.double().sum(0), half_step(db.dtype) * dy.double().sum(0).abs() + 8 * U * dy.double().abs().sum(0) + smallest(db.dtype), "db")


# ---- launches that large calls alone reach ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows, cols, t, p", [(70000, 513, "fp32", "fp32"), (70000, 1027, "bf16", "fp32"), (70001, 1025, "fp16", "fp16"),
                                              (300001, 57, "fp32", "fp32"), (140001, 129, "fp32", "fp32"), (140001, 253, "fp32", "fp32"),
                                              (140001, 259, "bf16", "bf16"), (300001, 128, "bf16", "bf16"), (20000, 1024, "fp32", "fp32"),
                                              (1100, 16001, "fp32", "fp32"), (2101, 16379, "bf16", "bf16"), (5000, 8196, "fp32", "fp32")])
def test_layer_norm_of_results_that_outgrow_the_cache(dev, rows, cols, t, p):
    """Results over 64 MB are written with another hint, by launches of their own: rows with edges of 16 and of 64 lanes, of one to 16
    wavefronts, and aligned ones."""
    g = torch.Generator(device=dev).manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=g, device=dev) * 2 + torch.randn(1, cols, generator=g, device=dev)).to(TYPES[t])
    w = (1 + 0.2 * torch.randn(cols, generator=g, device=dev)).to(TYPES[p])
    b = (0.3 * torch.randn(cols, generator=g, device=dev)).to(TYPES[p])
    dy = (0.1 * torch.randn(rows, cols, generator=g, device=dev)).to(TYPES[t])
    assert x.numel() * x.element_size() > 64 << 20
    check_norm(x, w, b, dy, what=f"{rows} x {cols}")


def test_layer_norm_of_long_rows_by_several_launches(dev):
    """Rows past the registers, 2^16 of them to a launch, and more elements than 32 bits count."""
    rows, cols = (1 << 17) + 37, 16392
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev).normal_()
    dy = torch.empty_like(x).normal_()
    w = torch.rand(cols, device=dev) + 0.5
    xs, ws = x.requires_grad_(), w.requires_grad_()
    y = pkg.layer_norm(xs, ws)
    dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    total, bound, size = (torch.zeros(cols, dtype=torch.float64, device=dev) for _ in range(3))
    for xp, dp, yp, gp in zip(*(v.detach().split(1 << 13) for v in (x, dy, y, dx))):
        want, tol = norm_reference(xp, w.detach(), None, dp, 1e-5)
        for a, v, e, name in ((yp, want[0], tol[0], "y"), (gp, want[1], tol[1], "dx")):
            assert_within(a, v, e + half_step(a.dtype) * (v.abs() + e) + smallest(a.dtype), name)
        total += want[2]
        bound += tol[2]
        size += tol[2] / (64 * U)   # at least the magnitudes that were added
    # a thread adds up a 64th of the rows
    assert_within(dw, total, bound + rows / 64 * U * size + half_step(dw.dtype) * total.abs(), "dw")


@pytest.mark.parametrize("tokens, table, cols, t, ids", [((1 << 22) + 37, 60000, 9, "bf16", torch.int64), ((1 << 22) + 37, 900, 9, "fp16", torch.int32),
                                                         ((1 << 23) + 5, 1000, 3, "fp32", torch.int64), ((1 << 22) + 3, 5000, 5, "fp32", torch.int32),
                                                         (300001, 5000, 136, "bf16", torch.int32), (140001, 700, 264, "fp16", torch.int64),
                                                         (16411, 9000, 4104, "bf16", torch.int64), (9001, 9000, 4099, "fp32", torch.int32)])
def test_embedding_of_results_that_outgrow_the_cache(dev, tokens, table, cols, t, ids):
    """Results over 64 MB are written with another hint; more than 2^22 tokens take several launches.  Copied rows are the same bits."""
    g = torch.Generator(device=dev).manual_seed(tokens)
    w = torch.randn(table, cols, generator=g, device=dev).to(TYPES[t]).requires_grad_()
    at = torch.randint(-2, table + 2, (tokens,), generator=g, device=dev).to(ids)   # some outside the table
    inside = (at >= 0) & (at < table)
    rows = torch.where(inside, at, 0).long()
    y = pkg.embedding(at, w)
    assert y.numel() * y.element_size() > 64 << 20
    assert torch.equal(y, w.detach()[rows].where(inside[:, None], torch.zeros((), dtype=w.dtype, device=dev)))
    assert torch.equal(pkg.embedding(at, w.detach(), 2.0), y.detach() * 2)
    dy = torch.randn(tokens, cols, generator=g, device=dev).to(TYPES[t])
    (dw,) = torch.autograd.grad(y, w, dy)
    total = torch.zeros(table, cols, dtype=torch.float64, device=dev).index_add_(0, rows[inside], dy[inside].double())
    size = torch.zeros_like(total).index_add_(0, rows[inside], dy[inside].double().abs())
    count = torch.bincount(rows[inside], minlength=table)[:, None]
    assert_within(dw, total, half_step(w.dtype) * total.abs() + (count + 4) * 2 * U * size + smallest(w.dtype), "dw")


def test_gradients_with_tangents_are_refused(dev):
    """Forward over reverse: a backward pass that dropped its gradient's tangent would return a wrong derivative."""
    x, w, table = (torch.randn(s, device=dev, requires_grad=True) for s in ((6, 32), (32,), (9, 32)))
    ids = torch.randint(0, 9, (6,), device=dev)
    dy = torch.randn(6, 32, device=dev)
    for make, leaf in ((lambda: pkg.layer_norm(x, w), x), (lambda: pkg.embedding(ids, table), table)):
        y = make()
        with torch.autograd.forward_ad.dual_level():
            up = torch.autograd.forward_ad.make_dual(dy, torch.ones_like(dy))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, up)
            (got,) = torch.autograd.grad(make(), leaf, dy)   # one without is taken inside of a level too
        (want,) = torch.autograd.grad(make(), leaf, dy)
        assert torch.equal(got, want)
