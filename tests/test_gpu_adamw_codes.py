"""The codes of 8-bit moments on the GPU, bit by bit, and the parameters beside them."""
import pytest
import torch

from fp8_gmm_amd import backend

pytestmark = pytest.mark.gpu


def test_codes_follow_the_stated_operations(dev):
    """m = 0.1 g, y = m (448 / largest), each rounded to fp32, and up where the fraction behind a code's 3 bits and the threshold's 20 bits
    make a whole: every step of it is exact or correctly rounded, so every code is known."""
    n, t = 1 << 26, 3
    g = torch.randn(n, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    p = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    codes = [torch.zeros(n, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2)]
    scales = [torch.zeros(n // 128, device=dev) for _ in range(2)]
    backend.multi_adamw([p], [g], [codes[0]], [codes[1]], t, 1e-3, scales=([scales[0]], [scales[1]]))
    part, wrong = 1 << 22, 0
    for at in range(0, n, part):
        m = (torch.tensor(1 - 0.9, dtype=torch.float32, device=dev) * g[at: at + part]).view(-1, 128)
        most = m.abs().amax(1, keepdim=True)
        assert torch.equal(scales[0][at // 128: (at + part) // 128], (most * torch.tensor(1 / 448, dtype=torch.float32, device=dev))[:, 0])
        y = (m * (448.0 / most)).clamp(-448, 448).flatten()
        h = (torch.arange(at, at + part, device=dev) * 0x6A09E667 + t * 0x9E3779B9) & 0xFFFFFFFF
        bits = y.view(torch.int32)
        up = (bits & 0xFFFFF) + (h >> 12) >= 1 << 20
        want = ((bits & ~0xFFFFF) + (up.to(torch.int32) << 20)).view(torch.float32).clamp(-448, 448)
        normal = y.abs() >= 2.0 ** -6
        assert normal.double().mean() > 0.999
        wrong += int((codes[0][at: at + part].float() != want)[normal].sum())
    assert wrong == 0, f"{wrong} of {n}"


@pytest.mark.parametrize("masters", [False, True])
def test_parameters_move_as_beside_moments_in_32_bits(dev, masters):
    """From moments of zeros the first step's parameters have the same bits with either kind of moments."""
    n = 1 << 20
    g = torch.randn(n, generator=torch.Generator(device=dev).manual_seed(1), device=dev) * 1e-2
    start = torch.randn(n, generator=torch.Generator(device=dev).manual_seed(2), device=dev) * 1e-3
    moved = []
    for bits in (32, 8):
        p = start.to(torch.bfloat16) if masters else start.clone()
        m, v = (torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.float8_e4m3fn, device=dev) for _ in range(2))
        scales = tuple([torch.zeros(n // 128, device=dev)] for _ in range(2)) if bits == 8 else None
        master = [start.clone()] if masters else None
        backend.multi_adamw([p], [g], [m], [v], 1, 1e-3, scales=scales, masters=master)
        moved.append((p, *(master or ())))
    assert all(torch.equal(a, b) for a, b in zip(*moved))


def test_a_square_that_fp32_does_not_hold_leaves_its_block_alone(dev):
    """A finite gradient whose second moment is infinite: its own parameter stands still but for the decay, as beside moments in 32 bits,
    and the others of its block go on, in this step and in the next ones."""
    n = 1000
    r = torch.Generator(device=dev).manual_seed(1)
    grads = [torch.randn(n, generator=r, device=dev) for _ in range(4)]
    grads[0][300], grads[0][301] = 1e25, -1e30
    p = torch.ones(n, device=dev)
    codes = [torch.zeros(n, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2)]
    scales = [torch.zeros(8, device=dev) for _ in range(2)]
    for t, g in enumerate(grads, 1):
        before = p.clone()
        backend.multi_adamw([p], [g], [codes[0]], [codes[1]], t, 1e-3, weight_decay=0.0, scales=([scales[0]], [scales[1]]))
        assert torch.isfinite(p).all() and all(torch.isfinite(s).all() for s in scales)
        assert all(torch.isfinite(c.float()).all() for c in codes)
        assert t > 1 or torch.equal(p[300:302], before[300:302])
        others = torch.cat([p[:256] != before[:256], p[384:] != before[384:]])
        assert others.all()
