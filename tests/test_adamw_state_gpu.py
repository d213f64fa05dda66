"""The 8-bit moments of adamw_step: their bytes against separate fp32 operations, and what becomes of them over many steps."""
import pytest
import torch

from holonomyawareattention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def state(n):
    return [torch.zeros(n, device=DEV).to(E4M3)], [torch.zeros(n, device=DEV).to(E4M3)], [torch.zeros(2, -(-n // 256), device=DEV)]


def bytes_of(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("n,at", [(600, 300), (600, 599), (2048, 0), (257, 256)])
def test_not_finite_stays_with_its_element(n, at, what):
    """One gradient that is not finite loses its own parameter, as with fp32 moments; the others go on as if it had been 0."""
    g = torch.Generator(device=DEV).manual_seed(n + at)
    runs = []
    for bad in (False, True):
        g.manual_seed(n + at)
        p, (m, v, s) = torch.ones(n, device=DEV), state(n)
        for t in range(1, 5):
            grad = torch.randn(n, device=DEV, generator=g)
            grad[at] = what if bad and t == 2 else 0.0
            ops.adamw_step([p], [grad], m, v, torch.full((1,), t, dtype=torch.int32, device=DEV), lr=1e-2, weight_decay=0.0, scales=s)
        runs.append((p, bytes_of(m[0]), bytes_of(v[0]), s[0]))
    one, two = runs
    rest = torch.arange(n, device=DEV) != at
    assert torch.isnan(two[0][at]) and torch.isfinite(two[0][rest]).all()
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(one[:3], two[:3])) and torch.equal(one[3], two[3])
    assert torch.isnan(two[1][at].view(E4M3).float()) and torch.isnan(two[2][at].view(E4M3).float())


def test_ended_gradients():
    """Weights whose gradients end come to rest, as with fp32 moments, while the rest of their block goes on."""
    n, steps = 64 * 256, 600
    g = torch.Generator(device=DEV).manual_seed(5)
    ended = torch.arange(n, device=DEV) % 2 == 0
    p, (m, v, s) = torch.zeros(n, device=DEV), state(n)
    at = []
    for t in range(1, steps + 1):
        grad = torch.randn(n, device=DEV, generator=g)
        if t > 50:
            grad[ended] = 0.0
        ops.adamw_step([p], [grad], m, v, torch.full((1,), t, dtype=torch.int32, device=DEV), lr=1.0, betas=(0.9, 0.95), weight_decay=0.0,
                       scales=s)
        if t in (300, steps):
            at.append(p.clone())
    # m falls by a tenth a step or a smallest step (2^-9 of 448 steps of its scale): after 250 steps nothing is left of it
    assert torch.equal(at[0][ended], at[1][ended]) and not m[0].float()[ended].any()
    assert bool((at[0][~ended] != at[1][~ended]).all())


def by_operations(m, v, s, grad, b1, b2):
    """(m's bytes, the root's, the scales) after a step, in separate fp32 operations."""
    n = grad.numel()
    pad = lambda t: torch.nn.functional.pad(t, (0, -n % 256)).view(-1, 256)  # noqa: E731
    g = pad(grad.float())
    old = s[0][:, None]
    mo = pad(m.float()) * old
    ro = pad(v.float()) * s[1][:, None]
    mn = mo * b1 + g * (1.0 - b1)
    r = ((ro * ro) * b2 + (g * g) * (1.0 - b2)).sqrt()
    by = torch.tensor(1.0, device=DEV) / 448.0
    ms, vs = mn.abs().amax(1, keepdim=True) * by, r.amax(1, keepdim=True) * by
    qm, qr = torch.where(ms > 0, mn / ms, 0.0), torch.where(vs > 0, r / vs, 0.0)
    ended = ((g.abs() * (1.0 - b1)) < 2.0 ** -10 * old) & (qm.abs() < 2.0 ** -5)
    qm = torch.where(ended, (qm * 512).trunc() / 512, qm)
    qr = torch.where((r > 0) & (qr < 2.0 ** -9), 2.0 ** -9, qr)
    back = lambda q: q.to(E4M3).reshape(-1)[:n].contiguous()  # noqa: E731
    return back(qm), back(qr), torch.stack([ms[:, 0], vs[:, 0]])


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.8, 0.9), (0.0, 0.5)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-9, 1e-13, 1e-18, 1e12, 1e17])       # (scales on both sides of 1e-12 and 1e12)
@pytest.mark.parametrize("n,at", [(40 * 256, 0), (40 * 256 + 77, 0), (5 * 256 + 9, 1), (3, 0)])
def test_bytes(n, at, size, betas):
    """The moments' bytes and scales are those of the same formula in separate fp32 operations with IEEE division and root,
    bit for bit (the kernel divides by a block's scale in three operations of its own), where a tensor starts on a 16-byte
    boundary and where it does not; blocks of zeros, partial ones, and ended gradients among them."""
    g = torch.Generator(device=DEV).manual_seed(n)
    new = lambda dt: torch.zeros(n + at, device=DEV).to(dt)[at:]  # noqa: E731
    m, v, p = new(E4M3), new(E4M3), new(torch.float32)
    s = torch.zeros(2, -(-n // 256), device=DEV)
    for t in range(1, 7):
        grad = size * torch.randn(n, device=DEV, generator=g) * 10.0 ** (3 * torch.rand(n, device=DEV, generator=g) - 2)
        grad[:min(n, 256)] = 0.0
        if t > 2:
            grad[::5] = 0.0
        want = by_operations(m, v, s, grad, *betas)
        ops.adamw_step([p], [grad], [m], [v], torch.full((1,), t, dtype=torch.int32, device=DEV), lr=0.1, betas=betas, scales=[s])
        assert torch.equal(s, want[2])
        assert torch.equal(m.float(), want[0].float()) and torch.equal(v.float(), want[1].float())
    assert m.float().any() or n < 256
