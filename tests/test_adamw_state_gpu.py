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


def noise(n, step):
    """The 32 random bits of each element in a step, as the kernel's comment defines them."""
    low = 0xffffffff
    i = torch.arange(n, device=DEV, dtype=torch.int64)
    x = ((((i & low) * 0x9e3779b1) & low) ^ (((i >> 32) * 0xb5297a4d) & low)) + ((step * 0x68e31da5) & low) & low
    for shift, by in ((16, 0x7a3f5c2b), (15, 0xc4d1e6b7)):
        x = x ^ (x >> shift)
        x = ((x >> 16) * by << 16) + (x & 0xffff) * by & low        # (no product passes 63 bits)
    return x ^ (x >> 16)


def by_chance(q, u):
    """q cut off after 16 random bits were added below its last place of e4m3 (2^-9 below 2^-6)."""
    q = q.double()
    place = torch.exp2(torch.frexp(q.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)
    return torch.copysign(((q.abs() / place + (u.double() + 0.5) / 65536).floor() * place), q).float()


def by_operations(m, v, s, grad, b1, b2, step=None):
    """(m's bytes, the root's, the scales) after a step, in separate fp32 operations; ``step``: rounded by chance."""
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
    if step is not None:
        u = torch.nn.functional.pad(noise(n, step), (0, -n % 256)).view(-1, 256)
        qm, qr = by_chance(qm, u >> 16), torch.where(r > 0, by_chance(qr, u & 0xffff).clamp(min=2.0 ** -9), qr)
        old = 0.0 * old
    ended = ((g.abs() * (1.0 - b1)) < 2.0 ** -10 * old) & (qm.abs() < 2.0 ** -5)
    qm = torch.where(ended, (qm * 512).trunc() / 512, qm)
    qr = torch.where((r > 0) & (qr < 2.0 ** -9), 2.0 ** -9, qr)
    back = lambda q: q.to(E4M3).reshape(-1)[:n].contiguous()  # noqa: E731
    return back(qm), back(qr), torch.stack([ms[:, 0], vs[:, 0]])


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.8, 0.9), (0.0, 0.5), (0.9375, 0.95), (0.9, 0.999), (0.95, 0.95), (0.9, 0.951)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-9, 1e-13, 1e-18, 1e12, 1e17])       # (scales on both sides of 1e-12 and 1e12)
@pytest.mark.parametrize("n,at", [(40 * 256, 0), (40 * 256 + 77, 0), (5 * 256 + 9, 1), (3, 0)])
def test_bytes(n, at, size, betas):
    """The moments' bytes and scales are those of the same formula in separate fp32 operations with IEEE division and root,
    bit for bit (the kernel divides by a block's scale in three operations of its own), where a tensor starts on a 16-byte
    boundary and where it does not; blocks of zeros, partial ones, and ended gradients among them.  The last three pairs of betas
    are on the side of the rule where the bytes are rounded by chance."""
    g = torch.Generator(device=DEV).manual_seed(n)
    new = lambda dt: torch.zeros(n + at, device=DEV).to(dt)[at:]  # noqa: E731
    m, v, p = new(E4M3), new(E4M3), new(torch.float32)
    s = torch.zeros(2, -(-n // 256), device=DEV)
    for t in range(1, 7):
        grad = size * torch.randn(n, device=DEV, generator=g) * 10.0 ** (3 * torch.rand(n, device=DEV, generator=g) - 2)
        grad[:min(n, 256)] = 0.0
        if t > 2:
            grad[::5] = 0.0
        want = by_operations(m, v, s, grad, *betas, step=t if betas[0] > 0.9375 or betas[1] > 0.95 else None)
        ops.adamw_step([p], [grad], [m], [v], torch.full((1,), t, dtype=torch.int32, device=DEV), lr=0.1, betas=betas, scales=[s])
        assert torch.equal(s, want[2])
        assert torch.equal(m.float(), want[0].float()) and torch.equal(v.float(), want[1].float())
    assert m.float().any() or n < 256


def test_noise():
    """The kernel's random bits: as many of each kind as chance gives, none like its neighbours' or the next step's."""
    u = torch.stack([noise(1 << 16, t) for t in range(1, 33)])
    for half in (u >> 16, u & 0xffff):
        f = (half.double() + 0.5) / 65536 - 0.5                      # (uniform: variance 1/12)
        sd = 1 / f.numel() ** 0.5
        assert abs(float(f.mean())) < 5 * sd / 12 ** 0.5
        for a, b in ((f[1:], f[:-1]), (f[2:], f[:-2]), (f[:, 1:], f[:, :-1]), (f[:, 8:], f[:, :-8]), (f[:, 256:], f[:, :-256])):
            assert abs(float((a * b).mean()) * 12) < 5.5 * sd        # (the products: standard deviation 1/12)
    count = torch.bincount((u >> 24).reshape(-1), minlength=256).double()
    each = u.numel() / 256
    assert abs(float(((count - each) ** 2 / each).sum()) - 255) < 6 * (2 * 255) ** 0.5


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.99), (0.9, 0.96)])
@pytest.mark.parametrize("change", [0.1, 1.0, 10.0])
def test_roots_follow(change, betas):
    """Half of the gradients change their size at step 200: the held roots follow those of fp32 moments.

    By chance a step moves a root by delta = (1 - b2) / 2 |g^2 / v - 1| on average, in jumps of a last place s <= 2^-3 of it,
    so with a variance of delta s at most, against a decay of (1 - b2) a step: a standard deviation of sqrt(s / 4) at most,
    0.15 with the mean s of 0.09.  While v falls it is delta that grows, to (1 - b2) / 2 itself: no more.  Six of them: a
    factor of 2.5.  The means are exact but for 1 / x of a spread x (0.15^2) and last places: 8%."""
    n = 64 * 256
    g = torch.Generator(device=DEV).manual_seed(int(change * 10))
    changed = torch.arange(n, device=DEV) % 2 == 0
    p, (m, v, s) = torch.zeros(n, device=DEV), state(n)
    p2, m2, v2 = p.clone(), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    steps = 200 + int(3 / (1 - betas[1]))
    for t in range(1, steps + 1):
        grad = torch.randn(n, device=DEV, generator=g)
        if t > 200:
            grad[changed] *= change
        step = torch.full((1,), t, dtype=torch.int32, device=DEV)
        ops.adamw_step([p], [grad], m, v, step, lr=1e-3, betas=betas, weight_decay=0.0, scales=s)
        ops.adamw_step([p2], [grad], [m2], [v2], step, lr=1e-3, betas=betas, weight_decay=0.0)
    held = v[0].double() * s[0][1].double().repeat_interleave(256)
    ratio = (held / v2.double().sqrt())[changed].sort().values
    low, mid, high = (float(ratio[int(f * (ratio.numel() - 1))]) for f in (0.01, 0.5, 0.99))
    assert 0.4 < low and high < 2.5 and abs(mid - 1) < 0.08, (low, mid, high)


def test_ended_gradients_by_chance():
    """... and weights whose gradients end come to rest at the default betas too."""
    n = 64 * 256
    g = torch.Generator(device=DEV).manual_seed(6)
    ended = torch.arange(n, device=DEV) % 2 == 0
    p, (m, v, s) = torch.zeros(n, device=DEV), state(n)
    for t in range(1, 601):
        grad = torch.randn(n, device=DEV, generator=g)
        if t > 50:
            grad[ended] = 0.0
        ops.adamw_step([p], [grad], m, v, torch.full((1,), t, dtype=torch.int32, device=DEV), lr=1.0, weight_decay=0.0, scales=s)
        if t == 350:
            at = p.clone()
    # m's mean falls as 0.9^t: from 448 at most to 2^-9 in 120 steps, and to 1e-8 of that, one chance in 1e8, in 300
    assert torch.equal(at[ended], p[ended]) and not m[0].float()[ended].any()
