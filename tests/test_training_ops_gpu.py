"""The training operators against plain 64-bit torch: attn_fwd_lse, attn_bwd, path_bwd, adamw_step.

Tolerances.  fp32 results of sums of n terms, each product rounded once: a relative error (2-norm) of a few
eps = 2^-24 times a factor that grows slower than sqrt(n); 1e-5 (170 eps) is above every such sum here.  bf16
results: the value's own rounding, at most half a step, finfo.eps / 2 = 2^-8 of it, and that of one bf16 factor of
every term (P or dS), at most 2^-8 of the term.  The factors' errors are independent, so in the 2-norm they add up as
the terms themselves do (squares of both sides: (2^-8)^2 times the terms' squares): at most 2^-8 of the sum's norm.
Together at most 2^-8 + 2^-8 = 2^-7.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32_TOL = 1e-5
BF16_TOL = 2.0 ** -7


def rel(x, y):
    y = y.double()
    return float((x.double() - y).norm() / y.norm().clamp(min=1e-300))


def randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attn_case(BH, Tq, Tk, off, d, dt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, do = randn(g, BH, Tq, d).to(dt), randn(g, BH, Tq, d).to(dt)
    k, v = randn(g, BH, Tk, d).to(dt), randn(g, BH, Tk, d).to(dt)
    return q, k, v, do


def attn_ref(q, k, v, do, scale, off):
    q, k, v = (x.double().requires_grad_() for x in (q, k, v))
    z = q @ k.transpose(1, 2) * scale
    unseen = torch.ones(q.shape[1], k.shape[1], dtype=torch.bool, device=DEV).triu(off + 1)
    z = z.masked_fill(unseen, float("-inf"))
    o = torch.softmax(z, -1) @ v
    grads = torch.autograd.grad((o * do.double()).sum(), (q, k, v))
    return o.detach(), torch.logsumexp(z, -1).detach(), grads


ATTN = [(2, 1, 1, 0, 48), (1, 1, 300, 299, 16), (3, 2, 2, 0, 8), (2, 17, 17, 0, 96), (1, 63, 64, 1, 64), (2, 64, 64, 0, 32),
        (1, 65, 129, 64, 80), (2, 127, 130, 0, 112), (1, 128, 128, 0, 120), (3, 129, 129, 0, 128), (1, 200, 777, 500, 96),
        (2, 333, 333, 0, 56), (1, 130, 700, 0, 24), (5, 257, 300, 43, 104), (1, 1000, 1000, 0, 72), (2, 100, 100, 0, 5), (1, 150, 190, 7, 50)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("BH,Tq,Tk,off,d", ATTN)
def test_attn_bwd(BH, Tq, Tk, off, d, dt):
    from holonomyawareattention_b200 import ops
    q, k, v, do = attn_case(BH, Tq, Tk, off, d, dt, seed=Tq + d)
    scale = d ** -0.5
    o, lse = ops.attn_fwd_lse(q, k, v, scale, off)
    ro, rl, (rq, rk, rv) = attn_ref(q, k, v, do, scale, off)
    tol = F32_TOL if dt is torch.float32 else BF16_TOL
    assert o.dtype is torch.float32 and rel(o, ro) < tol and float((lse - rl).abs().max()) < 2e-5
    dq, dk, dv = ops.attn_bwd(q, k, v, o, lse, do, scale, off)
    ops.check_status()
    assert dq.dtype is dt and dk.dtype is dt and dv.dtype is dt
    assert rel(dv, rv) < tol
    # where every query sees one key alone ds is exactly 0, and what remains is the rounding of do . v - do . o
    size = float((do.double().norm() * v.double().norm() * q.double().norm()) * scale)
    for x, r in ((dq, rq), (dk, rk)):
        assert float((x.double() - r).norm()) < tol * float(r.norm()) + 1e-6 * size
    # keys that no query sees
    assert not dk[:, off + Tq:].any() and not dv[:, off + Tq:].any()
    # the same bits again
    again = ops.attn_bwd(q, k, v, o, lse, do, scale, off)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), again))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attn_bwd_differences(dt):
    """The directional derivative of sum(o . do), by central differences of the fp64 forward on the same inputs."""
    from holonomyawareattention_b200 import ops
    q, k, v, do = attn_case(2, 70, 70, 0, 48, dt, seed=3)
    scale = 48 ** -0.5
    o, lse = ops.attn_fwd_lse(q, k, v, scale)
    grads = ops.attn_bwd(q, k, v, o, lse, do, scale)
    g = torch.Generator(device=DEV).manual_seed(9)
    for i in range(3):
        u = torch.randn(grads[i].shape, device=DEV, generator=g, dtype=torch.float64)
        h = 1e-5

        def loss(s):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + s * u
            return (attn_ref(*x, do, scale, 0)[0] * do.double()).sum()

        want = float((loss(h) - loss(-h)) / (2 * h))
        got = float((grads[i].double() * u).sum())
        # the error of a projection of n rounded values: their 2-norm error spread over directions
        tol = (F32_TOL if dt is torch.float32 else BF16_TOL) * float(grads[i].double().norm()) * 4 + 1e-6 * abs(want)
        assert abs(got - want) < tol


def test_attn_bwd_large_scores_and_late_rows():
    """Scores of +-100: probabilities of 0 and 1, no overflow.  Rows far behind the first shard's keys."""
    from holonomyawareattention_b200 import ops
    for dt, tol in ((torch.float32, F32_TOL), (torch.bfloat16, BF16_TOL)):
        q, k, v, do = attn_case(2, 140, 400, 260, 64, dt, seed=5)
        q, k = (q * 4).to(dt), (k * 4).to(dt)
        o, lse = ops.attn_fwd_lse(q, k, v, 0.125, 260)
        ro, rl, ref = attn_ref(q, k, v, do, 0.125, 260)
        got = ops.attn_bwd(q, k, v, o, lse, do, 0.125, 260)
        # (an error of a score of 100 is 100 eps of fp32 in its probability)
        for x, r in zip(got, ref):
            assert bool(torch.isfinite(x).all()) and rel(x, r) < tol + 200 * 2.0 ** -24


def test_attn_bwd_unaligned():
    """bf16 tensors from an address that TMA does not take run on the CUDA cores."""
    from holonomyawareattention_b200 import ops
    q, k, v, do = attn_case(2, 70, 70, 0, 48, torch.bfloat16, seed=4)
    odd = []
    for t in (q, k, v, do):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        odd.append(buf[1:].view(t.shape).copy_(t))
    o, lse = ops.attn_fwd_lse(*odd[:3], 0.2)
    got = ops.attn_bwd(*odd[:3], o, lse, odd[3], 0.2)
    ref = attn_ref(q, k, v, do, 0.2, 0)
    assert rel(o, ref[0]) < BF16_TOL
    for x, r in zip(got, ref[2]):
        assert rel(x, r) < BF16_TOL


def test_attn_bwd_refusals():
    from holonomyawareattention_b200 import ops
    q, k, v, do = attn_case(2, 8, 8, 0, 16, torch.float32)
    o, lse = ops.attn_fwd_lse(q, k, v, 0.25)
    with pytest.raises(ValueError, match="queries"):
        ops.attn_bwd(q, k, v, o, lse, do, 0.25, 1)
    with pytest.raises(ValueError, match="contiguous"):
        ops.attn_bwd(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, o, lse, do, 0.25)
    with pytest.raises(ValueError, match="do"):
        ops.attn_bwd(q, k, v, o, lse, do.bfloat16(), 0.25)
    with pytest.raises(ValueError, match="lse"):
        ops.attn_bwd(q, k, v, o, lse[:, :4].contiguous(), do, 0.25)
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.attn_bwd(q.half(), k.half(), v.half(), o, lse, do.half(), 0.25)
    with pytest.raises(NotImplementedError, match="head dim"):
        big = torch.zeros(1, 4, 136, device=DEV)
        ops.attn_fwd_lse(big, big, big, 0.1)


# ---------------------------------------------------------------------------
# the path
# ---------------------------------------------------------------------------
def skew(a, d):
    i, j = torch.triu_indices(d, d, 1, device=a.device)
    A = torch.zeros(*a.shape[:-1], d, d, dtype=a.dtype, device=a.device)
    A[..., i, j] = a
    return A - A.transpose(-1, -2)


def path_case(B, T, H, d, chunk, scale, dt, seed=0, amp=0.3):
    """Inputs, with R and C from the forward's own kernels' contract, composed here in fp64 and rounded."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    a = amp * randn(g, B, T, H * (d * (d - 1) // 2))
    gen = a.view(B, T, H, -1).permute(0, 2, 1, 3).reshape(B * H, T, -1).double()
    G = torch.linalg.matrix_exp(skew(scale * gen, d))
    P, R, C = [], [], []
    p = torch.eye(d, dtype=torch.float64, device=DEV).expand(B * H, d, d)
    r = p
    for t in range(T):
        if t % chunk == 0:
            C.append(p)
            r = torch.eye(d, dtype=torch.float64, device=DEV).expand(B * H, d, d)
        P.append(p)
        R.append(r)
        p, r = G[:, t] @ p, G[:, t] @ r
    hats = [randn(g, B * H, T, d).to(dt) for _ in range(3)] + [randn(g, B * H, T, d)]
    dhats = [randn(g, B * H, T, d).to(dt) for _ in range(4)]
    return a, torch.stack(R, 1).float(), torch.stack(C, 1).float(), torch.stack(P, 1), hats, dhats


def path_ref(a, P, hats, dhats, H, scale):
    """By autograd through the products themselves: loss = <dq^, P^T q> + ... + <P o, dout> with q = P q^ etc. held fixed."""
    B, T, _ = a.shape
    d = P.shape[-1]
    qkv = [torch.einsum("ctij,ctj->cti", P, x.double()) for x in hats[:3]]
    dout = torch.einsum("ctij,ctj->cti", P, dhats[3].double())
    leaf = a.double().requires_grad_()
    gen = leaf.view(B, T, H, -1).permute(0, 2, 1, 3).reshape(B * H, T, -1)
    G = torch.linalg.matrix_exp(skew(scale * gen, d))
    p = torch.eye(d, dtype=torch.float64, device=DEV).expand(B * H, d, d)
    loss = 0.0
    for t in range(T):
        for x, y in zip(qkv, dhats[:3]):
            loss = loss + (torch.einsum("cij,ci->cj", p, x[:, t]) * y[:, t].double()).sum()
        loss = loss + (torch.einsum("cij,cj->ci", p, hats[3][:, t].double()) * dout[:, t]).sum()
        p = G[:, t] @ p
    if T > 1:
        (da,) = torch.autograd.grad(loss, leaf)
    else:
        da = torch.zeros_like(leaf)
    dqkv = torch.stack([torch.einsum("ctij,ctj->cti", P, x.double()) for x in dhats[:3]], 2)        # (BH, T, 3, d)
    dqkv = dqkv.view(B, H, T, 3, d).permute(0, 2, 1, 3, 4).reshape(B, T, 3 * H * d)
    return da, dqkv


PATH = [(1, 1, 1, 8, 16, 0.1), (2, 2, 1, 5, 16, 0.1), (1, 17, 2, 16, 16, 0.1), (1, 40, 1, 20, 7, 0.5), (2, 33, 3, 24, 33, 0.05),
        (1, 70, 2, 32, 64, 0.1), (1, 65, 2, 40, 32, 0.3), (2, 37, 4, 48, 16, 0.05), (1, 48, 2, 50, 48, 0.2), (1, 20, 2, 64, 40, 0.05),
        (1, 35, 1, 72, 35, 0.1), (1, 18, 2, 80, 16, 0.1), (1, 40, 2, 96, 16, 0.05), (1, 9, 1, 104, 4, 0.1), (1, 20, 1, 112, 20, 0.05),
        (1, 12, 2, 120, 12, 0.05), (3, 5, 1, 2, 2, 1.5), (1, 30, 2, 3, 8, 1.5)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,d,chunk,scale", PATH)
def test_path_bwd(B, T, H, d, chunk, scale, dt):
    from holonomyawareattention_b200 import ops
    a, R, C, P, hats, dhats = path_case(B, T, H, d, chunk, scale, dt, seed=T + d)
    da, dqkv = ops.path_bwd(a, R, C, chunk, H, scale, hats, dhats)
    ops.check_status()
    ra, rqkv = path_ref(a, P, hats, dhats, H, scale)
    assert da.dtype is torch.float32 and dqkv.dtype is dt
    assert rel(dqkv, rqkv) < (F32_TOL if dt is torch.float32 else BF16_TOL)
    assert not da[:, T - 1].any()
    if T > 1:
        assert rel(da[:, :T - 1], ra[:, :T - 1]) < F32_TOL
    again = ops.path_bwd(a, R, C, chunk, H, scale, hats, dhats)
    assert torch.equal(da, again[0]) and torch.equal(dqkv, again[1])


# (bound on 2 ||A|| from about 4, where the series changes, to the several hundred it ends at)
@pytest.mark.parametrize("d,amp", [(16, 0.5), (16, 1.0), (48, 0.4), (48, 1.5), (96, 0.6), (96, 2.0), (120, 0.3), (120, 1.5), (5, 40.0), (33, 3.0)])
def test_path_bwd_large_norms(d, amp):
    from holonomyawareattention_b200 import ops
    a, R, C, P, hats, dhats = path_case(1, 6, 2, d, 4, 1.0, torch.float32, seed=d, amp=amp)
    da, _ = ops.path_bwd(a, R, C, 4, 2, 1.0, hats, dhats)
    ra, _ = path_ref(a, P, hats, dhats, 2, 1.0)
    # a rotation by an angle of n radians is off by n eps in fp32
    angle = float(torch.linalg.matrix_norm(skew(a.view(1, 6, 2, -1).double(), d), 2).max())
    assert rel(da, ra) < F32_TOL + 4 * angle * 2.0 ** -24


def test_path_bwd_magnitudes():
    """Gradients of 1e-20 and 1e20 times the ordinary: the scales of the products follow."""
    from holonomyawareattention_b200 import ops
    a, R, C, P, hats, dhats = path_case(1, 40, 2, 48, 16, 0.05, torch.float32, seed=2)
    da, dqkv = ops.path_bwd(a, R, C, 16, 2, 0.05, hats, dhats)
    for f in (2.0 ** -66, 2.0 ** 66):
        # (o enters the sums beside the others: all of a pair's sides are scaled)
        x, y = ops.path_bwd(a, R, C, 16, 2, 0.05, hats, [t * f for t in dhats])
        assert torch.equal(x, da * f) and torch.equal(y, dqkv * f)
    zero = [torch.zeros_like(t) for t in dhats]
    x, y = ops.path_bwd(a, R, C, 16, 2, 0.05, hats, zero)
    assert not x.any() and not y.any()


def test_path_bwd_nan():
    """A NaN in position t's gradient reaches the generators before t and no later one; one in a generator its own alone."""
    from holonomyawareattention_b200 import ops
    a, R, C, P, hats, dhats = path_case(1, 70, 1, 32, 16, 0.05, torch.float32, seed=6)
    dhats[1][0, 40, 3] = float("nan")
    da, _ = ops.path_bwd(a, R, C, 16, 1, 0.05, hats, dhats)
    nan = torch.isnan(da[0]).any(1)
    assert nan[:40].all() and not nan[40:].any()
    dhats[1][0, 40, 3] = 0.0
    a[0, 20, 7] = float("inf")
    da, _ = ops.path_bwd(a, R, C, 16, 1, 0.05, hats, dhats)
    nan = torch.isnan(da[0]).any(1)
    assert nan[20] and int(nan.sum()) == 1
    # a norm beyond the series' range
    a[0, 20] = 1e4
    da, _ = ops.path_bwd(a, R, C, 16, 1, 0.05, hats, dhats)
    assert torch.isnan(da[0, 20]).all() and int(torch.isnan(da[0]).any(1).sum()) == 1


@pytest.mark.parametrize("d", [32, 64, 96])
def test_path_bwd_banked_and_bias(d):
    from holonomyawareattention_b200 import ops
    a, R, C, P, hats, dhats = path_case(2, 21, 2, d, 8, 0.1, torch.bfloat16, seed=d)
    g = torch.Generator(device=DEV).manual_seed(1)
    bias = 0.1 * randn(g, a.shape[-1])
    da, dqkv = ops.path_bwd(a, R, C, 8, 2, 0.1, hats, dhats)
    x, y = ops.path_bwd(a - bias, R, C, 8, 2, 0.1, hats, dhats, a_bias=bias, out_dtype=torch.float32)
    # (a - bias) + bias is a to an ulp of the larger
    assert rel(x, da) < F32_TOL and y.dtype is torch.float32 and rel(y, dqkv) < BF16_TOL
    b, yb = ops.path_bwd(ops.gen_to_banked(a, 2, d), R, C, 8, 2, 0.1, hats, dhats, gen_layout="banked")
    assert torch.equal(ops.gen_from_banked(b, 2, d), da) and torch.equal(yb, dqkv)
    S = ops.gen_stride(d, "banked")
    unused = torch.ones(2 * S, dtype=torch.bool)
    unused[ops.gen_banked_index(d, 2)] = False
    assert not b[..., unused.to(DEV)].any()


def test_path_bwd_refusals():
    from holonomyawareattention_b200 import ops
    a, R, C, P, hats, dhats = path_case(1, 10, 2, 16, 4, 0.1, torch.float32)
    with pytest.raises(ValueError, match="C must"):
        ops.path_bwd(a, R, C, 5, 2, 0.1, hats, dhats)
    with pytest.raises(ValueError, match="a_all"):
        ops.path_bwd(a[..., :-1].contiguous(), R, C, 4, 2, 0.1, hats, dhats)
    with pytest.raises(ValueError, match="o must"):
        ops.path_bwd(a, R, C, 4, 2, 0.1, [h.bfloat16() for h in hats], dhats)
    with pytest.raises(ValueError, match="dk"):
        ops.path_bwd(a, R, C, 4, 2, 0.1, hats, [dhats[0], dhats[1].bfloat16(), *dhats[2:]])
    with pytest.raises(NotImplementedError, match="fp32 generators"):
        ops.path_bwd(a.bfloat16(), R, C, 4, 2, 0.1, hats, dhats)
    with pytest.raises(NotImplementedError, match="banked"):
        ops.path_bwd(a, R, C, 4, 2, 0.1, hats, dhats, gen_layout="banked")


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
def values8(q, scale):
    n = q.numel()
    return (q.reshape(-1).double() * scale.double().repeat_interleave(256)[:n]).view(q.shape)


def adamw_ref(x, g, m, v, t, lr, b1, b2, eps, wd):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return x * (1 - lr * wd) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


SHAPES = [(1,), (7,), (255,), (256,), (257,), (33, 65), (2048,), (2049,), (3, 5, 1111), (0,), (70001,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_dt,g_dt,masters", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, True),
                                               (torch.bfloat16, torch.float32, False), (torch.float32, torch.bfloat16, False)])
def test_adamw_steps(bits, p_dt, g_dt, masters):
    from holonomyawareattention_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(0)
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    full = [randn(g, *s) for s in SHAPES]
    p = [x.to(p_dt) for x in full]
    ms = [x.clone() for x in full] if masters else None
    if bits == 32:
        m, v, scales = [torch.zeros_like(x) for x in full], [torch.zeros_like(x) for x in full], None
    else:
        m, v = ([torch.zeros(s, device=DEV).to(torch.float8_e4m3fn) for s in SHAPES] for _ in range(2))
        scales = [torch.zeros(2, -(-x.numel() // 256), device=DEV) for x in full]
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    for t in range(1, 4):
        grads = [(randn(g, *s) * 10.0 ** -t).to(g_dt) for s in SHAPES]
        want = []
        for i, s in enumerate(SHAPES):
            x = (ms[i] if masters else p[i]).double()
            mo = m[i].double() if bits == 32 else values8(m[i], scales[i][0])
            vo = v[i].double() if bits == 32 else values8(v[i], scales[i][1]) ** 2
            want.append(adamw_ref(x, grads[i].double(), mo, vo, t, 1e-2, 0.9, 0.95, 1e-8, 0.1))
        step.add_(1)
        ops.adamw_step(p, grads, m, v, step, masters=ms, scales=scales, **hyper)
        for i in range(len(SHAPES)):
            if not p[i].numel():
                continue
            x, mn, vn = want[i]
            if masters:
                assert torch.allclose(ms[i].double(), x, rtol=1e-6, atol=1e-7)
                assert torch.equal(p[i], ms[i].to(p_dt))
            else:
                eps = torch.finfo(p_dt).eps / 2
                assert torch.allclose(p[i].double(), x, rtol=1.001 * eps + 1e-6, atol=1e-7)
            if bits == 32:
                # the sum of two terms, each rounded: 2 eps of the larger
                assert torch.allclose(m[i].double(), mn, rtol=1e-6, atol=1e-7 * float(mn.abs().max()))
                assert torch.allclose(v[i].double(), vn, rtol=1e-6, atol=0)
            else:
                # half a step of e4m3: 2^-4 of the value, or 2^-10 of the block's scale for its smallest values; a root in
                # (0, 2^-10) of the scale is held as 2^-9 of it by definition (never as 0), so it is off by up to 2^-9
                for got, new, low in ((values8(m[i], scales[i][0]), mn, 2.0 ** -10), (values8(v[i], scales[i][1]), vn.sqrt(), 2.0 ** -9)):
                    top = torch.zeros(-(-new.numel() // 256) * 256, dtype=torch.float64, device=DEV)
                    top[:new.numel()] = new.reshape(-1).abs()
                    sc = (top.view(-1, 256).amax(1) / 448).repeat_interleave(256)[:new.numel()].view(new.shape)
                    assert bool(((got - new).abs() <= 2.0 ** -4 * 1.0001 * new.abs() + low * 1.0001 * sc).all())
                root = values8(v[i], scales[i][1])
                assert bool((root[vn > 0] > 0).all())


def test_adamw_same_as_separate_operations():
    """The new moments are bit for bit those of separate fp32 operations, so the 8-bit values are too."""
    from holonomyawareattention_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(1)
    n = 100 * 256 + 77
    m, v = 1e-3 * randn(g, n), (1e-3 * randn(g, n)).square()
    grad, p = 1e-3 * randn(g, n), randn(g, n)
    wm = m * 0.9 + grad * (1.0 - 0.9)
    wv = v * 0.999 + (grad * grad) * (1.0 - 0.999)
    step = torch.ones(1, dtype=torch.int32, device=DEV)
    ops.adamw_step([p], [grad], [m], [v], step, lr=1e-3)
    assert torch.equal(m, wm) and torch.equal(v, wv)


def test_adamw_many_tensors_and_unaligned():
    from holonomyawareattention_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(2)
    sizes = [(i * 37) % 500 + 1 for i in range(600)]
    flat = [randn(g, sum(sizes) + 1)[1:] for _ in range(2)] + [torch.zeros(sum(sizes) + 1, device=DEV)[1:] for _ in range(2)]
    parts = [list(t.split(sizes)) for t in flat]
    p0, g0 = flat[0].clone(), flat[1].clone()
    step = torch.ones(1, dtype=torch.int32, device=DEV)
    ops.adamw_step(*parts, step, lr=1e-2, weight_decay=0.0)
    x, m, v = adamw_ref(p0.double(), g0.double(), 0.0 * p0.double(), 0.0 * p0.double(), 1, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    assert torch.allclose(flat[0].double(), x, rtol=1e-6, atol=1e-7) and torch.allclose(flat[2].double(), m, rtol=1e-6, atol=1e-9)


def test_adamw_zero_and_nan():
    from holonomyawareattention_b200 import ops
    for bits in (32, 8):
        n = 600
        p = torch.ones(n, device=DEV)
        grad = torch.zeros(n, device=DEV)
        if bits == 32:
            m, v, sc = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), None
        else:
            m, v = (torch.zeros(n, device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
            sc = [torch.zeros(2, 3, device=DEV)]
        step = torch.ones(1, dtype=torch.int32, device=DEV)
        ops.adamw_step([p], [grad], [m], [v], step, lr=0.1, weight_decay=0.0, scales=sc)
        assert bool((p == 1).all()) and not m.float().any() and not v.float().any()
        grad[300] = float("nan")
        ops.adamw_step([p], [grad], [m], [v], step, lr=0.1, weight_decay=0.0, scales=sc)
        assert torch.isnan(p[300]) and int(torch.isnan(p).sum()) == 1


def test_adamw_refusals():
    from holonomyawareattention_b200 import ops
    x = [torch.zeros(8, device=DEV)]
    step = torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="grads"):
        ops.adamw_step(x, [], x, x, step, lr=0.1)
    with pytest.raises(ValueError, match="exp_avg"):
        ops.adamw_step(x, x, [torch.zeros(8, device=DEV).bfloat16()], x, step, lr=0.1)
    with pytest.raises(ValueError, match="step"):
        ops.adamw_step(x, x, x, x, torch.ones(1, device=DEV), lr=0.1)
    with pytest.raises(ValueError, match="scales"):
        q = [torch.zeros(8, device=DEV).to(torch.float8_e4m3fn)]
        ops.adamw_step(x, x, q, q, step, lr=0.1, scales=[torch.zeros(2, 2, device=DEV)])
    with pytest.raises(ValueError, match="different"):
        ops.adamw_step(x * 2, x * 2, x * 2, x * 2, step, lr=0.1)
    with pytest.raises(ValueError, match="betas"):
        ops.adamw_step(x, x, x, x, step, lr=0.1, betas=(1.0, 0.9))
    with pytest.raises(NotImplementedError, match="dtype"):
        h = [torch.zeros(8, device=DEV).half()]
        ops.adamw_step(h, h, x, x, step, lr=0.1)
