"""Training through the module: its gradients against autograd of the float64 restatement of the reference, the
optimizer, one training step.

Tolerances (2-norm, relative).  fp32: the forward's bar is 1e-5 and the way to a weight's gradient is about twice as long
again: 3e-5.  bf16: at most 11 roundings of half a step (2^-8) on the way to a weight's gradient - x to qkv, the hats, the
heads and y; their gradients back to qkv; the generators', the hidden layer's two and the weight's own: 11 * 2^-8 = 4.3e-2.
"""
import pytest
import torch

from holonomyawareattention_b200 import AdamW, PathOrderedGeometricMHA, ops, train_step, training
from oracle import torch_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 3e-5, torch.bfloat16: 11 * 2.0 ** -8}


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


def tril(L):
    return torch.ones(L, L, dtype=torch.bool, device=DEV).tril()


def module(D, H, dtype, es=0.05, seed=0):
    torch.manual_seed(seed)
    return PathOrderedGeometricMHA(D, n_heads=H, edge_scale=es).to(DEV, dtype)


def reference_grads(m, x, w):
    sd = {k: v.detach().double().requires_grad_() for k, v in m.state_dict().items()}
    xd = x.detach().double().requires_grad_()
    y = torch_ref.module_forward(sd, xd, m.h, m.edge_scale, torch.float64, batch_slice=x.shape[0])
    (y * w.double()).sum().backward()
    return y.detach(), xd.grad, {k: v.grad for k, v in sd.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,H,B,L,es", [(32, 4, 2, 12, 0.1), (192, 4, 2, 70, 0.05), (64, 4, 1, 40, 1.5), (384, 4, 1, 65, 0.05), (240, 2, 2, 33, 0.05),
                                        (128, 2, 3, 1, 0.1), (20, 4, 1, 30, 0.1), (128, 4, 2, 150, 0.1)])
def test_gradients(D, H, B, L, es, dtype):
    m = module(D, H, dtype, es, seed=D)
    x = torch.randn(B, L, D, device=DEV).to(dtype).requires_grad_()
    w = torch.randn(B, L, D, device=DEV).to(dtype)
    y, geom = m(x, attn_mask=tril(L))
    assert geom is None
    (y * w).sum().backward()
    ops.check_status()
    yr, xr, gr = reference_grads(m, x, w)
    tol = TOL[dtype] * (10 if es > 1 else 1)            # (at edge_scale 1.5 angles of several radians: that many more ulps, bf16 steps of A too)
    if not (dtype is torch.bfloat16 and es > 1):         # (bf16 generators of that size turn the path by far more than their rounding)
        assert rel(y, yr) < (1e-5 if dtype is torch.float32 else 2e-2) * (3 if es > 1 else 1)
        assert rel(x.grad, xr) < tol
        for k, p in m.named_parameters():
            if k.startswith("g"):
                assert p.grad is None                    # not on the interaction link's path, as in the reference
            elif L > 1 or not k.startswith("edge"):
                assert rel(p.grad, gr[k]) < tol, k
            else:
                assert not p.grad.any()                  # one position: no edge
    else:
        assert all(bool(torch.isfinite(p.grad).all()) for k, p in m.named_parameters() if not k.startswith("g"))


def test_gradients_additive_link_and_split():
    m = module(64, 4, torch.float32, 0.1, seed=1)
    m.link_mode = "additive"
    x = torch.randn(2, 30, 64, device=DEV, requires_grad=True)
    w = torch.randn(2, 30, 64, device=DEV)
    (m(x, attn_mask=tril(30))[0] * w).sum().backward()
    assert all(p.grad is None for k, p in m.named_parameters() if k.startswith("edge"))
    # against differences of the forward (no_grad) along a direction of the generators' weights
    u = torch.randn_like(m.gqproj.weight)
    got = float((m.gqproj.weight.grad.double() * u.double()).sum())
    vals = []
    with torch.no_grad():
        base = m.gqproj.weight.clone()
        for h in (3e-3, -3e-3):
            m.gqproj.weight.copy_(base + h * u)
            vals.append(float((m(x, attn_mask=tril(30))[0].double() * w.double()).sum()))
        m.gqproj.weight.copy_(base)
    # y is good to 1e-5 of its norm: so is the difference to 1e-5 |y| |w| / (2 h); the curvature adds h^2 of the third derivative
    y = m(x, attn_mask=tril(30))[0]
    noise = 1e-5 * float(y.norm() * w.norm()) / 6e-3
    assert abs(got - (vals[0] - vals[1]) / 6e-3) < noise + 1e-2 * abs(got)
    # every form of the bf16 generators has the same gradients up to bf16
    m = module(192, 4, torch.bfloat16, 0.05, seed=2)
    x = torch.randn(1, 48, 192, device=DEV).to(torch.bfloat16)
    grads = {}
    for mode in ("bf16", "split", "split8"):
        m.generator_precision = mode
        m.zero_grad()
        m(x, attn_mask=tril(48))[0].float().square().sum().backward()
        grads[mode] = m.edge_mlp[2].weight.grad.clone()
    for mode in ("split", "split8"):
        assert rel(grads[mode], grads["bf16"]) < 2 * TOL[torch.bfloat16]


def test_forward_is_the_same_with_and_without_gradients():
    for dtype in (torch.float32, torch.bfloat16):
        m = module(192, 4, dtype, seed=3)
        x = torch.randn(3, 90, 192, device=DEV).to(dtype)
        with torch.no_grad():
            y0 = m(x, attn_mask=tril(90))[0]
        y1 = m(x, attn_mask=tril(90))[0]
        assert y1.requires_grad and rel(y1.detach(), y0) < (2e-5 if dtype is torch.float32 else 4e-2)
        # pieces of the batch
        m.PIECE_TOKENS = 90
        y2 = m(x, attn_mask=tril(90))[0]
        y2.sum().backward()
        g2 = m.edge_mlp[2].weight.grad.clone()
        m.zero_grad()
        y1.sum().backward()
        assert rel(y2.detach(), y1.detach()) < (2e-5 if dtype is torch.float32 else 4e-2)
        assert rel(g2, m.edge_mlp[2].weight.grad) < 2 * TOL[dtype]


def test_refusals():
    m = module(64, 4, torch.float32)
    x = torch.randn(1, 10, 64, device=DEV)
    with pytest.raises(NotImplementedError, match="tril"):
        m(x, attn_mask=None)
    with pytest.raises(NotImplementedError, match="geometry"):
        m(x, attn_mask=tril(10), return_geometry=True)
    with pytest.raises(NotImplementedError, match="causal"):
        PathOrderedGeometricMHA(64, n_heads=4, mode="inert").to(DEV)(x, attn_mask=tril(10))
    with pytest.raises(NotImplementedError, match="dropout"):
        PathOrderedGeometricMHA(64, n_heads=4, dropout=0.1).to(DEV).train()(x, attn_mask=tril(10))


def test_other_stream_and_accumulation():
    m = module(96, 2, torch.float32, seed=5)
    x = torch.randn(2, 40, 96, device=DEV)
    m(x, attn_mask=tril(40))[0].sum().backward()
    once = m.qkv.weight.grad.clone()
    m(x, attn_mask=tril(40))[0].sum().backward()
    assert rel(m.qkv.weight.grad, 2 * once) < 1e-6
    m.zero_grad()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m(x, attn_mask=tril(40))[0].sum().backward()
    s.synchronize()
    assert torch.equal(m.qkv.weight.grad, once)


def test_autocast():
    """fp32 weights, bf16 linears: what the core region is given then gives the same bits without autocast."""
    m = module(96, 3, torch.float32, seed=9)
    x, w = torch.randn(2, 50, 96, device=DEV), torch.randn(2, 50, 96, device=DEV)
    with torch.autocast("cuda", torch.bfloat16):
        y, _ = m(x, attn_mask=tril(50))
    (y * w).sum().backward()
    got = {k: p.grad for k, p in m.named_parameters()}
    m.zero_grad()
    with torch.autocast("cuda", torch.bfloat16):
        qkv, a = m.qkv(x), m.edge_mlp(torch.cat([x, torch.roll(x, -1, 1)], -1))
    assert qkv.dtype is a.dtype is torch.bfloat16
    heads = training.PathCore.apply(a.float(), qkv, None, m.h, m.edge_scale, m.scale, ops.plan_chunk(2, m.h, 50, m.d, x.device), "packed")
    with torch.autocast("cuda", torch.bfloat16):
        z = m.out(heads)
    (z * w).sum().backward()
    assert y.dtype is torch.bfloat16 and torch.equal(y, z)
    for k, p in m.named_parameters():
        assert (got[k] is None and p.grad is None) or (torch.equal(got[k], p.grad) and bool(p.grad.any())), k


def test_checkpointed_layers():
    """Two layers, each recomputed in the backward pass (torch.utils.checkpoint): the same gradients."""
    from torch.utils.checkpoint import checkpoint
    layers = [module(64, 4, torch.bfloat16, 0.1, seed=i) for i in (10, 11)]
    x = torch.randn(2, 40, 64, device=DEV).to(torch.bfloat16).requires_grad_()

    def run(wrap):
        y = x
        for m in layers:
            y = y + wrap(lambda t, m=m: m(t, attn_mask=tril(40))[0], y)
        y.float().square().sum().backward()
        grads = [x.grad] + [p.grad for m in layers for p in m.parameters() if p.grad is not None]
        x.grad = None
        for m in layers:
            m.zero_grad()
        return grads

    plain = run(lambda f, y: f(y))
    again = run(lambda f, y: checkpoint(f, y, use_reentrant=False))
    assert len(plain) == len(again) == 13 and all(torch.equal(a, b) for a, b in zip(plain, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_train_step_is_torch_adamw(dtype):
    m = module(64, 4, dtype, 0.1, seed=6)
    twin = module(64, 4, torch.float32, 0.1, seed=6)
    twin.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    x = torch.randn(2, 50, 64, device=DEV).to(dtype)
    target = torch.randn(2, 50, 64, device=DEV)
    opt = AdamW(m.parameters(), lr=1e-3, weight_decay=0.05)
    ref = torch.optim.AdamW(twin.parameters(), lr=1e-3, weight_decay=0.05)
    for _ in range(3):
        # the reference takes the gradients that this module has
        loss = (m(x, attn_mask=tril(50))[0].float() - target).square().mean()
        loss.backward()
        for p, q in zip(m.parameters(), twin.parameters()):
            q.grad = None if p.grad is None else p.grad.float()
        ref.step()
        opt.zero_grad()
        got = train_step(m, x, opt, lambda y: (y.float() - target).square().mean())
        assert got.shape == () and not got.requires_grad and rel(got, loss.detach()) < 1e-6
        assert all(p.grad is None for p in m.parameters())
        for (k, p), q in zip(m.named_parameters(), twin.parameters()):
            # (fp32: a few roundings of the update and of the value)
            x32 = opt.state[p].get("master", p) if p in opt.state else p
            assert torch.allclose(x32.float(), q, rtol=1e-6, atol=2e-8), k
            if dtype is torch.bfloat16 and "master" in opt.state.get(p, {}):
                assert torch.equal(p, x32.to(dtype))
    # the forward sees the new weights (nothing laid out from the old ones is used)
    fresh = module(64, 4, dtype, 0.1, seed=7)
    fresh.load_state_dict(m.state_dict())
    with torch.no_grad():
        assert torch.equal(m(x, attn_mask=tril(50))[0], fresh(x, attn_mask=tril(50))[0])


def test_train_step_clips_and_takes_8_bits():
    m = module(128, 4, torch.bfloat16, 0.05, seed=8)
    x = torch.randn(2, 64, 128, device=DEV).to(torch.bfloat16)
    opt = AdamW(m.parameters(), lr=1e-3, state_bits=8)
    before = {k: p.detach().clone() for k, p in m.named_parameters()}
    for _ in range(2):
        train_step(m, x, opt, lambda y: y.float().square().sum(), max_grad_norm=1.0)
    ops.check_status()
    s = opt.state[m.edge_mlp[2].weight]
    assert s["exp_avg"].dtype is torch.float8_e4m3fn and s["exp_avg_sq"].dtype is torch.float8_e4m3fn and s["step"] == 2
    for k, p in m.named_parameters():
        assert bool(torch.isfinite(p).all()) and torch.equal(p, before[k]) == k.startswith("g")
    # the state travels as it is
    opt2 = AdamW(m.parameters(), lr=1e-3, state_bits=8)
    opt2.load_state_dict(opt.state_dict())
    for p in m.parameters():
        for k, v in opt.state.get(p, {}).items():
            w = opt2.state[p][k]
            if torch.is_tensor(v):
                assert w.dtype is v.dtype and w.data_ptr() != v.data_ptr() and torch.equal(w.float(), v.float())
            else:
                assert w == v


def test_adamw_refusals():
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([torch.zeros(4, device=DEV, requires_grad=True)], state_bits=4)
    with pytest.raises(ValueError, match="betas"):
        AdamW([torch.zeros(4, device=DEV, requires_grad=True)], betas=(0.9, 1.0))
    p = torch.zeros(4, requires_grad=True)
    p.grad = torch.ones(4)
    with pytest.raises(NotImplementedError, match="CUDA"):
        AdamW([p]).step()
    q = torch.zeros(4, 6, device=DEV).t().requires_grad_()
    q.grad = torch.ones(6, 4, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([q]).step()
