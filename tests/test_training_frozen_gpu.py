"""Modules of which parts are frozen: the gradients of the rest are those of the whole, and what nobody asks for is not computed."""
import pytest
import torch

from holonomyawareattention_b200 import PathOrderedGeometricMHA, ops, training

pytestmark = pytest.mark.gpu
DEV = "cuda"
L = 40


def module(dtype, seed=0):
    torch.manual_seed(seed)
    return PathOrderedGeometricMHA(128, n_heads=4, edge_scale=0.1).to(DEV, dtype)


def grads(m, x, w):
    m.zero_grad()
    x.grad = None
    (m(x, attn_mask=torch.ones(L, L, dtype=torch.bool, device=DEV).tril())[0] * w).sum().backward()
    return {**{k: p.grad for k, p in m.named_parameters() if p.grad is not None}, **({"x": x.grad} if x.requires_grad else {})}


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("x_grad", [False, True])
@pytest.mark.parametrize("frozen", [("edge_mlp",), ("edge_mlp.0",), ("edge_mlp.2",), ("edge_mlp.0.bias", "edge_mlp.2.weight"), ("qkv",), ("qkv", "out"),
                                    ("qkv", "edge_mlp.0", "edge_mlp.2.bias")])
def test_frozen(frozen, x_grad, dtype, monkeypatch):
    m = module(dtype)
    x = torch.randn(2, L, 128, device=DEV).to(dtype).requires_grad_(x_grad)
    w = torch.randn(2, L, 128, device=DEV).to(dtype)
    whole = grads(m, x, w)
    for k, p in m.named_parameters():
        p.requires_grad_(not k.startswith(frozen))
    calls = []
    for mod, name in ((ops, "path_bwd"), (training, "_weight_grad")):
        real = getattr(mod, name)
        monkeypatch.setattr(mod, name, lambda *a, n=name, f=real: calls.append(n) or f(*a))
    part = grads(m, x, w)
    ops.check_status()
    assert set(part) == {k for k in whole if not k.startswith(frozen)}
    no_generators = not x_grad and frozen == ("edge_mlp",)
    assert calls.count("path_bwd") == (0 if no_generators else 1)
    if dtype is torch.bfloat16:
        assert calls.count("_weight_grad") == sum(k.startswith("edge_mlp") and k.endswith("weight") for k in part)
    for k in part:
        if no_generators and k == "qkv.weight":
            # (P d by fp32 FMAs in one place, by split f16 in the other: both far below a rounding of dqkv, which may fall the other way)
            assert rel(part[k], whole[k]) < (2e-6 if dtype is torch.float32 else 2.0 ** -8), k
        else:
            assert torch.equal(part[k], whole[k]), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bias_of_the_core(dtype):
    """One row of generators for all positions: its gradient is the sum of theirs."""
    m = module(torch.float32, seed=1)
    g = torch.Generator(device=DEV).manual_seed(1)
    a = 0.3 * torch.randn(2, L, m.h * m.m_dim, device=DEV, generator=g)
    qkv = torch.randn(2, L, 384, device=DEV, generator=g).to(dtype)
    w = torch.randn(2, L, 128, device=DEV, generator=g).to(dtype)
    bias = (0.1 * torch.randn(a.shape[-1], device=DEV, generator=g)).requires_grad_()
    got = torch.autograd.grad((training.PathCore.apply(a, qkv, bias, m.h, 0.1, m.scale, 8, "packed") * w).sum(), bias)[0]
    both = (a + bias.detach()).requires_grad_()
    want = torch.autograd.grad((training.PathCore.apply(both, qkv, None, m.h, 0.1, m.scale, 8, "packed") * w).sum(), both)[0].sum((0, 1))
    assert rel(got, want) < 2e-6
