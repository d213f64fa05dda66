"""The copies of weights that the module lays out for its kernels, in training and between training steps: each forward sees
the weights that are there."""
import pytest
import torch

from holonomyawareattention_b200 import AdamW, PathOrderedGeometricMHA, ops, train_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tril(L):
    return torch.ones(L, L, dtype=torch.bool, device=DEV).tril()


def module(D, H, dtype=torch.bfloat16, es=0.05, seed=0):
    torch.manual_seed(seed)
    return PathOrderedGeometricMHA(D, n_heads=H, edge_scale=es).to(DEV, dtype)


def grads_of(m, x):
    m.zero_grad()
    m(x, attn_mask=tril(x.shape[1]))[0].float().square().sum().backward()
    return {k: p.grad for k, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("D,H", [(192, 4), (128, 4)])                 # packed and banked generators
@pytest.mark.parametrize("mode", ["auto", "split", "split8"])
def test_evaluated_in_inference_mode_between_steps(D, H, mode):
    x = torch.randn(2, 48, D, device=DEV).to(torch.bfloat16)
    seen = []
    for evaluate in (False, True):
        m = module(D, H, seed=1)
        m.generator_precision = mode
        opt = AdamW(m.parameters(), lr=1e-3)
        for _ in range(2):
            train_step(m, x, opt, lambda y: y.float().square().sum())
            if evaluate:
                with torch.inference_mode():
                    m(x, attn_mask=tril(48))
        if evaluate:
            with torch.inference_mode():
                m(x, attn_mask=tril(48))
        seen.append(grads_of(m, x))
    ops.check_status()
    assert seen[0].keys() == seen[1].keys() and all(torch.equal(seen[0][k], seen[1][k]) for k in seen[0])
