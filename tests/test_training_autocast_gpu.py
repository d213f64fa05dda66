"""fp32 weights behind a bf16 input: what torch.autocast makes of a module that follows another linear."""
import pytest
import torch

from holonomyawareattention_b200 import PathOrderedGeometricMHA, ops
from oracle import torch_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("D,H", [(192, 4), (128, 4)])                 # packed and banked generators
@pytest.mark.parametrize("mode", ["bf16", "split", "split8"])
def test_attention_behind_a_linear(D, H, mode):
    torch.manual_seed(0)
    first = torch.nn.Linear(64, D).to(DEV)
    m = PathOrderedGeometricMHA(D, n_heads=H, edge_scale=0.05).to(DEV)
    m.generator_precision = mode
    z, w = torch.randn(2, 48, 64, device=DEV), torch.randn(2, 48, D, device=DEV)
    tril = torch.ones(48, 48, dtype=torch.bool, device=DEV).tril()
    with torch.autocast("cuda", torch.bfloat16):
        x = first(z)
        x.retain_grad()
        y, _ = m(x, attn_mask=tril)
    assert x.dtype is torch.bfloat16
    (y * w).sum().backward()                                          # (outside autocast, as torch advises)
    ops.check_status()
    sd = {k: v.detach().double().requires_grad_() for k, v in m.state_dict().items()}
    xd = x.detach().double().requires_grad_()
    yd = torch_ref.module_forward(sd, xd, m.h, m.edge_scale, torch.float64, batch_slice=2)
    (yd * w.double()).sum().backward()
    # bf16 all the way (half a step, 2^-8, each): the 11 roundings of the bf16 module and those of the four weights
    tol = 15 * 2.0 ** -8
    assert rel(x.grad, xd.grad) < tol and first.weight.grad.dtype is torch.float32
    for k, p in m.named_parameters():
        if not k.startswith("g"):
            assert p.grad.dtype is torch.float32 and rel(p.grad, sd[k].grad) < tol, k
        if k.startswith("edge"):
            assert not torch.equal(p.grad, p.grad.bfloat16().float()), k      # (sums in fp32, not rounded on their way)
