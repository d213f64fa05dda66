"""attn_bwd in bf16 is off by the rounding of its results and no more."""
import math

import pytest
import torch

from holonomyawareattention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("BH,Tq,Tk,off,d", [(1, 2, 39, 37, 104), (2, 6, 14, 8, 112), (3, 41, 41, 0, 48), (2, 35, 35, 0, 5), (1, 19, 19, 0, 16),
                                            (113, 2, 2, 0, 40), (1, 4, 4, 0, 112), (6, 51, 195, 20, 20), (16, 300, 300, 0, 96),
                                            (4, 200, 333, 100, 128), (8, 700, 700, 0, 64), (2, 1500, 1500, 0, 50)])
@pytest.mark.parametrize("sharp", [1.0, 4.0])
def test_rounded_once(BH, Tq, Tk, off, d, sharp):
    """Against 64 bits, from o and the log-sum-exp of 64 bits rounded to fp32.  Scores, exponentials and sums are fp32 and p
    and ds are taken to 2^-16: with terms that cancel to a tenth of their size that is 2^-12, and in squares beside the
    results' own rounding (2^-8 at most, a third of it on average) below 5%."""
    g = torch.Generator(device=DEV).manual_seed(BH * Tk + d)
    q, k, v, do = (torch.randn(BH, t, d, device=DEV, generator=g).bfloat16() for t in (Tq, Tk, Tk, Tq))
    scale = sharp / math.sqrt(d)
    x = [t.double().requires_grad_() for t in (q, k, v)]
    s = x[0] @ x[1].transpose(1, 2) * scale
    seen = torch.arange(Tk, device=DEV)[None, :] <= off + torch.arange(Tq, device=DEV)[:, None]
    s = s.masked_fill(~seen, -math.inf)
    o, lse = torch.softmax(s, -1) @ x[2], torch.logsumexp(s, -1)
    want = torch.autograd.grad((o * do.double()).sum(), x)
    got = ops.attn_bwd(q, k, v, o.detach().float(), lse.detach().float(), do, scale, off)
    ops.check_status()
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        once = float((b.bfloat16().double() - b).norm())
        assert float((a.double() - b).norm()) <= 1.05 * once, (name, float((a.double() - b).norm()) / once)
