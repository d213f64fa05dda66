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
