"""AdamW's fp32 master copies and parameters that something else writes between steps."""
import copy

import pytest
import torch

from holonomyawareattention_b200 import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"


def stepped(steps=2, seed=0):
    torch.manual_seed(seed)
    ps = [torch.randn(s, device=DEV).bfloat16().requires_grad_() for s in ((300,), (7, 33))]
    opt = AdamW(ps, lr=1e-3, weight_decay=0.0)
    for _ in range(steps):
        step(opt, ps)
    return ps, opt


def step(opt, ps, value=1.0):
    for p in ps:
        p.grad = torch.full_like(p, value)
    opt.step()


def masters(ps, opt):
    return [opt.state[p]["master"].clone() for p in ps]


def test_written_parameters_are_stepped_on():
    """load_state_dict, a clamp, an average: the step goes on from what was written, element by element."""
    ps, opt = stepped()
    before = masters(ps, opt)
    assert any(not torch.equal(m, m.bfloat16().float()) for m in before)
    with torch.no_grad():
        ps[0].clamp_(-0.5, 0.5)
    was = ps[0].detach().clone()
    cut = was.float() != before[0].bfloat16().float()
    assert 50 < int(cut.sum()) < 250
    step(opt, ps, 0.0)
    moved = before[0] - masters(ps, opt)[0]
    # (the step of the elements that were not written is that of the master; of the others, that of the written value)
    want = torch.where(cut, was.float(), before[0])
    first = masters(ps, opt)[0]
    assert float((first - want).abs().max()) < 2e-3 and float(moved[~cut].abs().max()) < 2e-3
    assert torch.equal(ps[0], first.bfloat16())
    with torch.no_grad():
        ps[1].copy_(torch.zeros_like(ps[1]))
    step(opt, ps, 0.0)
    assert float(masters(ps, opt)[1].abs().max()) < 2e-3 and float(ps[1].float().abs().max()) < 2e-3


def test_unwritten_parameters_keep_their_masters():
    """Steps in turn, a reloaded optimizer state, loaded before or after the parameters: the low bits stay."""
    ps, opt = stepped(3)
    twins = [p.detach().clone().requires_grad_() for p in ps]
    opt2 = AdamW(twins, lr=1e-3, weight_decay=0.0)
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    with torch.no_grad():
        for p, t in zip(ps, twins):
            t.copy_(p)                                           # (the same values again, as a resumed run loads them)
    for _ in range(2):
        step(opt, ps)
        step(opt2, twins)
    assert all(torch.equal(a, b) for a, b in zip(masters(ps, opt), masters(twins, opt2)))
    assert all(torch.equal(a, b) for a, b in zip(ps, twins))
    assert set(opt.state_dict()["state"][0]) == {"step", "exp_avg", "exp_avg_sq", "master"}


def test_replaced_memory():
    ps, opt = stepped()
    ps[0].data = torch.zeros_like(ps[0])
    step(opt, ps, 0.0)
    assert float(masters(ps, opt)[0].abs().max()) < 2e-3
    both = copy.deepcopy((ps, opt))                              # (optimizers are copied and pickled with their parameters)
    step(both[1], both[0])
    step(opt, ps)
    assert all(torch.equal(a, b) for a, b in zip(masters(ps, opt), masters(*both)))
