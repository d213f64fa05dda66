"""AdamW's arguments and errors: groups of their own, and steps that are refused before anything changes."""
import pytest
import torch

from holonomyawareattention_b200 import AdamW


def param(*shape, **kw):
    p = torch.ones(*shape, **kw).requires_grad_()
    p.grad = torch.ones_like(p)
    return p


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(betas=(0.9, 1.0)), dict(state_bits=16), dict(lr=float("nan"))])
def test_groups_are_checked(bad):
    with pytest.raises(ValueError):
        AdamW([dict(params=[param(3)], **bad)])
    opt = AdamW([param(3)])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[param(4)], **bad))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[param(4)], lr=0.0, state_bits=8))
    assert opt.param_groups[1]["state_bits"] == 8 and opt.param_groups[0]["state_bits"] == 32


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["cpu", "half", "stride", "grad"])
def test_refused_before_anything_changes(what):
    good = [param(5, device="cuda"), param(7, device="cuda", dtype=torch.bfloat16)]
    if what == "cpu":
        bad = param(3)
    elif what == "half":
        bad = param(3, device="cuda", dtype=torch.float16)
    elif what == "stride":
        bad = torch.ones(4, 6, device="cuda").t().requires_grad_()
        bad.grad = torch.ones(6, 4, device="cuda")
    else:
        bad = param(3, device="cuda")
        bad.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1), (3,), device="cuda")
    opt = AdamW([dict(params=good), dict(params=[bad])], lr=0.1)
    with pytest.raises((NotImplementedError, ValueError)):
        opt.step()
    assert all(bool((p == 1).all()) for p in good) and not opt.state
    bad.grad = None
    opt.step()
    assert all(bool((p < 1).all()) for p in good) and all(opt.state[p]["step"] == 1 for p in good)


@pytest.mark.gpu
def test_capture_refused_before_the_closure():
    p = param(5, device="cuda")
    opt, ran = AdamW([p]), []
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(NotImplementedError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(lambda: ran.append(1))
    assert not ran and opt.state[p]["step"] == 1


@pytest.mark.gpu
def test_default_type():
    """The state's types are their own, whatever torch's default type is."""
    old = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.float64)
        p = param(600, device="cuda", dtype=torch.bfloat16)
        opt = AdamW([p], state_bits=8)
        opt.step()
    finally:
        torch.set_default_dtype(old)
    # (the master: 1 - 1e-3 is 1 in bf16, whose values below 1 are 2^-8 apart)
    assert opt.state[p]["scales"].dtype is torch.float32 and bool((opt.state[p]["master"] < 1).all())
