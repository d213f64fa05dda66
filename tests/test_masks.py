"""Which masks the module takes for the causal one: each by what it holds, whatever lay in its memory before."""
import copy
import pickle

import pytest
import torch

from holonomyawareattention_b200 import PathOrderedGeometricMHA

L = 256


def tril(device="cpu", n=L):
    return torch.ones(n, n, dtype=torch.bool, device=device).tril()


def mask_at(address, like):
    """An uninitialised mask at ``address``, where the allocator gives that out."""
    held = []
    for _ in range(200):
        held.append(torch.empty_like(like))
        if held[-1].data_ptr() == address:
            return held[-1]
    pytest.skip("the allocator does not give the memory out again")


def check_freed(m, device, n=L):
    """Masks that take one another's memory: a tril mask is one, no other is."""
    other = torch.ones(n, n, dtype=torch.bool, device=device)
    for i in range(20):
        a = tril(device, n)
        assert m._mask_is_tril(a, n)
        at = a.data_ptr()
        del a
        b = mask_at(at, other)                       # (its version is 0, as the other's was)
        b.data.copy_(other)
        assert b._version == 0 and not m._mask_is_tril(b, n)
        del b


def test_freed_masks():
    check_freed(PathOrderedGeometricMHA(32, n_heads=4), "cpu")


def test_masks_written_and_viewed():
    m = PathOrderedGeometricMHA(32, n_heads=4)
    big = torch.ones(2 * L, 2 * L, dtype=torch.bool).tril()
    looked = []
    real = torch.equal
    try:
        torch.equal = lambda *a: looked.append(1) or real(*a)
        assert m._mask_is_tril(big[:L, :L], L) and m._mask_is_tril(big[:L, :L], L)
        assert len(looked) == 1                      # another view of the same memory is not looked at again
    finally:
        torch.equal = real
    assert not m._mask_is_tril(big[L:, :L], L)
    big[0, 5] = True
    assert not m._mask_is_tril(big[:L, :L], L)
    big[0, 5] = False
    assert m._mask_is_tril(big[:L, :L], L)
    assert not m._mask_is_tril(big[:L, :L].t(), L)
    with torch.inference_mode():                     # (torch counts no writes of this one)
        c = tril()
        assert m._mask_is_tril(c, L)
        c[0, 1] = True
        assert not m._mask_is_tril(c, L)


def test_module_copies():
    m = PathOrderedGeometricMHA(32, n_heads=4)
    a = tril()
    m._mask_is_tril(a, L)
    for twin in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert not twin._mask_is_tril(~a, L) and twin._mask_is_tril(a, L)


def test_pickles_of_earlier_versions():
    """A module that was pickled with a dictionary of masks and without copies of weights."""
    m = PathOrderedGeometricMHA(32, n_heads=4)
    m._tril_ok = {}
    del m._copies
    twin = pickle.loads(pickle.dumps(m))
    assert twin._mask_is_tril(tril(), L) and not twin._mask_is_tril(~tril(), L)
    twin.eval().train()


@pytest.mark.gpu
def test_freed_masks_on_the_gpu():
    """A freed causal mask's memory with another mask in it: the forward is that mask's, with gradients it is refused."""
    torch.manual_seed(0)
    n = 2048                                         # (4 MB: a block of its own, which the next mask of that size is given)
    m = PathOrderedGeometricMHA(64, n_heads=4).to("cuda")
    check_freed(m, "cuda", n)
    x = torch.randn(1, n, 64, device="cuda")
    window = torch.ones(n, n, dtype=torch.bool, device="cuda").tril().triu(-5)
    with torch.no_grad():
        a = tril("cuda", n)
        causal, at = m(x, attn_mask=a)[0], a.data_ptr()
        want = m(x, attn_mask=window)[0]
        assert float((want - causal).norm()) > 0.1 * float(causal.norm())
        del a
        b = mask_at(at, window)
        b.data.copy_(window)
        assert torch.equal(m(x, attn_mask=b)[0], want)
    del b
    a = tril("cuda", n)
    m(x, attn_mask=a)[0].sum().backward()
    del a
    b = window.clone()
    with pytest.raises(NotImplementedError, match="tril"):
        m(x, attn_mask=b)
