"""Generation through the module: prefill, fork, share, decode, free and compact against the module's own
full forward over each row's whole sequence.

Tolerances: both sides are within the module's bars of the exact result (fp32 1e-5, bf16 2e-2 rel-L2),
so they are within twice that of one another.
"""
import pytest
import torch

from holonomyawareattention_b200 import PathCache, PathOrderedGeometricMHA, _lib, decode, ops, prefill

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 2e-5, torch.bfloat16: 4e-2}


def full(attn, x):
    L = x.shape[0]
    mask = torch.tril(torch.ones(L, L, dtype=torch.bool, device=DEV))
    return attn(x[None], attn_mask=mask)[0][0]


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,H,page,link", [(192, 4, 16, "interaction"), (384, 4, 64, "interaction"), (240, 2, 24, "interaction"),
                                           (64, 4, 16, "additive")])
def test_generation_equals_the_full_forward(D, H, page, link, dtype):
    torch.manual_seed(D)
    attn = PathOrderedGeometricMHA(D, n_heads=H, edge_scale=0.05).to(DEV, dtype).eval()
    attn.link_mode = link
    rows = 5
    cache = PathCache(attn, rows=rows, max_tokens=200, page=page)
    seq = [torch.zeros(0, D, device=DEV, dtype=dtype) for _ in range(rows)]     # what each row was given
    got = [torch.zeros(0, D, device=DEV, dtype=dtype) for _ in range(rows)]

    def feed(x, rs):
        y = prefill(attn, x, cache, rs)
        for i, r in enumerate(rs):
            seq[r], got[r] = torch.cat([seq[r], x[i]]), torch.cat([got[r], y[i]])

    def step():
        x = torch.randn(rows, D, device=DEV).to(dtype)
        y = decode(attn, x, cache)
        for r in range(rows):
            if cache.tokens[r]:
                seq[r], got[r] = torch.cat([seq[r], x[r:r + 1]]), torch.cat([got[r], y[r:r + 1]])

    with torch.no_grad():
        feed(torch.randn(1, 70, D, device=DEV).to(dtype), [1])
        step()                                                    # rows 0 and 2-4 are idle
        cache.fork([1, 1, 1], [3, 0, 4])
        for r in (3, 0, 4):
            seq[r], got[r] = seq[1], got[1]
        assert cache.share(1) == 71 // page * page
        step()
        feed(torch.randn(2, 37, D, device=DEV).to(dtype), [0, 4])  # questions after the shared prompt
        for _ in range(3):
            step()
        cache.free([1, 3])
        for r in (1, 3):
            seq[r], got[r] = seq[r][:0], got[r][:0]
        live = cache.compact()
        assert int(live) == int((cache.refs > 0).sum()) and bool((cache.refs[int(live):] == 0).all())
        step()
        cache.share(0, 0)
        feed(torch.randn(2, 1, D, device=DEV).to(dtype), [2, 3])   # prompts of one token in new rows
        step()
        step()
        ops.check_status()
        for r in (0, 2, 3, 4):
            assert cache.tokens[r] == len(seq[r])
            assert rel(got[r], full(attn, seq[r])) <= TOL[dtype], r


def test_cache_refusals():
    attn = PathOrderedGeometricMHA(64, n_heads=2).to(DEV).eval()
    x = torch.randn(1, 20, 64, device=DEV)
    with torch.no_grad():
        cache = PathCache(attn, rows=3, max_tokens=40, n_pages=4, page=16)
        prefill(attn, x, cache, [0])
        with pytest.raises(ValueError, match="max_tokens"):
            prefill(attn, torch.cat([x, x], 1), cache, [0])
        with pytest.raises(ValueError, match="all be empty"):
            prefill(attn, torch.cat([x, x]), cache, [0, 1])
        with pytest.raises(ValueError, match="different rows"):
            cache.free([3])
        with pytest.raises(ValueError, match="empty"):
            cache.fork([0], [0])
        with pytest.raises(ValueError, match="with tokens"):
            cache.fork([1], [2])
        cache.share(0)
        with pytest.raises(ValueError, match="shared pages"):
            prefill(attn, x, cache, [1])
        cache.share(0, 0)
        prefill(attn, x, cache, [1])
        with pytest.raises(ValueError, match="fork"):
            cache.share(0)
        with pytest.raises(ValueError, match="must be"):
            decode(attn, x[0], cache)
        state = cache.table, cache.lens, cache.refs, list(cache.tokens)
        for call in (lambda: prefill(attn, x, cache, [2]), lambda: cache.fork([0], [2])):
            with pytest.raises(_lib.HoaError) as e:                # four pages are taken: none is left
                call()
            assert e.value.status == _lib.HOA_ERR_PAGES
        assert state[:3] == (cache.table, cache.lens, cache.refs) and state[3] == cache.tokens
        cache.free([1])
        cache.fork([0], [2])
        ops.check_status()
        assert int((cache.refs > 0).sum()) == len(cache._count) == 3
    with pytest.raises(NotImplementedError, match="forward-only"):
        decode(attn, torch.randn(3, 64, device=DEV), cache)
    with pytest.raises(NotImplementedError, match="causal"):
        PathCache(PathOrderedGeometricMHA(64, n_heads=2, mode="inert").to(DEV), 1, 8)
