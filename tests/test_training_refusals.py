"""What the training entry points refuse, without a GPU: CPU tensors, and bad sizes and types at the C ABI before any launch."""
import ctypes

import pytest
import torch

from holonomyawareattention_b200 import AdamW, PathOrderedGeometricMHA, _lib, ops, train_step

P = ctypes.c_void_p(256)           # (an address that no refused call looks at)
INVALID, UNSUPPORTED, WORKSPACE = _lib.HOA_ERR_INVALID_ARG, _lib.HOA_ERR_UNSUPPORTED, _lib.HOA_ERR_WORKSPACE


def test_cpu_tensors():
    x = torch.zeros(2, 4, 8)
    with pytest.raises(NotImplementedError, match="CUDA"):
        ops.attn_fwd_lse(x, x, x, 0.1)
    with pytest.raises(NotImplementedError, match="CUDA"):
        ops.attn_bwd(x, x, x, x, x[..., 0], x, 0.1)
    with pytest.raises(NotImplementedError, match="CUDA"):
        ops.path_bwd(torch.zeros(1, 4, 56), torch.zeros(2, 4, 8, 8), torch.zeros(2, 1, 8, 8), 4, 2, 0.1, [x] * 4, [x] * 4)
    with pytest.raises(NotImplementedError, match="CUDA"):
        ops.adamw_step([x], [x], [x], [x], torch.ones(1, dtype=torch.int32), lr=0.1)
    m = PathOrderedGeometricMHA(32, n_heads=4)
    with pytest.raises(NotImplementedError, match="CUDA"):
        train_step(m, torch.zeros(1, 4, 32), AdamW(m.parameters()), lambda y: y.sum())


def attn_bwd(dtype=_lib.HOA_BF16, BH=2, Tq=4, Tk=4, off=0, d=16, ws=1 << 20, q=P):
    return _lib.load().hoa_attn_bwd(q, P, P, P, P, P, dtype, P, P, P, 0.1, BH, Tq, Tk, off, d, P, ws, None, None)


def test_attn_bwd_abi():
    assert attn_bwd(q=None) == INVALID
    assert attn_bwd(BH=0) == INVALID and attn_bwd(Tq=0) == INVALID and attn_bwd(d=0) == INVALID
    assert attn_bwd(off=1) == INVALID and attn_bwd(off=-1) == INVALID and attn_bwd(Tq=5) == INVALID
    assert attn_bwd(off=2 ** 31 - 3, Tk=2 ** 31 - 1) == INVALID          # (the sum passes an int)
    assert attn_bwd(dtype=7) == UNSUPPORTED and attn_bwd(d=129) == UNSUPPORTED and attn_bwd(BH=65536) == UNSUPPORTED
    assert attn_bwd(Tk=2 ** 31 - 1) == UNSUPPORTED
    assert attn_bwd(ws=8) == WORKSPACE
    lib = _lib.load()
    f = lib.hoa_attn_bwd_workspace_bytes
    assert f(3, 5, 9, 16, _lib.HOA_F32, 0) == f(3, 5, 9, 16, _lib.HOA_BF16, 1) == 256 and f(0, 5, 9, 16, _lib.HOA_F32, 1) == 0
    # copies of 3 + 4 tensors, rows of 24 for 20, each from a 256-byte boundary
    assert f(3, 5, 9, 20, _lib.HOA_BF16, 1) == 256 + 3 * 768 + 4 * 1536 and f(3, 5, 9, 16, _lib.HOA_BF16, 0) > 256
    assert attn_bwd(d=20, ws=1024) == WORKSPACE
    assert lib.hoa_attn_fwd_lse(P, P, P, _lib.HOA_F32, P, None, 0.1, 1, 1, 1, 0, 8, None, None) == INVALID
    assert lib.hoa_attn_fwd_lse(P, P, P, 9, P, P, 0.1, 1, 1, 1, 0, 8, None, None) == UNSUPPORTED


@pytest.mark.parametrize("scale", [0.0, -0.25, float("inf"), float("-inf"), float("nan")])
def test_softmax_scale(scale):
    """A masked score is -infinity times the scale: only a positive, finite one leaves it masked."""
    lib = _lib.load()
    for dtype in (_lib.HOA_F32, _lib.HOA_BF16):
        assert lib.hoa_attn_fwd_lse(P, P, P, dtype, P, P, scale, 1, 1, 1, 0, 8, None, None) == INVALID
        assert lib.hoa_attn_bwd(P, P, P, P, P, P, dtype, P, P, P, scale, 1, 1, 1, 0, 8, P, 1 << 20, None, None) == INVALID


def path_bwd(a_dtype=_lib.HOA_F32, chunk=4, hat=_lib.HOA_F32, out=_lib.HOA_F32, B=1, H=2, T=8, d=8, ws=1 << 40, a=P, wsp=P):
    return _lib.load().hoa_path_bwd(a, a_dtype, None, 0.1, P, P, chunk, P, P, P, P, P, P, P, P, hat, P, P, out, B, H, T, d, wsp, ws, None, None)


def test_path_bwd_abi():
    assert path_bwd(a=None) == INVALID and path_bwd(wsp=None) == INVALID
    assert path_bwd(B=0) == INVALID and path_bwd(T=0) == INVALID and path_bwd(d=1) == INVALID and path_bwd(chunk=0) == INVALID
    assert path_bwd(d=121) == UNSUPPORTED and path_bwd(hat=5) == UNSUPPORTED and path_bwd(out=5) == UNSUPPORTED
    assert path_bwd(a_dtype=_lib.HOA_BF16) == UNSUPPORTED
    assert path_bwd(a_dtype=_lib.HOA_F32 | _lib.HOA_GEN_BANKED) == UNSUPPORTED      # (d % 32 != 0)
    assert path_bwd(B=65536, H=65536) == UNSUPPORTED
    assert path_bwd(ws=1024) == WORKSPACE
    assert path_bwd(wsp=ctypes.c_void_p(128)) == WORKSPACE                           # (256-byte boundaries)
    f = _lib.load().hoa_path_bwd_workspace_bytes
    assert f(1, 2, 8, 8, 4) > 0 and f(1, 2, 8, 8, 0) == 0 and f(1, 2, 8, 121, 4) == 0 and f(65536, 65536, 1, 8, 4) == 0
    # the matrices of a pass are bounded: a long input's workspace grows with its runs of 32 positions alone
    small, large = f(1, 16, 4096, 96, 64), f(1, 16, 65536, 96, 64)
    assert large - small < (65536 - 4096) // 32 * 16 * 96 * 96 * 4 * 1.01


def adamw(sizes=(4,), bits=32, p=P, p_dt=_lib.HOA_F32, g_dt=_lib.HOA_F32, scales=False, step=P):
    n = len(sizes)
    ptrs = (ctypes.c_void_p * n)(*([p] * n))
    return _lib.load().hoa_adamw_step(ptrs, p_dt, None, ptrs, g_dt, ptrs, ptrs, ptrs if scales else None, bits,
                                      (ctypes.c_longlong * n)(*sizes), n, step, 1e-3, 0.9, 0.99, 1e-8, 0.0, None)


def test_adamw_abi():
    assert adamw(step=None) == INVALID and adamw(p=None) == INVALID and adamw(sizes=(-1,)) == INVALID
    assert adamw(bits=16) == UNSUPPORTED and adamw(p_dt=3) == UNSUPPORTED and adamw(g_dt=3) == UNSUPPORTED
    assert adamw(bits=8) == INVALID                                                   # (no scales)
    assert adamw(sizes=(0, 0), p=None) == _lib.HOA_OK                                 # nothing to do


def test_adamw_arguments():
    w = [torch.zeros(3, requires_grad=True)]
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(weight_decay=-0.1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW(w, **bad)
