"""Generation operators: bad arguments are refused before anything runs (no GPU needed)."""
import ctypes

import pytest
import torch

from holonomyawareattention_b200 import _lib, ops


@pytest.fixture(scope="module")
def lib():
    from holonomyawareattention_b200 import _build
    _build.build()
    return _lib.load()


def z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    t, n, r = z(2, 3), z(2), z(4)
    kp = z(4, 1, 8, 16, dtype=torch.float32)
    for call in (lambda: ops.pages_reserve(t, n, r, n, 8), lambda: ops.pages_fork([kp], t, n, r, n, n, 8),
                 lambda: ops.pages_free(t, n, r, n, 8), lambda: ops.pages_compact([kp], t, r),
                 lambda: ops.pages_copy([kp], n, n), lambda: ops.pages_write(kp, kp, kp, kp, t, n),
                 lambda: ops.paged_attn_fwd(kp, kp, kp, t, n, 1.0),
                 lambda: ops.path_step(kp, kp, kp, 1, 1.0, kp, kp, t, n)):
        with pytest.raises(NotImplementedError, match="CUDA"):
            call()


def test_workspace_sizes(lib):
    assert lib.hoa_pages_workspace_bytes(-1, 4) == 0 and lib.hoa_pages_workspace_bytes(4, 0) == 0
    assert lib.hoa_pages_workspace_bytes(4, 100) >= 4 * 300
    ws = lib.hoa_paged_attn_workspace_bytes
    assert ws(0, 1, 4, 4, 48, 16, 0, 4, 148) == 0 and ws(2, 1, 4, 3, 48, 16, 0, 4, 148) == 0
    assert ws(2, 1, 4, 4, 48, 16, 0, 4, 148) > 0


def test_entry_points_refuse_bad_arguments(lib):
    p = ctypes.c_void_p(16)
    q = ctypes.c_void_p(32)
    none = None
    s3 = (ctypes.c_longlong * 3)(1, 1, 1)
    inv, uns, wsp = _lib.HOA_ERR_INVALID_ARG, _lib.HOA_ERR_UNSUPPORTED, _lib.HOA_ERR_WORKSPACE
    # reserve: null pointers, no rows, outputs that alias inputs, too many rows, small workspace
    assert lib.hoa_pages_reserve(none, p, p, p, q, q, q, 1, 1, 1, 1, p, 1000, none, none) == inv
    assert lib.hoa_pages_reserve(p, p, p, p, q, q, q, 0, 1, 1, 1, p, 1000, none, none) == inv
    assert lib.hoa_pages_reserve(p, p, p, p, p, q, q, 1, 1, 1, 1, p, 1000, none, none) == inv
    assert lib.hoa_pages_reserve(p, p, p, p, q, q, q, 65537, 1, 1, 1, p, 1 << 30, none, none) == uns
    assert lib.hoa_pages_reserve(p, p, p, p, q, q, q, 1, 1, 1, 1, p, 8, none, none) == wsp
    assert lib.hoa_pages_fork(p, p, p, p, p, 2, q, q, q, 1, 1, 1, 1, none, none, none, 0, p, 1000, none, none) == uns
    assert lib.hoa_pages_fork(p, p, p, none, p, 1, q, q, q, 1, 1, 1, 1, none, none, none, 0, p, 1000, none, none) == inv
    assert lib.hoa_pages_fork(p, p, p, p, p, 1, q, q, q, 1, 1, 1, 1, none, none, none, 1, p, 1000, none, none) == inv
    assert lib.hoa_pages_free(p, p, p, none, 1, q, q, q, 1, 1, 1, 1, none, none) == inv
    assert lib.hoa_pages_compact(p, p, q, q, none, 1, 1, 1, none, none, none, 0, p, 1000, none, none) == inv
    assert lib.hoa_pages_copy(none, none, none, 1, p, p, 1, 1, none, none) == inv
    assert lib.hoa_pages_copy(none, none, none, 0, p, p, 0, 1, none, none) == 0          # nothing to do
    w = lib.hoa_pages_write
    assert w(none, p, 0, s3, s3, p, p, 0, s3, p, 1, p, 1, 1, 1, 8, 4, 1, 1, none, none) == inv
    assert w(p, p, 7, s3, s3, p, p, 0, s3, p, 1, p, 1, 1, 1, 8, 4, 1, 1, none, none) == uns
    # attention: heads that do not divide, paths with several tokens, head dim, dtype, workspace
    f = lib.hoa_paged_attn_fwd

    def attn(q_=p, H=4, Hk=4, d=48, Tq=1, dtype=0, paths=none, n_shared=0, shared=none, W=1, page=16, nb=1 << 30):
        return f(q_, s3, p, p, s3, dtype, shared, n_shared, p, 1, W, p, paths, p, 0, p, 1.0, 1, Tq, H, Hk, d, page, 4,
                 148, p, nb, none, none)
    assert attn(q_=none) == inv and attn(H=4, Hk=3) == inv and attn(paths=p, Tq=2) == inv and attn(n_shared=1) == inv
    assert attn(d=129) == uns and attn(dtype=3) == uns and attn(W=2 ** 30, page=64) == uns and attn(nb=1) == wsp
    g = lib.hoa_path_step

    def step(a=p, adt=0, d=16, dtype=0, W=1):
        return g(a, adt, none, 1.0, p, p, p, 0, 48, p, p, p, dtype, s3, p, 1, W, p, 1, 1, d, 4, 4, none, none)
    assert step(a=none) == inv and step(d=1) == inv and step(W=0) == inv
    assert step(d=121) == uns and step(adt=1) == uns and step(dtype=2) == uns
    assert step(adt=_lib.HOA_GEN_BANKED) == uns                                          # 16 % 32 != 0
    assert b"page" in lib.hoa_status_string(_lib.HOA_ERR_PAGES)
