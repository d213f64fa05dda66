"""Building and loading: what one part needs, the other does without (no GPU needed)."""
import os

import pytest
import torch

from holonomyawareattention_b200 import _build, _lib, ops


def test_the_library_does_not_need_the_torch_side(monkeypatch, tmp_path):
    """libhoa.so is made (or found up to date) where the C++ host side cannot be: a warning, and the library's path."""
    def fails(force=False):
        raise RuntimeError("no headers here")

    monkeypatch.setattr(_build, "build_torch", fails)
    _build_lib = _build.LIB
    with pytest.warns(RuntimeWarning, match="no headers here"):
        assert _build.build() == _build_lib and os.path.exists(_build_lib)


def test_torch_side_is_rebuilt_for_another_torch(monkeypatch):
    """The C++ host side is made against one torch's headers: it is not taken for up to date under another one."""
    _build.build_torch()
    assert _build.torch_up_to_date()
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    assert not _build.torch_up_to_date()


def test_python_functions_take_over_without_the_torch_side(monkeypatch):
    """Where _hoa_torch.so cannot be loaded the Python functions take every call; said once."""
    import builtins
    real = builtins.__import__

    def no_host(name, globals=None, locals=None, fromlist=(), level=0):
        if fromlist and "_hoa_torch" in fromlist:
            raise ImportError("undefined symbol")
        return real(name, globals, locals, fromlist, level)

    monkeypatch.setattr(builtins, "__import__", no_host)
    monkeypatch.setattr(ops, "_HOST", None)
    with pytest.warns(RuntimeWarning, match="undefined symbol"):
        host = ops._host()
    assert ops._host() is host
    for name in ("pages_reserve", "pages_fork", "pages_free", "pages_compact", "paged_attn_fwd", "path_step", "device"):
        assert getattr(host, name)(1, 2, 3) is None
    t, n, r = (torch.zeros(*s, dtype=torch.int32) for s in ((2, 3), (2,), (4,)))
    with pytest.raises(NotImplementedError, match="CUDA"):
        ops.pages_free(t, n, r, n, 8)
    monkeypatch.undo()
    assert _lib.load() is not None
