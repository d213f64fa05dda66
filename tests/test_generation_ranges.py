"""Generation operators at the ends of their integer ranges: refused on the host before anything runs, or
shown on the index arithmetic alone (no GPU needed).
"""
import ctypes

import pytest
import torch

from holonomyawareattention_b200 import _lib, ops

UNS = _lib.HOA_ERR_UNSUPPORTED
BIG = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    from holonomyawareattention_b200 import _build
    _build.build()
    return _lib.load()


p, q, none = ctypes.c_void_p(16), ctypes.c_void_p(32), None
s3 = (ctypes.c_longlong * 3)(8, 8, 8)


@pytest.mark.parametrize("B,Tq,H", [(2 ** 31 - 1, 2, 1), (2 ** 20, 2 ** 11, 1), (1, 2 ** 30, 2), (2 ** 16, 2 ** 12, 8)])
def test_attention_rows_beyond_int(lib, B, Tq, H):
    """The kernels number the rows of a head, (b, t, g), with an int: 2^31 of them would come out negative."""
    assert lib.hoa_paged_attn_fwd(p, s3, p, p, s3, 0, p, 4, p, 1, 1, p, none, p, 0, p, 1.0, B, Tq, H, 1, 8, 16, 4, 148, p, 1 << 62,
                                  none, none) == UNS


@pytest.mark.parametrize("B,H", [(BIG, 1), (BIG - 200, 1), (2 ** 25 - 1, 64), (2 ** 30, 2)])
def test_path_step_units_beyond_int(lib, B, H):
    """A CTA steps from one (row, head) to the next by the size of the grid, also past the last one: with an int."""
    assert lib.hoa_path_step(p, 0, none, 1.0, p, p, p, 0, 6, p, p, p, 0, s3, p, 1, 1, p, B, H, 2, 4, 4, none, none) == UNS


@pytest.mark.parametrize("n_pages", [BIG, BIG - 100])
def test_pages_beyond_int(lib, n_pages):
    """The loops over pages and requests step past the last one with an int."""
    big = 1 << 62
    assert lib.hoa_pages_reserve(p, p, p, p, q, q, q, 1, 1, n_pages, 1, p, big, none, none) == UNS
    assert lib.hoa_pages_fork(p, p, p, p, p, 1, q, q, q, 1, 1, n_pages, 1, none, none, none, 0, p, big, none, none) == UNS
    assert lib.hoa_pages_free(p, p, p, p, 1, q, q, q, 1, 1, n_pages, 1, none, none) == UNS
    assert lib.hoa_pages_free(p, p, p, p, n_pages, q, q, q, 1, 1, 4, 1, none, none) == UNS
    assert lib.hoa_pages_compact(p, p, q, q, q, 1, 1, n_pages, none, none, none, 0, p, big, none, none) == UNS


def test_sizes_beyond_int_are_refused_in_python(monkeypatch):
    """Sizes that the C entry points take as int do not wrap on the way there."""
    monkeypatch.setattr(ops, "_index", lambda t: 0)
    monkeypatch.setattr(ops, "_ints", lambda *a: None)
    huge = torch.empty(1, dtype=torch.int32).expand(2 ** 32 + 5)
    small = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="2\\^31"):
        ops._books(small, None, huge, 4)
    with pytest.raises(ValueError, match="2\\^31"):
        ops._books(torch.empty(1, 1, dtype=torch.int32).expand(2 ** 16, 2 ** 16 + 1), None, small[0], 4)
    with pytest.raises(ValueError, match="2\\^31"):
        ops._books(small, None, small[0], 2 ** 32 + 1)


def test_a_pool_of_one_page_is_as_large_as_its_page():
    """A pool cut down to one page keeps the stride of the pool it was cut from, and counts as contiguous."""
    wide = torch.zeros(6, 4, 5)
    one = wide[::3][:1]
    assert one.is_contiguous() and one.stride(0) == 60
    keep, base, stride, size, n = ops._pool_args([one], 1, one.get_device())
    assert n == 1 and list(keep) == [one.data_ptr(), 240, 80]
