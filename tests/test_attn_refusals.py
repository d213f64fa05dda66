"""Sizes that the attention entry points refuse before any launch (no GPU needed): sums of offsets that pass an int."""
import ctypes

import pytest

from holonomyawareattention_b200 import _lib

P = ctypes.c_void_p(256)           # (an address that no refused call looks at)
F32, BF16 = _lib.HOA_F32, _lib.HOA_BF16


def calls(Tq, Tk, off):
    lib = _lib.load()
    yield lib.hoa_attn_fwd(P, P, P, F32, P, 0.1, 1, Tq, Tk, off, 8, None)
    yield lib.hoa_attn_fwd(P, P, P, BF16, P, 0.1, 1, Tq, Tk, off, 8, None)
    yield lib.hoa_attn_tc_fwd(P, P, P, P, None, 0.1, 1, Tq, Tk, off, 8, None)
    for dtype, d in ((F32, 8), (BF16, 8), (BF16, 5)):
        yield lib.hoa_attn_fwd_lse(P, P, P, dtype, P, P, 0.1, 1, Tq, Tk, off, d, None, None)


@pytest.mark.parametrize("Tq,Tk,off", [(4, 2 ** 31 - 1, 2 ** 31 - 3), (4, 9, 2 ** 31 - 1), (2 ** 31 - 1, 9, 2 ** 31 - 1), (4, 9, 6)])
def test_queries_past_the_keys(Tq, Tk, off):
    assert all(st == _lib.HOA_ERR_INVALID_ARG for st in calls(Tq, Tk, off))


def test_keys_past_an_int():
    """Tiles of keys start at multiples of up to 128, counted with ints."""
    assert all(st == _lib.HOA_ERR_UNSUPPORTED for st in calls(4, 2 ** 31 - 1, 0))
