"""Sizes that the head's losses cannot index with 32-bit numbers are refused before the device is touched."""
import ctypes

import pytest

import lancet_b200 as LB
from lancet_b200 import _capi

ONE = ctypes.c_void_p(256)
MOST = 1 << 30


@pytest.fixture(scope="module")
def L():
    LB.build.build()
    return _capi.lib()


def _fwd(L, rows, vocab):
    return L.lancet_distill_fwd(ONE, 1 << 40, ONE, 0, ONE, 2, 1.0, rows, vocab, 0, ONE, ONE, ONE, ONE, None, ONE, None)


def _bwd(L, rows, vocab, cols):
    return L.lancet_distill_bwd(ONE, 1 << 40, ONE, ONE, ONE, 2, 1.0, rows, vocab, cols, 0, ONE, None, None, 1.0, None, 1 << 40, None)


def test_distillation(L):
    # 2: sizes that are taken reach the check of the null pointer that is passed on purpose
    for size in (MOST, 1):
        assert _fwd(L, size, 5) == 2 and _fwd(L, 5, size) == 2
        assert _bwd(L, size, 5, 5) == 2 and _bwd(L, 5, 1, size) == 2
    for size in (MOST + 1, 2 ** 31 - 1):
        assert _fwd(L, size, 5) == 1 and _fwd(L, 5, size) == 1
        assert _bwd(L, size, 5, 5) == 1 and _bwd(L, 5, 1, size) == 1 and _bwd(L, 5, size, size) == 1


def test_copy_rows(L):
    assert L.lancet_copy_rows(None, 8, ONE, 8, MOST, 8, None) == 2
    for rows, width in ((MOST + 1, 8), (2 ** 31 - 1, 8), (4, MOST + 1)):
        assert L.lancet_copy_rows(None, 1 << 40, ONE, 1 << 40, rows, width, None) == 1
