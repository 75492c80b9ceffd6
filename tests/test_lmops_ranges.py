"""Refusals of ah_linear_ce at the ends of the integers' ranges (CPU, as in test_lmops_errors.py)."""
import ctypes as C

import pytest

import test_lmops_errors as TE
from anneal_amd import _lib as L

lib, H, P = TE.lib, TE.H, TE.P
FAR = 1 << 40


@pytest.mark.parametrize("kw", [dict(N=1 << 27, ldx=FAR), dict(V=1 << 27, ldw=FAR), dict(N=1 << 27, lddx=FAR), dict(V=1 << 27, lddw=FAR),
                                dict(N=(1 << 23) + 1, ldx=FAR, dX=None), dict(N=1 << 26, ldx=1 << 39)], ids=str)
def test_rows_that_span_more_than_the_address_space(kw):
    """Rows times stride pass 64 bits, where a span would come out negative and overlap nothing."""
    d, n = TE.lce(**kw), C.c_int64(-1)
    assert lib.ah_linear_ce_workspace(H, C.byref(d), C.byref(n)) == TE.INVALID and n.value == -1 and "span" in TE.last_error()
    d = TE.lce(ws_bytes=(1 << 63) - 1, **kw)
    assert lib.ah_linear_ce(H, C.byref(d)) == TE.INVALID and "span" in TE.last_error()
