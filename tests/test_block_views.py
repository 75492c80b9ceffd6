"""Which arrays of a call may lie between one another: rows of one stride side by side, as the halves of one array, are apart; anything that shares a
byte is refused. No device is needed: a call whose arrays are apart goes on to the check of its workspace, which is made to fail here."""
import ctypes as C

import pytest

from anneal_amd import _lib as L
from test_block_errors import H, INVALID, P, last_error, lib, linear, linear_grad, norm, norm_grad

F = 16
Q = 40 * P   # apart from all that a call has by default
WS = dict(ws=P, ws_bytes=P)   # over X, dY or Y alone


def refusal(fn, d):
    assert getattr(lib, fn)(H, C.byref(d)) == INVALID
    return last_error()


APART = [(4, Q, Q + 4 * F, 2 * F), (4, Q + 4 * F, Q, 2 * F), (4, Q, Q + 4 * (F + 5), 2 * F + 5), (3, Q, Q + 4 * F, 3 * F),
         (3, Q + 8 * F, Q, 3 * F), (4, Q, Q + 4 * (3 * F), 2 * F)]
SHARED = [(4, Q, Q + 4 * F - 4, 2 * F), (4, Q, Q + 4 * F + 4, 2 * F), (4, Q, Q + 8 * F, 2 * F), (4, Q, Q, 2 * F),
          (4, Q + 4, Q, 2 * F), (4, Q, Q + 4 * F, 2 * F - 1)]


@pytest.mark.parametrize("N,z,u,ld", APART)
def test_halves_are_apart(N, z, u, ld):
    d = linear(N=N, Z=z, U=u, ldz=ld, ldu=ld, **WS)
    assert "ws overlaps X" in refusal("ah_linear", d)
    d = linear_grad(N=N, dU=z, U=u, lddu=ld, ldu=ld, **WS)
    assert "ws overlaps X" in refusal("ah_linear_grad", d)


@pytest.mark.parametrize("N,z,u,ld", SHARED)
def test_what_shares_a_byte_is_refused(N, z, u, ld):
    assert "Z overlaps U" in refusal("ah_linear", linear(N=N, Z=z, U=u, ldz=ld, ldu=ld, **WS))
    assert "dU overlaps U" in refusal("ah_linear_grad", linear_grad(N=N, dU=z, U=u, lddu=ld, ldu=ld, **WS))


def test_other_strides_between_one_another_are_refused():
    assert "Z overlaps U" in refusal("ah_linear", linear(Z=Q, U=Q + 4 * F, ldz=2 * F, ldu=4 * F))
    assert "Z overlaps bias" in refusal("ah_linear", linear(Z=Q, bias=Q + 4 * F, ldz=2 * F))


def test_strides_count_in_bytes():
    """An f32 array's rows beside an f16 one's, in rows of the same bytes."""
    d = linear_grad(dtype=L.AH_F16, dW=Q, lddw=24, W=Q + 32, ldw=48, D=8, ws=5 * P, ws_bytes=P)
    assert "ws overlaps dY" in refusal("ah_linear_grad", d)
    d = linear_grad(dtype=L.AH_F16, dW=Q, lddw=24, W=Q + 30, ldw=48, D=8, ws=5 * P, ws_bytes=P)
    assert "dW overlaps W" in refusal("ah_linear_grad", d)


def test_norms():
    assert "ws overlaps Y" in refusal("ah_residual_norm_grad", norm_grad(dY=Q, lddy=16, dH=Q + 32, lddh=16, **WS))
    assert "dH overlaps dY" in refusal("ah_residual_norm_grad", norm_grad(dY=Q, lddy=16, dH=Q + 28, lddh=16, **WS))
    assert "H_out overlaps O" in refusal("ah_residual_norm", norm(H_out=Q + 28, ldh_out=16, O=Q, ldo=16))
