"""Argument checks of ah_linear_ce, ah_orthogonalize and ah_muon_step: refused before any device work (no device needed; the
handle is a block of zeroed host memory that no refusal reads beyond)."""
import ctypes as C

import pytest

from anneal_amd import _lib as L

lib = L.load()
INVALID, UNSUPPORTED = 1, 3
_HANDLE = C.create_string_buffer(1 << 16)
H = C.addressof(_HANDLE)
P = 1 << 20   # an address that is never read


def last_error():
    return (lib.ah_last_error() or b"").decode()


def lce(**kw):
    # X, W, ... lie far apart
    d = dict(dtype=L.AH_F32, grad_dtype=L.AH_F32, N=4, D=8, V=16, mean=1, X=P, ldx=8, W=2 * P, ldw=8, bias=3 * P, labels=4 * P, loss=5 * P,
             rowloss=6 * P, lse=7 * P, dX=8 * P, lddx=8, dW=9 * P, lddw=8, dbias=10 * P, grad_scale=1.0, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    return L.ah_linear_ce_desc(**d)


LCE_BAD = [(dict(dtype=L.AH_BF16), UNSUPPORTED), (dict(grad_dtype=L.AH_I32), UNSUPPORTED), (dict(grad_dtype=L.AH_F16), UNSUPPORTED),
           (dict(N=0), INVALID), (dict(N=-3), INVALID), (dict(D=0), INVALID), (dict(V=0), INVALID), (dict(D=(1 << 20) + 1), INVALID),
           (dict(X=None), INVALID), (dict(W=None), INVALID), (dict(labels=None), INVALID), (dict(loss=None), INVALID),
           (dict(ldx=7), INVALID), (dict(ldw=-8), INVALID), (dict(lddx=7), INVALID), (dict(lddw=0), INVALID), (dict(ldw=1 << 41), INVALID),
           (dict(grad_scale=float("nan")), INVALID), (dict(grad_scale=float("inf")), INVALID), (dict(piece_mb=-1), INVALID),
           (dict(X=P + 2), INVALID), (dict(dX=8 * P + 1), INVALID), (dict(labels=4 * P + 2), INVALID)]
LCE_BAD_CALL = [(dict(ws=None), INVALID), (dict(ws=16 * P + 4), INVALID), (dict(ws_bytes=100), INVALID), (dict(dX=P), INVALID),
                (dict(dX=P + 64), INVALID), (dict(dW=2 * P), INVALID), (dict(dW=8 * P + 96), INVALID), (dict(rowloss=5 * P), INVALID),
                (dict(dbias=3 * P), INVALID), (dict(loss=16 * P + 64), INVALID), (dict(ws=2 * P - 1024), INVALID)]


@pytest.mark.parametrize("kw,code", LCE_BAD + LCE_BAD_CALL, ids=lambda v: str(v)[:40])
def test_linear_ce_refuses(kw, code):
    d = lce(**kw)
    assert lib.ah_linear_ce(H, C.byref(d)) == code and "ah_linear_ce" in last_error()
    n = C.c_int64(-1)
    if (kw, code) in LCE_BAD:
        assert lib.ah_linear_ce_workspace(H, C.byref(d), C.byref(n)) == code and n.value == -1
    else:
        assert lib.ah_linear_ce_workspace(H, C.byref(d), C.byref(n)) == 0 and n.value > 0


def orth(**kw):
    d = dict(dtype=L.AH_F32, out_dtype=L.AH_F32, rows=8, cols=16, batch=2, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, G=P, ldg=16, stride_g=128,
             O=2 * P, ldo=16, stride_o=128, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    return L.ah_orthogonalize_desc(**d)


NS_BAD = [(dict(dtype=L.AH_BF16), UNSUPPORTED), (dict(rows=0), INVALID), (dict(cols=-1), INVALID), (dict(batch=0), INVALID), (dict(batch=65536), INVALID),
          (dict(rows=(1 << 20) + 1), INVALID), (dict(steps=0), INVALID), (dict(steps=65), INVALID), (dict(a=20.0), INVALID), (dict(b=float("nan")), INVALID),
          (dict(eps=-1.0), INVALID), (dict(eps=float("inf")), INVALID), (dict(G=None), INVALID), (dict(ldg=15), INVALID), (dict(stride_g=-1), INVALID),
          (dict(G=P + 1), INVALID)]
ORTH_BAD = NS_BAD + [(dict(out_dtype=L.AH_U32), UNSUPPORTED), (dict(O=None), INVALID), (dict(ldo=15), INVALID), (dict(stride_o=127), INVALID)]
ORTH_BAD_CALL = [(dict(ws=None), INVALID), (dict(ws_bytes=64), INVALID), (dict(ws=P), INVALID), (dict(O=16 * P + 256), INVALID)]


@pytest.mark.parametrize("kw,code", ORTH_BAD + ORTH_BAD_CALL, ids=lambda v: str(v)[:40])
def test_orthogonalize_refuses(kw, code):
    d = orth(**kw)
    assert lib.ah_orthogonalize(H, C.byref(d)) == code and "ah_orthogonalize" in last_error()
    n = C.c_int64(-1)
    assert lib.ah_orthogonalize_workspace(H, C.byref(d), C.byref(n)) == (code if (kw, code) in ORTH_BAD else 0)


def muon(**kw):
    d = dict(dtype=L.AH_F32, rows=8, cols=16, batch=2, steps=5, nesterov=1, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, G=P, ldg=16, stride_g=128, M=2 * P,
             M_out=3 * P, W=4 * P, W_out=5 * P, W16_out=6 * P, ldw=16, stride_w=128, lr=0.1, momentum=0.9, decay=0.0, scale=1.0, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    return L.ah_muon_desc(**d)


MUON_BAD = NS_BAD + [(dict(M=None), INVALID), (dict(M_out=None), INVALID), (dict(W=None), INVALID), (dict(W_out=None), INVALID), (dict(ldw=15), INVALID),
                     (dict(stride_w=100), INVALID), (dict(lr=float("nan")), INVALID), (dict(momentum=float("inf")), INVALID),
                     (dict(decay=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(W16_out=6 * P + 1), INVALID)]
MUON_BAD_CALL = [(dict(ws=None), INVALID), (dict(ws_bytes=64), INVALID), (dict(M_out=P), INVALID), (dict(M_out=2 * P + 64), INVALID),
                 (dict(W_out=4 * P + 4), INVALID), (dict(W_out=3 * P), INVALID), (dict(W16_out=5 * P), INVALID), (dict(W_out=2 * P), INVALID)]


@pytest.mark.parametrize("kw,code", MUON_BAD + MUON_BAD_CALL, ids=lambda v: str(v)[:40])
def test_muon_step_refuses(kw, code):
    d = muon(**kw)
    assert lib.ah_muon_step(H, C.byref(d)) == code and "ah_muon_step" in last_error()
    n = C.c_int64(-1)
    assert lib.ah_muon_workspace(H, C.byref(d), C.byref(n)) == (code if (kw, code) in MUON_BAD else 0)


def test_null_arguments():
    n = C.c_int64()
    for call, size, d in ((lib.ah_linear_ce, lib.ah_linear_ce_workspace, lce()), (lib.ah_orthogonalize, lib.ah_orthogonalize_workspace, orth()),
                          (lib.ah_muon_step, lib.ah_muon_workspace, muon())):
        assert call(None, C.byref(d)) == INVALID and call(H, None) == INVALID
        assert size(None, C.byref(d), C.byref(n)) == INVALID and size(H, None, C.byref(n)) == INVALID and size(H, C.byref(d), None) == INVALID
