"""Argument checks of ah_linear, ah_linear_grad, ah_residual_norm, ah_residual_norm_grad and ah_clip_norm: refused before any device work (no
device needed; the handle is a block of zeroed host memory that no refusal reads beyond), and their descriptors' layouts."""
import ctypes as C
import os
import subprocess

import pytest

from anneal_amd import _lib as L

lib = L.load()
INVALID, UNSUPPORTED = 1, 3
_HANDLE = C.create_string_buffer(1 << 16)
H = C.addressof(_HANDLE)
P = 1 << 20   # an address that is never read
FAR = 1 << 40
NAN, INF = float("nan"), float("inf")


def last_error():
    return (lib.ah_last_error() or b"").decode()


def linear(**kw):
    d = dict(dtype=L.AH_F32, act=L.ACT_GELU, N=4, D=8, F=16, scale=1.0, X=P, ldx=8, W=2 * P, ldw=8, bias=3 * P, U=4 * P, ldu=16, R=5 * P, ldr=16, Y=6 * P,
             ldy=16, Z=7 * P, ldz=16, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    return L.ah_linear_desc(**d)


def linear_grad(**kw):
    d = dict(dtype=L.AH_F32, grad_dtype=L.AH_F32, act=L.ACT_GELU, N=4, D=8, F=16, scale=1.0, X=P, ldx=8, W=2 * P, ldw=8, Z=3 * P, ldz=16, U=4 * P, ldu=16,
             dY=5 * P, lddy=16, dX=6 * P, lddx=8, dW=7 * P, lddw=8, dbias=8 * P, dU=9 * P, lddu=16, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    return L.ah_linear_grad_desc(**d)


def norm(**kw):
    d = dict(dtype=L.AH_F32, res_dtype=L.AH_F32, N=6, D=8, post=L.NORM_LAYER, pre=L.NORM_LAYER, rows_per_gate=2, eps=1e-6, skip=1.0, scale=1.0, H=P, ldh=8,
             Y=2 * P, ldy=8, gate=3 * P, ldgate=8, post_w=4 * P, post_b=5 * P, pre_w=6 * P, pre_b=7 * P, H_out=8 * P, ldh_out=8, O=9 * P, ldo=8)
    d.update(kw)
    return L.ah_residual_norm_desc(**d)


def norm_grad(**kw):
    d = dict(dtype=L.AH_F32, res_dtype=L.AH_F32, N=6, D=8, post=L.NORM_LAYER, pre=L.NORM_LAYER, rows_per_gate=2, eps=1e-6, skip=1.0, scale=1.0, Y=P, ldy=8,
             gate=2 * P, ldgate=8, post_w=3 * P, post_b=4 * P, pre_w=5 * P, H_out=6 * P, ldh_out=8, dH_out=7 * P, lddh_out=8, dO=8 * P, lddo=8, dH=9 * P,
             lddh=8, dY=10 * P, lddy=8, dgate=11 * P, lddgate=8, dpost_w=12 * P, dpost_b=13 * P, dpre_w=14 * P, dpre_b=15 * P, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    return L.ah_residual_norm_grad_desc(**d)


LINEAR = [(dict(dtype=L.AH_BF16), UNSUPPORTED), (dict(act=5), UNSUPPORTED), (dict(act=-1), UNSUPPORTED), (dict(N=0), INVALID), (dict(N=(1 << 21) + 1), INVALID),
          (dict(D=0), INVALID), (dict(F=-1), INVALID), (dict(F=(1 << 20) + 1), INVALID), (dict(D=(1 << 20) + 1), INVALID), (dict(scale=NAN), INVALID),
          (dict(X=P + 2), INVALID), (dict(ldx=7), INVALID), (dict(ldw=-8), INVALID), (dict(ldu=15), INVALID), (dict(ldx=FAR + 1), INVALID),
          (dict(N=1 << 21, ldx=FAR), INVALID)]
LINEAR_BAD = LINEAR + [(dict(X=None), INVALID), (dict(W=None), INVALID), (dict(Y=None), INVALID), (dict(ldr=15), INVALID), (dict(ldy=15), INVALID),
                       (dict(ldz=0), INVALID), (dict(bias=3 * P + 1), INVALID), (dict(Z=7 * P + 2), INVALID)]
LINEAR_CALL = [(dict(ws=None), INVALID), (dict(ws=16 * P + 4), INVALID), (dict(ws_bytes=8), INVALID), (dict(ws=P), INVALID), (dict(ws=6 * P + 64), INVALID),
               (dict(Y=P), INVALID), (dict(Y=7 * P), INVALID), (dict(Y=5 * P + 64), INVALID), (dict(Y=5 * P, ldy=32), INVALID), (dict(Z=5 * P), INVALID),
               (dict(Z=4 * P + 16), INVALID), (dict(Y=3 * P), INVALID)]
LINEAR_GRAD_BAD = LINEAR + [(dict(grad_dtype=L.AH_F16), UNSUPPORTED), (dict(grad_dtype=L.AH_I32), UNSUPPORTED), (dict(dY=None), INVALID),
                            (dict(dX=None, dW=None, dbias=None, dU=None), INVALID), (dict(W=None), INVALID), (dict(X=None), INVALID), (dict(U=None), INVALID),
                            (dict(Z=None), INVALID), (dict(Z=None, act=0), INVALID), (dict(lddy=15), INVALID), (dict(lddx=7), INVALID), (dict(lddw=7), INVALID),
                            (dict(lddu=15), INVALID), (dict(dbias=8 * P + 2), INVALID)]
LINEAR_GRAD_CALL = [(dict(ws=None), INVALID), (dict(ws_bytes=64), INVALID), (dict(dX=P), INVALID), (dict(dW=2 * P), INVALID), (dict(dU=5 * P), INVALID),
                    (dict(dbias=7 * P + 32), INVALID), (dict(dX=7 * P), INVALID), (dict(ws=3 * P), INVALID)]
NORM = [(dict(dtype=L.AH_I32), UNSUPPORTED), (dict(res_dtype=L.AH_F16), UNSUPPORTED), (dict(post=3), UNSUPPORTED), (dict(pre=-1), UNSUPPORTED), (dict(N=0), INVALID),
        (dict(N=(1 << 27) + 1), INVALID), (dict(D=0), INVALID), (dict(D=(1 << 20) + 1), INVALID), (dict(rows_per_gate=-1), INVALID), (dict(eps=-1e-9), INVALID),
        (dict(eps=INF), INVALID), (dict(skip=NAN), INVALID), (dict(scale=INF), INVALID), (dict(ldy=7), INVALID), (dict(ldgate=7), INVALID), (dict(ldh_out=0), INVALID),
        (dict(Y=P + 3), INVALID), (dict(N=1 << 27, ldy=FAR), INVALID), (dict(post=L.NORM_NONE), INVALID), (dict(post=L.NORM_RMS), INVALID),
        (dict(pre=L.NORM_RMS), INVALID), (dict(pre=L.NORM_NONE), INVALID)]
NORM_BAD = NORM + [(dict(H=None, Y=None), INVALID), (dict(Y=None), INVALID), (dict(Y=None, gate=None), INVALID), (dict(O=None), INVALID),
                   (dict(O=None, H_out=None, pre=L.NORM_NONE, pre_w=None, pre_b=None), INVALID), (dict(pre=L.NORM_NONE, pre_w=None, pre_b=None), INVALID),
                   (dict(O=P), INVALID), (dict(H_out=2 * P), INVALID), (dict(H_out=P, ldh_out=16), INVALID), (dict(H_out=P + 32), INVALID),
                   (dict(O=8 * P + 64), INVALID), (dict(O=2 * P), INVALID), (dict(O=3 * P + 64), INVALID), (dict(H_out=5 * P), INVALID)]
NORM_GRAD_BAD = NORM + [(dict(dO=None), INVALID), (dict(H_out=None), INVALID), (dict(Y=None), INVALID), (dict(post=0, post_w=None, post_b=None), INVALID),
                        (dict(dH=None, dY=None, dgate=None, dpost_w=None, dpost_b=None, dpre_w=None, dpre_b=None), INVALID),
                        (dict(pre=0, pre_w=None, dpre_w=None, dpre_b=None), INVALID), (dict(pre=0, pre_w=None, dpre_w=None, dpre_b=None, dO=None, dH_out=None), INVALID),
                        (dict(lddh=7), INVALID), (dict(lddgate=7), INVALID), (dict(dpre_b=15 * P + 1), INVALID)]
NORM_GRAD_CALL = [(dict(ws=None), INVALID), (dict(ws_bytes=8), INVALID), (dict(dH=7 * P + 32), INVALID), (dict(dH=7 * P, lddh=9), INVALID), (dict(dY=8 * P), INVALID),
                  (dict(dY=P), INVALID), (dict(dgate=2 * P + 64), INVALID), (dict(dpre_w=15 * P), INVALID), (dict(ws=9 * P), INVALID)]
CASES = {"ah_linear": (linear, LINEAR_BAD, LINEAR_CALL), "ah_linear_grad": (linear_grad, LINEAR_GRAD_BAD, LINEAR_GRAD_CALL),
         "ah_residual_norm": (norm, NORM_BAD, []), "ah_residual_norm_grad": (norm_grad, NORM_GRAD_BAD, NORM_GRAD_CALL)}


@pytest.mark.parametrize("fn,kw,code,size", [(f, k, c, True) for f, (_, bad, _) in CASES.items() for k, c in bad] +
                         [(f, k, c, False) for f, (_, _, call) in CASES.items() for k, c in call], ids=lambda v: str(v)[:40])
def test_refuses(fn, kw, code, size):
    """size: the workspace call refuses it too."""
    d = CASES[fn][0](**kw)
    assert getattr(lib, fn)(H, C.byref(d)) == code and fn in last_error(), last_error()
    if fn != "ah_residual_norm":
        n = C.c_int64(-1)
        assert getattr(lib, fn + "_workspace")(H, C.byref(d), C.byref(n)) == (code if size else 0)
        assert (n.value == -1) == size


def clip(tensors=None, **kw):
    t = [(P, 2 * P, 100, 0, 0), (3 * P, 4 * P, 50, 1, 0), (5 * P, 5 * P, 7, 1, 1), (6 * P, None, 9, 0, 0)] if tensors is None else tensors
    a = (L.ah_tensor * max(1, len(t)))(*t)
    d = dict(n=len(t), max_norm=1.0, eps=1e-6, unscale=1.0, tensors=C.addressof(a), norm=7 * P, coef=8 * P, ws=16 * P, ws_bytes=1 << 30)
    d.update(kw)
    out = L.ah_clip_desc(**d)
    out.keep = a
    return out


CLIP_BAD = [(dict(n=0), INVALID), (dict(n=-1), INVALID), (dict(n=(1 << 16) + 1), INVALID), (dict(tensors=[]), INVALID), (dict(max_norm=-1.0), INVALID),
            (dict(max_norm=NAN), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=INF), INVALID), (dict(unscale=0.0), INVALID), (dict(unscale=-1.0), INVALID),
            (dict(unscale=INF), INVALID), (dict(unscale=NAN), INVALID), (dict(norm=7 * P + 2), INVALID), (dict(coef=8 * P + 1), INVALID),
            (dict(tensors=[(P, 2 * P, -1, 0, 0)]), INVALID), (dict(tensors=[(None, 2 * P, 1, 0, 0)]), INVALID), (dict(tensors=[(P + 2, 2 * P, 1, 0, 0)]), INVALID),
            (dict(tensors=[(P, 2 * P + 1, 1, 1, 1)]), INVALID), (dict(tensors=[(P, 2 * P, 1, 0, 1)]), UNSUPPORTED), (dict(tensors=[(P, 2 * P, 1, 2, 0)]), UNSUPPORTED),
            (dict(tensors=[(P, 2 * P, 1, 0, 3)]), UNSUPPORTED), (dict(tensors=[(P, None, 1 << 40, 0, 0), (2 * P, None, 1, 0, 0)]), INVALID)]
CLIP_CALL = [(dict(ws=None), INVALID), (dict(ws=16 * P + 8), INVALID), (dict(ws_bytes=16), INVALID), (dict(tensors=[(P, P + 4, 100, 0, 0)]), INVALID),
             (dict(tensors=[(P, P, 100, 1, 0)]), INVALID), (dict(tensors=[(P, 2 * P, 100, 0, 0), (3 * P, 2 * P + 396, 1, 0, 0)]), INVALID),
             (dict(tensors=[(P, P, 100, 0, 0), (P, P, 100, 0, 0)]), INVALID), (dict(tensors=[(P, P, 100, 0, 0), (P + 40, None, 3, 0, 0)]), INVALID),
             (dict(norm=2 * P + 8), INVALID), (dict(norm=8 * P), INVALID), (dict(norm=P + 16), INVALID), (dict(ws=4 * P), INVALID)]


@pytest.mark.parametrize("kw,code", CLIP_BAD + CLIP_CALL, ids=lambda v: str(v)[:50])
def test_clip_norm_refuses(kw, code):
    d = clip(**kw)
    assert lib.ah_clip_norm(H, C.byref(d)) == code and "ah_clip_norm" in last_error()
    n = C.c_int64(-1)
    assert lib.ah_clip_norm_workspace(H, C.byref(d), C.byref(n)) == (code if (kw, code) in CLIP_BAD else 0)


def test_null_arguments():
    n = C.c_int64()
    for fn, d in (("ah_linear", linear()), ("ah_linear_grad", linear_grad()), ("ah_residual_norm", norm()), ("ah_residual_norm_grad", norm_grad()),
                  ("ah_clip_norm", clip())):
        call = getattr(lib, fn)
        assert call(None, C.byref(d)) == INVALID and call(H, None) == INVALID
        if fn != "ah_residual_norm":
            size = getattr(lib, fn + "_workspace")
            assert size(None, C.byref(d), C.byref(n)) == INVALID and size(H, None, C.byref(n)) == INVALID and size(H, C.byref(d), None) == INVALID


def test_workspaces_grow_with_what_is_asked_for():
    def size(fn, d):
        n = C.c_int64()
        L.check(getattr(lib, fn + "_workspace")(H, C.byref(d), C.byref(n)))
        return n.value
    big = dict(N=4096, D=1024, F=4096, ldx=1024, ldw=1024, ldu=4096)
    f16 = size("ah_linear", linear(dtype=L.AH_F16, ldr=4096, ldy=4096, ldz=4096, **big))
    f32 = size("ah_linear", linear(ldr=4096, ldy=4096, ldz=4096, **big))
    assert f16 <= 64 << 20 and (4096 + 4096) * 1024 * 4 <= f32 <= f16 + (65 << 20)   # aligned f16 rows are read as they lie
    g = dict(ldz=4096, lddy=4096, lddx=1024, lddw=1024, lddu=4096, **big)
    only = size("ah_linear_grad", linear_grad(dX=None, dW=None, **g))
    assert only < 2 << 20 <= 4096 * 4096 * 4 <= size("ah_linear_grad", linear_grad(**g))
    assert size("ah_clip_norm", clip()) <= 1 << 15


@pytest.mark.parametrize("name", ["ah_linear_desc", "ah_linear_grad_desc", "ah_residual_norm_desc", "ah_residual_norm_grad_desc", "ah_tensor", "ah_clip_desc"])
def test_ctypes_mirror_matches_the_c_header(tmp_path, name):
    cls = getattr(L, name)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "anneal_hip.h"\nint main(void) {\n    printf("%zu\\n", sizeof(' + name + "));\n" +
                   "".join(f'    printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]
