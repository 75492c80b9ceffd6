"""Workspaces of ah_linear_ce: what they are made of, and what piece_mb bounds (CPU: the sizes need no device)."""
import ctypes as C

import pytest

from anneal_amd import _lib as L

lib = L.load()
_HANDLE = C.create_string_buffer(1 << 16)
P = 1 << 20   # addresses that are never read
MB = 1 << 20


def workspace(want, **kw):
    d = dict(dtype=L.AH_F16, grad_dtype=L.AH_F16, mean=1, X=P, W=2 * P, labels=4 * P, loss=5 * P, grad_scale=1.0)
    d.update(kw)
    for k in ("ldx", "ldw", "lddx", "lddw"):
        d.setdefault(k, d["D"])
    for i, k in enumerate(want):
        d[k] = (8 + i) * P
    n = C.c_int64()
    L.check(lib.ah_linear_ce_workspace(C.addressof(_HANDLE), C.byref(L.ah_linear_ce_desc(**d)), C.byref(n)))
    return n.value


@pytest.mark.parametrize("N,V", [(16384, 131072), (4096, 50304), (8192, 1000003)])
def test_the_loss_alone_keeps_two_floats_a_row_and_wave_tile(N, V):
    """128 classes a wave tile at these sizes, 8 bytes each; X's rows and a few words a row beside them."""
    assert workspace((), N=N, D=1024, V=V) <= N * (V + 255) // 128 * 8 + N * 1024 * 2 + 64 * N + 8 * MB


@pytest.mark.parametrize("dtype", [L.AH_F16, L.AH_F32], ids=["f16", "f32"])
@pytest.mark.parametrize("mb", [0, 64, 4096])
def test_piece_mb_bounds_the_statistics(mb, dtype):
    """8 million classes: as many rows as piece_mb holds statistics of (or 256). f32 operands are packed beside them; 256 MB of partial
    tiles at most."""
    N, D, V = 16384, 64, 8 << 20
    e = 1 if dtype == L.AH_F16 else 2
    packed = 2 * e * D * (N + (V + (1 << 17) if e == 2 else 0))
    bound = max((mb or 2048) * MB, 256 * V // 32 * 8) + packed + 64 * N + 256 * MB
    assert workspace((), N=N, D=D, V=V, dtype=dtype, grad_dtype=dtype, piece_mb=mb) <= bound


@pytest.mark.parametrize("dtype", [L.AH_F16, L.AH_F32], ids=["f16", "f32"])
@pytest.mark.parametrize("mb", [0, 512])
def test_a_bias_adds_a_64th_of_a_piece(mb, dtype):
    """db's partial sums are a float a class for 64 rows of the piece that is worked on, not of all rows."""
    kw = dict(N=1 << 20, D=64, V=131072, dtype=dtype, grad_dtype=dtype, piece_mb=mb)
    assert workspace(("dX", "dbias"), **kw) - workspace(("dX",), **kw) <= (mb or 2048) * MB // 64 + 4096
