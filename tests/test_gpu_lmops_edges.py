"""Single roundings, limits and rare states of ah_linear_ce, ah_orthogonalize and ah_muon_step (GPU). Tolerances as in
test_gpu_linear_ce.py and test_gpu_muon.py where none is derived here."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_linear_ce as TL
import test_gpu_lmops_run as TR
import test_gpu_muon as TM
from anneal_amd import _lib as L

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -11, 2.0 ** -24


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("D,N", [(64, 1), (64, 140), (72, 3), (65, 2)])
def test_f16_gradients_round_p_once(dev, D, N, bias):
    """dW of one row of powers of two: row v is s P_v X exactly, and P_v in f16 needs no second rounding on the way out. So it is within
    half a step of f16 of s P_v X; two roundings would be up to a whole step off. Logits below 4 in f32 move P by (D/32 + 40) U32 * 16."""
    V = 3000
    c = TL.Case(N, D, V, dtype=L.AH_F16, grad_dtype=L.AH_F16, bias=bias, labels=[7] + [-1] * (N - 1))
    c.X[:] = np.where(c.X < 0, -0.5, 0.5)
    got = TL.run(dev, c, want=("loss", "dX", "dW") + (("dbias",) if bias else ()), grad_scale=2.0 ** 12)
    X = c.X[0].astype(np.float64)
    z = c.W.astype(np.float64) @ X + (c.b.astype(np.float64) if bias else 0.0)
    P = np.exp(z - z.max())
    P /= P.sum()
    P[7] -= 1.0
    want = 2.0 ** 12 * P[:, None] * X
    assert np.abs(want).min() > 2.0 ** -14   # f16 has its full 11 bits
    tol = (U16 + (D / 32 + 40) * U32 * 16) * np.abs(want)
    worst = np.abs(got["dW"] - want) / tol
    assert worst.max() <= 1.0, worst.max()


# rows, features, classes, and pieces of how many MiB: tiles of 64 features and more, either sum split, few rows of unaligned W, pieces
LABELLED = [(130, 64, 1000, 0), (777, 96, 3003, 0), (2, 41, 300, 0), (100, 65, 2049, 0), (2500, 64, 200, 0), (150, 264, 20011, 0), (900, 130, 2100, 1),
            (3000, 520, 5003, 0)]


@pytest.mark.parametrize("labels", ["uniform", "few", "one"])
@pytest.mark.parametrize("shape", LABELLED, ids=lambda s: "%dx%dx%d_%d" % s)
def test_f16_gradients_keep_p_at_the_label(dev, shape, labels):
    """P at the label is the largest entry of most rows. It takes part with 22 bits, as f16 and what that leaves, so a gradient is off
    by its own rounding, by U16 of the other entries' share, and by f32 sums: with P at the label in f16 alone it is up to twice as far."""
    N, D, V, mb = shape
    r = np.random.default_rng([N, D])
    y = {"uniform": r.integers(0, V, N), "few": np.exp(r.uniform(0, np.log(V), N)).astype(int) - 1, "one": np.full(N, V // 2)}[labels]
    if N > 2:
        y[r.random(N) < 0.2] = -1
    c = TL.Case(N, D, V, dtype=L.AH_F16, grad_dtype=L.AH_F16, labels=y, bias=False)
    s = 2.0 ** 10
    got = TL.run(dev, c, want=("loss", "dX", "dW"), mean=False, grad_scale=s, piece_mb=mb)
    X, W, on = c.X.astype(np.float64), c.W.astype(np.float64), np.flatnonzero(y >= 0)
    X = X[on]
    z = X @ W.T
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    at = np.arange(len(on)), y[on]
    dz = (np.abs(X) @ np.abs(W).T).max(1, keepdims=True) * (D / 32 + 32) * U32
    dP = p * (3 * dz + (V / 64 + 40) * U32 + 2.0 ** -20) + U16 * p   # the logits, the statistics, exp; f16
    P = p.copy()
    P[at] -= 1.0
    dP[at] = p[at] * (3 * dz[:, 0] + (V / 64 + 40) * U32 + 2.0 ** -20) + 2.0 ** -21 * np.abs(P[at])
    dP += 2.0 ** -39
    pieces = 4 if mb else 1
    for name, a, da, b in (("dX", P, dP, W), ("dW", P.T, dP.T, X)):
        want = a @ b * s
        tol = s * (da @ np.abs(b) + (a.shape[1] / 32 + 32 * pieces) * U32 * (np.abs(a) @ np.abs(b))) + U16 * 1.01 * np.abs(want) + 2.0 ** -25
        g = got[name][on] if name == "dX" else got[name]
        over = np.abs(want) > 65504 - tol   # past f16's range (many rows of one label): infinite, or the largest value
        assert np.all(np.sign(g[over]) == np.sign(want[over])) and np.all(np.abs(g[over]) >= np.minimum(np.abs(want), 65504)[over] - tol[over])
        worst = np.where(over, 0.0, np.abs(np.where(over, 0.0, g) - want) / tol)
        assert worst.max() <= 1.0, (name, worst.max(), np.argwhere(worst > 1)[:4].tolist())


# ── more rows or classes than one array of panels holds ────────────────────────

def _repeated(dev, base, rows, dtype=L.AH_F32):
    """Device memory of `rows` rows, row r that of base's r % len(base)."""
    b = dev.buffer(rows * base.shape[1], dtype)
    chunk = np.ascontiguousarray(np.tile(base.astype(TL.NP[dtype]), (256, 1)))
    for r in range(0, rows, len(chunk)):
        n = min(len(chunk), rows - r) * base.shape[1] * chunk.itemsize
        L.check(dev.lib.ah_upload_bytes(dev.h, b.ptr + r * base.shape[1] * chunk.itemsize, chunk.ctypes.data, n))
    return b


def _run(dev, **args):
    ws = dev.buffer(dev.linear_ce_workspace(**args) // 4 + 4)
    dev.linear_ce(ws=ws, **args)
    dev.sync()
    ws.free()


@pytest.mark.parametrize("dtype,N,D,V", [(L.AH_F32, 2048, 256, 5_000_000), (L.AH_F16, 300, 257, 4_300_003)], ids=["f32", "f16"])
def test_millions_of_classes(dev, dtype, N, D, V):
    """Packed W of more rows than a tile's 32-bit offsets span, with 256-wide tiles of dX in the f32 case: loss and dX against 64 bits. W
    repeats 1021 rows, so that the sums over classes are short here. A row's P is off by a share e of it, from its logit and the
    statistics, and dX by e |P| |W| and by f32 sums over V / splits, splits >= 8."""
    r = np.random.default_rng(V)
    base, X = (D ** -0.5 * r.standard_normal((1021, D))).astype(TL.NP[dtype]), r.standard_normal((N, D)).astype(TL.NP[dtype])
    y = r.integers(0, V, N).astype(np.int32)
    s, u16 = (1024.0, U16) if dtype == L.AH_F16 else (1.0, 0.0)
    b = {"X": dev.buffer(X, dtype), "W": _repeated(dev, base, V, dtype), "labels": dev.buffer(y, L.AH_I32), "loss": dev.buffer(1), "rowloss": dev.buffer(N),
         "dX": dev.buffer(N * D, dtype)}
    _run(dev, dtype=dtype, grad_dtype=dtype, N=N, D=D, V=V, mean=False, grad_scale=s, piece_mb=48000, **b)
    rowloss, dX = b["rowloss"].read(), b["dX"].read().reshape(N, D).astype(np.float64)
    for v in b.values():
        v.free()
    X, base = X.astype(np.float64), base.astype(np.float64)
    z = X @ base.T
    times = np.bincount(np.arange(V) % 1021, minlength=1021)
    m = z.max(1, keepdims=True)
    lse = m + np.log((np.exp(z - m) * times).sum(1, keepdims=True))
    want = lse[:, 0] - z[np.arange(N), y % 1021]
    dz = (np.abs(X) @ np.abs(base).T).max(1) * ((3 * 2.0 ** -22 if dtype == L.AH_F32 else 0.0) + (D / 32 + 32) * U32)
    # V / 128 = 39063 wave tiles, joined by a wave in chains of 610 f32 sums; lse is up to 18
    dlse = dz + (640 + 64 + 40) * U32 + 18 * 2 * U32
    assert np.all(np.abs(rowloss - want) <= dlse + dz + 20 * U32)
    p = np.exp(z - lse) * times   # the repeated rows' P, summed
    own = base[y % 1021]
    e = 2 * dz + dlse + 2.0 ** -20 + (V / 8 / 32 + 64) * U32
    want = p @ base - own
    tol = (e + u16)[:, None] * (p @ np.abs(base)) + (e + 2.0 ** -20)[:, None] * np.abs(own) + 2.0 ** -39 * np.abs(base).sum(0) * V / 1021
    off = np.abs(dX - s * want) / (s * (tol + (u16 + 2 * U32) * 1.01 * np.abs(want)) + 2.0 ** -25)
    assert off.max() <= 1.0, off.max()


def test_millions_of_rows(dev):
    """dW over 5 million packed rows of X in pieces, with 256-wide tiles, against 64 bits; X repeats 1021 rows. e as above; f32 sums over a
    piece's 262144 rows in at least 8 splits, and over 20 pieces."""
    N, D, V = 5_000_000, 256, 2048
    r = np.random.default_rng(N)
    W, base = (D ** -0.5 * r.standard_normal((V, D))).astype(np.float32), r.standard_normal((1021, D)).astype(np.float32)
    y = (np.arange(N, dtype=np.int64) * 7 % V).astype(np.int32)
    b = {"X": _repeated(dev, base, N), "W": dev.buffer(W), "labels": dev.buffer(y, L.AH_I32), "loss": dev.buffer(1), "dW": dev.buffer(V * D)}
    _run(dev, dtype=L.AH_F32, N=N, D=D, V=V, mean=False, **b)
    loss, dW = float(b["loss"].read()[0]), b["dW"].read().reshape(V, D).astype(np.float64)
    for v in b.values():
        v.free()
    base, W = base.astype(np.float64), W.astype(np.float64)
    z = base @ W.T
    m = z.max(1, keepdims=True)
    lse = m + np.log(np.exp(z - m).sum(1, keepdims=True))
    kind = np.arange(N) % 1021
    times = np.bincount(kind, minlength=1021)
    pairs = np.bincount(kind * V + y, minlength=1021 * V).reshape(1021, V).astype(np.float64)   # rows of each kind with each label
    dz = float((np.abs(base) @ np.abs(W).T).max()) * (3 * 2.0 ** -22 + (D / 32 + 32) * U32)
    total = (times * lse[:, 0]).sum() - (pairs * z).sum()
    assert abs(loss - total) <= N * (2 * dz + 80 * U32 + 16 * 2 * U32) + 2 * U32 * total
    p = np.exp(z - lse)
    e = 3 * dz + 2.0 ** -19 + (262144 / 8 / 32 + 64 + 20) * U32
    want = (p * times[:, None] - pairs).T @ base
    off = np.abs(dW - want) / (e * ((p * times[:, None] + pairs).T @ np.abs(base)) + 2.0 ** -39 * N)
    assert off.max() <= 1.0, off.max()


# ── polynomials whose iterates come near the largest singular value that is allowed, 4 ──

FAR = [(2, (4.15, -1.25, 0.1)), (2, (3.375, -0.375, 0.0)), (3, (3.375, -0.375, 0.0)), (2, (4.0, 0.0, 0.0)), (2, (-4.0, 0.0, 0.0)), (2, (2.0, 1.0, 1.0)),
       (2, (14.0, -0.5, 0.5))]


@pytest.mark.parametrize("shape", [(1, 1), (20, 30), (50, 90), (130, 100), (280, 260), (300, 700), (640, 300)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("steps,coef", FAR, ids=str)
@pytest.mark.parametrize("axis", [False, True], ids=["", "axis"])
def test_singular_values_up_to_4(dev, shape, steps, coef, axis):
    """A single value, which starts at 1, and matrices with one strong direction, spread out or along an axis (where one entry of the Gram
    matrix has all of its eigenvalue). The bound is iterate()'s, with (14, -0.5, 0.5) after one
    step at 14, which only the last iterate may be."""
    if coef[0] == 14.0:
        steps = 1
    r = np.random.default_rng(shape)
    G = np.outer(r.standard_normal(shape[0]), r.standard_normal(shape[1])) + 0.02 * r.standard_normal(shape)
    if axis:
        G = 1e-4 * r.standard_normal(shape)
        G[shape[0] // 2, shape[1] // 3] = 1.0
    G = G.astype(np.float32)
    want, err = TM.iterate(G.astype(np.float64), steps, coef)
    a, b, c = coef
    s = np.linalg.svd(G.astype(np.float64), compute_uv=False)
    s = s / np.linalg.norm(s)
    for _ in range(steps - 1):
        s = a * s + b * s ** 3 + c * s ** 5
        assert np.abs(s).max() <= 4.0
    got = TM.ortho(dev, G, L.AH_F32, steps=steps, coef=coef)[0]
    assert np.linalg.norm(got - want) <= err + U32 * np.linalg.norm(want), (np.linalg.norm(got - want), err, np.linalg.norm(want))


# ── zero and tiny matrices ─────────────────────────────────────────────────────

@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-36, 1e-7])
@pytest.mark.parametrize("shape", [(1, 1), (40, 70), (128, 300), (300, 280), (700, 300)], ids=lambda s: "%dx%d" % s)
def test_zero_matrices_and_tiny_ones_in_a_batch(dev, shape, eps):
    """Zero stays zero without a norm to divide by, beside others, and values of 2^-130 and less, whose norm's inverse passes f32's range, are
    orthogonalised as they are. Planes end at 2^-24 of values scaled by 2^12: X is off by 2^-37 an entry where eps leaves it that small, and
    five steps raise that by at most 3.4445^5 = 485."""
    r = np.random.default_rng(shape)
    big = TM.gradient(r, *shape, L.AH_F32)
    tiny = (big * np.float32(2.0 ** -60)) * np.float32(2.0 ** -60)
    G = np.stack([big, 0 * big, tiny, 0 * big])
    assert 0 < np.abs(tiny).max() < 2.0 ** -120
    got = TM.ortho(dev, G, L.AH_F32, eps=eps)
    assert not got[1].any() and not got[3].any()
    for z in (0, 2):
        want, err = TM.iterate(G[z].astype(np.float64), eps=eps)
        assert np.linalg.norm(got[z] - want) <= err + U32 * np.linalg.norm(want) + 485 * 2.0 ** -37 * want.size ** 0.5, z


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (40, 70), (300, 128), (300, 280)], ids=lambda s: "%dx%d" % s)
def test_a_matrix_that_is_not_finite_is_nan_alone(dev, shape, bad):
    G = np.stack([TM.gradient(np.random.default_rng([z, *shape]), *shape, L.AH_F32) for z in range(3)])
    alone = [TM.ortho(dev, g, L.AH_F32)[0] for g in G]
    G[1, shape[0] // 2, shape[1] // 3] = bad
    got = TM.ortho(dev, G, L.AH_F32)
    assert np.isnan(got[1]).all()
    for z in (0, 2):
        np.testing.assert_allclose(got[z], alone[z], rtol=0, atol=2e-5 * np.linalg.norm(alone[z]))


@pytest.mark.parametrize("eps", [0.0, 1e-45])
@pytest.mark.parametrize("shape", [(64, 100), (300, 280)], ids=lambda s: "%dx%d" % s)
def test_a_step_without_a_gradient_decays_the_weights(dev, shape, eps):
    W = np.random.default_rng(3).standard_normal(shape).astype(np.float32)
    bG, bM, bW, b16 = dev.buffer(np.zeros(shape, np.float32)), dev.buffer(np.zeros(shape, np.float32)), dev.buffer(W), dev.buffer(W.size, L.AH_F16)
    args = dict(dtype=L.AH_F32, rows=shape[0], cols=shape[1], G=bG, M=bM, W=bW, W16_out=b16, lr=0.125, decay=0.5, eps=eps)
    ws = dev.buffer(dev.muon_step_workspace(**args) // 4 + 4)
    dev.muon_step(ws=ws, **args)
    dev.sync()
    want = np.float32(1 - 0.125 * 0.5) * W
    np.testing.assert_array_equal(bW.read().reshape(shape), want)
    np.testing.assert_array_equal(b16.read().reshape(shape), want.astype(np.float16))
    assert not bM.read().any()
    for b in (bG, bM, bW, b16, ws):
        b.free()


# ── a key's workspace, which all of its launches share ─────────────────────────

def _traps(dev, mib):
    """Memory of the sizes that a workspace may have left behind, filled with NaN."""
    return [dev.buffer(np.full(m << 18, np.nan, np.float32)) for m in mib]


def _untouched(traps):
    for t in traps:
        assert np.isnan(t.read()).all()
        t.free()


def test_plans_of_one_key_with_other_batches(dev):
    """A second plan's larger batch moves the workspace that the first one's graph holds."""
    key = dict(dtype=L.AH_F32, bias=True)
    small, large = TL.Case(70, 47, 530, **key), TL.Case(900, 47, 530, **key)
    item = TR._head_item(small, sym=True)[0]
    plans = [TR.Plan(dev, [item], graph=True) for _ in range(2)]
    TL.compare(TR._head_values(small, plans[0].run(TR._head_item(small)[1], {"n": 70})), small.exact())
    TL.compare(TR._head_values(large, plans[1].run(TR._head_item(large)[1], {"n": 900})), large.exact())
    traps = _traps(dev, (1, 1, 2, 2, 4))
    for seed in (1, 2):
        c = TL.Case(70, 47, 530, seed=seed, **key)
        TL.compare(TR._head_values(c, plans[0].run(TR._head_item(c)[1], {"n": 70})), c.exact())
    TL.compare(TR._head_values(large, plans[1].run(TR._head_item(large)[1], {"n": 900})), large.exact())
    _untouched(traps)
    captures, replays = plans[0].stats()
    assert captures <= 2 and replays >= 1   # captured again at most once
    for p in plans:
        p.close()


def test_a_callers_graph_keeps_the_workspace(dev):
    """A launch of a key that the caller captured replays soundly after a larger launch of the key."""
    c, large = TL.Case(66, 43, 270, dtype=L.AH_F32, bias=True), TL.Case(1000, 43, 270, dtype=L.AH_F32, bias=True)
    key = ("tmpl:linear_ce;dtype=f32;grad=f32;N=sym;D=43;V=270;bias=1").encode()
    k = C.c_void_p()
    L.check(dev.lib.ah_module_get(dev.h, key, b"kernel", C.byref(k)))

    def launch(c, b):
        order = [b[n].ptr for n in ("dX", "X", "W", "labels", "bias", "dW", "loss", "dbias")]
        one = (C.c_uint32 * 3)(1, 1, 1)
        L.check(dev.lib.ah_launch(dev.h, k, one, one, (C.c_void_p * 8)(*order), 8, (C.c_int32 * 4)(*[c.N] * 4), 4))

    want = ("dX", "dW", "loss", "dbias")
    bufs = [TL.buffers(dev, x, want) for x in (c, large)]
    launch(c, bufs[0])
    dev.sync()
    g = C.c_void_p()
    L.check(dev.lib.ah_graph_begin(dev.h))
    launch(c, bufs[0])
    L.check(dev.lib.ah_graph_end(dev.h, C.byref(g)))
    launch(large, bufs[1])
    dev.sync()
    traps = _traps(dev, (1, 1, 2))
    for _ in range(3):
        for n in want:
            bufs[0][n].write(np.zeros(bufs[0][n].n, np.float32))
        L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.sync()
        shapes = {"dX": (c.N, c.D), "dW": (c.V, c.D)}
        TL.compare({n: bufs[0][n].read().astype(np.float64).reshape(shapes.get(n, -1)) for n in want}, c.exact())
    _untouched(traps)
    dev.lib.ah_graph_destroy(g)
    for b in bufs:
        for v in b.values():
            v.free()


# ── pieces ─────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
def test_the_loss_alone_in_pieces(dev, dtype):
    """Statistics of 1 MiB: 256 rows at a time, the same losses bit for bit."""
    y = np.random.default_rng(4).integers(-5000, 30001, 900)
    c = TL.Case(900, 64, 30001, dtype=dtype, grad_dtype=dtype, labels=y)
    want = ("loss", "rowloss", "lse")
    one, many = TL.run(dev, c, want=want), TL.run(dev, c, want=want, piece_mb=1)
    TL.compare(one, c.exact())
    for k in want:
        np.testing.assert_array_equal(one[k], many[k], err_msg=k)


@pytest.mark.parametrize("types", TL.TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_db_adds_up_over_pieces_in_order(dev, types):
    """db is summed in place over pieces, some of which have no row that counts. (Pieces of other sizes may have other tiles, whose statistics
    round otherwise: each result has the bound of the whole, and repeats bit for bit by itself.)"""
    y = np.random.default_rng(6).integers(0, 2100, 1100)
    y[300:900] = -1
    c = TL.Case(1100, 72, 2100, dtype=types[0], grad_dtype=types[1], labels=y)
    one, many, again = (TL.run(dev, c, want=("loss", "dX", "dbias"), piece_mb=mb) for mb in (0, 1, 1))
    for got in (one, many):
        TL.compare(got, c.exact())
    np.testing.assert_array_equal(many["dbias"], again["dbias"])


# ── rows that are not finite ───────────────────────────────────────────────────

@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("scale", [1e6, 1e-6, 1.0])
@pytest.mark.parametrize("N", [60, 200])
@pytest.mark.parametrize("types", TL.TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_rows_that_are_not_finite_leave_the_others(dev, types, N, scale, bad):
    """A counted row with an infinity or NaN has a NaN loss and dX, and the weights' gradients are NaN; the other rows are as they are without
    it, whatever the size of their values (f32 operands share one power of two)."""
    if types[0] == L.AH_F16 and scale != 1.0:
        scale = 2.0 ** 8 if scale > 1 else 2.0 ** -6
    c = TL.Case(N, 64, 300, dtype=types[0], grad_dtype=types[1], std=scale, wstd=0.125 / scale)
    c.X[9, 3] = bad
    s = 64.0 * (scale if types[1] == L.AH_F16 else 1.0)
    got = TL.run(dev, c, want=("loss", "rowloss", "lse", "dX", "dW"), mean=False, grad_scale=s)
    c.labels[9] = -1   # the oracle without the row
    exact = c.exact(mean=False, grad_scale=s)
    keep = np.arange(N) != 9
    for k in ("rowloss", "lse", "dX"):
        assert np.isnan(got[k][9]).all()
        v, tol = exact[k]
        assert np.all(np.abs(got[k][keep] - v[keep]) <= tol[keep]), k
    assert np.isnan(got["loss"][0]) and np.isnan(got["dW"]).all()


@pytest.mark.parametrize("N", [40, 150])
@pytest.mark.parametrize("types", TL.TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_a_label_that_is_ruled_out(dev, types, N):
    """A bias of -inf at some rows' labels: their loss is infinite, and P there -1, as the formulas have it."""
    c = TL.Case(N, 64, 300, dtype=types[0], grad_dtype=types[1], labels=np.arange(N) * 5 % 300)
    c.b[::10] = -np.inf
    out = c.labels % 10 == 0
    got, exact = TL.run(dev, c, want=("rowloss", "lse", "loss", "dX", "dW", "dbias")), c.exact()
    assert np.isposinf(got["rowloss"][out]).all() and np.isposinf(got["loss"][0])
    for k in ("lse", "dX", "dW", "dbias"):
        v, tol = exact[k]
        assert np.all(np.abs(got[k] - v) <= tol), k
    v, tol = exact["rowloss"]
    assert np.all(np.abs(got["rowloss"][~out] - v[~out]) <= tol[~out])
