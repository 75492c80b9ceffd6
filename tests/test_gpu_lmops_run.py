"""The linear cross-entropy and the orthogonalised update as a program uses them (GPU): sizes that take each tile width and split,
pieces, the "tmpl:" keys through the executor and replayed plans, two device handles at once, and a training run of ah_gemm,
ah_linear_ce and ah_muon_step together, eager and captured. Tolerances as in test_gpu_linear_ce.py and test_gpu_muon.py."""
import ctypes as C
import threading

import numpy as np
import pytest

import test_gpu_linear_ce as TL
import test_gpu_muon as TM
from anneal_amd import _lib as L
from anneal_amd.backend import Device
from anneal_amd.executor import Buffer, ExecItem, Executor, Plan

pytestmark = pytest.mark.gpu
NP = {L.AH_F16: np.float16, L.AH_F32: np.float32}


# ── sizes ──────────────────────────────────────────────────────────────────────

# rows, features, classes: 256-, 128- and 64-wide tiles, whole and split over K, ragged edges of each
LARGE = [(1100, 520, 9000), (3000, 1201, 5003), (700, 333, 20011), (2, 4097, 3001), (513, 64, 30001)]


@pytest.mark.parametrize("types", TL.TYPES, ids=["f32", "f16", "f16_f32grad"])
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: "%dx%dx%d" % s)
def test_large_heads(dev, shape, types):
    y = np.random.default_rng(shape).integers(-shape[2] // 4, shape[2], shape[0])   # a fifth does not count
    c = TL.Case(*shape, dtype=types[0], grad_dtype=types[1], labels=y, bias=shape[0] % 2 == 0)
    want = ("loss", "rowloss", "lse", "dX", "dW") + (("dbias",) if c.b is not None else ())
    TL.compare(TL.run(dev, c, want=want, grad_scale=64.0), c.exact(grad_scale=64.0))


@pytest.mark.parametrize("types", TL.TYPES, ids=["f32", "f16", "f16_f32grad"])
@pytest.mark.parametrize("bias", [True, False])
def test_pieces(dev, types, bias):
    """A workspace of 1 MiB of logits: the rows are worked on 256 at a time, and dW adds up over the pieces."""
    y = np.random.default_rng(2).integers(0, 2100, 900)
    y[200:640] = -1   # a piece and more in which no row counts, after the rest has moved up
    c = TL.Case(900, 130, 2100, dtype=types[0], grad_dtype=types[1], labels=y, bias=bias)
    want = ("loss", "rowloss", "dX", "dW") + (("dbias",) if bias else ())
    one, many = TL.run(dev, c, want=want), TL.run(dev, c, want=want, piece_mb=1)
    exact = c.exact()
    # each further piece adds dW in f32 (the accumulator's rounding: 2^-23 of what it holds, at most the sum of magnitudes)
    X = np.where(((y >= 0) & (y < c.V))[:, None], c.X.astype(np.float64), 0.0)
    v, tol = exact["dW"]
    exact["dW"] = (v, tol + 4 * 2.0 ** -23 * np.abs(X).sum(0) / max(1, int((y >= 0).sum())))
    TL.compare(one, exact)
    TL.compare(many, exact)
    np.testing.assert_array_equal(one["rowloss"], many["rowloss"])


def test_smaller_pieces_take_less_workspace(dev):
    c = TL.Case(4096, 64, 50000, dtype=L.AH_F16, grad_dtype=L.AH_F16, bias=False)
    b = TL.buffers(dev, c, ("loss", "dX"))
    args = dict(dtype=c.dtype, grad_dtype=c.grad_dtype, N=c.N, D=c.D, V=c.V, **b)
    full, small = dev.linear_ce_workspace(**args), dev.linear_ce_workspace(piece_mb=64, **args)
    loss_alone = dev.linear_ce_workspace(**{k: v for k, v in args.items() if k != "dX"})
    assert small < full / 4 and loss_alone < full / 4 and full > 4096 * 50000 * 2
    for v in b.values():
        v.free()


@pytest.mark.parametrize("shape", [(3700, 4300), (4300, 3700), (2200, 2200), (1300, 2500), (520, 4100), (4097, 260)], ids=lambda s: "%dx%d" % s)
def test_large_orthogonalisation(dev, shape):
    """As near to 64 bits as 32-bit products come (the bound of iterate() with its norms of whole matrices is far wider here)."""
    G = TM.gradient(np.random.default_rng(shape), *shape, L.AH_F32)
    got = TM.ortho(dev, G, L.AH_F32)[0]
    a, b, c = (float(np.float32(v)) for v in TM.COEF)
    X = (G if shape[0] <= shape[1] else G.T).astype(np.float64)
    X = X / (np.linalg.norm(X) + float(np.float32(1e-7)))
    for _ in range(5):
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    d = (got if shape[0] <= shape[1] else got.T) - X
    assert np.linalg.norm(d) <= 1e-5 * np.linalg.norm(X)
    assert np.abs(d).max() <= 8e-4 * np.linalg.norm(X) / X.size ** 0.5


@pytest.mark.parametrize("shape", [(3, 64, 65), (5, 128, 1000), (4, 900, 100), (16, 20, 33), (2, 300, 500)], ids=lambda s: "%dx%dx%d" % s)
def test_batches_are_each_matrix_alone(dev, shape):
    G = np.stack([TM.gradient(np.random.default_rng([z, *shape]), *shape[1:], L.AH_F32) * 10.0 ** z for z in range(shape[0])])
    got = TM.ortho(dev, G.astype(np.float32), L.AH_F32)
    for z in range(shape[0]):
        want, err = TM.iterate(G[z].astype(np.float32).astype(np.float64))
        assert np.linalg.norm(got[z] - want) <= min(err, 2e-5 * np.linalg.norm(want))


@pytest.mark.parametrize("steps", range(1, 9))
@pytest.mark.parametrize("shape", [(40, 300), (300, 280)])
def test_every_number_of_steps(dev, shape, steps):
    """Each way that steps are put into groups."""
    G = TM.gradient(np.random.default_rng(steps), *shape, L.AH_F32)
    want, err = TM.iterate(G.astype(np.float64), steps)
    assert np.linalg.norm(TM.ortho(dev, G, L.AH_F32, steps=steps)[0] - want) <= min(err, 4e-5 * np.linalg.norm(want))


@pytest.mark.parametrize("coef", [(6.0, -6.0, 2.0), (1.5, -0.5, 0.0), (4.5, -5.0, 1.6)], ids=str)
@pytest.mark.parametrize("shape", [(60, 90), (300, 800)])
def test_polynomials_that_take_shorter_groups(dev, shape, coef):
    G = TM.gradient(np.random.default_rng(1), *shape, L.AH_F32)
    want, err = TM.iterate(G.astype(np.float64), 2, coef)
    assert np.linalg.norm(TM.ortho(dev, G, L.AH_F32, steps=2, coef=coef)[0] - want) <= err


# ── the executor's keys ────────────────────────────────────────────────────────

def _raw(a):
    return np.ascontiguousarray(a, np.int32).view(np.float32)


def _head_item(c, sym=False, **key):
    N, D, V = c.N, c.D, c.V
    t = {L.AH_F16: "f16", L.AH_F32: "f32"}
    k = ";".join(["tmpl:linear_ce", "dtype=" + t[c.dtype], "grad=" + t[c.grad_dtype], "N=" + ("sym" if sym else str(N)), "D=%d" % D, "V=%d" % V] +
                 ["%s=%s" % kv for kv in key.items()] + (["bias=1"] if c.b is not None else []))
    n = 0 if sym else N
    bufs = [Buffer(10, n * D, [n, D], c.grad_dtype), Buffer(1, n * D, [n, D], c.dtype), Buffer(2, V * D, [V, D], c.dtype), Buffer(3, n, [n], L.AH_I32)]
    if c.b is not None:
        bufs.append(Buffer(4, V, [V], c.dtype))
    bufs += [Buffer(11, V * D, [V, D], c.grad_dtype), Buffer(12, 1, [1])]
    if c.b is not None:
        bufs.append(Buffer(13, V, [V]))
    ins = {1: c.X.astype(np.float32).ravel(), 2: c.W.astype(np.float32).ravel(), 3: _raw(c.labels)}
    if c.b is not None:
        ins[4] = c.b.astype(np.float32)
    return ExecItem(k, bufs, sym_vars=["n"] if sym else []), ins


def _head_values(c, out):
    got = {"dX": out[10].astype(np.float64).reshape(c.N, c.D), "dW": out[11].astype(np.float64).reshape(c.V, c.D), "loss": out[12].astype(np.float64)}
    if c.b is not None:
        got["dbias"] = out[13].astype(np.float64)
    return got


@pytest.mark.parametrize("types", TL.TYPES, ids=["f32", "f16", "f16_f32grad"])
@pytest.mark.parametrize("bias", [True, False])
def test_head_key(dev, types, bias):
    c = TL.Case(90, 72, 500, dtype=types[0], grad_dtype=types[1], bias=bias)
    item, ins = _head_item(c, scale=32.0)
    TL.compare(_head_values(c, Executor(dev).run([item], ins)), c.exact(grad_scale=32.0))
    plan = Plan(dev, [item], graph=True)
    for seed in (1, 2, 1):   # captured once, replayed with other leaves
        c = TL.Case(90, 72, 500, dtype=types[0], grad_dtype=types[1], bias=bias, seed=seed)
        TL.compare(_head_values(c, plan.run(_head_item(c)[1])), c.exact(grad_scale=32.0))
    plan.close()


def test_head_key_with_a_symbolic_batch(dev):
    for n in (3, 70, 1):
        c = TL.Case(n, 40, 130, dtype=L.AH_F32, bias=True)
        item, ins = _head_item(c, sym=True)
        TL.compare(_head_values(c, Executor(dev).run_symbolic([item], ins, {"n": n})), c.exact())


def test_update_keys(dev):
    r = np.random.default_rng(9)
    G, M, W = TM.gradient(r, 96, 150, L.AH_F32), 1e-2 * r.standard_normal((96, 150)).astype(np.float32), r.standard_normal((96, 150)).astype(np.float32)
    n = G.size
    shape = [96, 150]
    orth = ExecItem("tmpl:orthogonalize;rows=96;cols=150", [Buffer(20, n, shape), Buffer(1, n, shape)])
    step = ExecItem("tmpl:muon;rows=96;cols=150;lr=0.125;wd=0.5;mu=0.5;scale=2",
                    [Buffer(21, n, shape), Buffer(3, n, shape), Buffer(1, n, shape), Buffer(2, n, shape), Buffer(22, n, shape)])
    out = Executor(dev).run([orth, step], {1: G.ravel(), 2: M.ravel(), 3: W.ravel()})
    want, err = TM.iterate(G.astype(np.float64))
    assert np.linalg.norm(out[20].reshape(shape) - want) <= err
    M1 = 0.5 * M.astype(np.float64) + G
    assert np.all(np.abs(out[22].reshape(shape) - M1) <= 2 * TM.U32 * (np.abs(M) + np.abs(M1)))
    O, err = TM.iterate(G + 0.5 * out[22].reshape(shape).astype(np.float64))
    want = (1 - 0.125 * 0.5) * W.astype(np.float64) - 0.25 * O
    assert np.linalg.norm(out[21].reshape(shape) - want) <= 0.25 * 2 * err + 4 * TM.U32 * np.linalg.norm(W)


@pytest.mark.parametrize("key", ["linear_ce;N=4;D=8", "linear_ce;N=0;D=8;V=4", "linear_ce;N=4;D=8;V=4;dtype=f32;grad=f16", "linear_ce;N=4;D=8;V=4;dtype=bf16",
                                 "linear_ce;N=4;D=8;V=4;scale=inf", "orthogonalize;rows=4", "orthogonalize;rows=4;cols=0", "orthogonalize;rows=4;cols=4;steps=0",
                                 "orthogonalize;rows=4;cols=4;a=40", "orthogonalize;rows=4;cols=4;out=i32", "muon;rows=4;cols=4", "muon;rows=4;cols=4;lr=nan"])
def test_bad_keys(dev, key):
    k = C.c_void_p()
    assert dev.lib.ah_module_get(dev.h, ("tmpl:" + key).encode(), b"kernel", C.byref(k)) in (1, 3)


def test_short_buffers_are_refused(dev):
    item = ExecItem("tmpl:orthogonalize;rows=8;cols=8", [Buffer(20, 64, [64]), Buffer(1, 63, [63])])
    with pytest.raises(L.AnnealHipError):
        Executor(dev).run([item], {1: np.ones(63, np.float32)})


# ── calls side by side ─────────────────────────────────────────────────────────

def test_two_handles_at_once(dev):
    """Two device handles, each with its workspace, driven from two threads: the bits of each alone."""
    cases = [TL.Case(300, 128, 3000, dtype=L.AH_F16, grad_dtype=L.AH_F16, seed=s) for s in (1, 2)]
    want = ("loss", "dX", "dW", "dbias")
    alone = [TL.run(dev, c, want=want) for c in cases]
    G = TM.gradient(np.random.default_rng(3), 200, 300, L.AH_F32)
    ortho_alone = TM.ortho(dev, G, L.AH_F32)
    wrong = []

    def work(handle, c, ref):
        for _ in range(10):
            got = TL.run(handle, c, want=want)
            if any(not np.array_equal(got[k], ref[k]) for k in want) or not np.array_equal(TM.ortho(handle, G, L.AH_F32), ortho_alone):
                wrong.append(c)

    with Device(0) as other:
        threads = [threading.Thread(target=work, args=a) for a in zip((dev, other), cases, alone)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong


def test_calls_share_a_workspace_and_nothing_is_left_in_it(dev):
    """Calls of all three operators one after the other through one workspace, and two captured graphs that hold it."""
    c = TL.Case(200, 96, 1500, dtype=L.AH_F16, grad_dtype=L.AH_F32)
    want = ("loss", "dX", "dW")
    b = TL.buffers(dev, c, want)
    head = dict(dtype=c.dtype, grad_dtype=c.grad_dtype, N=c.N, D=c.D, V=c.V, **b)
    G = TM.gradient(np.random.default_rng(3), 300, 200, L.AH_F32)
    bG, bO = dev.buffer(G), dev.buffer(G.size)
    orth = dict(dtype=L.AH_F32, rows=300, cols=200, G=bG, O=bO)
    ws = dev.buffer(max(dev.linear_ce_workspace(**head), dev.orthogonalize_workspace(**orth)) // 4 + 4)
    graphs = []
    for call, args in ((dev.linear_ce, head), (dev.orthogonalize, orth)):
        call(ws=ws, **args)
        dev.sync()
        g = C.c_void_p()
        L.check(dev.lib.ah_graph_begin(dev.h))
        call(ws=ws, **args)
        L.check(dev.lib.ah_graph_end(dev.h, C.byref(g)))
        graphs.append(g)
    first = {k: b[k].read() for k in want}, bO.read()
    for _ in range(4):
        for g in graphs:
            L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.linear_ce(ws=ws, **head)
        for g in reversed(graphs):
            L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.sync()
        for k in want:
            np.testing.assert_array_equal(b[k].read(), first[0][k])
        np.testing.assert_array_equal(bO.read(), first[1])
    for g in graphs:
        dev.lib.ah_graph_destroy(g)
    for v in list(b.values()) + [bG, bO, ws]:
        v.free()


# ── a training run ─────────────────────────────────────────────────────────────

def test_training_run(dev):
    """H = X W1^T + b1 (ah_gemm), loss and dH, dW2 of the head (ah_linear_ce), dW1 = dH^T X (ah_gemm), both weights by
    ah_muon_step: four steps captured as one graph each, and each step's weights against 64 bits on the state before it."""
    B, D, H, V = 192, 160, 136, 700
    r = np.random.default_rng(11)
    X = r.standard_normal((B, D)).astype(np.float32)
    y = r.integers(-80, V, B).astype(np.int32)
    W1, b1 = (D ** -0.5 * r.standard_normal((H, D))).astype(np.float32), (0.1 * r.standard_normal(H)).astype(np.float32)
    W2 = (H ** -0.5 * r.standard_normal((V, H))).astype(np.float32)
    buf = {k: dev.buffer(v) for k, v in dict(X=X, W1=W1, b1=b1, W2=W2, M1=np.zeros_like(W1), M2=np.zeros_like(W2)).items()}
    buf["y"] = dev.buffer(y, L.AH_I32)
    for k, n in (("H", B * H), ("dH", B * H), ("dW1", H * D), ("dW2", V * H), ("loss", 1)):
        buf[k] = dev.buffer(n)
    lr, mu = float(np.float32(0.02)), float(np.float32(0.9))
    head = dict(dtype=L.AH_F32, N=B, D=H, V=V, X=buf["H"], W=buf["W2"], labels=buf["y"], loss=buf["loss"], dX=buf["dH"], dW=buf["dW2"])
    up1 = dict(dtype=L.AH_F32, rows=H, cols=D, G=buf["dW1"], M=buf["M1"], W=buf["W1"], lr=lr, momentum=mu)
    up2 = dict(dtype=L.AH_F32, rows=V, cols=H, G=buf["dW2"], M=buf["M2"], W=buf["W2"], lr=lr, momentum=mu)
    ws = dev.buffer(max(dev.linear_ce_workspace(**head), dev.muon_step_workspace(**up1), dev.muon_step_workspace(**up2)) // 4 + 4)

    def step():
        dev.gemm(dtype=L.AH_F32, epi=L.EPI_BIAS, ta=0, tb=0, M=B, N=H, K=D, A=buf["X"], B=buf["W1"], lda=D, ldb=D, C_out=buf["H"], ldc=H, bias=buf["b1"])
        dev.linear_ce(ws=ws, **head)
        dev.gemm(dtype=L.AH_F32, epi=L.EPI_STORE, ta=1, tb=1, M=H, N=D, K=B, A=buf["dH"], B=buf["X"], lda=H, ldb=D, C_out=buf["dW1"], ldc=D)
        dev.muon_step(ws=ws, **up1)
        dev.muon_step(ws=ws, **up2)

    def check(before, W, M, dW, err_dW):
        """W and M after the step against 64 bits, given the gradient that the device used and how far it may be off."""
        M64 = mu * before[1].astype(np.float64) + dW
        U = dW + mu * M64
        O, err = TM.iterate(U)
        # the update moves by at most 485 |dU| / |U|; dU: the gradient's own error and the roundings of M and U
        dU = 2 * np.linalg.norm(err_dW) + 8 * TM.U32 * np.linalg.norm(np.abs(U) + np.abs(M64))
        tol = lr * (err + 2 * 485 * dU / np.linalg.norm(U)) + 4 * TM.U32 * np.linalg.norm(before[0])
        assert np.linalg.norm(W - (before[0].astype(np.float64) - lr * O)) <= tol
        assert np.linalg.norm(M - M64) <= dU

    step()
    dev.sync()
    for k, v in (("W1", W1), ("W2", W2), ("M1", 0 * W1), ("M2", 0 * W2)):
        buf[k].write(v)
    g = C.c_void_p()
    L.check(dev.lib.ah_graph_begin(dev.h))
    step()
    L.check(dev.lib.ah_graph_end(dev.h, C.byref(g)))
    losses = []
    for _ in range(4):
        L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.sync()
        got = {k: buf[k].read().reshape(s) for k, s in (("W1", (H, D)), ("W2", (V, H)), ("M1", (H, D)), ("M2", (V, H)), ("H", (B, H)), ("dH", (B, H)),
                                                       ("dW1", (H, D)), ("dW2", (V, H)), ("loss", (1,)))}
        if not losses:
            W, M = {"1": W1, "2": W2}, {"1": 0 * W1, "2": 0 * W2}
        H64 = X.astype(np.float64) @ W["1"].astype(np.float64).T + b1
        assert np.abs(got["H"] - H64).max() <= (D / 4 + 8) * TM.U32 * (np.abs(X) @ np.abs(W["1"]).T + np.abs(b1)).max()
        c = TL.Case(B, H, V, dtype=L.AH_F32, bias=False, labels=y)   # the head on the hidden states that the device holds
        c.X, c.W = got["H"], W["2"]
        e = c.exact()
        TL.compare({"loss": got["loss"].astype(np.float64), "dX": got["dH"].astype(np.float64), "dW": got["dW2"].astype(np.float64)}, e)
        dW1 = got["dH"].astype(np.float64).T @ X
        tol1 = (B / 4 + 8) * TM.U32 * (np.abs(got["dH"]).T.astype(np.float64) @ np.abs(X))
        assert np.all(np.abs(got["dW1"] - dW1) <= tol1)
        check((W["1"], M["1"]), got["W1"], got["M1"], dW1, tol1)
        check((W["2"], M["2"]), got["W2"], got["M2"], *e["dW"])
        W, M = {"1": got["W1"], "2": got["W2"]}, {"1": got["M1"], "2": got["M2"]}
        losses.append(float(got["loss"][0]))
    dev.lib.ah_graph_destroy(g)
    for v in list(buf.values()) + [ws]:
        v.free()


# ── gradients against differences ──────────────────────────────────────────────

def test_gradients_against_differences(dev):
    """Central differences of the call's own loss along random directions. The loss is an f32 near 6, so a difference over 2 h
    is off by about 2^-23 * 6 / h, and by h^2 / 6 times the third derivative, which is at most the direction's logits cubed."""
    c = TL.Case(64, 48, 300, dtype=L.AH_F32)
    g = TL.run(dev, c, mean=False)
    r = np.random.default_rng(0)
    h = 2.0 ** -6
    for name, grad in (("X", "dX"), ("W", "dW"), ("b", "dbias")):
        base = getattr(c, name).copy()
        d = r.standard_normal(base.shape).astype(np.float32)
        d /= np.float32(np.linalg.norm(d))
        values = []
        for s in (h, -h):
            setattr(c, name, (base + np.float32(s) * d).astype(np.float32))
            values.append(TL.run(dev, c, want=("loss", "rowloss"))["rowloss"].sum())
        setattr(c, name, base)
        want = (values[0] - values[1]) / (2 * h)
        got = float((g[grad].reshape(base.shape) * d).sum())
        assert abs(got - want) <= 64 * 2.0 ** -22 * 8 / h + h * h * 8, name
