"""Host-side handles over the C ABI: Device, DeviceBuffer and Trainer.

Device mirrors the reference's backend.Executor owner (backend/webgpu/open.go:89, backend/device.go:10-37):
one handle, one HIP stream, calls serialized by the caller. Trainer runs one BASELINE config's training
step with parameters resident on the device (the reference re-uploads parameters and realizes each
gradient separately every step: examples/mlp.go:112-142).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib as L

_NP_DTYPES = {L.AH_F32: np.float32, L.AH_F16: np.float16, L.AH_I32: np.int32, L.AH_U32: np.uint32}


class DeviceBuffer:
    def __init__(self, dev: "Device", n: int, dtype: int):
        self.dev, self.n, self.dtype = dev, int(n), dtype
        p = C.c_void_p()
        L.check(dev.lib.ah_buf_alloc(dev.h, self.n, dtype, C.byref(p)))
        self.ptr = p.value

    @property
    def nbytes(self) -> int:
        return self.n * (2 if self.dtype == L.AH_F16 else 4)

    def write(self, arr: np.ndarray) -> "DeviceBuffer":
        a = np.ascontiguousarray(arr, dtype=_NP_DTYPES[self.dtype])
        if a.size > self.n:
            raise ValueError(f"array of {a.size} elements does not fit a buffer of {self.n}")
        L.check(self.dev.lib.ah_upload_bytes(self.dev.h, self.ptr, a.ctypes.data, a.nbytes))
        return self

    def read(self, n: int | None = None) -> np.ndarray:
        n = self.n if n is None else n
        out = np.empty(n, dtype=_NP_DTYPES[self.dtype])
        L.check(self.dev.lib.ah_download_bytes(self.dev.h, out.ctypes.data, self.ptr, out.nbytes))
        return out

    def free(self) -> None:
        if self.ptr:
            self.dev.lib.ah_buf_free(self.dev.h, self.ptr)
            self.ptr = None


class Device:
    def __init__(self, ordinal: int = 0):
        self.lib = L.load()
        h = C.c_void_p()
        L.check(self.lib.ah_open(ordinal, C.byref(h)))
        self.h = h.value

    def caps(self) -> dict:
        c = L.ah_caps()
        L.check(self.lib.ah_get_caps(self.h, C.byref(c)))
        return {"arch": c.arch.decode(), "cu_count": c.cu_count, "wavefront": c.wavefront,
                "hbm_bytes": c.hbm_bytes, "lds_bytes_per_block": c.lds_bytes_per_block,
                "has_f16": bool(c.has_f16), "has_bf16": bool(c.has_bf16)}

    def buffer(self, arr_or_n, dtype: int = L.AH_F32) -> DeviceBuffer:
        if isinstance(arr_or_n, np.ndarray):
            b = DeviceBuffer(self, arr_or_n.size, dtype)
            return b.write(arr_or_n)
        return DeviceBuffer(self, int(arr_or_n), dtype)

    def sync(self) -> None:
        L.check(self.lib.ah_sync(self.h))

    def timer_start(self) -> None:
        L.check(self.lib.ah_timer_start(self.h))

    def timer_stop(self) -> float:
        """Milliseconds of device-stream time since timer_start (waits for the stream)."""
        ms = C.c_double()
        L.check(self.lib.ah_timer_stop(self.h, C.byref(ms)))
        return ms.value

    @staticmethod
    def _gemm_desc(dtype, epi, ta, tb, M, N, K, A, B, lda, ldb, C_out=None, ldc=0, bias=None, aux=None, ldaux=0,
                   scale=1.0, colsum=None, W32=None, W16=None, lr=0.0, gout=None, lossacc=None, tile=0, variant=0):
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        return L.ah_gemm_desc(dtype=dtype, epi=epi, ta=ta, tb=tb, M=M, N=N, K=K, A=p(A), B=p(B), lda=lda, ldb=ldb,
                              C=p(C_out), ldc=ldc, bias=p(bias), aux=p(aux), ldaux=ldaux, scale=scale,
                              colsum=p(colsum), W32=p(W32), W16=p(W16), lr=lr, gout=p(gout), lossacc=p(lossacc),
                              tile=tile, variant=variant)

    def gemm(self, **kw):
        """One contraction with a fused epilogue (keyword arguments mirror ah_gemm_desc)."""
        d = self._gemm_desc(**kw)
        L.check(self.lib.ah_gemm(self.h, C.byref(d)))

    def gemm_tune(self, iterations: int = 3, **kw):
        """Times every f16 variant (or f32 configuration) of the contraction and caches the fastest;
        returns (variant or configuration index, mean us), variant 0 where the kernel that an f16 call runs
        by itself is no variant and the fastest (nothing is cached then)."""
        d = self._gemm_desc(**kw)
        v, us = C.c_int32(), C.c_double()
        L.check(self.lib.ah_gemm_tune(self.h, C.byref(d), iterations, C.byref(v), C.byref(us)))
        return v.value, us.value

    def gemm_tune_cache(self, path: str, save: bool) -> None:
        """Saves the tuned f16 variants and f32 configurations to path, or merges a saved file into this device's cache."""
        L.check(self.lib.ah_gemm_tune_cache(self.h, str(path).encode(), 1 if save else 0))

    def softmax_ce(self, z: DeviceBuffer, labels: DeviceBuffer, B: int, Cn: int, dz: DeviceBuffer,
                   loss: DeviceBuffer) -> None:
        L.check(self.lib.ah_softmax_ce(self.h, z.ptr, labels.ptr, B, Cn, dz.ptr, loss.ptr))

    def chain_step(self, X, g, R, Cc, dX, dg, loss) -> None:
        L.check(self.lib.ah_chain_step(self.h, X.ptr, g.ptr, R, Cc, dX.ptr, dg.ptr, loss.ptr))

    def chain_step_noalloc(self, X, g, R, Cc, dX, dg, loss) -> None:
        """chain_step with the workspace in the library's per-GPU static array (enqueues only)."""
        L.check(self.lib.ah_chain_step_noalloc(self.h, X.ptr, g.ptr, R, Cc, dX.ptr, dg.ptr, loss.ptr))

    def _sized(self, fn, d) -> int:
        n = C.c_int64()
        L.check(fn(self.h, C.byref(d), C.byref(n)))
        return n.value

    @staticmethod
    def _linear_ce_desc(dtype, N, D, V, X, W, labels, loss, grad_dtype=L.AH_F32, bias=None, rowloss=None, lse=None, dX=None, dW=None,
                        dbias=None, grad_scale=1.0, mean=True, piece_mb=0, ldx=None, ldw=None, lddx=None, lddw=None, ws=None, ws_bytes=None):
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        ld = lambda v: D if v is None else v        # noqa: E731
        return L.ah_linear_ce_desc(dtype=dtype, grad_dtype=grad_dtype, N=N, D=D, V=V, mean=1 if mean else 0, X=p(X), ldx=ld(ldx), W=p(W),
                                   ldw=ld(ldw), bias=p(bias), labels=p(labels), loss=p(loss), rowloss=p(rowloss), lse=p(lse), dX=p(dX),
                                   lddx=ld(lddx), dW=p(dW), lddw=ld(lddw), dbias=p(dbias), grad_scale=grad_scale, piece_mb=piece_mb, ws=p(ws),
                                   ws_bytes=ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def linear_ce(self, **kw) -> None:
        """Softmax cross-entropy of the linear head X W^T + bias, its logits in pieces of piece_mb MiB; with dX, dW or dbias given also
        those gradients (keyword arguments mirror ah_linear_ce_desc; strides default to contiguous rows, ws_bytes to ws.nbytes)."""
        L.check(self.lib.ah_linear_ce(self.h, C.byref(self._linear_ce_desc(**kw))))

    def linear_ce_workspace(self, **kw) -> int:
        """Bytes of workspace that linear_ce needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_linear_ce_workspace, self._linear_ce_desc(**kw))

    #: Coefficients (a, b, c) of the quintic that raises small singular values fastest while it keeps all of them below 1.3.
    NS_COEF = (3.4445, -4.7750, 2.0315)

    @classmethod
    def _orthogonalize_desc(cls, dtype, rows, cols, G, O, out_dtype=L.AH_F32, batch=1, steps=5, coef=None, eps=1e-7, ldg=None, stride_g=None,
                            ldo=None, stride_o=None, ws=None, ws_bytes=None):
        a, b, c = cls.NS_COEF if coef is None else coef
        ldg, ldo = cols if ldg is None else ldg, cols if ldo is None else ldo
        return L.ah_orthogonalize_desc(dtype=dtype, out_dtype=out_dtype, rows=rows, cols=cols, batch=batch, steps=steps, a=a, b=b, c=c, eps=eps,
                                       G=G.ptr, ldg=ldg, stride_g=rows * ldg if stride_g is None else stride_g, O=O.ptr, ldo=ldo,
                                       stride_o=rows * ldo if stride_o is None else stride_o, ws=None if ws is None else ws.ptr,
                                       ws_bytes=ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def orthogonalize(self, **kw) -> None:
        """O = the steps-th Newton-Schulz iterate of G / (|G| + eps), for one matrix or a batch (keyword arguments mirror
        ah_orthogonalize_desc; coef is (a, b, c), strides default to contiguous matrices, ws_bytes to ws.nbytes)."""
        L.check(self.lib.ah_orthogonalize(self.h, C.byref(self._orthogonalize_desc(**kw))))

    def orthogonalize_workspace(self, **kw) -> int:
        """Bytes of workspace that orthogonalize needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_orthogonalize_workspace, self._orthogonalize_desc(**kw))

    @classmethod
    def _muon_desc(cls, dtype, rows, cols, G, M, W, lr, M_out=None, W_out=None, W16_out=None, batch=1, steps=5, coef=None, eps=1e-7, momentum=0.95,
                   nesterov=True, decay=0.0, scale=1.0, ldg=None, stride_g=None, ldw=None, stride_w=None, ws=None, ws_bytes=None):
        a, b, c = cls.NS_COEF if coef is None else coef
        ldg, ldw = cols if ldg is None else ldg, cols if ldw is None else ldw
        return L.ah_muon_desc(dtype=dtype, rows=rows, cols=cols, batch=batch, steps=steps, nesterov=1 if nesterov else 0, a=a, b=b, c=c, eps=eps,
                              G=G.ptr, ldg=ldg, stride_g=rows * ldg if stride_g is None else stride_g, M=M.ptr,
                              M_out=M.ptr if M_out is None else M_out.ptr, W=W.ptr, W_out=W.ptr if W_out is None else W_out.ptr,
                              W16_out=None if W16_out is None else W16_out.ptr, ldw=ldw, stride_w=rows * ldw if stride_w is None else stride_w,
                              lr=lr, momentum=momentum, decay=decay, scale=scale, ws=None if ws is None else ws.ptr,
                              ws_bytes=ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def muon_step(self, **kw) -> None:
        """One weight update by orthogonalised momentum (keyword arguments mirror ah_muon_desc; M and W are updated in place
        unless M_out and W_out are given, strides default to contiguous matrices, ws_bytes to ws.nbytes)."""
        L.check(self.lib.ah_muon_step(self.h, C.byref(self._muon_desc(**kw))))

    def muon_step_workspace(self, **kw) -> int:
        """Bytes of workspace that muon_step needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_muon_workspace, self._muon_desc(**kw))

    @staticmethod
    def _linear_desc(dtype, N, D, F, X, W, Y, act=L.ACT_NONE, scale=1.0, bias=None, U=None, R=None, Z=None, ldx=None, ldw=None, ldu=None, ldr=None,
                     ldy=None, ldz=None, ws=None, ws_bytes=None):
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        ld = lambda v, n: n if v is None else v     # noqa: E731
        return L.ah_linear_desc(dtype, act, N, D, F, scale, X.ptr, ld(ldx, D), W.ptr, ld(ldw, D), p(bias), p(U), ld(ldu, F), p(R), ld(ldr, F), Y.ptr,
                                ld(ldy, F), p(Z), ld(ldz, F), p(ws), ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def linear(self, **kw) -> None:
        """Y = R + scale act(Z) U, Z = X W^T + bias (keyword arguments mirror ah_linear_desc; bias, U, R and Z may be left out, strides
        default to contiguous rows, ws_bytes to ws.nbytes)."""
        L.check(self.lib.ah_linear(self.h, C.byref(self._linear_desc(**kw))))

    def linear_workspace(self, **kw) -> int:
        """Bytes of workspace that linear needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_linear_workspace, self._linear_desc(**kw))

    @staticmethod
    def _linear_grad_desc(dtype, N, D, F, dY, grad_dtype=L.AH_F32, act=L.ACT_NONE, scale=1.0, X=None, W=None, Z=None, U=None, dX=None, dW=None, dbias=None,
                          dU=None, ldx=None, ldw=None, ldz=None, ldu=None, lddy=None, lddx=None, lddw=None, lddu=None, ws=None, ws_bytes=None):
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        ld = lambda v, n: n if v is None else v     # noqa: E731
        return L.ah_linear_grad_desc(dtype, grad_dtype, act, N, D, F, scale, p(X), ld(ldx, D), p(W), ld(ldw, D), p(Z), ld(ldz, F), p(U), ld(ldu, F), dY.ptr,
                                     ld(lddy, F), p(dX), ld(lddx, D), p(dW), ld(lddw, D), p(dbias), p(dU), ld(lddu, F), p(ws),
                                     ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def linear_grad(self, **kw) -> None:
        """The gradients of linear that are given buffers: dX, dW, dbias, dU (keyword arguments mirror ah_linear_grad_desc)."""
        L.check(self.lib.ah_linear_grad(self.h, C.byref(self._linear_grad_desc(**kw))))

    def linear_grad_workspace(self, **kw) -> int:
        """Bytes of workspace that linear_grad needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_linear_grad_workspace, self._linear_grad_desc(**kw))

    def residual_norm(self, dtype, N, D, res_dtype=None, post=L.NORM_NONE, pre=L.NORM_NONE, rows_per_gate=0, eps=1e-6, skip=1.0, scale=1.0, H=None, Y=None,
                      gate=None, post_w=None, post_b=None, pre_w=None, pre_b=None, H_out=None, O=None, ldh=None, ldy=None, ldgate=None, ldh_out=None,
                      ldo=None) -> None:
        """H_out = skip H + scale gate post(Y), O = pre(H_out) (arguments mirror ah_residual_norm_desc; res_dtype defaults to dtype, arrays may
        be left out as ah_residual_norm says, strides default to contiguous rows)."""
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        ld = lambda v: D if v is None else v        # noqa: E731
        d = L.ah_residual_norm_desc(dtype, dtype if res_dtype is None else res_dtype, N, D, post, pre, rows_per_gate, eps, skip, scale, p(H), ld(ldh), p(Y),
                                    ld(ldy), p(gate), ld(ldgate), p(post_w), p(post_b), p(pre_w), p(pre_b), p(H_out), ld(ldh_out), p(O), ld(ldo))
        L.check(self.lib.ah_residual_norm(self.h, C.byref(d)))

    @staticmethod
    def _residual_norm_grad_desc(dtype, N, D, res_dtype=None, post=L.NORM_NONE, pre=L.NORM_NONE, rows_per_gate=0, eps=1e-6, skip=1.0, scale=1.0, Y=None,
                                 gate=None, post_w=None, post_b=None, pre_w=None, H_out=None, dH_out=None, dO=None, dH=None, dY=None, dgate=None,
                                 dpost_w=None, dpost_b=None, dpre_w=None, dpre_b=None, ldy=None, ldgate=None, ldh_out=None, lddh_out=None, lddo=None,
                                 lddh=None, lddy=None, lddgate=None, ws=None, ws_bytes=None):
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        ld = lambda v: D if v is None else v        # noqa: E731
        return L.ah_residual_norm_grad_desc(dtype, dtype if res_dtype is None else res_dtype, N, D, post, pre, rows_per_gate, eps, skip, scale, p(Y), ld(ldy),
                                            p(gate), ld(ldgate), p(post_w), p(post_b), p(pre_w), p(H_out), ld(ldh_out), p(dH_out), ld(lddh_out), p(dO),
                                            ld(lddo), p(dH), ld(lddh), p(dY), ld(lddy), p(dgate), ld(lddgate), p(dpost_w), p(dpost_b), p(dpre_w), p(dpre_b),
                                            p(ws), ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def residual_norm_grad(self, **kw) -> None:
        """The gradients of residual_norm that are given buffers: dH, dY, dgate and the weights' (keyword arguments mirror
        ah_residual_norm_grad_desc)."""
        L.check(self.lib.ah_residual_norm_grad(self.h, C.byref(self._residual_norm_grad_desc(**kw))))

    def residual_norm_grad_workspace(self, **kw) -> int:
        """Bytes of workspace that residual_norm_grad needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_residual_norm_grad_workspace, self._residual_norm_grad_desc(**kw))

    @staticmethod
    def tensor_list(tensors):
        """The tensors of clip_norm, to be kept by a program whose gradients stay where they are: (src, dst or None, count, dtype,
        out_dtype) each."""
        return (L.ah_tensor * len(tensors))(*[(s.ptr, None if o is None else o.ptr, n, t, to) for s, o, n, t, to in tensors])

    def _clip_desc(self, tensors, max_norm, norm=None, coef=None, eps=1e-6, unscale=1.0, ws=None, ws_bytes=None):
        p = lambda b: None if b is None else b.ptr  # noqa: E731
        return L.ah_clip_desc(n=len(tensors), max_norm=max_norm, eps=eps, unscale=unscale, tensors=C.addressof(tensors), norm=p(norm), coef=p(coef),
                              ws=p(ws), ws_bytes=ws_bytes if ws_bytes is not None else 0 if ws is None else ws.nbytes)

    def clip_norm(self, **kw) -> None:
        """norm = unscale times the norm of all tensors together, coef = min(1, max_norm / (norm + eps)), dst = unscale coef src for each
        (tensors: a tensor_list; the other keyword arguments mirror ah_clip_desc)."""
        L.check(self.lib.ah_clip_norm(self.h, C.byref(self._clip_desc(**kw))))

    def clip_norm_workspace(self, **kw) -> int:
        """Bytes of workspace that clip_norm needs for the same arguments (ws left out)."""
        return self._sized(self.lib.ah_clip_norm_workspace, self._clip_desc(**kw))

    def close(self) -> None:
        if self.h:
            self.lib.ah_close(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


class Trainer:
    """One BASELINE config's device-resident training step (slot numbering in include/anneal_hip.h)."""

    SLOTS = {
        L.TRAIN_MLP_CE: ["x", "labels", "W1", "b1", "W2", "b2", "loss", "dW1", "db1", "dW2", "db2", "H1"],
        L.TRAIN_CONVNET: ["x", "labels", "cw1", "cb1", "cw2", "cb2", "fw", "fb", "loss", "dcw1", "dcb1", "dcw2",
                          "dcb2", "dfw", "dfb"],
        L.TRAIN_MLP3_F16: ["x", "t", "W1", "b1", "W2", "b2", "W3", "b3", "loss", "dW1", "db1", "dW2", "db2", "dW3",
                           "db3", "loss_sum", "H1", "H2", "d"],
        L.TRAIN_CHAIN: ["X", "g", "loss", "dX", "dg"],
    }

    def __init__(self, dev: Device, kind: int, dims, lr: float = 0.0):
        self.dev, self.kind, self.dims = dev, kind, list(dims)
        arr = (C.c_int64 * len(dims))(*dims)
        h = C.c_void_p()
        L.check(dev.lib.ah_trainer_create(dev.h, kind, arr, len(dims), C.c_float(lr), C.byref(h)))
        self.h = h.value
        self.slots = {n: i for i, n in enumerate(self.SLOTS[kind])}

    def set(self, name: str, arr: np.ndarray) -> None:
        a = np.ascontiguousarray(arr)
        if a.dtype not in (np.float32, np.int32):
            a = a.astype(np.float32)
        L.check(self.dev.lib.ah_trainer_set(self.h, self.slots[name], a.ctypes.data, a.size))

    def get(self, name: str, n: int, dtype=np.float32) -> np.ndarray:
        out = np.empty(n, dtype=dtype)
        L.check(self.dev.lib.ah_trainer_get(self.h, self.slots[name], out.ctypes.data, n))
        return out

    def step(self, batch: int, store_grads: bool = False, graph: bool = False) -> None:
        flags = (L.STEP_STORE_GRADS if store_grads else 0) | (L.STEP_GRAPH if graph else 0)
        L.check(self.dev.lib.ah_trainer_step(self.h, int(batch), flags))

    def steps(self, batch: int, n: int, store_grads: bool = False, graph: bool = False) -> None:
        """n consecutive steps; with graph=True as hipGraph launches of up to 16 steps each."""
        flags = (L.STEP_STORE_GRADS if store_grads else 0) | (L.STEP_GRAPH if graph else 0)
        L.check(self.dev.lib.ah_trainer_steps(self.h, int(batch), flags, int(n)))

    def probe(self, kernel_index: int) -> None:
        L.check(self.dev.lib.ah_trainer_probe(self.h, kernel_index))

    def probe_span(self, first: int, last: int) -> None:
        """hipEvents before launch `first` and after launch `last` of each following step."""
        L.check(self.dev.lib.ah_trainer_probe_span(self.h, first, last))

    def probe_read(self):
        ms, n = C.c_double(), C.c_int64()
        L.check(self.dev.lib.ah_trainer_probe_read(self.h, C.byref(ms), C.byref(n)))
        return ms.value, n.value

    def kernel_count(self, batch: int) -> int:
        c = C.c_int32()
        L.check(self.dev.lib.ah_trainer_kernel_count(self.h, int(batch), C.byref(c)))
        return c.value

    def kernel_names(self, batch: int) -> list:
        """Names of the step's launches in order (ah_trainer_kernel_count, then ah_trainer_kernel_name)."""
        n = self.kernel_count(batch)
        buf = C.create_string_buffer(64)
        out = []
        for i in range(n):
            L.check(self.dev.lib.ah_trainer_kernel_name(self.h, i, buf, 64))
            out.append(buf.value.decode())
        return out

    def close(self) -> None:
        if self.h:
            self.dev.lib.ah_trainer_destroy(self.h)
            self.h = None
