// blockops.cpp — C entries of the linear layers, the norms around a block and clipping by the global norm: argument checks, then
// linear.hip, resnorm.hip and clip.hip.
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#include "clip.h"
#include "linear.h"
#include "lm_args.h"
#include "resnorm.h"

using namespace ah;

namespace {

bool is_float(int32_t t) { return t == AH_F32 || t == AH_F16; }

// A strided array [rows, cols] of a call.
struct Array {
    const char *name;
    const void *p;
    int64_t rows, ld, cols;
    int esz;
    Span span() const { return ::span(name, p, rows, ld, cols, esz); }
};

int check_arrays(const char *fn, const Array *a, int n) {
    for (int i = 0; i < n; i++) {
        if (!a[i].p) continue;
        if (a[i].ld < a[i].cols || a[i].ld > kMaxStride)
            return set_error(AH_ERR_INVALID, "%s: %s's row stride %lld is less than its %lld columns or past 2^40", fn, a[i].name, (long long)a[i].ld,
                             (long long)a[i].cols);
        if (a[i].rows > 1 && a[i].ld > kMaxSpan / (a[i].rows - 1)) return set_error(AH_ERR_INVALID, "%s: %s's rows span more than 2^48 elements", fn, a[i].name);
        if (int rc = aligned(fn, a[i].name, a[i].p, a[i].esz)) return rc;
    }
    return AH_OK;
}

// Whether two arrays share a byte. Rows of one stride may lie side by side, as the halves of one [N, 2 F] array do; between rows of another
// stride nothing else may lie.
bool shared(const Array &a, const Array &b) {
    if (!overlap(a.span(), b.span())) return false;
    const int64_t ld = a.ld * a.esz;
    if (ld != b.ld * b.esz) return true;
    const int64_t by = (int64_t)((intptr_t)b.p - (intptr_t)a.p) % ld, at = by < 0 ? by + ld : by;   // where b's rows begin, from a's on
    return at < a.cols * a.esz || at + b.cols * b.esz > ld;
}

// Outputs (the first n_out) against one another and the inputs. same[i]: the array that output i may be, or -1.
int check_outputs(const char *fn, const Array *a, int n, int n_out, const int *same) {
    for (int i = 0; i < n_out; i++)
        for (int j = i + 1; j < n; j++) {
            if (same && same[i] == j && a[i].p == a[j].p && a[i].ld == a[j].ld) continue;
            if (shared(a[i], a[j])) return set_error(AH_ERR_INVALID, "%s: %s overlaps %s", fn, a[i].name, a[j].name);
        }
    return AH_OK;
}

// A workspace against the arrays of a call.
int check_ws_apart(const char *fn, const void *ws, int64_t bytes, const Array *a, int n) {
    const Span w{"ws", (const char *)ws, bytes};
    for (int i = 0; i < n; i++)
        if (overlap(w, a[i].span())) return set_error(AH_ERR_INVALID, "%s: ws overlaps %s", fn, a[i].name);
    return AH_OK;
}

// ── linear layers ──────────────────────────────────────────────────────────────

constexpr int64_t kMaxTokens = 1 << 21;

int linear_shape(const char *fn, int32_t dtype, int32_t act, int32_t N, int32_t D, int32_t F, float scale) {
    if (!is_float(dtype)) return set_error(AH_ERR_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (act < AH_ACT_NONE || act > AH_ACT_SILU) return set_error(AH_ERR_UNSUPPORTED, "%s: act %d", fn, act);
    if (N < 1 || D < 1 || F < 1 || N > kMaxTokens || D > kMaxSide || F > kMaxSide)
        return set_error(AH_ERR_INVALID, "%s: N=%d D=%d F=%d (1 to 2^21 rows, 1 to 2^20 features)", fn, N, D, F);
    if (!std::isfinite(scale)) return set_error(AH_ERR_INVALID, "%s: scale is not finite", fn);
    return AH_OK;
}

struct LinearArrays {
    Array a[7];
    explicit LinearArrays(const ah_linear_desc &d) {
        const int e = esize(d.dtype);
        const Array v[7] = {{"Y", d.Y, d.N, d.ldy, d.F, e}, {"Z", d.Z, d.N, d.ldz, d.F, e}, {"X", d.X, d.N, d.ldx, d.D, e}, {"W", d.W, d.F, d.ldw, d.D, e},
                            {"bias", d.bias, 1, d.F, d.F, e}, {"U", d.U, d.N, d.ldu, d.F, e}, {"R", d.R, d.N, d.ldr, d.F, e}};
        std::copy(v, v + 7, a);
    }
};

int linear_args(ah_device *dev, const ah_linear_desc *d) {
    const char *fn = "ah_linear";
    if (!dev || !d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (int rc = linear_shape(fn, d->dtype, d->act, d->N, d->D, d->F, d->scale)) return rc;
    if (!d->X || !d->W || !d->Y) return set_error(AH_ERR_INVALID, "%s: null X, W or Y", fn);
    return check_arrays(fn, LinearArrays(*d).a, 7);
}

struct LinearGradArrays {
    Array a[9];
    explicit LinearGradArrays(const ah_linear_grad_desc &d) {
        const int e = esize(d.dtype), g = esize(d.grad_dtype);
        const Array v[9] = {{"dX", d.dX, d.N, d.lddx, d.D, g}, {"dW", d.dW, d.F, d.lddw, d.D, g}, {"dbias", d.dbias, 1, d.F, d.F, 4},
                            {"dU", d.dU, d.N, d.lddu, d.F, e}, {"X", d.X, d.N, d.ldx, d.D, e}, {"W", d.W, d.F, d.ldw, d.D, e},
                            {"Z", d.Z, d.N, d.ldz, d.F, e}, {"U", d.U, d.N, d.ldu, d.F, e}, {"dY", d.dY, d.N, d.lddy, d.F, e}};
        std::copy(v, v + 9, a);
    }
};

int linear_grad_args(ah_device *dev, const ah_linear_grad_desc *d) {
    const char *fn = "ah_linear_grad";
    if (!dev || !d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (int rc = linear_shape(fn, d->dtype, d->act, d->N, d->D, d->F, d->scale)) return rc;
    if (!is_float(d->grad_dtype)) return set_error(AH_ERR_UNSUPPORTED, "%s: gradients of dtype %d", fn, d->grad_dtype);
    if (d->dtype == AH_F32 && d->grad_dtype != AH_F32) return set_error(AH_ERR_UNSUPPORTED, "%s: f32 operands have f32 gradients", fn);
    if (!d->dY) return set_error(AH_ERR_INVALID, "%s: null dY", fn);
    if (!d->dX && !d->dW && !d->dbias && !d->dU) return set_error(AH_ERR_INVALID, "%s: no output", fn);
    if (d->dX && !d->W) return set_error(AH_ERR_INVALID, "%s: dX needs W", fn);
    if (d->dW && !d->X) return set_error(AH_ERR_INVALID, "%s: dW needs X", fn);
    if (d->dU && !d->U) return set_error(AH_ERR_INVALID, "%s: dU without U", fn);
    if ((d->act != AH_ACT_NONE || d->dU) && !d->Z) return set_error(AH_ERR_INVALID, "%s: an activation or dU needs Z", fn);
    return check_arrays(fn, LinearGradArrays(*d).a, 9);
}

// ── norms ──────────────────────────────────────────────────────────────────────

bool is_norm(int32_t k) { return k >= AH_NORM_NONE && k <= AH_NORM_LAYER; }

int norm_shape(const char *fn, int32_t dtype, int32_t res, int32_t N, int32_t D, int32_t post, int32_t pre, int32_t per, float eps, float skip, float scale) {
    if (!is_float(dtype) || !is_float(res) || (dtype == AH_F32 && res == AH_F16))
        return set_error(AH_ERR_UNSUPPORTED, "%s: dtype %d with a residual stream of dtype %d", fn, dtype, res);
    if (!is_norm(post) || !is_norm(pre)) return set_error(AH_ERR_UNSUPPORTED, "%s: post %d, pre %d", fn, post, pre);
    if (N < 1 || D < 1 || N > kMaxRows || D > kMaxSide) return set_error(AH_ERR_INVALID, "%s: N=%d D=%d (1 to 2^27 rows of 1 to 2^20)", fn, N, D);
    if (per < 0) return set_error(AH_ERR_INVALID, "%s: rows_per_gate=%d", fn, per);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return set_error(AH_ERR_INVALID, "%s: eps is negative or not finite", fn);
    if (!std::isfinite(skip) || !std::isfinite(scale)) return set_error(AH_ERR_INVALID, "%s: skip or scale is not finite", fn);
    return AH_OK;
}

int norm_weights(const char *fn, const char *which, int32_t kind, const void *w, const void *b) {
    if (kind == AH_NORM_NONE && w) return set_error(AH_ERR_INVALID, "%s: a weight without a %s norm", fn, which);
    if (kind != AH_NORM_LAYER && b) return set_error(AH_ERR_INVALID, "%s: a bias without a %s layer norm", fn, which);
    return AH_OK;
}

int64_t gates_of(int32_t N, int32_t per) { return per ? ((int64_t)N + per - 1) / per : 1; }

struct NormArrays {
    Array a[9];
    explicit NormArrays(const ah_residual_norm_desc &d) {
        const int e = esize(d.dtype), r = esize(d.res_dtype);
        const Array v[9] = {{"H_out", d.H_out, d.N, d.ldh_out, d.D, r}, {"O", d.O, d.N, d.ldo, d.D, e}, {"H", d.H, d.N, d.ldh, d.D, r},
                            {"Y", d.Y, d.N, d.ldy, d.D, e}, {"gate", d.gate, gates_of(d.N, d.rows_per_gate), d.ldgate, d.D, e},
                            {"post_w", d.post_w, 1, d.D, d.D, e}, {"post_b", d.post_b, 1, d.D, d.D, e}, {"pre_w", d.pre_w, 1, d.D, d.D, e},
                            {"pre_b", d.pre_b, 1, d.D, d.D, e}};
        std::copy(v, v + 9, a);
    }
};

int norm_args(ah_device *dev, const ah_residual_norm_desc *d) {
    const char *fn = "ah_residual_norm";
    if (!dev || !d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (int rc = norm_shape(fn, d->dtype, d->res_dtype, d->N, d->D, d->post, d->pre, d->rows_per_gate, d->eps, d->skip, d->scale)) return rc;
    if (int rc = norm_weights(fn, "post", d->post, d->post_w, d->post_b)) return rc;
    if (int rc = norm_weights(fn, "pre", d->pre, d->pre_w, d->pre_b)) return rc;
    if (!d->H && !d->Y) return set_error(AH_ERR_INVALID, "%s: neither H nor Y", fn);
    if (!d->Y && (d->gate || d->post != AH_NORM_NONE)) return set_error(AH_ERR_INVALID, "%s: a gate or a post norm without Y", fn);
    if (!d->H_out && !d->O) return set_error(AH_ERR_INVALID, "%s: neither H_out nor O", fn);
    if ((d->O != nullptr) != (d->pre != AH_NORM_NONE)) return set_error(AH_ERR_INVALID, "%s: O goes with a pre norm", fn);
    return check_arrays(fn, NormArrays(*d).a, 9);
}

struct NormGradArrays {
    Array a[15];
    explicit NormGradArrays(const ah_residual_norm_grad_desc &d) {
        const int e = esize(d.dtype), r = esize(d.res_dtype);
        const int64_t gates = gates_of(d.N, d.rows_per_gate);
        const Array v[15] = {{"dH", d.dH, d.N, d.lddh, d.D, r}, {"dY", d.dY, d.N, d.lddy, d.D, e}, {"dgate", d.dgate, gates, d.lddgate, d.D, e},
                             {"dpost_w", d.dpost_w, 1, d.D, d.D, 4}, {"dpost_b", d.dpost_b, 1, d.D, d.D, 4}, {"dpre_w", d.dpre_w, 1, d.D, d.D, 4},
                             {"dpre_b", d.dpre_b, 1, d.D, d.D, 4}, {"Y", d.Y, d.N, d.ldy, d.D, e}, {"gate", d.gate, gates, d.ldgate, d.D, e},
                             {"post_w", d.post_w, 1, d.D, d.D, e}, {"post_b", d.post_b, 1, d.D, d.D, e}, {"pre_w", d.pre_w, 1, d.D, d.D, e},
                             {"H_out", d.H_out, d.N, d.ldh_out, d.D, r}, {"dH_out", d.dH_out, d.N, d.lddh_out, d.D, r}, {"dO", d.dO, d.N, d.lddo, d.D, e}};
        std::copy(v, v + 15, a);
    }
};

int norm_grad_args(ah_device *dev, const ah_residual_norm_grad_desc *d) {
    const char *fn = "ah_residual_norm_grad";
    if (!dev || !d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (int rc = norm_shape(fn, d->dtype, d->res_dtype, d->N, d->D, d->post, d->pre, d->rows_per_gate, d->eps, d->skip, d->scale)) return rc;
    if (int rc = norm_weights(fn, "post", d->post, d->post_w, d->post_b)) return rc;
    if (int rc = norm_weights(fn, "post", d->post, d->dpost_w, d->dpost_b)) return rc;
    if (int rc = norm_weights(fn, "pre", d->pre, d->pre_w, nullptr)) return rc;
    if (int rc = norm_weights(fn, "pre", d->pre, d->dpre_w, d->dpre_b)) return rc;
    if (!d->dH && !d->dY && !d->dgate && !d->dpost_w && !d->dpost_b && !d->dpre_w && !d->dpre_b) return set_error(AH_ERR_INVALID, "%s: no output", fn);
    if (d->pre != AH_NORM_NONE && (!d->dO || !d->H_out)) return set_error(AH_ERR_INVALID, "%s: a pre norm needs dO and H_out", fn);
    if (d->pre == AH_NORM_NONE && (d->dO || !d->dH_out)) return set_error(AH_ERR_INVALID, "%s: without a pre norm dH_out is needed, and there is no dO", fn);
    if ((d->post != AH_NORM_NONE || d->dgate) && !d->Y) return set_error(AH_ERR_INVALID, "%s: a post norm or dgate needs Y", fn);
    return check_arrays(fn, NormGradArrays(*d).a, 15);
}

// ── clipping ───────────────────────────────────────────────────────────────────

constexpr int kMaxTensors = 1 << 16;

int clip_args(ah_device *dev, const ah_clip_desc *d) {
    const char *fn = "ah_clip_norm";
    if (!dev || !d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (d->n < 1 || d->n > kMaxTensors || !d->tensors) return set_error(AH_ERR_INVALID, "%s: %d tensors (1 to 2^16)", fn, d->n);
    if (!(d->max_norm >= 0.0f)) return set_error(AH_ERR_INVALID, "%s: max_norm is negative or NaN", fn);
    if (!(d->eps >= 0.0f) || !std::isfinite(d->eps)) return set_error(AH_ERR_INVALID, "%s: eps is negative or not finite", fn);
    if (!(d->unscale > 0.0f) || !std::isfinite(d->unscale)) return set_error(AH_ERR_INVALID, "%s: unscale is not positive and finite", fn);
    int64_t total = 0;
    for (int i = 0; i < d->n; i++) {
        const ah_tensor &t = d->tensors[i];
        if (!is_float(t.dtype) || (t.dst && (!is_float(t.out_dtype) || (t.dtype == AH_F32 && t.out_dtype == AH_F16))))
            return set_error(AH_ERR_UNSUPPORTED, "%s: tensor %d of dtype %d to dtype %d", fn, i, t.dtype, t.out_dtype);
        if (t.count < 0 || t.count > kMaxElems || (total += t.count) > kMaxElems)
            return set_error(AH_ERR_INVALID, "%s: tensor %d has %lld elements (0 or more, at most 2^40 in all)", fn, i, (long long)t.count);
        if (t.count && !t.src) return set_error(AH_ERR_INVALID, "%s: tensor %d is null", fn, i);
        if (int rc = aligned(fn, "a tensor", t.src, esize(t.dtype))) return rc;
        if (int rc = aligned(fn, "an output", t.dst, esize(t.out_dtype))) return rc;
    }
    int rc;
    if ((rc = aligned(fn, "norm", d->norm, 4)) || (rc = aligned(fn, "coef", d->coef, 4))) return rc;
    return AH_OK;
}

// Every output against everything else, by one pass over the spans in the order of their addresses.
int clip_apart(const ah_clip_desc *d) {
    struct Range {
        const char *from, *to;
        bool out;
    };
    std::vector<Range> r;
    r.reserve(2 * (size_t)d->n + 3);
    const auto add = [&](const void *p, int64_t bytes, bool out) {
        if (p && bytes) r.push_back({(const char *)p, (const char *)p + bytes, out});
    };
    add(d->ws, d->ws_bytes, true);
    add(d->norm, 4, true);
    add(d->coef, 4, true);
    for (int i = 0; i < d->n; i++) {
        const ah_tensor &t = d->tensors[i];
        const bool in_place = t.src == t.dst && t.dtype == t.out_dtype;
        if (!in_place) add(t.src, t.count * esize(t.dtype), false);
        add(t.dst, t.count * esize(t.out_dtype), true);
    }
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
    const char *any = nullptr, *out = nullptr;   // ends of what has been passed: of everything, of outputs
    for (const Range &x : r) {
        if (x.from < out || (x.out && x.from < any)) return set_error(AH_ERR_INVALID, "ah_clip_norm: an output overlaps another array");
        any = std::max(any, x.to);
        if (x.out) out = std::max(out, x.to);
    }
    return AH_OK;
}

}  // namespace

extern "C" {

int ah_linear_workspace(ah_device *dev, const ah_linear_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_linear_workspace: null bytes");
    if (int rc = linear_args(dev, d)) return rc;
    *bytes = linear_workspace(*d);
    return AH_OK;
}

int ah_linear(ah_device *dev, const ah_linear_desc *d) {
    if (int rc = linear_args(dev, d)) return rc;
    if (int rc = check_ws("ah_linear", d->ws, d->ws_bytes, linear_workspace(*d))) return rc;
    const LinearArrays v(*d);
    const int same[2] = {6, -1};   // Y may be R
    if (int rc = check_outputs("ah_linear", v.a, 7, 2, same)) return rc;
    if (int rc = check_ws_apart("ah_linear", d->ws, d->ws_bytes, v.a, 7)) return rc;
    OnDevice on(dev);
    AH_HIP(linear(*d, dev->stream));
    return AH_OK;
}

int ah_linear_grad_workspace(ah_device *dev, const ah_linear_grad_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_linear_grad_workspace: null bytes");
    if (int rc = linear_grad_args(dev, d)) return rc;
    *bytes = linear_grad_workspace(*d);
    return AH_OK;
}

int ah_linear_grad(ah_device *dev, const ah_linear_grad_desc *d) {
    if (int rc = linear_grad_args(dev, d)) return rc;
    if (int rc = check_ws("ah_linear_grad", d->ws, d->ws_bytes, linear_grad_workspace(*d))) return rc;
    const LinearGradArrays v(*d);
    if (int rc = check_outputs("ah_linear_grad", v.a, 9, 4, nullptr)) return rc;
    if (int rc = check_ws_apart("ah_linear_grad", d->ws, d->ws_bytes, v.a, 9)) return rc;
    OnDevice on(dev);
    AH_HIP(linear_grad(*d, dev->stream));
    return AH_OK;
}

int ah_residual_norm(ah_device *dev, const ah_residual_norm_desc *d) {
    if (int rc = norm_args(dev, d)) return rc;
    const NormArrays v(*d);
    const int same[2] = {2, -1};   // H_out may be H
    if (int rc = check_outputs("ah_residual_norm", v.a, 9, 2, same)) return rc;
    OnDevice on(dev);
    AH_HIP(residual_norm(*d, dev->stream));
    return AH_OK;
}

int ah_residual_norm_grad_workspace(ah_device *dev, const ah_residual_norm_grad_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_residual_norm_grad_workspace: null bytes");
    if (int rc = norm_grad_args(dev, d)) return rc;
    *bytes = residual_norm_grad_workspace(*d);
    return AH_OK;
}

int ah_residual_norm_grad(ah_device *dev, const ah_residual_norm_grad_desc *d) {
    if (int rc = norm_grad_args(dev, d)) return rc;
    if (int rc = check_ws("ah_residual_norm_grad", d->ws, d->ws_bytes, residual_norm_grad_workspace(*d))) return rc;
    const NormGradArrays v(*d);
    const int same[7] = {13, -1, -1, -1, -1, -1, -1};   // dH may be dH_out
    if (int rc = check_outputs("ah_residual_norm_grad", v.a, 15, 7, same)) return rc;
    if (int rc = check_ws_apart("ah_residual_norm_grad", d->ws, d->ws_bytes, v.a, 15)) return rc;
    OnDevice on(dev);
    AH_HIP(residual_norm_grad(*d, dev->stream));
    return AH_OK;
}

int ah_clip_norm_workspace(ah_device *dev, const ah_clip_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_clip_norm_workspace: null bytes");
    if (int rc = clip_args(dev, d)) return rc;
    *bytes = clip_workspace(*d);
    return AH_OK;
}

int ah_clip_norm(ah_device *dev, const ah_clip_desc *d) {
    if (int rc = clip_args(dev, d)) return rc;
    if (int rc = check_ws("ah_clip_norm", d->ws, d->ws_bytes, clip_workspace(*d))) return rc;
    try {
        if (int rc = clip_apart(d)) return rc;
    } catch (const std::bad_alloc &) {
        return set_error(AH_ERR_NOMEM, "ah_clip_norm: no host memory for %d tensors", d->n);
    }
    OnDevice on(dev);
    AH_HIP(clip_norm(*d, dev->stream));
    return AH_OK;
}

}  // extern "C"
