// lmops.cpp — C entries of the linear cross-entropy and of the orthogonalised updates: argument checks, then linear_ce.hip and
// muon.hip.
#include <math.h>

#include "linear_ce.h"
#include "lm_args.h"
#include "muon.h"

using namespace ah;

namespace {

int linear_ce_args(ah_device *dev, const ah_linear_ce_desc *d, LinearCe *o) {
    const char *fn = "ah_linear_ce";
    if (!dev || !d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if ((d->dtype != AH_F32 && d->dtype != AH_F16) || (d->grad_dtype != AH_F32 && d->grad_dtype != AH_F16))
        return set_error(AH_ERR_UNSUPPORTED, "%s: dtype %d with gradients of dtype %d", fn, d->dtype, d->grad_dtype);
    if (d->dtype == AH_F32 && d->grad_dtype != AH_F32) return set_error(AH_ERR_UNSUPPORTED, "%s: f32 operands have f32 gradients", fn);
    if (d->N < 1 || d->D < 1 || d->V < 1 || d->N > kMaxRows || d->V > kMaxRows || d->D > kMaxSide)
        return set_error(AH_ERR_INVALID, "%s: N=%d D=%d V=%d (1 to %lld rows and classes, 1 to %lld features)", fn, d->N, d->D, d->V,
                         (long long)kMaxRows, (long long)kMaxSide);
    if ((int64_t)d->N * d->D > kMaxElems || (int64_t)d->V * d->D > kMaxElems) return set_error(AH_ERR_INVALID, "%s: more than 2^40 elements", fn);
    if (!d->X || !d->W || !d->labels || !d->loss) return set_error(AH_ERR_INVALID, "%s: null X, W, labels or loss", fn);
    if (d->ldx < d->D || d->ldw < d->D || (d->dX && d->lddx < d->D) || (d->dW && d->lddw < d->D) || d->ldx > kMaxStride || d->ldw > kMaxStride ||
        (d->dX && d->lddx > kMaxStride) || (d->dW && d->lddw > kMaxStride))
        return set_error(AH_ERR_INVALID, "%s: a row stride is less than D=%d or past 2^40", fn, d->D);
    const auto spans = [](int64_t rows, int64_t ld) { return rows > 1 && ld > kMaxSpan / (rows - 1); };
    if (spans(d->N, d->ldx) || spans(d->V, d->ldw) || (d->dX && spans(d->N, d->lddx)) || (d->dW && spans(d->V, d->lddw)))
        return set_error(AH_ERR_INVALID, "%s: rows that span more than 2^48 elements", fn);
    if (!std::isfinite(d->grad_scale)) return set_error(AH_ERR_INVALID, "%s: grad_scale is not finite", fn);
    if (d->piece_mb < 0) return set_error(AH_ERR_INVALID, "%s: piece_mb=%d", fn, d->piece_mb);
    const int e = esize(d->dtype), g = esize(d->grad_dtype);
    int rc;
    if ((rc = aligned(fn, "X", d->X, e)) || (rc = aligned(fn, "W", d->W, e)) || (rc = aligned(fn, "bias", d->bias, e)) ||
        (rc = aligned(fn, "labels", d->labels, 4)) || (rc = aligned(fn, "loss", d->loss, 4)) || (rc = aligned(fn, "rowloss", d->rowloss, 4)) ||
        (rc = aligned(fn, "lse", d->lse, 4)) || (rc = aligned(fn, "dX", d->dX, g)) || (rc = aligned(fn, "dW", d->dW, g)) ||
        (rc = aligned(fn, "dbias", d->dbias, 4)))
        return rc;
    *o = LinearCe{};
    o->f16 = d->dtype == AH_F16;
    o->g16 = d->grad_dtype == AH_F16;
    o->N = d->N; o->D = d->D; o->V = d->V;
    o->X = d->X; o->W = d->W; o->bias = d->bias; o->ldx = d->ldx; o->ldw = d->ldw;
    o->labels = d->labels; o->loss = d->loss; o->rowloss = d->rowloss; o->lse = d->lse;
    o->dX = d->dX; o->dW = d->dW; o->lddx = d->lddx; o->lddw = d->lddw; o->dbias = d->dbias;
    o->grad_scale = d->grad_scale;
    o->mean = d->mean != 0;
    o->piece_mb = d->piece_mb;
    return AH_OK;
}

int ns_common(const char *fn, ah_device *dev, int32_t dtype, int32_t rows, int32_t cols, int32_t batch, int32_t steps, float a, float b, float c,
              float eps, const void *G, int64_t ldg, int64_t sg) {
    if (!dev) return set_error(AH_ERR_INVALID, "%s: null device", fn);
    if (dtype != AH_F32 && dtype != AH_F16) return set_error(AH_ERR_UNSUPPORTED, "%s: dtype %d", fn, dtype);
    if (rows < 1 || cols < 1 || batch < 1 || rows > kMaxSide || cols > kMaxSide || batch > 65535)
        return set_error(AH_ERR_INVALID, "%s: %d matrices of %d x %d (sides 1 to %lld, 1 to 65535 matrices)", fn, batch, rows, cols, (long long)kMaxSide);
    if ((int64_t)(rows + 63) * (cols + 63) * batch > kMaxElems) return set_error(AH_ERR_INVALID, "%s: more than 2^40 elements", fn);
    if (steps < 1 || steps > 64) return set_error(AH_ERR_INVALID, "%s: %d steps (1 to 64)", fn, steps);
    if (!(fabsf(a) + fabsf(b) + fabsf(c) <= 15.0f)) return set_error(AH_ERR_INVALID, "%s: |a| + |b| + |c| is over 15", fn);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return set_error(AH_ERR_INVALID, "%s: eps is negative or not finite", fn);
    if (!G) return set_error(AH_ERR_INVALID, "%s: null G", fn);
    if (ldg < cols || ldg > kMaxStride || (batch > 1 && (sg < 0 || sg > kMaxStride)))
        return set_error(AH_ERR_INVALID, "%s: G's strides %lld, %lld", fn, (long long)ldg, (long long)sg);
    return aligned(fn, "G", G, esize(dtype));
}

int out_strides(const char *fn, int32_t rows, int32_t cols, int32_t batch, int64_t ld, int64_t stride) {
    if (ld < cols || ld > kMaxStride || (batch > 1 && (stride > kMaxStride || stride < (int64_t)(rows - 1) * ld + cols)))
        return set_error(AH_ERR_INVALID, "%s: strides %lld, %lld make the outputs' rows or matrices overlap", fn, (long long)ld, (long long)stride);
    return AH_OK;
}

int64_t extent(int32_t rows, int32_t cols, int32_t batch, int64_t ld, int64_t stride) {
    return (batch > 1 ? (int64_t)(batch - 1) * stride : 0) + (int64_t)(rows - 1) * ld + cols;
}

int orthogonalize_args(ah_device *dev, const ah_orthogonalize_desc *d, Muon *o) {
    const char *fn = "ah_orthogonalize";
    if (!d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (int rc = ns_common(fn, dev, d->dtype, d->rows, d->cols, d->batch, d->steps, d->a, d->b, d->c, d->eps, d->G, d->ldg, d->stride_g)) return rc;
    if (d->out_dtype != AH_F32 && d->out_dtype != AH_F16) return set_error(AH_ERR_UNSUPPORTED, "%s: out_dtype %d", fn, d->out_dtype);
    if (!d->O) return set_error(AH_ERR_INVALID, "%s: null O", fn);
    if (int rc = aligned(fn, "O", d->O, esize(d->out_dtype))) return rc;
    if (int rc = out_strides(fn, d->rows, d->cols, d->batch, d->ldo, d->stride_o)) return rc;
    *o = Muon{};
    o->f16 = d->dtype == AH_F16;
    o->rows = d->rows; o->cols = d->cols; o->batch = d->batch;
    o->G = d->G; o->ldg = d->ldg; o->sg = d->stride_g;
    o->steps = d->steps; o->a = d->a; o->b = d->b; o->c = d->c; o->eps = d->eps;
    o->O = d->O; o->ldo = d->ldo; o->so = d->stride_o; o->out16 = d->out_dtype == AH_F16;
    return AH_OK;
}

int muon_args(ah_device *dev, const ah_muon_desc *d, Muon *o) {
    const char *fn = "ah_muon_step";
    if (!d) return set_error(AH_ERR_INVALID, "%s: null argument", fn);
    if (int rc = ns_common(fn, dev, d->dtype, d->rows, d->cols, d->batch, d->steps, d->a, d->b, d->c, d->eps, d->G, d->ldg, d->stride_g)) return rc;
    if (!d->M || !d->M_out || !d->W || !d->W_out) return set_error(AH_ERR_INVALID, "%s: null M, W or an output of theirs", fn);
    int rc;
    if ((rc = aligned(fn, "M", d->M, 4)) || (rc = aligned(fn, "M_out", d->M_out, 4)) || (rc = aligned(fn, "W", d->W, 4)) ||
        (rc = aligned(fn, "W_out", d->W_out, 4)) || (rc = aligned(fn, "W16_out", d->W16_out, 2)))
        return rc;
    if ((rc = out_strides(fn, d->rows, d->cols, d->batch, d->ldw, d->stride_w))) return rc;
    if (!std::isfinite(d->lr) || !std::isfinite(d->momentum) || !std::isfinite(d->decay) || !std::isfinite(d->scale))
        return set_error(AH_ERR_INVALID, "%s: lr, momentum, decay or scale is not finite", fn);
    *o = Muon{};
    o->f16 = d->dtype == AH_F16;
    o->rows = d->rows; o->cols = d->cols; o->batch = d->batch;
    o->G = d->G; o->ldg = d->ldg; o->sg = d->stride_g;
    o->steps = d->steps; o->a = d->a; o->b = d->b; o->c = d->c; o->eps = d->eps;
    o->M = d->M; o->M_out = d->M_out; o->W = d->W; o->W_out = d->W_out; o->W16_out = d->W16_out;
    o->ldw = d->ldw; o->sw = d->stride_w;
    o->lr = d->lr; o->momentum = d->momentum; o->decay = d->decay; o->scale = d->scale;
    o->nesterov = d->nesterov != 0;
    return AH_OK;
}

}  // namespace

extern "C" {

int ah_linear_ce_workspace(ah_device *dev, const ah_linear_ce_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_linear_ce_workspace: null bytes");
    LinearCe o;
    if (int rc = linear_ce_args(dev, d, &o)) return rc;
    *bytes = linear_ce_workspace(o);
    return AH_OK;
}

int ah_linear_ce(ah_device *dev, const ah_linear_ce_desc *d) {
    LinearCe o;
    if (int rc = linear_ce_args(dev, d, &o)) return rc;
    if (int rc = check_ws("ah_linear_ce", d->ws, d->ws_bytes, linear_ce_workspace(o))) return rc;
    const int e = esize(d->dtype), g = esize(d->grad_dtype);
    const Span s[] = {span("ws", d->ws, 1, 0, d->ws_bytes, 1), span("loss", d->loss, 1, 0, 1, 4), span("rowloss", d->rowloss, 1, 0, d->N, 4),
                      span("lse", d->lse, 1, 0, d->N, 4), span("dX", d->dX, d->N, d->lddx, d->D, g), span("dW", d->dW, d->V, d->lddw, d->D, g),
                      span("dbias", d->dbias, 1, 0, d->V, 4), span("X", d->X, d->N, d->ldx, d->D, e), span("W", d->W, d->V, d->ldw, d->D, e),
                      span("bias", d->bias, 1, 0, d->V, e), span("labels", d->labels, 1, 0, d->N, 4)};
    if (int rc = check_overlap("ah_linear_ce", s, 11, 7)) return rc;
    OnDevice on(dev);
    AH_HIP(linear_ce(o, d->ws, dev->stream));
    return AH_OK;
}

int ah_orthogonalize_workspace(ah_device *dev, const ah_orthogonalize_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_orthogonalize_workspace: null bytes");
    Muon o;
    if (int rc = orthogonalize_args(dev, d, &o)) return rc;
    *bytes = muon_workspace(o);
    return AH_OK;
}

int ah_orthogonalize(ah_device *dev, const ah_orthogonalize_desc *d) {
    Muon o;
    if (int rc = orthogonalize_args(dev, d, &o)) return rc;
    if (int rc = check_ws("ah_orthogonalize", d->ws, d->ws_bytes, muon_workspace(o))) return rc;
    // G is read before O is written, so they may overlap
    const Span s[] = {span("ws", d->ws, 1, 0, d->ws_bytes, 1), {"G", (const char *)d->G, extent(d->rows, d->cols, d->batch, d->ldg, d->stride_g) * esize(d->dtype)},
                      {"O", (const char *)d->O, extent(d->rows, d->cols, d->batch, d->ldo, d->stride_o) * esize(d->out_dtype)}};
    if (int rc = check_overlap("ah_orthogonalize", s, 3, 1)) return rc;
    OnDevice on(dev);
    AH_HIP(muon(o, d->ws, dev->stream));
    return AH_OK;
}

int ah_muon_workspace(ah_device *dev, const ah_muon_desc *d, int64_t *bytes) {
    if (!bytes) return set_error(AH_ERR_INVALID, "ah_muon_workspace: null bytes");
    Muon o;
    if (int rc = muon_args(dev, d, &o)) return rc;
    *bytes = muon_workspace(o);
    return AH_OK;
}

int ah_muon_step(ah_device *dev, const ah_muon_desc *d) {
    Muon o;
    if (int rc = muon_args(dev, d, &o)) return rc;
    if (int rc = check_ws("ah_muon_step", d->ws, d->ws_bytes, muon_workspace(o))) return rc;
    const int64_t n = extent(d->rows, d->cols, d->batch, d->ldw, d->stride_w) * 4;
    const Span s[] = {span("ws", d->ws, 1, 0, d->ws_bytes, 1), {"M_out", (const char *)d->M_out, n}, {"W_out", (const char *)d->W_out, n},
                      {"W16_out", (const char *)d->W16_out, n / 2},
                      {"G", (const char *)d->G, extent(d->rows, d->cols, d->batch, d->ldg, d->stride_g) * esize(d->dtype)},
                      {"M", d->M == d->M_out ? nullptr : (const char *)d->M, n}, {"W", d->W == d->W_out ? nullptr : (const char *)d->W, n}};
    if (int rc = check_overlap("ah_muon_step", s, 7, 4)) return rc;
    OnDevice on(dev);
    AH_HIP(muon(o, d->ws, dev->stream));
    return AH_OK;
}

}  // extern "C"
