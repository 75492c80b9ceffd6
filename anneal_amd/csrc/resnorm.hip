// resnorm.hip — norms after and before a block, fused with its gate and the residual sum, and their gradients.
//
//   u = post(Y),  h = skip H + scale g u,  O = pre(h)             norm(x) = (x - m) r w + b,  r = 1 / sqrt(mean (x - m)^2 + eps)
//   t = dh + r_h (q - mean(q xh) xh - mean(q)),  q = dO w_pre     (m, b, mean(q): layer norms alone; xh = (h - m) r_h, yh likewise)
//   dH = skip t,  dg = sum scale t u,  dY = r_y (p - mean(p yh) yh - mean(p)),  p = scale g t w_post
//   dw_pre = sum dO xh,  db_pre = sum dO,  dw_post = sum scale g t yh,  db_post = sum scale g t
//
// Bound by memory: each array is read and written once, a row's statistics are taken from registers. A row belongs to TPR threads, eight
// columns to each; up to 64 threads (512 columns) rows share a wave and are joined by shuffles alone, above that they are a workgroup.
// The backward pass holds the columns' sums in registers: a group of threads (a worker) walks down a run of neighbouring rows with the next
// row's loads in flight, and leaves its sums in the workspace, where a second launch adds them in the workers' order. A run that begins or
// ends inside a gate's rows leaves that gate's part there too; the sums of gates whose rows are all its own it writes itself.
// Rows past 8192 columns (1024 threads) are read again for each of their passes, from caches mostly, and their columns' sums are a launch of
// their own with the rows' statistics given.
#include "resnorm.h"

#include <algorithm>

#include "ah_common.h"

namespace ah {
namespace {

constexpr int kVec = 8;            // columns of a thread
constexpr int kWide = 8192;        // columns that a workgroup's registers hold

struct f8 {
    float v[kVec];
};
template <class T>
struct Raw {   // eight values as they lie; rows may start anywhere
    typedef T type __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
};
template <class T>
__device__ __forceinline__ typename Raw<T>::type load_raw(const T *row, int c, int D) {
    typename Raw<T>::type x = {};
    if (c + kVec <= D) {
        x = *(const typename Raw<T>::type *)(row + c);
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k++)
            if (c + k < D) x[k] = row[c + k];
    }
    return x;
}
template <class V>
__device__ __forceinline__ f8 widen(V x) {
    f8 r;
#pragma unroll
    for (int k = 0; k < kVec; k++) r.v[k] = (float)x[k];
    return r;
}
template <class T>
__device__ __forceinline__ f8 load8(const T *row, int c, int D) {
    return widen(load_raw(row, c, D));
}
__device__ __forceinline__ f8 all8(float x) {
    f8 r;
#pragma unroll
    for (int k = 0; k < kVec; k++) r.v[k] = x;
    return r;
}
template <class T>
__device__ __forceinline__ f8 load8_or(const T *row, int c, int D, float other) {
    return row ? load8(row, c, D) : all8(other);
}
template <class T>
__device__ __forceinline__ void store8(T *row, int c, int D, const f8 &x) {
    typename Raw<T>::type o;
#pragma unroll
    for (int k = 0; k < kVec; k++) o[k] = (T)x.v[k];
    if (c + kVec <= D) {
        *(typename Raw<T>::type *)(row + c) = o;
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k++)
            if (c + k < D) row[c + k] = o[k];
    }
}

// K sums over the TPR threads of a row, in every one of them. Over several waves through LDS: `turn` alternates between two
// buffers, so that one barrier a sum is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&s)[K], int &turn) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o >= 1; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; k++) s[k] += __shfl_xor(s[k], o, 64);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        __shared__ float red[2][2][W];
        static_assert(K <= 2, "two sums at a time");
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) red[turn][k][threadIdx.x >> 6] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            s[k] = red[turn][k][0];
#pragma unroll
            for (int w = 1; w < W; w++) s[k] += red[turn][k][w];
        }
        turn ^= 1;
    }
}

// Mean and inverse deviation of two rows at once (a, b: their eight columns from c on here, for every c).
struct Stats {
    float m, r;
};
// each(f): f(c, a, b) for each of this thread's column groups. One pass for the sums, and one for layer norms' squares about the mean.
template <int TPR, class Each>
__device__ __forceinline__ void stats2(int D, int ka, int kb, float eps, Each each, Stats &A, Stats &B, int &turn) {
    const float n = 1.0f / (float)D;
    float s[2] = {};
    if (ka == AH_NORM_LAYER || kb == AH_NORM_LAYER) {
        each([&](int, const f8 &a, const f8 &b) {
#pragma unroll
            for (int k = 0; k < kVec; k++) {
                s[0] += a.v[k];
                s[1] += b.v[k];
            }
        });
        row_sums<TPR>(s, turn);
    }
    A.m = ka == AH_NORM_LAYER ? s[0] * n : 0.0f;
    B.m = kb == AH_NORM_LAYER ? s[1] * n : 0.0f;
    s[0] = s[1] = 0.0f;
    each([&](int c, const f8 &a, const f8 &b) {
#pragma unroll
        for (int k = 0; k < kVec; k++) {
            const float x = c + k < D ? a.v[k] - A.m : 0.0f, y = c + k < D ? b.v[k] - B.m : 0.0f;
            s[0] = fmaf(x, x, s[0]);
            s[1] = fmaf(y, y, s[1]);
        }
    });
    row_sums<TPR>(s, turn);
    A.r = 1.0f / sqrtf(s[0] * n + eps);
    B.r = 1.0f / sqrtf(s[1] * n + eps);
}
template <int TPR, class Each>
__device__ __forceinline__ Stats stats1(int D, int kind, float eps, Each each, int &turn) {
    const float n = 1.0f / (float)D;
    Stats S{};
    float s[1] = {};
    if (kind == AH_NORM_LAYER) {
        each([&](int, const f8 &a) {
#pragma unroll
            for (int k = 0; k < kVec; k++) s[0] += a.v[k];
        });
        row_sums<TPR>(s, turn);
        S.m = s[0] * n;
        s[0] = 0.0f;
    }
    each([&](int c, const f8 &a) {
#pragma unroll
        for (int k = 0; k < kVec; k++) {
            const float x = c + k < D ? a.v[k] - S.m : 0.0f;
            s[0] = fmaf(x, x, s[0]);
        }
    });
    row_sums<TPR>(s, turn);
    S.r = 1.0f / sqrtf(s[0] * n + eps);
    return S;
}

// ── forward ────────────────────────────────────────────────────────────────────

// T: Y, O, gate and weights; R: the residual stream. VPT: column groups that a thread holds; 0: rows are read again for each pass.
template <class T, class R, int TPR, int VPT>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void resnorm_kernel(ah_residual_norm_desc d) {
    constexpr int PER = TPR <= 64 ? 256 / TPR : 1, V = VPT ? VPT : 1;
    const int t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, D = d.D;
    int turn = 0;
    const T *pw = (const T *)d.post_w, *pb = (const T *)d.post_b, *nw = (const T *)d.pre_w, *nb = (const T *)d.pre_b;
    for (long r = (long)blockIdx.x * PER + (TPR <= 64 ? threadIdx.x / TPR : 0); r < ((d.N + PER - 1) / PER) * (long)PER; r += (long)gridDim.x * PER) {
        const bool on = PER == 1 || r < d.N;   // lanes past the last row keep their wave company
        const long row = on ? r : d.N - 1;
        const R *H = d.H ? (const R *)d.H + row * d.ldh : nullptr;
        const T *Y = d.Y ? (const T *)d.Y + row * d.ldy : nullptr;
        const T *G = d.gate ? (const T *)d.gate + (long)(d.rows_per_gate ? (int)row / d.rows_per_gate : 0) * d.ldgate : nullptr;
        f8 y[V], h[V];
        const auto groups = [&](auto f) {   // f(v, c): this thread's column groups
            if constexpr (VPT == 0) {
                for (int c = t * kVec; c < D; c += TPR * kVec) f(0, c);
            } else {
#pragma unroll
                for (int v = 0; v < VPT; v++)
                    if ((v * TPR + t) * kVec < D) f(v, (v * TPR + t) * kVec);
            }
        };
        if constexpr (VPT > 0)
            groups([&](int v, int c) {
                if (Y) y[v] = load8(Y, c, D);
                if (H) h[v] = load8(H, c, D);
            });
        const auto y_at = [&](int v, int c) {
            if constexpr (VPT == 0) return load8(Y, c, D);
            else return y[v];
        };
        Stats P{0.0f, 1.0f};
        if (Y && d.post != AH_NORM_NONE)
            P = stats1<TPR>(D, d.post, d.eps, [&](auto f) { groups([&](int v, int c) { f(c, y_at(v, c)); }); }, turn);
        const auto sum_at = [&](int v, int c) {
            f8 s = {};
            if (Y) {
                s = y_at(v, c);
                if (d.post != AH_NORM_NONE) {
                    const f8 w = load8_or(pw, c, D, 1.0f);
#pragma unroll
                    for (int k = 0; k < kVec; k++) s.v[k] = (s.v[k] - P.m) * P.r * w.v[k];
                    if (d.post == AH_NORM_LAYER && pb) {
                        const f8 b = load8(pb, c, D);
#pragma unroll
                        for (int k = 0; k < kVec; k++) s.v[k] += b.v[k];
                    }
                }
                const f8 g = load8_or(G, c, D, 1.0f);
#pragma unroll
                for (int k = 0; k < kVec; k++) s.v[k] *= d.scale * g.v[k];
            }
            if (H) {
                f8 x;
                if constexpr (VPT == 0) x = load8(H, c, D);
                else x = h[v];
#pragma unroll
                for (int k = 0; k < kVec; k++) s.v[k] = fmaf(d.skip, x.v[k], s.v[k]);
            }
            return s;
        };
        if constexpr (VPT > 0)
            groups([&](int v, int c) {
                h[v] = sum_at(v, c);
                if (d.H_out && on) store8((R *)d.H_out + row * d.ldh_out, c, D, h[v]);
            });
        const auto h_at = [&](int v, int c) {
            if constexpr (VPT == 0) return sum_at(v, c);
            else return h[v];
        };
        Stats Q{0.0f, 1.0f};
        if (d.O) Q = stats1<TPR>(D, d.pre, d.eps, [&](auto f) { groups([&](int v, int c) { f(c, h_at(v, c)); }); }, turn);
        if (d.O || VPT == 0)
            groups([&](int v, int c) {
                f8 s = h_at(v, c);
                if (VPT == 0 && d.H_out) store8((R *)d.H_out + row * d.ldh_out, c, D, s);   // after the row's last reading: H_out may be H
                if (!d.O) return;
                const f8 w = load8_or(nw, c, D, 1.0f);
#pragma unroll
                for (int k = 0; k < kVec; k++) s.v[k] = (s.v[k] - Q.m) * Q.r * w.v[k];
                if (d.pre == AH_NORM_LAYER && nb) {
                    const f8 b = load8(nb, c, D);
#pragma unroll
                    for (int k = 0; k < kVec; k++) s.v[k] += b.v[k];
                }
                if (on) store8((T *)d.O + row * d.ldo, c, D, s);
            });
    }
}

// ── backward ───────────────────────────────────────────────────────────────────

// Workers' runs and where their sums go.
struct Runs {
    int workers, n;        // rows n, worker w has [w n / workers, (w + 1) n / workers)
    int per;               // rows of a gate (n where one serves all)
    int arrays;            // column sums of a worker that are wanted: places 0 .. arrays-1
    int wpre, bpre, wpost, bpost;   // their places, -1: not wanted
    float *sums;           // [worker][arrays][D]
    float *gates;          // [worker][2][D]: the gate that began before the run, the one that goes on after it (null: every gate is whole)
    __host__ __device__ int row(int w) const { return (int)((long)w * n / workers); }
};

// What a row's gradient needs of its statistics.
struct RowStats {
    Stats y, h;
    float q1, qx, p1, px;  // means of q, q xh, p, p yh
};

struct Slots {   // a thread's sums over rows
    f8 wpre, bpre, wpost, bpost, gate;
};

struct RowCols {   // a row's values in a thread's columns
    f8 y, h, dh, dO, g;
};

// t from the row's values: the gradient of h.
__device__ __forceinline__ f8 grad_h(const RowCols &x, const f8 &wn, const RowStats &s, int pre) {
    f8 t = x.dh;
    if (pre != AH_NORM_NONE) {
#pragma unroll
        for (int k = 0; k < kVec; k++) {
            const float xh = (x.h.v[k] - s.h.m) * s.h.r, q = x.dO.v[k] * wn.v[k];
            t.v[k] += s.h.r * (q - s.qx * xh - s.q1);
        }
    }
    return t;
}

// The columns' sums gain a row. layer: some norm has a bias.
template <bool LAYER>
__device__ __forceinline__ void add_row(Slots &a, const RowCols &x, const f8 &t, const f8 &wp, const f8 &bp, const RowStats &s, float scale) {
#pragma unroll
    for (int k = 0; k < kVec; k++) {
        const float xh = (x.h.v[k] - s.h.m) * s.h.r, yh = (x.y.v[k] - s.y.m) * s.y.r, v = scale * t.v[k];
        a.wpre.v[k] = fmaf(x.dO.v[k], xh, a.wpre.v[k]);
        a.wpost.v[k] = fmaf(v * x.g.v[k], yh, a.wpost.v[k]);
        float u = yh * wp.v[k];
        if constexpr (LAYER) {
            a.bpre.v[k] += x.dO.v[k];
            a.bpost.v[k] = fmaf(v, x.g.v[k], a.bpost.v[k]);
            u += bp.v[k];
        }
        a.gate.v[k] = fmaf(v, u, a.gate.v[k]);
    }
}

// Gate `index`, whose rows the run [a, b) of worker w has come to the end of: into dgate if they are all in the run, else into one
// of the worker's two places.
template <class T>
__device__ __forceinline__ void put_gate(const ah_residual_norm_grad_desc &d, const Runs &u, int w, int a, int b, long index, int c, const f8 &v) {
    const long first = index * u.per, end = min(first + (long)u.per, (long)u.n);
    if (first >= a && end <= b) store8((T *)d.dgate + index * d.lddgate, c, d.D, v);
    else store8(u.gates + ((long)w * 2 + (first < a ? 0 : 1)) * d.D, c, d.D, v);
}

__device__ __forceinline__ void put_sums(const Runs &u, int w, int c, int D, const Slots &s) {
    float *p = u.sums + (long)w * u.arrays * D;
    if (u.wpre >= 0) store8(p + (long)u.wpre * D, c, D, s.wpre);
    if (u.bpre >= 0) store8(p + (long)u.bpre * D, c, D, s.bpre);
    if (u.wpost >= 0) store8(p + (long)u.wpost * D, c, D, s.wpost);
    if (u.bpost >= 0) store8(p + (long)u.bpost * D, c, D, s.bpost);
}

// Rows of up to 8 TPR columns, TPR threads a worker. AHEAD: the next row's loads go out before this row's work (its values as they lie, 20
// or 40 registers).
template <class T, class R, int TPR, bool LAYER, bool AHEAD>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void resnorm_grad_kernel(ah_residual_norm_grad_desc d, Runs u) {
    constexpr int PER = TPR <= 64 ? 256 / TPR : 1;
    const int t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, D = d.D, c = t * kVec;
    const int w = blockIdx.x * PER + (TPR <= 64 ? threadIdx.x / TPR : 0);
    if (PER > 1 && w >= u.workers) return;   // whole groups of lanes; shuffles stay within a group
    const int a = u.row(w), b = u.row(w + 1);
    const bool in = c < D, ln_pre = d.pre == AH_NORM_LAYER, ln_post = d.post == AH_NORM_LAYER;
    const bool rd_y = in && d.Y, rd_h = in && d.H_out, rd_dh = in && d.dH_out, rd_dO = in && d.dO, rd_g = in && d.gate;
    int turn = 0;
    typedef typename Raw<T>::type rawT;
    typedef typename Raw<R>::type rawR;
    struct Line {
        rawT y, dO, g;
        rawR h, dh;
    };
    const auto fetch = [&](int r, long gate) {
        Line l = {};
        if (rd_y) l.y = load_raw((const T *)d.Y + (long)r * d.ldy, c, D);
        if (rd_dO) l.dO = load_raw((const T *)d.dO + (long)r * d.lddo, c, D);
        if (rd_h) l.h = load_raw((const R *)d.H_out + (long)r * d.ldh_out, c, D);
        if (rd_dh) l.dh = load_raw((const R *)d.dH_out + (long)r * d.lddh_out, c, D);
        if (rd_g) l.g = load_raw((const T *)d.gate + gate * d.ldgate, c, D);
        return l;
    };
    f8 wn = all8(1.0f), wp = all8(1.0f), bp = all8(0.0f);
    if (in) {
        if (d.pre_w) wn = load8((const T *)d.pre_w, c, D);
        if (d.post_w) wp = load8((const T *)d.post_w, c, D);
        if (LAYER && ln_post && d.post_b) bp = load8((const T *)d.post_b, c, D);
    }
    Slots sums = {};
    long gate = a / u.per;
    int left = (int)min((long)u.per - a % u.per, (long)0x7fffffff);   // rows to the gate's end
    Line next = {};
    if (AHEAD && a < b) next = fetch(a, gate);
    const float n = 1.0f / (float)D;
    for (int r = a; r < b; r++) {
        Line l;
        const long gate_next = left == 1 ? gate + 1 : gate;
        if constexpr (AHEAD) {
            l = next;
            if (r + 1 < b) next = fetch(r + 1, gate_next);
        } else {
            l = fetch(r, gate);
        }
        RowCols x{widen(l.y), widen(l.h), widen(l.dh), widen(l.dO), rd_g ? widen(l.g) : all8(1.0f)};
        RowStats s{{0.0f, 1.0f}, {0.0f, 1.0f}, 0.0f, 0.0f, 0.0f, 0.0f};
        if (d.pre != AH_NORM_NONE || d.post != AH_NORM_NONE) {
            stats2<TPR>(D, d.post, d.pre, d.eps, [&](auto f) { f(c, x.y, x.h); }, s.y, s.h, turn);
            if (d.post == AH_NORM_NONE) s.y = {0.0f, 1.0f};
            if (d.pre == AH_NORM_NONE) s.h = {0.0f, 1.0f};
        }
        if (d.pre != AH_NORM_NONE) {
            float m[2] = {};
#pragma unroll
            for (int k = 0; k < kVec; k++) {   // dO is 0 past the last column
                const float q = x.dO.v[k] * wn.v[k];
                m[0] = fmaf(q, (x.h.v[k] - s.h.m) * s.h.r, m[0]);
                m[1] += q;
            }
            row_sums<TPR>(m, turn);
            s.qx = m[0] * n;
            s.q1 = ln_pre ? m[1] * n : 0.0f;
        }
        const f8 tt = grad_h(x, wn, s, d.pre);
        if (d.dH && in) {
            f8 o;
#pragma unroll
            for (int k = 0; k < kVec; k++) o.v[k] = d.skip * tt.v[k];
            store8((R *)d.dH + (long)r * d.lddh, c, D, o);
        }
        if (d.dY) {
            f8 p;
#pragma unroll
            for (int k = 0; k < kVec; k++) p.v[k] = d.scale * x.g.v[k] * tt.v[k];
            if (d.post != AH_NORM_NONE) {
                float m[2] = {};
#pragma unroll
                for (int k = 0; k < kVec; k++) {
                    p.v[k] = c + k < D ? p.v[k] * wp.v[k] : 0.0f;
                    m[0] = fmaf(p.v[k], (x.y.v[k] - s.y.m) * s.y.r, m[0]);
                    m[1] += p.v[k];
                }
                row_sums<TPR>(m, turn);
                s.px = m[0] * n;
                s.p1 = ln_post ? m[1] * n : 0.0f;
#pragma unroll
                for (int k = 0; k < kVec; k++) p.v[k] = s.y.r * (p.v[k] - s.px * ((x.y.v[k] - s.y.m) * s.y.r) - s.p1);
            }
            if (in) store8((T *)d.dY + (long)r * d.lddy, c, D, p);
        }
        add_row<LAYER>(sums, x, tt, wp, bp, s, d.scale);
        if (--left == 0 || r + 1 == b) {
            if (d.dgate && in) put_gate<T>(d, u, w, a, b, gate, c, sums.gate);
            sums.gate = all8(0.0f);
            gate = gate_next;
            left = u.per;
        }
    }
    if (u.arrays && in) put_sums(u, w, c, D, sums);
}

// Rows of any width, a workgroup a row: dH and dY by several readings of the row, and its statistics for the columns' sums.
constexpr int kWideT = 1024;
template <class T, class R>
__global__ __launch_bounds__(kWideT) void resnorm_grad_wide_kernel(ah_residual_norm_grad_desc d, RowStats *rows) {
    const int D = d.D;
    const float n = 1.0f / (float)D;
    const T *wn = (const T *)d.pre_w, *wp = (const T *)d.post_w;
    int turn = 0;
    const auto groups = [&](auto f) {
        for (int c = threadIdx.x * kVec; c < D; c += kWideT * kVec) f(c);
    };
    for (long r = blockIdx.x; r < d.N; r += gridDim.x) {
        const T *Y = d.Y ? (const T *)d.Y + r * d.ldy : nullptr, *dO = d.dO ? (const T *)d.dO + r * d.lddo : nullptr;
        const T *G = d.gate ? (const T *)d.gate + (long)(d.rows_per_gate ? (int)r / d.rows_per_gate : 0) * d.ldgate : nullptr;
        const R *H = d.H_out ? (const R *)d.H_out + r * d.ldh_out : nullptr, *dh = d.dH_out ? (const R *)d.dH_out + r * d.lddh_out : nullptr;
        RowStats s{{0.0f, 1.0f}, {0.0f, 1.0f}, 0.0f, 0.0f, 0.0f, 0.0f};
        if (d.post != AH_NORM_NONE) s.y = stats1<kWideT>(D, d.post, d.eps, [&](auto f) { groups([&](int c) { f(c, load8(Y, c, D)); }); }, turn);
        if (d.pre != AH_NORM_NONE) {
            s.h = stats1<kWideT>(D, d.pre, d.eps, [&](auto f) { groups([&](int c) { f(c, load8(H, c, D)); }); }, turn);
            float m[2] = {};
            groups([&](int c) {
                const f8 h = load8(H, c, D), g = load8(dO, c, D), w = load8_or(wn, c, D, 1.0f);
#pragma unroll
                for (int k = 0; k < kVec; k++) {
                    const float q = g.v[k] * w.v[k];
                    m[0] = fmaf(q, (h.v[k] - s.h.m) * s.h.r, m[0]);
                    m[1] += q;
                }
            });
            row_sums<kWideT>(m, turn);
            s.qx = m[0] * n;
            s.q1 = d.pre == AH_NORM_LAYER ? m[1] * n : 0.0f;
        }
        const auto t_at = [&](int c) {
            RowCols x{};
            if (H) x.h = load8(H, c, D);
            if (dO) x.dO = load8(dO, c, D);
            if (dh) x.dh = load8(dh, c, D);
            return grad_h(x, load8_or(wn, c, D, 1.0f), s, d.pre);
        };
        const auto p_at = [&](int c) {
            f8 t = t_at(c);
            const f8 g = load8_or(G, c, D, 1.0f), w = d.post != AH_NORM_NONE ? load8_or(wp, c, D, 1.0f) : all8(1.0f);
#pragma unroll
            for (int k = 0; k < kVec; k++) t.v[k] = c + k < D ? d.scale * g.v[k] * t.v[k] * w.v[k] : 0.0f;
            return t;
        };
        if (d.dY && d.post != AH_NORM_NONE) {
            float m[2] = {};
            groups([&](int c) {
                const f8 p = p_at(c), y = load8(Y, c, D);
#pragma unroll
                for (int k = 0; k < kVec; k++) {
                    m[0] = fmaf(p.v[k], (y.v[k] - s.y.m) * s.y.r, m[0]);
                    m[1] += p.v[k];
                }
            });
            row_sums<kWideT>(m, turn);
            s.px = m[0] * n;
            s.p1 = d.post == AH_NORM_LAYER ? m[1] * n : 0.0f;
        }
        groups([&](int c) {
            if (d.dY) {
                f8 p = p_at(c);
                if (d.post != AH_NORM_NONE) {
                    const f8 y = load8(Y, c, D);
#pragma unroll
                    for (int k = 0; k < kVec; k++) p.v[k] = s.y.r * (p.v[k] - s.px * ((y.v[k] - s.y.m) * s.y.r) - s.p1);
                }
                store8((T *)d.dY + r * d.lddy, c, D, p);
            }
        });
        if (rows && threadIdx.x == 0) rows[r] = s;
    }
}
// The columns' sums, and dH last of all: it may be dH_out, which the rows' gradients are read from. A workgroup has 2048 columns.
template <class T, class R>
__global__ __launch_bounds__(256) void resnorm_grad_columns_kernel(ah_residual_norm_grad_desc d, Runs u, const RowStats *rows) {
    const int D = d.D, c = (blockIdx.x * 256 + threadIdx.x) * kVec, w = blockIdx.y;
    if (c >= D) return;
    const int a = u.row(w), b = u.row(w + 1);
    const f8 wn = load8_or((const T *)d.pre_w, c, D, 1.0f), wp = load8_or((const T *)d.post_w, c, D, 1.0f);
    const f8 bp = load8_or(d.post == AH_NORM_LAYER ? (const T *)d.post_b : nullptr, c, D, 0.0f);
    Slots sums = {};
    long gate = a / u.per;
    int left = u.per - a % u.per;
    for (int r = a; r < b; r++) {
        RowCols x{};
        if (d.Y) x.y = load8((const T *)d.Y + (long)r * d.ldy, c, D);
        if (d.H_out) x.h = load8((const R *)d.H_out + (long)r * d.ldh_out, c, D);
        if (d.dH_out) x.dh = load8((const R *)d.dH_out + (long)r * d.lddh_out, c, D);
        if (d.dO) x.dO = load8((const T *)d.dO + (long)r * d.lddo, c, D);
        x.g = load8_or(d.gate ? (const T *)d.gate + gate * d.ldgate : nullptr, c, D, 1.0f);
        const RowStats s = rows[r];
        const f8 t = grad_h(x, wn, s, d.pre);
        if (d.dH) {
            f8 o;
#pragma unroll
            for (int k = 0; k < kVec; k++) o.v[k] = d.skip * t.v[k];
            store8((R *)d.dH + (long)r * d.lddh, c, D, o);
        }
        add_row<true>(sums, x, t, wp, bp, s, d.scale);
        if (--left == 0 || r + 1 == b) {
            if (d.dgate) put_gate<T>(d, u, w, a, b, gate, c, sums.gate);
            sums.gate = all8(0.0f);
            gate++;
            left = u.per;
        }
    }
    if (u.arrays) put_sums(u, w, c, D, sums);
}

// The workers' sums added in order: 64 columns a workgroup, 16 threads a column with neighbouring workers each. blockIdx.y: an array, or past
// those a gate that several workers have rows of: gate by gate, or where there are more gates than bounds between runs, bound by bound.
template <class T>
__global__ __launch_bounds__(1024) void resnorm_join_kernel(ah_residual_norm_grad_desc d, Runs u, int gates, int by_bound) {
    __shared__ float red[16][64];
    const int D = d.D, c = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    int w0 = 0, w1 = u.workers;   // the workers that are added
    long gate = -1, first = 0;
    if ((int)blockIdx.y >= u.arrays) {
        gate = blockIdx.y - u.arrays;
        if (by_bound) {
            w0 = (int)gate + 1;
            const int a = u.row(w0);
            gate = a / u.per;
            first = gate * u.per;
            if (first == a || u.row(w0 - 1) > first) return;   // no gate, or one of an earlier bound
            w0--;
        } else {
            first = gate * u.per;
            w0 = (int)(((first + 1) * u.workers - 1) / u.n);   // the last worker that begins at or before `first`
        }
        const long end = min(first + (long)u.per, (long)u.n);
        if (u.row(w0 + 1) >= end) return;   // all rows in one run
        w1 = (int)((end * u.workers + u.n - 1) / u.n);         // the first worker that begins at or after `end`
    }
    const int each = (w1 - w0 + 15) / 16, lo = w0 + part * each, hi = min(w1, lo + each);
    float s = 0.0f;
    if (c < D) {
        if (gate < 0) {
#pragma unroll 8
            for (int w = lo; w < hi; w++) s += u.sums[((long)w * u.arrays + blockIdx.y) * D + c];
        } else {
#pragma unroll 8
            for (int w = lo; w < hi; w++) s += u.gates[((long)w * 2 + (w == w0 ? 1 : 0)) * D + c];
        }
    }
    red[part][threadIdx.x & 63] = s;
    __syncthreads();
    if (part || c >= D) return;
    for (int k = 1; k < 16; k++) s += red[k][threadIdx.x];
    if (gate >= 0) {
        ((T *)d.dgate)[gate * d.lddgate + c] = (T)s;
        return;
    }
    float *out = (int)blockIdx.y == u.wpre ? d.dpre_w : (int)blockIdx.y == u.bpre ? d.dpre_b : (int)blockIdx.y == u.wpost ? d.dpost_w : d.dpost_b;
    out[c] = s;
}

// ── host ───────────────────────────────────────────────────────────────────────

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Threads a row: the power of two that holds it in groups of eight columns.
int threads_of(int D) {
    int t = 8;
    while (t < 1024 && t * kVec < D) t *= 2;
    return t;
}

template <class T, class R>
void launch_forward(const ah_residual_norm_desc &d, hipStream_t s) {
    const int tpr = threads_of(d.D), per = tpr <= 64 ? 256 / tpr : 1;
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(d.N, per), 16384)), block(tpr <= 64 ? 256 : tpr);
    switch (d.D > kWide ? 0 : tpr) {
        case 8: hipLaunchKernelGGL((resnorm_kernel<T, R, 8, 1>), grid, block, 0, s, d); break;
        case 16: hipLaunchKernelGGL((resnorm_kernel<T, R, 16, 1>), grid, block, 0, s, d); break;
        case 32: hipLaunchKernelGGL((resnorm_kernel<T, R, 32, 1>), grid, block, 0, s, d); break;
        case 64: hipLaunchKernelGGL((resnorm_kernel<T, R, 64, 1>), grid, block, 0, s, d); break;
        case 128: hipLaunchKernelGGL((resnorm_kernel<T, R, 128, 1>), grid, block, 0, s, d); break;
        case 256: hipLaunchKernelGGL((resnorm_kernel<T, R, 256, 1>), grid, block, 0, s, d); break;
        case 512: hipLaunchKernelGGL((resnorm_kernel<T, R, 512, 1>), grid, block, 0, s, d); break;
        case 1024: hipLaunchKernelGGL((resnorm_kernel<T, R, 1024, 1>), grid, block, 0, s, d); break;
        default: hipLaunchKernelGGL((resnorm_kernel<T, R, 1024, 0>), grid, block, 0, s, d);
    }
}

struct Plan {
    int tpr;             // 0: wide rows
    Runs u;
    int gates, by_bound; // gates that workers may share, and how the join finds them
    int64_t rows, total; // of the workspace: the wide rows' statistics
};

Plan plan_of(const ah_residual_norm_grad_desc &d) {
    Plan p{};
    p.tpr = d.D > kWide ? 0 : threads_of(d.D);
    Runs &u = p.u;
    u.n = d.N;
    u.per = d.rows_per_gate && d.rows_per_gate < d.N ? d.rows_per_gate : d.N;
    u.wpre = u.bpre = u.wpost = u.bpost = -1;
    if (d.dpre_w) u.wpre = u.arrays++;
    if (d.dpre_b) u.bpre = u.arrays++;
    if (d.dpost_w) u.wpost = u.arrays++;
    if (d.dpost_b) u.bpost = u.arrays++;
    // Workers: enough to fill the chip, with at least four rows each where there are many (a worker's sums cross memory twice).
    const int cap = p.tpr == 0 ? 256 : p.tpr <= 64 ? 512 * (256 / p.tpr) : p.tpr == 128 ? 1024 : p.tpr == 256 ? 512 : 256;
    u.workers = std::max(1, std::min(cap, std::max(std::min(d.N, 256), d.N / 4)));
    u.workers = std::min(u.workers, d.N);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at = (at + bytes + 255) & ~255ll;
        return o;
    };
    u.sums = (float *)take((int64_t)u.workers * u.arrays * d.D * 4);
    const int gates = ceil_div(d.N, u.per);
    const bool shared = d.dgate && u.per > 1 && u.workers > 1;
    u.gates = (float *)take(shared ? (int64_t)u.workers * 2 * d.D * 4 : 0);
    if (shared) {
        p.by_bound = gates > u.workers - 1;
        p.gates = std::min(gates, u.workers - 1);
    }
    p.rows = take(p.tpr == 0 ? (int64_t)d.N * sizeof(RowStats) : 0);
    p.total = std::max<int64_t>(at, 16);
    return p;
}

template <class T, class R, int TPR>
void launch_grad_rows(const ah_residual_norm_grad_desc &d, const Plan &p, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(p.u.workers, TPR <= 64 ? 256 / TPR : 1)), block(TPR <= 64 ? 256 : TPR);
    constexpr bool AHEAD = TPR <= 512;
    if (d.pre == AH_NORM_LAYER || d.post == AH_NORM_LAYER) hipLaunchKernelGGL((resnorm_grad_kernel<T, R, TPR, true, AHEAD>), grid, block, 0, s, d, p.u);
    else hipLaunchKernelGGL((resnorm_grad_kernel<T, R, TPR, false, AHEAD>), grid, block, 0, s, d, p.u);
}

template <class T, class R>
void launch_grad(const ah_residual_norm_grad_desc &d, Plan p, hipStream_t s) {
    char *ws = (char *)d.ws;
    p.u.sums = (float *)(ws + (uintptr_t)p.u.sums);
    p.u.gates = (float *)(ws + (uintptr_t)p.u.gates);
    switch (p.tpr) {
        case 8: launch_grad_rows<T, R, 8>(d, p, s); break;
        case 16: launch_grad_rows<T, R, 16>(d, p, s); break;
        case 32: launch_grad_rows<T, R, 32>(d, p, s); break;
        case 64: launch_grad_rows<T, R, 64>(d, p, s); break;
        case 128: launch_grad_rows<T, R, 128>(d, p, s); break;
        case 256: launch_grad_rows<T, R, 256>(d, p, s); break;
        case 512: launch_grad_rows<T, R, 512>(d, p, s); break;
        case 1024: launch_grad_rows<T, R, 1024>(d, p, s); break;
        default: {
            RowStats *rows = (RowStats *)(ws + p.rows);
            hipLaunchKernelGGL((resnorm_grad_wide_kernel<T, R>), dim3((unsigned)std::min(d.N, 16384)), dim3(kWideT), 0, s, d, rows);
            hipLaunchKernelGGL((resnorm_grad_columns_kernel<T, R>), dim3((unsigned)ceil_div(d.D, 256 * kVec), (unsigned)p.u.workers), dim3(256), 0, s, d, p.u, rows);
        }
    }
    if (p.u.arrays + p.gates)
        hipLaunchKernelGGL(resnorm_join_kernel<T>, dim3((unsigned)ceil_div(d.D, 64), (unsigned)(p.u.arrays + p.gates)), dim3(1024), 0, s, d, p.u, p.gates, p.by_bound);
}

}  // namespace

hipError_t residual_norm(const ah_residual_norm_desc &d, hipStream_t s) {
    if (d.dtype == AH_F32) launch_forward<float, float>(d, s);
    else if (d.res_dtype == AH_F32) launch_forward<half_t, float>(d, s);
    else launch_forward<half_t, half_t>(d, s);
    return hipGetLastError();
}

int64_t residual_norm_grad_workspace(const ah_residual_norm_grad_desc &d) { return plan_of(d).total; }

hipError_t residual_norm_grad(const ah_residual_norm_grad_desc &d, hipStream_t s) {
    const Plan p = plan_of(d);
    if (d.dtype == AH_F32) launch_grad<float, float>(d, p, s);
    else if (d.res_dtype == AH_F32) launch_grad<half_t, float>(d, p, s);
    else launch_grad<half_t, half_t>(d, p, s);
    return hipGetLastError();
}

}  // namespace ah
