// resnorm.hip — norms after and before a block, fused with its gate and the residual sum, and their gradients.
//
//   u = post(Y),  h = skip H + scale g u,  O = pre(h)             norm(x) = (x - m) r w + b,  r = 1 / sqrt(mean (x - m)^2 + eps)
//   t = dh + r_h (q - mean(q xh) xh - mean(q)),  q = dO w_pre     (m, b, mean(q): layer norms alone; xh = (h - m) r_h, yh likewise)
//   dH = skip t,  dg = sum scale t u,  dY = r_y (p - mean(p yh) yh - mean(p)),  p = scale g t w_post
//   dw_pre = sum dO xh,  db_pre = sum dO,  dw_post = sum scale g t yh,  db_post = sum scale g t
//
// Bound by memory: each array is read and written once, a row's statistics are taken from registers (f16 on an f32 stream, 16384 x 4096 rms twice:
// 150 us, 5.4 TB/s). A row belongs to TPR threads, eight columns to each (sixteen from 8192 to 16384 columns; longer rows are read again for
// each pass, from caches mostly); up to 64 threads rows share a wave and are joined by lane exchanges alone, above that they are a workgroup.
// The backward pass holds the columns' sums in registers: a group of threads (a worker) walks down a run of neighbouring rows with the next
// row's loads in flight, and leaves its sums in the workspace, where a second launch adds them in the workers' order (f16, the same size: 178 us,
// 4.6 TB/s; f32, 1999 x 1001 with layer norms: 23, latency). A run that begins or ends inside a gate's rows leaves that gate's part there too;
// the sums of gates whose rows are all its own it writes itself. Rows that 1024 threads do not hold take two launches, the rows' terms and
// then the columns (4000 x 12000 f16: 239 us, 4000 x 6000 f32 with layer norms 217; one launch with fewer threads' registers spilled 280).
#include "resnorm.h"

#include <algorithm>
#include <type_traits>

#include "vec8.h"

namespace ah {
namespace {

constexpr int kVec = 8;            // columns of a thread
constexpr int kWide = 8192;        // columns that a workgroup's registers hold
constexpr int kTermsT = 512;       // threads of a row whose terms are a launch of their own

template <class T>
__device__ __forceinline__ f8 load8_or(const T *row, int c, int D, float other) {
    return row ? load8(row, c, D) : all_of<kVec>(other);
}

// x from another lane of the row of 16: CTRL is a lane permutation of the cross-lane adder.
template <int CTRL>
__device__ __forceinline__ float lane_of(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xF, 0xF, true));
}
// Sum over groups of G lanes, in each of them: neighbours, pairs, then mirrored within 8 and 16 lanes, and the halves of 32 and 64 exchanged.
template <int G>
__device__ __forceinline__ float lanes_sum(float x) {
    if constexpr (G >= 2) x += lane_of<0xB1>(x);    // 1 0 3 2
    if constexpr (G >= 4) x += lane_of<0x4E>(x);    // 2 3 0 1
    if constexpr (G >= 8) x += lane_of<0x141>(x);   // 7 .. 0
    if constexpr (G >= 16) x += lane_of<0x140>(x);  // 15 .. 0
    if constexpr (G >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    if constexpr (G >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    return x;
}
// K sums over the TPR threads of a row, in every one of them. Over several waves through LDS, where each lane then reads one wave's sums
// and groups of lanes add those: `turn` alternates between two buffers, so that one barrier is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&s)[K], int &turn) {
#pragma unroll
    for (int k = 0; k < K; k++) s[k] = lanes_sum<TPR < 64 ? TPR : 64>(s[k]);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64, KP = K + (K & 1);   // (8-byte accesses)
        __shared__ __attribute__((aligned(16))) float red[2][W][KP];
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) red[turn][threadIdx.x >> 6][k] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) s[k] = red[turn][threadIdx.x & (W - 1)][k];
#pragma unroll
        for (int k = 0; k < K; k++) s[k] = lanes_sum<W>(s[k]);
        turn ^= 1;
    }
}

// A row whose mean square v (with eps) is past f32's range, or so small that the squares have lost bits, is scaled by a power of two before it is
// squared again: |x| up to 2^128 to 2^52 at most, and from 2^-149 to below 2^-48 (where eps, below 2^-96 then, keeps its share) past 2^-59.
__device__ __forceinline__ float rescale(float v) { return v < 0x1p-96f ? 0x1p90f : v < __builtin_inff() ? 1.0f : 0x1p-76f; }

struct Stats {
    float m, r, up;   // the norm is ((x - m) up) r
};
// Mean and inverse deviation of a row. each(f): f(c, a) for each of this thread's column groups. One pass for the sum, and one for layer
// norms' squares about the mean.
template <int TPR, class Each>
__device__ __forceinline__ Stats stats1(int D, int kind, float eps, Each each, int &turn) {
    const float n = 1.0f / (float)D;
    Stats S{0.0f, 0.0f, 1.0f};
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
    const auto square = [&] {
        s[0] = 0.0f;
        each([&](int c, const f8 &a) {
#pragma unroll
            for (int k = 0; k < kVec; k++) {
                const float x = c + k < D ? (a.v[k] - S.m) * S.up : 0.0f;
                s[0] = fmaf(x, x, s[0]);
            }
        });
        row_sums<TPR>(s, turn);
        return fmaf(s[0], n, eps * S.up * S.up);
    };
    float v = square();
    S.up = rescale(v);
    if (S.up != 1.0f) v = square();
    S.r = 1.0f / sqrtf(v);
    return S;
}

// x less its mean, zeros past the row's end.
template <int V, bool LAYER>
__device__ __forceinline__ fN<V> less(fN<V> x, float m, int c, int D) {
    if constexpr (LAYER)
#pragma unroll
        for (int k = 0; k < V; k++) x.v[k] = c + k < D ? x.v[k] - m : 0.0f;
    return x;
}
template <int V>
__device__ __forceinline__ fN<V> times(float s, fN<V> a, const fN<V> &b) {   // s a b
#pragma unroll
    for (int k = 0; k < V; k++) a.v[k] = s * a.v[k] * b.v[k];
    return a;
}

// ── forward ────────────────────────────────────────────────────────────────────

// T: Y, O, gate and weights; R: the residual stream. Rows of up to 8 TPR columns. Weights are loaded where they are needed, from L2: held from the
// start they cost half the waves (16384 x 4096: 232 us against 160).
// G: groups of eight columns that a thread has.
template <class T, class R, int TPR, int G>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR, G == 1 ? 8 : 4) void resnorm_kernel(ah_residual_norm_desc d) {
    constexpr int PER = TPR <= 64 ? 256 / TPR : 1, V = kVec;
    constexpr bool NARROW = TPR == 8;   // there may be fewer than eight columns
    const int t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, D = d.D;
    int c0 = t * V, turn = 0;
    const auto col = [&](int g) { return c0 + g * TPR * V; };
    const auto weights = [&](const void *w, int g, float other) {
        return w && col(g) < D ? widen<V>(settle<T, V, NARROW>(load_raw<T, V, NARROW>((const T *)w, col(g), D), col(g), D)) : all_of<V>(other);
    };
    const auto normed = [&](int kind, f8 (&x)[G], const void *w, const void *b) {
        const float n = 1.0f / (float)D;
        float s[1] = {};
        if (kind == AH_NORM_LAYER) {
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < V; k++) s[0] += x[g].v[k];
            row_sums<TPR>(s, turn);
            const float m = s[0] * n;
#pragma unroll
            for (int g = 0; g < G; g++) x[g] = less<V, true>(x[g], m, col(g), D);
        }
        float up = 1.0f;
        const auto square = [&] {
            s[0] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < V; k++) s[0] = fmaf(x[g].v[k], x[g].v[k], s[0]);
            row_sums<TPR>(s, turn);
            return fmaf(s[0], n, d.eps * up * up);
        };
        float v = square();
        up = rescale(v);
        if (up != 1.0f) {   // the same in all of a row's threads
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int k = 0; k < V; k++) x[g].v[k] *= up;
            v = square();
        }
        const float r = 1.0f / sqrtf(v);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const f8 ww = weights(w, g, 1.0f), bb = weights(b, g, 0.0f);
#pragma unroll
            for (int k = 0; k < V; k++) x[g].v[k] = fmaf(x[g].v[k] * r, ww.v[k], bb.v[k]);
        }
    };
    for (long r = (long)blockIdx.x * PER + (TPR <= 64 ? threadIdx.x / TPR : 0); r < ((d.N + PER - 1) / PER) * (long)PER; r += (long)gridDim.x * PER) {
        asm volatile("" : "+v"(c0));   // addresses are formed anew for each row: kept, they cost waves
        const bool on = PER == 1 || r < d.N;   // lanes past the last row keep their wave company
        const long row = on ? r : d.N - 1;
        typename RawN<T, V>::type ry[G] = {};
        typename RawN<R, V>::type rh[G] = {};
#pragma unroll
        for (int g = 0; g < G; g++) {
            if (col(g) >= D) continue;
            if (d.Y) ry[g] = load_raw<T, V, NARROW>((const T *)d.Y + row * d.ldy, col(g), D);
            if (d.H) rh[g] = load_raw<R, V, NARROW>((const R *)d.H + row * d.ldh, col(g), D);
        }
        f8 s[G] = {};
        if (d.Y) {
#pragma unroll
            for (int g = 0; g < G; g++) s[g] = widen<V>(settle<T, V, NARROW>(ry[g], col(g), D));
            if (d.post != AH_NORM_NONE) normed(d.post, s, d.post_w, d.post_b);
            const T *gate = d.gate ? (const T *)d.gate + (long)(d.rows_per_gate ? (int)row / d.rows_per_gate : 0) * d.ldgate : nullptr;
#pragma unroll
            for (int g = 0; g < G; g++) s[g] = times<V>(d.scale, weights(gate, g, 1.0f), s[g]);
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            if (d.H) {
                const f8 h = widen<V>(settle<R, V, NARROW>(rh[g], col(g), D));
#pragma unroll
                for (int k = 0; k < V; k++) s[g].v[k] = fmaf(d.skip, h.v[k], s[g].v[k]);
            }
            if (d.H_out && on && col(g) < D) store8((R *)d.H_out + row * d.ldh_out, col(g), D, s[g]);
        }
        if (!d.O) continue;
        normed(d.pre, s, d.pre_w, d.pre_b);
#pragma unroll
        for (int g = 0; g < G; g++)
            if (on && col(g) < D) store8((T *)d.O + row * d.ldo, col(g), D, s[g]);
    }
}

// Rows of any width, a workgroup a row: read again for each pass.
constexpr int kWideT = 1024;
template <class T, class R>
__global__ __launch_bounds__(kWideT) void resnorm_wide_kernel(ah_residual_norm_desc d) {
    const int D = d.D;
    int turn = 0;
    const T *pw = (const T *)d.post_w, *pb = (const T *)d.post_b, *nw = (const T *)d.pre_w, *nb = (const T *)d.pre_b;
    const auto groups = [&](auto f) {
        for (int c = threadIdx.x * kVec; c < D; c += kWideT * kVec) f(c);
    };
    for (long r = blockIdx.x; r < d.N; r += gridDim.x) {
        const R *H = d.H ? (const R *)d.H + r * d.ldh : nullptr;
        const T *Y = d.Y ? (const T *)d.Y + r * d.ldy : nullptr;
        const T *G = d.gate ? (const T *)d.gate + (long)(d.rows_per_gate ? (int)r / d.rows_per_gate : 0) * d.ldgate : nullptr;
        Stats P{0.0f, 1.0f, 1.0f}, Q{0.0f, 1.0f, 1.0f};
        if (d.post != AH_NORM_NONE) P = stats1<kWideT>(D, d.post, d.eps, [&](auto f) { groups([&](int c) { f(c, load8(Y, c, D)); }); }, turn);
        const auto sum_at = [&](int c) {
            f8 s = {};
            if (Y) {
                s = load8(Y, c, D);
                if (d.post != AH_NORM_NONE) {
                    const f8 w = load8_or(pw, c, D, 1.0f), b = load8_or(pb, c, D, 0.0f);
#pragma unroll
                    for (int k = 0; k < kVec; k++) s.v[k] = fmaf((s.v[k] - P.m) * P.up * P.r, w.v[k], b.v[k]);
                }
                const f8 g = load8_or(G, c, D, 1.0f);
#pragma unroll
                for (int k = 0; k < kVec; k++) s.v[k] *= d.scale * g.v[k];
            }
            if (H) {
                const f8 h = load8(H, c, D);
#pragma unroll
                for (int k = 0; k < kVec; k++) s.v[k] = fmaf(d.skip, h.v[k], s.v[k]);
            }
            return s;
        };
        if (d.O) Q = stats1<kWideT>(D, d.pre, d.eps, [&](auto f) { groups([&](int c) { f(c, sum_at(c)); }); }, turn);
        groups([&](int c) {
            f8 s = sum_at(c);
            if (d.H_out) store8((R *)d.H_out + r * d.ldh_out, c, D, s);   // after the row's last reading: H_out may be H
            if (!d.O) return;
            const f8 w = load8_or(nw, c, D, 1.0f), b = load8_or(nb, c, D, 0.0f);
#pragma unroll
            for (int k = 0; k < kVec; k++) s.v[k] = fmaf((s.v[k] - Q.m) * Q.up * Q.r, w.v[k], b.v[k]);
            store8((T *)d.O + r * d.ldo, c, D, s);
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

// What a row's gradients need of its sums:
//   t = dh + c1 (q - c2 h) - c0,  c1 = r_h,  c2 = r_h (r_h mean(q h)),  c0 = r_h mean(q)
//   dY = r_y (p - px y) - p1,     px = r_y (r_y mean(p y)),  p1 = r_y mean(p),  p = a t,  a = scale g w_post
// (y, h less their means my, mh; c0, p1 of layer norms alone). c2 h and px y are as large as q and p whatever the rows' size; r^3 leaves f32's range where
// y or h is past 2^42 or, with a small eps, below 2^-42. The sums of p come from those of t's terms, so that all are taken at once:
//   sum p y = sum a y dh + c1 (sum a y q - c2 sum a y h) - c0 sum a y,  and sum p likewise
struct RowTerms {
    float my, mh, ry, c1, c2, c0, px, p1;
};
template <bool LAYER>
constexpr int kSums = LAYER ? 12 : 6;
template <int V, bool LAYER>
__device__ __forceinline__ void add_terms(float (&s)[kSums<LAYER>], const fN<V> &y, const fN<V> &h, const fN<V> &q, const fN<V> &dh, const fN<V> &a, int c, int D) {
#pragma unroll
    for (int k = 0; k < V; k++) {
        const float ay = a.v[k] * y.v[k];
        s[0] = fmaf(y.v[k], y.v[k], s[0]);
        s[1] = fmaf(h.v[k], h.v[k], s[1]);
        s[2] = fmaf(q.v[k], h.v[k], s[2]);
        s[3] = fmaf(ay, dh.v[k], s[3]);
        s[4] = fmaf(ay, q.v[k], s[4]);
        s[5] = fmaf(ay, h.v[k], s[5]);
        if constexpr (LAYER) {
            s[6] += q.v[k];
            s[7] = fmaf(a.v[k], dh.v[k], s[7]);
            s[8] = fmaf(a.v[k], q.v[k], s[8]);
            s[9] = fmaf(a.v[k], h.v[k], s[9]);
            s[10] += c + k < D ? a.v[k] : 0.0f;
            s[11] += ay;
        }
    }
}
// 1 / sqrt(v) of a mean square with eps; NaN where squares are past f32's range, or below its normal numbers and not hidden by eps: not a gradient of 0.
__device__ __forceinline__ float inverse(float v, float eps) {
    return (v >= 0x1p-126f || v == eps) && v < __builtin_inff() ? 1.0f / sqrtf(v) : __builtin_nanf("");
}
template <bool LAYER>
__device__ __forceinline__ RowTerms terms_of(const ah_residual_norm_grad_desc &d, const float (&m)[2], const float (&s)[kSums<LAYER>], float n) {
    const bool pre = d.pre != AH_NORM_NONE, post = d.post != AH_NORM_NONE;
    RowTerms x{m[0], m[1], 1.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (post) x.ry = inverse(s[0] * n + d.eps, d.eps);
    if (pre) {
        x.c1 = inverse(s[1] * n + d.eps, d.eps);
        x.c2 = x.c1 * (x.c1 * (s[2] * n));
    }
    float py = s[3] + x.c1 * (s[4] - x.c2 * s[5]);
    if constexpr (LAYER) {
        if (d.pre == AH_NORM_LAYER) x.c0 = x.c1 * (s[6] * n);
        py -= x.c0 * s[11];
        if (d.post == AH_NORM_LAYER) x.p1 = x.ry * (n * (s[7] + x.c1 * (s[8] - x.c2 * s[9]) - x.c0 * s[10]));
    }
    if (post) x.px = x.ry * (x.ry * (n * py));
    return x;
}
template <int V>
struct Slots {   // a thread's sums over rows
    fN<V> wpre, bpre, wpost, bpost;
};

// Gate `index`, whose rows the run [a, b) of worker w has come to the end of: into dgate if they are all in the run, else into one
// of the worker's two places.
template <class T, int V>
__device__ __forceinline__ void put_gate(const ah_residual_norm_grad_desc &d, const Runs &u, int w, int a, int b, long index, int c, const fN<V> &v) {
    const long first = index * u.per, end = min(first + (long)u.per, (long)u.n);
    if (first >= a && end <= b) store_cols<T, V>((T *)d.dgate + index * d.lddgate, c, d.D, v);
    else store_cols<float, V>(u.gates + ((long)w * 2 + (first < a ? 0 : 1)) * d.D, c, d.D, v);
}

template <int V>
__device__ __forceinline__ void put_sums(const Runs &u, int w, int c, int D, const Slots<V> &s) {
    float *p = u.sums + (long)w * u.arrays * D;
    if (u.wpre >= 0) store_cols<float, V>(p + (long)u.wpre * D, c, D, s.wpre);
    if (u.bpre >= 0) store_cols<float, V>(p + (long)u.bpre * D, c, D, s.bpre);
    if (u.wpost >= 0) store_cols<float, V>(p + (long)u.wpost * D, c, D, s.wpost);
    if (u.bpost >= 0) store_cols<float, V>(p + (long)u.bpost * D, c, D, s.bpost);
}

// Rows of up to V TPR columns, TPR threads a worker. The next row's loads go out before this row's work; a row costs its threads one barrier (two
// with layer norms, which need the means first). GIVEN: rows of any width whose terms are known, V TPR columns a workgroup. The gradients of the
// gate and the second norm's weights share sums over a gate's rows: sum t yh and sum t. LAYER: some norm has a mean and a bias.
template <class T, class R, int TPR, int V, bool LAYER, bool GIVEN>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR, TPR <= 64 ? 3 : 4) void resnorm_grad_kernel(ah_residual_norm_grad_desc d, Runs u, const RowTerms *rows) {
    constexpr int PER = TPR <= 64 ? 256 / TPR : 1;
    const int t = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x, D = d.D;
    int c = (GIVEN ? (int)blockIdx.y * TPR + t : t) * V;
    const int w = blockIdx.x * PER + (TPR <= 64 ? threadIdx.x / TPR : 0);
    if (PER > 1 && w >= u.workers) return;   // whole groups of lanes; sums stay within a group
    const int a = u.row(w), b = u.row(w + 1);
    const bool in = c < D, pre = d.pre != AH_NORM_NONE, post = d.post != AH_NORM_NONE;
    const bool rd_y = in && d.Y, rd_h = in && pre, rd_dh = in && d.dH_out, rd_g = in && d.gate;
    constexpr bool NARROW = TPR == 8;   // there may be fewer than V columns
    int turn = 0;
    typedef typename RawN<T, V>::type rawT;
    typedef typename RawN<R, V>::type rawR;
    struct Line {
        rawT y, dO;
        rawR h, dh;
    };
    const auto fetch = [&](int r) {
        Line l = {};
        if (rd_y) l.y = load_raw<T, V, NARROW>((const T *)d.Y + (long)r * d.ldy, c, D);
        if (rd_dh) l.dh = load_raw<R, V, NARROW>((const R *)d.dH_out + (long)r * d.lddh_out, c, D);
        if (rd_h) {
            l.h = load_raw<R, V, NARROW>((const R *)d.H_out + (long)r * d.ldh_out, c, D);
            l.dO = load_raw<T, V, NARROW>((const T *)d.dO + (long)r * d.lddo, c, D);
        }
        return l;
    };
    rawT rg = {}, rwn = {}, rwp = {}, rbp = {};   // gate and weights as they lie: half the registers in f16
    const auto fetch_gate = [&](long gate) {
        if (rd_g) rg = settle<T, V, NARROW>(load_raw<T, V, NARROW>((const T *)d.gate + gate * d.ldgate, c, D), c, D);
    };
    if (in && d.pre_w) rwn = settle<T, V, NARROW>(load_raw<T, V, NARROW>((const T *)d.pre_w, c, D), c, D);
    if (in && d.post_w) rwp = settle<T, V, NARROW>(load_raw<T, V, NARROW>((const T *)d.post_w, c, D), c, D);
    if (in && LAYER && d.post_b) rbp = settle<T, V, NARROW>(load_raw<T, V, NARROW>((const T *)d.post_b, c, D), c, D);
    const auto or_one = [&](bool there, rawT x) { return there ? widen<V>(x) : all_of<V>(1.0f); };
    Slots<V> sums = {};
    fN<V> ty = {}, ts = {};   // of a gate's rows: sum t yh, sum t
    long gate = a / u.per;
    int left = (int)min((long)u.per - a % u.per, (long)0x7fffffff);   // rows to the gate's end
    Line next = {};
    if (a < b) {
        next = fetch(a);
        fetch_gate(gate);
    }
    const float n = 1.0f / (float)D;
    for (int r = a; r < b; r++) {
        asm volatile("" : "+v"(c));   // addresses are formed anew for each row: kept, they spill
        Line l = next;
        if (r + 1 < b) next = fetch(r + 1);
        l.y = settle<T, V, NARROW>(l.y, c, D);
        l.h = settle<R, V, NARROW>(l.h, c, D);
        l.dO = settle<T, V, NARROW>(l.dO, c, D);
        l.dh = settle<R, V, NARROW>(l.dh, c, D);
        const auto gain = [&] { return times<V>(d.scale, or_one(d.gate, rg), or_one(d.post_w, rwp)); };
        const auto grad = [&] { return times<V>(1.0f, widen<V>(l.dO), or_one(d.pre_w, rwn)); };
        if constexpr (LAYER) {
            const fN<V> q = widen<V>(l.dO);
#pragma unroll
            for (int k = 0; k < V; k++) sums.bpre.v[k] += q.v[k];
        }
        RowTerms x;
        if constexpr (GIVEN) {
            x = rows[r];
        } else {
            float m[2] = {}, s[kSums<LAYER>] = {};
            if constexpr (LAYER) {
                const fN<V> y = widen<V>(l.y), h = widen<V>(l.h);
#pragma unroll
                for (int k = 0; k < V; k++) {
                    m[0] += y.v[k];
                    m[1] += h.v[k];
                }
                row_sums<TPR>(m, turn);
                m[0] = d.post == AH_NORM_LAYER ? m[0] * n : 0.0f;
                m[1] = d.pre == AH_NORM_LAYER ? m[1] * n : 0.0f;
            }
            if (pre || post) {
                add_terms<V, LAYER>(s, less<V, LAYER>(widen<V>(l.y), m[0], c, D), less<V, LAYER>(widen<V>(l.h), m[1], c, D), grad(), widen<V>(l.dh), gain(), c, D);
                row_sums<TPR>(s, turn);
            }
            x = terms_of<LAYER>(d, m, s, n);
        }
        // the row as it lies is widened again, rather than kept
        asm volatile("" : "+v"(l.y), "+v"(l.h), "+v"(l.dO), "+v"(l.dh));
        const fN<V> y = less<V, LAYER>(widen<V>(l.y), x.my, c, D);
        fN<V> tt, o;
        {
            const fN<V> h = less<V, LAYER>(widen<V>(l.h), x.mh, c, D), dO = widen<V>(l.dO), q = grad(), dh = widen<V>(l.dh);
#pragma unroll
            for (int k = 0; k < V; k++) {
                tt.v[k] = dh.v[k];
                if (pre) tt.v[k] += fmaf(x.c1, fmaf(-x.c2, h.v[k], q.v[k]), -x.c0);
                sums.wpre.v[k] = fmaf(dO.v[k], x.c1 * h.v[k], sums.wpre.v[k]);
                ty.v[k] = fmaf(tt.v[k], x.ry * y.v[k], ty.v[k]);
                if constexpr (LAYER) ts.v[k] += tt.v[k];
            }
        }
        if (d.dH && in) {
#pragma unroll
            for (int k = 0; k < V; k++) o.v[k] = d.skip * tt.v[k];
            store_cols<R, V>((R *)d.dH + (long)r * d.lddh, c, D, o);
        }
        if (d.dY && in) {
            const fN<V> gw = gain();
#pragma unroll
            for (int k = 0; k < V; k++) o.v[k] = fmaf(x.ry, fmaf(-x.px, y.v[k], gw.v[k] * tt.v[k]), -x.p1);
            store_cols<T, V>((T *)d.dY + (long)r * d.lddy, c, D, o);
        }
        if (--left == 0 || r + 1 == b) {
            const fN<V> g = or_one(d.gate, rg), wp = or_one(d.post_w, rwp), bp = widen<V>(rbp);
#pragma unroll
            for (int k = 0; k < V; k++) {
                sums.wpost.v[k] = fmaf(d.scale * g.v[k], ty.v[k], sums.wpost.v[k]);
                if constexpr (LAYER) sums.bpost.v[k] = fmaf(d.scale * g.v[k], ts.v[k], sums.bpost.v[k]);
                o.v[k] = d.scale * fmaf(wp.v[k], ty.v[k], LAYER ? bp.v[k] * ts.v[k] : 0.0f);
            }
            if (d.dgate && in) put_gate<T, V>(d, u, w, a, b, gate, c, o);
            ty = ts = all_of<V>(0.0f);
            gate++;
            left = u.per;
            if (r + 1 < b) fetch_gate(gate);
        }
    }
    if (u.arrays && in) put_sums(u, w, c, D, sums);
}

// The terms of rows of any width, a workgroup a row; layer norms read it again, from caches.
template <class T, class R, bool LAYER>
__global__ __launch_bounds__(kTermsT) void resnorm_grad_terms_kernel(ah_residual_norm_grad_desc d, RowTerms *rows) {
    const int D = d.D;
    const float n = 1.0f / (float)D;
    const bool pre = d.pre != AH_NORM_NONE, post = d.post != AH_NORM_NONE;
    int turn = 0;
    for (long r = blockIdx.x; r < d.N; r += gridDim.x) {
        const T *Y = d.Y ? (const T *)d.Y + r * d.ldy : nullptr, *G = d.gate ? (const T *)d.gate + (long)(d.rows_per_gate ? (int)r / d.rows_per_gate : 0) * d.ldgate : nullptr;
        const T *dO = pre ? (const T *)d.dO + r * d.lddo : nullptr;
        const R *H = pre ? (const R *)d.H_out + r * d.ldh_out : nullptr, *dh = d.dH_out ? (const R *)d.dH_out + r * d.lddh_out : nullptr;
        float m[2] = {}, s[kSums<LAYER>] = {};
        if constexpr (LAYER) {
            for (int c = threadIdx.x * kVec; c < D; c += kTermsT * kVec) {
                const f8 y = load8_or(Y, c, D, 0.0f), h = load8_or(H, c, D, 0.0f);
#pragma unroll
                for (int k = 0; k < kVec; k++) {
                    m[0] += y.v[k];
                    m[1] += h.v[k];
                }
            }
            row_sums<kTermsT>(m, turn);
            m[0] = d.post == AH_NORM_LAYER ? m[0] * n : 0.0f;
            m[1] = d.pre == AH_NORM_LAYER ? m[1] * n : 0.0f;
        }
        if (pre || post) {
            for (int c = threadIdx.x * kVec; c < D; c += kTermsT * kVec) {
                const f8 y = load8_or(Y, c, D, 0.0f), h = load8_or(H, c, D, 0.0f), q = load8_or(dO, c, D, 0.0f), g = load8_or(dh, c, D, 0.0f);
                const f8 a = times<kVec>(d.scale, load8_or(G, c, D, 1.0f), load8_or((const T *)d.post_w, c, D, 1.0f));
                add_terms<kVec, LAYER>(s, less<kVec, LAYER>(y, m[0], c, D), less<kVec, LAYER>(h, m[1], c, D), times<kVec>(1.0f, q, load8_or((const T *)d.pre_w, c, D, 1.0f)),
                                       g, a, c, D);
            }
            row_sums<kTermsT>(s, turn);
        }
        const RowTerms x = terms_of<LAYER>(d, m, s, n);
        if (threadIdx.x == 0) rows[r] = x;
    }
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

// Threads a row: the power of two that holds it in groups of `cols` columns.
int threads_of(int D, int cols) {
    int t = 8;
    while (t < 1024 && t * cols < D) t *= 2;
    return t;
}
bool has_layer(const ah_residual_norm_grad_desc &d) { return d.pre == AH_NORM_LAYER || d.post == AH_NORM_LAYER; }

template <class T, class R>
void launch_forward(const ah_residual_norm_desc &d, hipStream_t s) {
    const int tpr = threads_of(d.D, kVec), per = tpr <= 64 ? 256 / tpr : 1;
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(d.N, per), 16384)), block(tpr <= 64 ? 256 : tpr);
    switch (d.D > 2 * kWide ? 0 : d.D > kWide ? 2048 : tpr) {
        case 8: hipLaunchKernelGGL((resnorm_kernel<T, R, 8, 1>), grid, block, 0, s, d); break;
        case 16: hipLaunchKernelGGL((resnorm_kernel<T, R, 16, 1>), grid, block, 0, s, d); break;
        case 32: hipLaunchKernelGGL((resnorm_kernel<T, R, 32, 1>), grid, block, 0, s, d); break;
        case 64: hipLaunchKernelGGL((resnorm_kernel<T, R, 64, 1>), grid, block, 0, s, d); break;
        case 128: hipLaunchKernelGGL((resnorm_kernel<T, R, 128, 1>), grid, block, 0, s, d); break;
        case 256: hipLaunchKernelGGL((resnorm_kernel<T, R, 256, 1>), grid, block, 0, s, d); break;
        case 512: hipLaunchKernelGGL((resnorm_kernel<T, R, 512, 1>), grid, block, 0, s, d); break;
        case 1024: hipLaunchKernelGGL((resnorm_kernel<T, R, 1024, 1>), grid, block, 0, s, d); break;
        case 2048: hipLaunchKernelGGL((resnorm_kernel<T, R, 1024, 2>), grid, block, 0, s, d); break;
        default: hipLaunchKernelGGL((resnorm_wide_kernel<T, R>), grid, block, 0, s, d);
    }
}

struct Plan {
    int tpr;             // threads of a row (0: wide rows)
    Runs u;
    int gates, by_bound; // gates that workers may share, and how the join finds them
    int64_t rows, total; // of the workspace: the wide rows' terms
};

Plan plan_of(const ah_residual_norm_grad_desc &d) {
    Plan p{};
    // Eight columns a thread where its registers hold them and the next row's; four for f32 streams and for layer norms' sums. Rows past
    // 1024 threads' columns take two launches (4000 x 12000 f16 239 us; 410 by several readings of whole rows).
    const int cols = d.res_dtype == AH_F32 || has_layer(d) ? 4 : kVec;
    p.tpr = d.D > 1024 * cols ? 0 : threads_of(d.D, cols);
    Runs &u = p.u;
    u.n = d.N;
    u.per = d.rows_per_gate && d.rows_per_gate < d.N ? d.rows_per_gate : d.N;
    u.wpre = u.bpre = u.wpost = u.bpost = -1;
    if (d.dpre_w) u.wpre = u.arrays++;
    if (d.dpre_b) u.bpre = u.arrays++;
    if (d.dpost_w) u.wpost = u.arrays++;
    if (d.dpost_b) u.bpost = u.arrays++;
    // Workers: enough to fill the chip, with at least four rows each where there are many (a worker's sums cross memory twice).
    const int cap = p.tpr == 0 ? 256 : p.tpr <= 64 ? 512 * (256 / p.tpr) : p.tpr == 1024 ? 256 : (1 << 18) / p.tpr;
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
    p.rows = take(p.tpr == 0 ? (int64_t)d.N * sizeof(RowTerms) : 0);
    p.total = std::max<int64_t>(at, 16);
    return p;
}

template <class T, class R, int V, bool LAYER>
void launch_grad_rows(const ah_residual_norm_grad_desc &d, const Plan &p, RowTerms *rows, hipStream_t s) {
    const auto go = [&](auto tpr) {
        constexpr int TPR = tpr;
        const dim3 grid((unsigned)ceil_div(p.u.workers, TPR <= 64 ? 256 / TPR : 1)), block(TPR <= 64 ? 256 : TPR);
        hipLaunchKernelGGL((resnorm_grad_kernel<T, R, TPR, V, LAYER, false>), grid, block, 0, s, d, p.u, rows);
    };
    switch (p.tpr) {
        case 8: return go(std::integral_constant<int, 8>());
        case 16: return go(std::integral_constant<int, 16>());
        case 32: return go(std::integral_constant<int, 32>());
        case 64: return go(std::integral_constant<int, 64>());
        case 128: return go(std::integral_constant<int, 128>());
        case 256: return go(std::integral_constant<int, 256>());
        case 512: return go(std::integral_constant<int, 512>());
        case 1024: return go(std::integral_constant<int, 1024>());
    }
    hipLaunchKernelGGL((resnorm_grad_terms_kernel<T, R, LAYER>), dim3((unsigned)std::min(d.N, 16384)), dim3(kTermsT), 0, s, d, rows);
    hipLaunchKernelGGL((resnorm_grad_kernel<T, R, 256, V, LAYER, true>), dim3((unsigned)p.u.workers, (unsigned)ceil_div(d.D, 256 * V)), dim3(256), 0, s, d, p.u, rows);
}

template <class T, class R>
void launch_grad(const ah_residual_norm_grad_desc &d, Plan p, hipStream_t s) {
    char *ws = (char *)d.ws;
    p.u.sums = (float *)(ws + (uintptr_t)p.u.sums);
    p.u.gates = (float *)(ws + (uintptr_t)p.u.gates);
    RowTerms *rows = (RowTerms *)(ws + p.rows);
    if (has_layer(d)) launch_grad_rows<T, R, 4, true>(d, p, rows, s);
    else launch_grad_rows<T, R, sizeof(R) == 2 ? 8 : 4, false>(d, p, rows, s);
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
