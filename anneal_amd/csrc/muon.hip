// muon.hip — Newton-Schulz orthogonalisation, and the momentum step whose update it orthogonalises.
//
//   X = U / (|U|_F + eps);  steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X      (U wide)
//                                         A = X^T X,                    X <- a X + X B      (U tall)
//
// The iteration raises small singular values by a = 3.4 a step, 480-fold in five: what is lost of X to rounding grows as much. So X, A
// and B are carried as two f16 planes (22 bits, plane_gemm.h) and every product is three f16 products in an f32 accumulator;
// against 64 bits the result is as far off as 32-bit products leave it (2e-6 to 4e-6), and takes 3/16 of the f32 MFMAs' time.
// The planes hold 2^12 X, 2^13 A and 2^11 B: with the singular values of X at most 1.2, as the iteration keeps them, entries
// stay far below f16's largest value, and entries down to 2^-22 of the matrix's norm keep 22 bits less what they are below 2^-14.
//
// A and B are symmetric: only tiles on and above the diagonal are computed and each is stored twice. a X is added in the last
// product's epilogue: folded into B as a I it would be rounded with B, and where singular values are small a X is all there is.
// X, A and B stay padded with zeros to multiples of 64, where no product needs a bound.
#include "muon.h"

#include <algorithm>

#include "plane_gemm.h"

namespace ah {
namespace {

using pg::h4;

constexpr int kSX = 12, kSA = 13, kSB = 11;   // powers of two of the planes
constexpr int kBlocks = 1024;                 // blocks of an elementwise pass over a matrix, at most

// Four values from column c of a row of `cols`, zeros past its end; vec: rows start at multiples of four elements.
template <class T>
__device__ __forceinline__ floatx4 load4(const T *row, int c, int cols, bool vec) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    floatx4 v = {};
    if (vec && c + 3 < cols) {
        const t4 x = *(const t4 *)(row + c);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)x[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (c + k < cols) v[k] = (float)row[c + k];
    }
    return v;
}

template <class T>
__device__ __forceinline__ void store4(T *row, int c, int cols, bool vec, floatx4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 x;
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] = (T)v[k];
    if (vec && c + 3 < cols) *(t4 *)(row + c) = x;
    else
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (c + k < cols) row[c + k] = x[k];
}

__device__ __forceinline__ floatx4 load_g(const Muon &d, long z, int r, int c) {
    const long at = z * d.sg + r * d.ldg;
    return d.f16 ? load4((const half_t *)d.G + at, c, d.cols, d.vec_g) : load4((const float *)d.G + at, c, d.cols, d.vec_g);
}

// U from G and the new momentum.
__device__ __forceinline__ floatx4 update_of(const Muon &d, floatx4 g, floatx4 m) {
    const float mu = d.momentum;
    if (!d.nesterov) return m;
#pragma unroll
    for (int k = 0; k < 4; k++) g[k] += mu * m[k];
    return g;
}

// The elementwise passes give a wave one segment of a row at a time.
constexpr int kSegment = 1024;

// Sums of squares of U per block in f64 (f32 squares of small gradients would vanish); with momentum also M_out.
__global__ __launch_bounds__(256) void muon_norm_kernel(Muon d, double *part) {
    __shared__ double red[4];
    const long z = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, segs = (d.cols + kSegment - 1) / kSegment;
    const float mu = d.momentum;
    double s = 0.0;
    for (long q = (long)blockIdx.x * 4 + wave; q < (long)d.rows * segs; q += (long)gridDim.x * 4) {
        const int r = (int)(q / segs), c0 = (int)(q - (long)r * segs) * kSegment + lane * 4;
#pragma unroll
        for (int i = 0; i < kSegment; i += 256) {
            const int c = c0 + i;
            if (c >= d.cols) continue;
            floatx4 u = load_g(d, z, r, c);
            if (d.W) {
                const long at = z * d.sw + r * d.ldw;
                floatx4 m = load4(d.M + at, c, d.cols, d.vec_w);
#pragma unroll
                for (int k = 0; k < 4; k++) m[k] = mu * m[k] + u[k];
                store4(d.M_out + at, c, d.cols, d.vec_w, m);
                u = update_of(d, u, m);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) s += (double)u[k] * (double)u[k];
        }
    }
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[z * gridDim.x + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// X's planes: U / (|U| + eps), zeros past the matrix.
__global__ __launch_bounds__(256) void muon_pack_kernel(Muon d, const double *part, int parts, half_t *X, int Rp, int Cp) {
    __shared__ double red[4];
    const long z = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, segs = (Cp + kSegment - 1) / kSegment;
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) s += part[z * parts + i];
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    const float inv = (float)((double)(1 << kSX) / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)d.eps));
    half_t *out = X + z * (long)Rp * Cp * 2;
    for (long q = (long)blockIdx.x * 4 + wave; q < (long)Rp * segs; q += (long)gridDim.x * 4) {
        const int r = (int)(q / segs), c0 = (int)(q - (long)r * segs) * kSegment + lane * 4;
#pragma unroll
        for (int i = 0; i < kSegment; i += 256) {
            const int c = c0 + i;
            if (c >= Cp) continue;
            floatx4 v = {};
            if (r < d.rows && c < d.cols) {
                v = load_g(d, z, r, c);
                if (d.W) v = update_of(d, v, load4(d.M_out + z * d.sw + r * d.ldw, c, d.cols, d.vec_w));
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] *= inv;
            }
            pg::plane_store(out + pg::panel_at<2>(Rp, r, c), v);
        }
    }
}

// ── the products ───────────────────────────────────────────────────────────────

enum { NS_GRAM = 0, NS_POLY = 1, NS_NEXT = 2, NS_LAST = 3 };

struct NsArgs {
    pg::Operand A, B;
    long sA, sB;            // bytes from matrix to matrix
    int M, N, nk;           // padded sizes
    int tiles_m, tiles_n;
    int tiles;              // of one matrix
    pg::Work w;
    const half_t *Q;        // planes added in the epilogue: the Gram matrix (NS_POLY), X (NS_NEXT, NS_LAST)
    half_t *out;            // planes
    long sQ, so;            // halves
    int rows;               // of Q's and out's panels
};

template <class C, int WHAT>
__device__ __forceinline__ void ns_tile(const NsArgs &p, int tile, long &z, int &m0, int &n0) {
    z = tile / p.tiles;
    int tr, tc;
    if constexpr (WHAT == NS_GRAM || WHAT == NS_POLY) pg::tri_tile(tile - (int)z * p.tiles, p.tiles_m, tr, tc);
    else pg::grouped_tile(tile - (int)z * p.tiles, p.tiles_m, p.tiles_n, tr, tc);
    m0 = tr * C::BM;
    n0 = tc * C::BN;
}

// The planes that row m's epilogue adds, summed.
template <class C>
__device__ __forceinline__ void ns_load(const NsArgs &p, long z, int m, int n0, floatx4 (&q)[C::FB]) {
    const half_t *base = p.Q + z * p.sQ;
#pragma unroll
    for (int j = 0; j < C::FB; j++) {
        const int n = n0 + 16 * j;
        if (m >= p.M || n >= p.N) continue;
        const half_t *s = base + pg::panel_at<2>(p.rows, m, n);
        const h4 hi = *(const h4 *)s, lo = *(const h4 *)(s + 32);
#pragma unroll
        for (int r = 0; r < 4; r++) q[j][r] = (float)hi[r] + (float)lo[r];
    }
}

// What follows a product, for row m of it.
template <class C, int WHAT>
__device__ __forceinline__ void ns_row(const NsArgs &p, const Muon &d, long z, int m, int n0, bool mirror, const floatx4 (&acc)[C::FB],
                                       const floatx4 (&q)[C::FB]) {
    constexpr bool SYM = WHAT == NS_GRAM || WHAT == NS_POLY;
    if (m >= p.M) return;
    const float ca = d.a, cb = d.b, cc = d.c, keep = 1.0f - d.lr * d.decay, step = d.lr * d.scale;
#pragma unroll
    for (int j = 0; j < C::FB; j++) {
        const int n = n0 + 16 * j;
        if (n >= p.N) continue;
        floatx4 v = acc[j];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if constexpr (WHAT == NS_GRAM) v[r] *= 1.0f / (1 << (2 * kSX - kSA));
            else if constexpr (WHAT == NS_POLY) v[r] = cc * (v[r] * (1.0f / (1 << (2 * kSA - kSB)))) + cb * (q[j][r] * (1.0f / (1 << (kSA - kSB))));
            else v[r] = ca * q[j][r] + v[r] * (1.0f / (1 << kSB));
        }
        if constexpr (WHAT != NS_LAST) {
            half_t *o = p.out + z * p.so;
            pg::plane_store(o + pg::panel_at<2>(p.rows, m, n), v);
            if (SYM && mirror) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const half_t hi = (half_t)v[r];
                    half_t *t = o + pg::panel_at<2>(p.rows, n + r, m);
                    t[0] = hi;
                    t[32] = (half_t)(v[r] - (float)hi);
                }
            }
        } else {
            if (m >= d.rows || n >= d.cols) continue;
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] *= 1.0f / (1 << kSX);
            if (d.W) {
                const long w0 = z * d.sw + (long)m * d.ldw;
                const floatx4 w = load4(d.W + w0, n, d.cols, d.vec_w);
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = keep * w[r] - step * v[r];
                store4(d.W_out + w0, n, d.cols, d.vec_w, v);
                if (d.W16_out) store4((half_t *)d.W16_out + w0, n, d.cols, d.vec_o, v);
            } else {
                const long o0 = z * d.so + (long)m * d.ldo;
                if (d.out16) store4((half_t *)d.O + o0, n, d.cols, d.vec_o, v);
                else store4((float *)d.O + o0, n, d.cols, d.vec_o, v);
            }
        }
    }
}

// NR accumulator rows from row i0; what a row adds is loaded while the one before it is worked on.
template <class C, int WHAT, int NR>
__device__ __forceinline__ void ns_rows(const NsArgs &p, const Muon &d, long z, int m0, int n0, int i0, const floatx4 (&acc)[NR][C::FB]) {
    const pg::Place<C> at(m0, n0);
    const int m1 = at.m + 16 * i0;
    floatx4 q[2][C::FB] = {};
    if constexpr (WHAT != NS_GRAM) ns_load<C>(p, z, m1, at.n, q[0]);
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const pg::Place<C> row(m0, n0);   // fresh addresses for each row
        if constexpr (WHAT != NS_GRAM)
            if (i + 1 < NR) ns_load<C>(p, z, m1 + 16 * (i + 1), row.n, q[(i + 1) & 1]);
        ns_row<C, WHAT>(p, d, z, m1 + 16 * i, row.n, m0 != n0, acc[i], q[i & 1]);
    }
}

template <class C, int WHAT>
__global__ __launch_bounds__(C::NT, 2) void ns_product_kernel(NsArgs p, Muon d) {
    __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
    int tile, slot, first, count, m0, n0;
    long z;
    pg::pick(p.w, blockIdx.x, p.nk, tile, slot, first, count);
    ns_tile<C, WHAT>(p, tile, z, m0, n0);
    pg::Operand A = p.A, B = p.B;
    A.p += z * p.sA;
    B.p += z * p.sB;
    floatx4 acc[C::FA][C::FB];
    pg::contract<C>(A, B, m0, n0, first, count, smem, acc);
    if (slot >= 0) {
        pg::store_partials<C>(p.w.part, slot, acc);
        return;
    }
    ns_rows<C, WHAT, C::FA>(p, d, z, m0, n0, 0, acc);
}

template <class C, int WHAT>
__global__ __launch_bounds__(C::NT) void ns_join_kernel(NsArgs p, Muon d) {
    int m0, n0;
    long z;
    ns_tile<C, WHAT>(p, p.w.whole + blockIdx.x, z, m0, n0);
    floatx4 v[1][C::FB];
    pg::sum_partials<C>(p.w, blockIdx.x, blockIdx.y, v[0]);
    ns_rows<C, WHAT, 1>(p, d, z, m0, n0, blockIdx.y, v);
}

// ── host ───────────────────────────────────────────────────────────────────────

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct Layout {
    int Rp, Cp, S;   // padded sides, the short one
    int parts;
    int64_t part, X0, X1, A, B, sums, total;
};

bool symmetric(int what) { return what == NS_GRAM || what == NS_POLY; }

// Tiles of one product over the batch and how they are split, for M x N results summed over k.
pg::Plan ns_plan(int what, int batch, int M, int N, int k) {
    const auto tiles = [&](int w) -> long {
        const long m = ceil_div(M, w), n = ceil_div(N, w);
        return batch * (symmetric(what) ? m * (m + 1) / 2 : m * n);
    };
    return pg::plan(tiles(256), tiles(128), k, 2, 2);
}

Layout layout(const Muon &d) {
    Layout l{};
    l.Rp = (d.rows + 63) & ~63;
    l.Cp = (d.cols + 63) & ~63;
    l.S = d.rows <= d.cols ? l.Rp : l.Cp;
    l.parts = (int)std::min<int64_t>(kBlocks, ((int64_t)d.rows * ceil_div(d.cols, kSegment) + 3) / 4);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        at = (at + 255) & ~255ll;
        const int64_t o = at;
        at += bytes;
        return o;
    };
    l.part = take((int64_t)d.batch * l.parts * 8);
    l.X0 = take((int64_t)d.batch * l.Rp * l.Cp * 4);
    l.X1 = take((int64_t)d.batch * l.Rp * l.Cp * 4);
    l.A = take((int64_t)d.batch * l.S * l.S * 4);
    l.B = take((int64_t)d.batch * l.S * l.S * 4);
    const int K = d.rows <= d.cols ? l.Cp : l.Rp;
    l.sums = take(std::max({ns_plan(NS_GRAM, d.batch, l.S, l.S, K).part_bytes(), ns_plan(NS_POLY, d.batch, l.S, l.S, l.S).part_bytes(),
                            ns_plan(NS_NEXT, d.batch, l.Rp, l.Cp, l.S).part_bytes()}));
    l.total = (at + 255) & ~255ll;
    return l;
}

template <class C, int WHAT>
void launch(NsArgs p, const Muon &d, hipStream_t s) {
    p.tiles_m = ceil_div(p.M, C::BM);
    p.tiles_n = ceil_div(p.N, C::BN);
    p.tiles = symmetric(WHAT) ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
    hipLaunchKernelGGL((ns_product_kernel<C, WHAT>), dim3((unsigned)p.w.blocks()), dim3(C::NT), 0, s, p, d);
    if (p.w.splits > 1) hipLaunchKernelGGL((ns_join_kernel<C, WHAT>), dim3((unsigned)p.w.rest, C::FA), dim3(C::NT), 0, s, p, d);
}

template <int TA, int TB, int WHAT>
void product(NsArgs p, const Muon &d, float *part, hipStream_t s) {
    const pg::Plan plan = ns_plan(WHAT, d.batch, p.M, p.N, p.nk * 32);
    p.w = plan.w;
    p.w.part = part;
    if (plan.big) launch<pg::Tile<256, 256, 4, 2, TA, TB, 2, 2, 2>, WHAT>(p, d, s);
    else launch<pg::Tile<128, 128, 2, 2, TA, TB, 2, 2, 2>, WHAT>(p, d, s);
}

}  // namespace

int64_t muon_workspace(const Muon &d) { return layout(d).total; }

hipError_t muon(const Muon &in, void *wsp, hipStream_t s) {
    Muon d = in;
    const auto vec = [&](const void *p, long ld, long stride, int esz) {
        return !p || (((uintptr_t)p % (4 * esz)) == 0 && ld % 4 == 0 && (d.batch == 1 || stride % 4 == 0));
    };
    d.vec_g = vec(d.G, d.ldg, d.sg, d.f16 ? 2 : 4);
    d.vec_w = vec(d.M, d.ldw, d.sw, 4) && vec(d.M_out, d.ldw, d.sw, 4) && vec(d.W, d.ldw, d.sw, 4) && vec(d.W_out, d.ldw, d.sw, 4);
    d.vec_o = d.W ? vec(d.W16_out, d.ldw, d.sw, 2) : vec(d.O, d.ldo, d.so, d.out16 ? 2 : 4);
    const Layout l = layout(d);
    char *ws = (char *)wsp;
    double *part = (double *)(ws + l.part);
    float *sums = (float *)(ws + l.sums);
    half_t *X = (half_t *)(ws + l.X0), *Xn = (half_t *)(ws + l.X1), *A = (half_t *)(ws + l.A), *B = (half_t *)(ws + l.B);
    const bool wide = d.rows <= d.cols;
    hipLaunchKernelGGL(muon_norm_kernel, dim3((unsigned)l.parts, (unsigned)d.batch), dim3(256), 0, s, d, part);
    hipLaunchKernelGGL(muon_pack_kernel, dim3((unsigned)std::min<int64_t>(kBlocks, (int64_t)l.Rp / 4 * ceil_div(l.Cp, kSegment)), (unsigned)d.batch),
                       dim3(256), 0, s, d, part, l.parts, X, l.Rp, l.Cp);
    const long sx = (long)l.Rp * l.Cp * 4, ss = (long)l.S * l.S * 4;
    for (int k = 0; k < d.steps; k++) {
        NsArgs g{};   // A = X X^T or X^T X
        g.M = g.N = l.S;
        g.out = A;
        g.so = ss / 2;
        g.rows = l.S;
        g.sA = g.sB = sx;
        g.A = g.B = pg::panels(X, l.Rp, l.S, wide ? l.Cp : l.Rp);
        g.nk = (wide ? l.Cp : l.Rp) / 32;
        if (wide) product<0, 0, NS_GRAM>(g, d, sums, s);
        else product<1, 1, NS_GRAM>(g, d, sums, s);

        NsArgs q = g;   // B = b A + c A A
        q.Q = A;
        q.sQ = ss / 2;
        q.out = B;
        q.sA = q.sB = ss;
        q.A = q.B = pg::panels(A, l.S, l.S, l.S);
        q.nk = l.S / 32;
        product<0, 0, NS_POLY>(q, d, sums, s);

        NsArgs n{};   // a X + B X or a X + X B (B is symmetric: its rows serve as columns)
        n.Q = X;
        n.sQ = sx / 2;
        n.M = l.Rp;
        n.N = l.Cp;
        n.out = Xn;
        n.so = sx / 2;
        n.rows = l.Rp;
        const pg::Operand b = pg::panels(B, l.S, l.S, l.S);
        if (wide) {
            n.A = b;
            n.sA = ss;
            n.B = pg::panels(X, l.Rp, l.Cp, l.Rp);
            n.sB = sx;
        } else {
            n.A = pg::panels(X, l.Rp, l.Rp, l.Cp);
            n.sA = sx;
            n.B = b;
            n.sB = ss;
        }
        n.nk = l.S / 32;
        const bool last = k + 1 == d.steps;
        if (wide) last ? product<0, 1, NS_LAST>(n, d, sums, s) : product<0, 1, NS_NEXT>(n, d, sums, s);
        else last ? product<0, 0, NS_LAST>(n, d, sums, s) : product<0, 0, NS_NEXT>(n, d, sums, s);
        std::swap(X, Xn);
    }
    return hipGetLastError();
}

}  // namespace ah
