// muon.hip — Newton-Schulz orthogonalisation, and the momentum step whose update it orthogonalises.
//
//   X = U / (|U|_F + eps);  steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X      (U wide)
//                                         A = X^T X,                    X <- a X + X B      (U tall)
//
// The iteration raises small singular values by a = 3.4 a step, 480-fold in five: what is lost of X to rounding grows as much. So
// all matrices are carried as two f16 planes (22 bits, plane_gemm.h) and every product is three f16 products in an f32
// accumulator; against 64 bits the result is about as far off as 32-bit products leave it, in 3/16 of the f32 MFMAs' time. Each
// matrix is scaled by a power of two (kSX, Scales), by how far the polynomial can take the singular values, up to 4: entries stay
// below f16's largest value. Where they stay at 1.2, entries down to 2^-22 of the matrix's norm keep 22 bits less what they are below 2^-14.
//
// Several steps in one. A + (a I + B) A (a I + B) = the next step's A: all are polynomials of one symmetric matrix and commute. So a
// group of g steps can be run on the s x s side (s the short side, l the long one) and applied to X once:
//   Q = a I + B;  then g - 1 times:  A <- (a I + B) A (a I + B),  B = b A + c A A,  Q <- (a I + B) Q;      X <- Q X
// All products but X's own are symmetric, half the tiles: a group costs s^2 l + (4 g - 3) s^3 + 2 s^2 l multiply-adds against
// g (3 s^2 l + s^3) step by step. Every A after a group's first carries the rounding of the one before, a^2-fold, and Q and qi I
// cancel where singular values are near 1, so groups have at most 3 steps (muon_dev.h). Which way is faster goes by the modelled
// time of the products (plan).
//
// A, B, Q are symmetric: only tiles on and above the diagonal are computed and each is stored twice. Multiples of I stay outside
// the planes (a X is added in the last product's epilogue): folded in they would be rounded with the rest, and where singular
// values are small they are all there is. Matrices stay padded with zeros to multiples of 64, where no product needs a bound.
#include "muon.h"

#include <algorithm>
#include <cmath>

#include "muon_dev.h"

namespace ah {
namespace {

using namespace ns;

constexpr int kBlocks = 1024;   // blocks of an elementwise pass over a matrix, at most

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
                floatx4 m = load4(d.M + at, c, d.cols);
#pragma unroll
                for (int k = 0; k < 4; k++) m[k] = mu * m[k] + u[k];
                store4(d.M_out + at, c, d.cols, m);
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
    const double inv = inverse_norm<256>(d, part, parts, z, red);
    half_t *out = X + z * (long)Rp * Cp * 2;
    for (long q = (long)blockIdx.x * 4 + wave; q < (long)Rp * segs; q += (long)gridDim.x * 4) {
        const int r = (int)(q / segs), c0 = (int)(q - (long)r * segs) * kSegment + lane * 4;
#pragma unroll
        for (int i = 0; i < kSegment; i += 256) {
            const int c = c0 + i;
            if (c >= Cp) continue;
            pg::plane_store(out + pg::panel_at<2>(Rp, r, c), scaled_update(d, z, r, c, inv));
        }
    }
}

// ── the products ───────────────────────────────────────────────────────────────

// NS_SYM: a symmetric matrix, stored on both sides of the diagonal. NS_NEXT: planes. NS_LAST: the caller's output.
enum { NS_SYM = 0, NS_NEXT = 1, NS_LAST = 2 };

struct NsArgs {
    pg::Operand A, B;
    long sA, sB;            // bytes from matrix to matrix
    int M, N, nk;           // padded sizes
    int tiles_m, tiles_n;
    int tiles;              // of one matrix
    pg::Work w;
    const half_t *P1, *P2;  // planes added in the epilogue, or null
    half_t *out;            // planes
    long sp, so;            // halves from matrix to matrix of P1 and P2, of out
    int rows;               // of their panels
    float k0, k1, k2;       // out = k0 (the product) + k1 P1 + k2 P2
};

template <class C, int WHAT>
__device__ __forceinline__ void ns_tile(const NsArgs &p, int tile, long &z, int &m0, int &n0) {
    z = tile / p.tiles;
    int tr, tc;
    if constexpr (WHAT == NS_SYM) pg::tri_tile(tile - (int)z * p.tiles, p.tiles_m, tr, tc);
    else pg::grouped_tile(tile - (int)z * p.tiles, p.tiles_m, p.tiles_n, tr, tc);
    m0 = tr * C::BM;
    n0 = tc * C::BN;
}

// q += k P at row m.
template <class C>
__device__ __forceinline__ void ns_add(const NsArgs &p, const half_t *P, float k, long z, int m, int n0, floatx4 (&q)[C::FB]) {
    const half_t *base = P + z * p.sp;
#pragma unroll
    for (int j = 0; j < C::FB; j++) {
        const int n = n0 + 16 * j;
        if (m >= p.M || n >= p.N) continue;
        const half_t *s = base + pg::panel_at<2>(p.rows, m, n);
        const h4 hi = *(const h4 *)s, lo = *(const h4 *)(s + 32);
#pragma unroll
        for (int r = 0; r < 4; r++) q[j][r] += k * ((float)hi[r] + (float)lo[r]);
    }
}

// What row m's epilogue adds to k0 times the product.
template <class C>
__device__ __forceinline__ void ns_load(const NsArgs &p, long z, int m, int n0, floatx4 (&q)[C::FB]) {
#pragma unroll
    for (int j = 0; j < C::FB; j++) q[j] = (floatx4){};
    if (p.P1) ns_add<C>(p, p.P1, p.k1, z, m, n0, q);
    if (p.P2) ns_add<C>(p, p.P2, p.k2, z, m, n0, q);
}

// What follows a product, for row m of it.
template <class C, int WHAT>
__device__ __forceinline__ void ns_row(const NsArgs &p, const Muon &d, long z, int m, int n0, bool mirror, const floatx4 (&acc)[C::FB],
                                       const floatx4 (&q)[C::FB]) {
    if (m >= p.M) return;
    const float k0 = p.k0;
#pragma unroll
    for (int j = 0; j < C::FB; j++) {
        const int n = n0 + 16 * j;
        if (n >= p.N) continue;
        floatx4 v = acc[j];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = k0 * v[r] + q[j][r];
        if constexpr (WHAT != NS_LAST) {
            half_t *o = p.out + z * p.so;
            pg::plane_store(o + pg::panel_at<2>(p.rows, m, n), v);
            if (WHAT == NS_SYM && mirror) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const half_t hi = (half_t)v[r];
                    half_t *t = o + pg::panel_at<2>(p.rows, n + r, m);
                    t[0] = hi;
                    t[32] = (half_t)(v[r] - (float)hi);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] *= 1.0f / (1 << kSX);
            store_result(d, z, m, n, v);
        }
    }
}

// NR accumulator rows from row i0; what a row adds is loaded while the one before it is worked on.
template <class C, int WHAT, int NR>
__device__ __forceinline__ void ns_rows(const NsArgs &p, const Muon &d, long z, int m0, int n0, int i0, const floatx4 (&acc)[NR][C::FB]) {
    const pg::Place<C> at(m0, n0);
    const int m1 = at.m + 16 * i0;
    floatx4 q[2][C::FB];
    ns_load<C>(p, z, m1, at.n, q[0]);
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const pg::Place<C> row(m0, n0);   // fresh addresses for each row
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

// Tiles of one product over the batch and how they are split, for M x N results summed over k.
pg::Plan ns_plan(bool symmetric, int batch, int M, int N, int k, long piece = 1l << 40) {
    const auto tiles = [&](int w) -> long {
        const long m = ceil_div(M, w), n = ceil_div(N, w);
        return batch * (symmetric ? m * (m + 1) / 2 : m * n);
    };
    return pg::plan(tiles, k, 2, 2, true, piece);
}

struct Layout {
    int Rp, Cp, S, K;   // padded sides; the short one, the long one
    bool wide;
    int group;          // steps of a group, at most
    int parts;
    pg::Plan gram, square, apply;
    int64_t part, small, X0, X1, square_at[6], sums, total;
};

Layout layout(const Muon &d) {
    Layout l{};
    l.Rp = (d.rows + 63) & ~63;
    l.Cp = (d.cols + 63) & ~63;
    l.wide = d.rows <= d.cols;
    l.S = l.wide ? l.Rp : l.Cp;
    l.K = l.wide ? l.Cp : l.Rp;
    // Sums over the long side in pieces of at most 2048 (or of the short side, which the other products sum over), added in the join:
    // in one chain of 7384 the diagonal's rounding errors cost the result 3.8e-6 at 9 x 7384 x 704, in pieces 2.2e-6, at no time.
    l.gram = ns_plan(true, d.batch, l.S, l.S, l.K, std::max(2048, l.S));
    l.square = ns_plan(true, d.batch, l.S, l.S, l.S);
    l.apply = ns_plan(false, d.batch, l.Rp, l.Cp, l.S);
    const int most = longest_group(d);
    double single = d.steps * (l.gram.us + l.square.us + l.apply.us), grouped = 0;
    for (int left = d.steps, index = 0; left > 0; index++) {
        const int g = group_size(most, index, left);
        grouped += l.gram.us + (4 * g - 3) * l.square.us + l.apply.us;
        left -= g;
    }
    l.group = grouped < single ? most : 1;
    l.parts = (int)std::min<int64_t>(kBlocks, ((int64_t)d.rows * ceil_div(d.cols, kSegment) + 3) / 4);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        at = (at + 255) & ~255ll;
        const int64_t o = at;
        at += bytes;
        return o;
    };
    l.part = take((int64_t)d.batch * l.parts * 8);
    if (std::min(d.rows, d.cols) <= kSmallSide) {
        l.small = take(muon_small_workspace(d));
        l.total = (at + 255) & ~255ll;
        return l;
    }
    l.X0 = take((int64_t)d.batch * l.Rp * l.Cp * 4);
    l.X1 = take((int64_t)d.batch * l.Rp * l.Cp * 4);
    for (int i = 0; i < (l.group > 1 ? 6 : 2); i++) l.square_at[i] = take((int64_t)d.batch * l.S * l.S * 4);
    l.sums = take(std::max({l.gram.part_bytes(), l.square.part_bytes(), l.apply.part_bytes()}));
    l.total = (at + 255) & ~255ll;
    return l;
}

template <class C, int WHAT>
void launch(NsArgs p, const Muon &d, hipStream_t s) {
    p.tiles_m = ceil_div(p.M, C::BM);
    p.tiles_n = ceil_div(p.N, C::BN);
    p.tiles = WHAT == NS_SYM ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
    hipLaunchKernelGGL((ns_product_kernel<C, WHAT>), dim3((unsigned)p.w.blocks()), dim3(C::NT), 0, s, p, d);
    if (p.w.splits > 1) hipLaunchKernelGGL((ns_join_kernel<C, WHAT>), dim3((unsigned)p.w.rest, C::FA), dim3(C::NT), 0, s, p, d);
}

template <int TA, int TB, int WHAT>
void product(NsArgs p, const pg::Plan &plan, const Muon &d, float *sums, hipStream_t s) {
    p.w = plan.w;
    p.w.part = sums;
    if (plan.width == 256) launch<pg::Tile256<TA, TB, 2, 2>, WHAT>(p, d, s);
    else if (plan.width == 128) launch<pg::Tile128<TA, TB, 2, 2>, WHAT>(p, d, s);
    else launch<pg::Tile64<TA, TB, 2, 2>, WHAT>(p, d, s);
}

// A symmetric s x s matrix in planes scaled by 2^e.
struct Square {
    half_t *p;
    int e;
};

}  // namespace

int64_t muon_workspace(const Muon &d) { return layout(d).total; }

hipError_t muon(const Muon &d, void *wsp, hipStream_t s) {
    const Layout l = layout(d);
    char *ws = (char *)wsp;
    double *part = (double *)(ws + l.part);
    float *sums = (float *)(ws + l.sums);
    half_t *X = (half_t *)(ws + l.X0), *Xn = (half_t *)(ws + l.X1);
    hipLaunchKernelGGL(muon_norm_kernel, dim3((unsigned)l.parts, (unsigned)d.batch), dim3(256), 0, s, d, part);
    if (std::min(d.rows, d.cols) <= kSmallSide) {
        muon_small(d, part, l.parts, ws + l.small, s);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(muon_pack_kernel, dim3((unsigned)std::min<int64_t>(kBlocks, (int64_t)l.Rp / 4 * ceil_div(l.Cp, kSegment)), (unsigned)d.batch),
                       dim3(256), 0, s, d, part, l.parts, X, l.Rp, l.Cp);

    const long sx = (long)l.Rp * l.Cp * 4, ss = (long)l.S * l.S * 4;
    const Scales sc = scales(d);
    const auto buf = [&](int i) { return (half_t *)(ws + l.square_at[i]); };
    const auto square = [&](const half_t *p) { return pg::panels(p, l.S, l.S, l.S); };
    // out = k (left right) + k1 p1 + k2 p2, matrices without their planes' scales
    const auto symmetric = [&](Square out, Square left, Square right, double k, double k1, Square p1, double k2, Square p2) {
        NsArgs q{};
        q.M = q.N = l.S;
        q.nk = l.S / 32;
        q.A = square(left.p);
        q.B = square(right.p);
        q.sA = q.sB = ss;
        q.out = out.p;
        q.so = q.sp = ss / 2;
        q.rows = l.S;
        q.k0 = (float)std::ldexp(k, out.e - left.e - right.e);
        q.P1 = p1.p;
        q.k1 = (float)std::ldexp(k1, out.e - p1.e);
        q.P2 = p2.p;
        q.k2 = (float)std::ldexp(k2, out.e - p2.e);
        product<0, 0, NS_SYM>(q, l.square, d, sums, s);
    };
    const Square none{nullptr, 0};
    for (int left = d.steps, index = 0; left > 0; index++) {
        const int g = group_size(l.group, index, left);
        left -= g;
        Square A{buf(0), sc.A}, B{buf(1), sc.B};
        NsArgs q{};   // A = X X^T or X^T X
        q.M = q.N = l.S;
        q.nk = l.K / 32;
        q.A = q.B = pg::panels(X, l.Rp, l.S, l.K);
        q.sA = q.sB = sx;
        q.out = A.p;
        q.so = ss / 2;
        q.rows = l.S;
        q.k0 = (float)std::ldexp(1.0, sc.A - 2 * kSX);
        if (l.wide) product<0, 0, NS_SYM>(q, l.gram, d, sums, s);
        else product<1, 1, NS_SYM>(q, l.gram, d, sums, s);

        symmetric(B, A, A, d.c, d.b, A, 0, none);   // B = b A + c A A
        Square Q = B;                               // the group's polynomial is qi I + Q
        double qi = d.a;
        for (int i = 1; i < g; i++) {
            const Square BA{buf(2), sc.BA}, Bn{buf(i == 1 ? 3 : 1), sc.B}, Qn{buf(3 + i), i == 1 ? sc.Q2 : sc.Q3};
            symmetric(BA, B, A, 1, d.a, A, 0, none);       // (a I + B) A
            symmetric(A, BA, B, 1, d.a, BA, 0, none);      // (a I + B) A (a I + B)
            symmetric(Bn, A, A, d.c, d.b, A, 0, none);
            symmetric(Qn, Bn, Q, 1, d.a, Q, qi, Bn);       // (a I + B) (qi I + Q) - a qi I
            B = Bn;
            Q = Qn;
            qi *= d.a;
        }
        NsArgs n{};   // X <- qi X + Q X or qi X + X Q (Q is symmetric: its rows serve as columns)
        n.M = l.Rp;
        n.N = l.Cp;
        n.nk = l.S / 32;
        n.out = Xn;
        n.so = n.sp = sx / 2;
        n.rows = l.Rp;
        n.P1 = X;
        n.k1 = (float)qi;
        n.k0 = (float)std::ldexp(1.0, -Q.e);
        if (l.wide) {
            n.A = square(Q.p);
            n.sA = ss;
            n.B = pg::panels(X, l.Rp, l.Cp, l.Rp);
            n.sB = sx;
            left ? product<0, 1, NS_NEXT>(n, l.apply, d, sums, s) : product<0, 1, NS_LAST>(n, l.apply, d, sums, s);
        } else {
            n.A = pg::panels(X, l.Rp, l.Rp, l.Cp);
            n.sA = sx;
            n.B = square(Q.p);
            n.sB = ss;
            left ? product<0, 0, NS_NEXT>(n, l.apply, d, sums, s) : product<0, 0, NS_LAST>(n, l.apply, d, sums, s);
        }
        std::swap(X, Xn);
    }
    return hipGetLastError();
}

}  // namespace ah
