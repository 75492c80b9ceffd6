// muon.hip — Newton-Schulz orthogonalisation, and the momentum step whose update it orthogonalises.
//
//   X = U / (|U|_F + eps);  steps times:  A = X X^T,  B = a I + b A + c A A,  X <- B X      (U wide)
//                                         A = X^T X,                          X <- X B      (U tall)
//
// The iteration raises small singular values by a = 3.4 a step, 480-fold in five: what is lost of X to rounding grows as much. So X, A
// and B are carried as two f16 planes (22 bits, plane_gemm.h) and every product is three f16 products in an f32 accumulator;
// against 64 bits the result is as far off as 32-bit products leave it (2e-6 to 4e-6), and takes 3/16 of the f32 MFMAs' time.
// The planes hold 2^12 X, 2^13 A and 2^11 B: with the singular values of X at most 1.2, as the iteration keeps them, entries
// stay far below f16's largest value, and entries down to 2^-22 of the matrix's norm keep 22 bits less what they are below 2^-14.
//
// A and B are symmetric: only tiles on and above the diagonal are computed and each is stored twice. a I is folded into B, so X
// is read by the last product alone. X, A and B stay padded with zeros to multiples of 64, where no product needs a bound.
#include "muon.h"

#include <algorithm>

#include "plane_gemm.h"

namespace ah {
namespace {

using pg::h4;

constexpr int kSX = 12, kSA = 13, kSB = 11;   // powers of two of the planes
constexpr int kParts = 256;                   // blocks that sum a matrix's squares, at most

__device__ __forceinline__ float load_g(const Muon &d, long i) {
    return d.f16 ? (float)((const half_t *)d.G)[i] : ((const float *)d.G)[i];
}

// U at (r, c) of matrix z, from G and the new momentum.
__device__ __forceinline__ float update_of(const Muon &d, float g, float m) { return d.nesterov ? g + d.momentum * m : m; }

// Sums of squares of U per block in f64 (f32 squares of small gradients would vanish); with momentum also M_out.
__global__ __launch_bounds__(256) void muon_norm_kernel(Muon d, double *part) {
    __shared__ double red[4];
    const long z = blockIdx.y, n = (long)d.rows * d.cols;
    double s = 0.0;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long r = i / d.cols, c = i - r * d.cols;
        float u = load_g(d, z * d.sg + r * d.ldg + c);
        if (d.W) {
            const long k = z * d.sw + r * d.ldw + c;
            const float m = d.momentum * d.M[k] + u;
            d.M_out[k] = m;
            u = update_of(d, u, m);
        }
        s += (double)u * (double)u;
    }
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[z * gridDim.x + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// X's planes: U / (|U| + eps), zeros past the matrix. A block takes whole stored rows.
__global__ __launch_bounds__(256) void muon_pack_kernel(Muon d, const double *part, int parts, half_t *X, int Rp, int Cp) {
    __shared__ float inv_s;
    const long z = blockIdx.y;
    if (threadIdx.x < 64) {
        double s = 0.0;
        for (int i = threadIdx.x; i < parts; i += 64) s += part[z * parts + i];
        for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
        if (threadIdx.x == 0) inv_s = (float)((double)(1 << kSX) / (sqrt(s) + (double)d.eps));
    }
    __syncthreads();
    const float inv = inv_s;
    for (int r = blockIdx.x; r < Rp; r += gridDim.x) {
        half_t *out = X + (z * Rp + r) * (long)Cp * 2;
        for (int c = threadIdx.x * 4; c < Cp; c += 1024) {
            floatx4 v = {};
            if (r < d.rows)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (c + k < d.cols) {
                        const float g = load_g(d, z * d.sg + r * d.ldg + c + k);
                        v[k] = (d.W ? update_of(d, g, d.M_out[z * d.sw + r * d.ldw + c + k]) : g) * inv;
                    }
            pg::plane_store(out + pg::plane_col<2>(c), v);
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
    const half_t *Q;        // NS_POLY: the Gram matrix's planes
    half_t *out;            // planes
    long sQ, so, ldo;       // halves
};

template <class C, int WHAT>
__global__ __launch_bounds__(C::NT) void ns_product_kernel(NsArgs p, Muon d) {
    __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
    constexpr bool SYM = WHAT == NS_GRAM || WHAT == NS_POLY;
    const long z = blockIdx.y;
    int tr, tc;
    const int L = pg::xcd_tile(blockIdx.x, gridDim.x);
    if constexpr (SYM) pg::tri_tile(L, tr, tc);
    else {
        tr = L / p.tiles_n;
        tc = L % p.tiles_n;
    }
    const int m0 = tr * C::BM, n0 = tc * C::BN;
    pg::Operand A = p.A, B = p.B;
    A.p += z * p.sA;
    B.p += z * p.sB;
    floatx4 acc[C::FA][C::FB];
    pg::contract<C>(A, B, m0, n0, 0, p.nk, smem, acc);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mb = m0 + (wave / C::WVN) * C::WM + (lane & 15), nb = n0 + (wave % C::WVN) * C::WN + 4 * (lane >> 4);
    const float ca = d.a, cb = d.b, cc = d.c, keep = 1.0f - d.lr * d.decay, step = d.lr * d.scale;
#pragma unroll
    for (int i = 0; i < C::FA; i++) {
        const int m = mb + 16 * i;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < C::FB; j++) {
            const int n = nb + 16 * j;
            if (n >= p.N) continue;
            floatx4 v = acc[i][j];
            if constexpr (WHAT == NS_GRAM) {
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] *= 1.0f / (1 << (2 * kSX - kSA));
            } else if constexpr (WHAT == NS_POLY) {
                const half_t *q = p.Q + z * p.sQ + (long)m * p.ldo + pg::plane_col<2>(n);
                const h4 hi = *(const h4 *)q, lo = *(const h4 *)(q + 32);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float g = (float)hi[r] + (float)lo[r];
                    v[r] = cc * (v[r] * (1.0f / (1 << (2 * kSA - kSB)))) + cb * (g * (1.0f / (1 << (kSA - kSB))));
                    if (n + r == m) v[r] += ca * (float)(1 << kSB);
                }
            } else if constexpr (WHAT == NS_NEXT) {
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] *= 1.0f / (1 << kSB);
            }
            if constexpr (WHAT != NS_LAST) {
                half_t *o = p.out + z * p.so;
                pg::plane_store(o + (long)m * p.ldo + pg::plane_col<2>(n), v);
                if (SYM && m0 != n0) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const half_t hi = (half_t)v[r];
                        half_t *t = o + (long)(n + r) * p.ldo + pg::plane_col<2>(m);
                        t[0] = hi;
                        t[32] = (half_t)(v[r] - (float)hi);
                    }
                }
            } else {
                if (m >= d.rows) continue;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (n + r >= d.cols) continue;
                    const float x = v[r] * (1.0f / (1 << (kSB + kSX)));
                    if (d.W) {
                        const long k = z * d.sw + (long)m * d.ldw + n + r;
                        const float w = keep * d.W[k] - step * x;
                        d.W_out[k] = w;
                        if (d.W16_out) ((half_t *)d.W16_out)[k] = (half_t)w;
                    } else {
                        const long k = z * d.so + (long)m * d.ldo + n + r;
                        if (d.out16) ((half_t *)d.O)[k] = (half_t)x;
                        else ((float *)d.O)[k] = x;
                    }
                }
            }
        }
    }
}

// ── host ───────────────────────────────────────────────────────────────────────

struct Layout {
    int Rp, Cp, S;   // padded sides, the short one
    int parts;
    int64_t part, X0, X1, A, B, total;
};

Layout layout(const Muon &d) {
    Layout l{};
    l.Rp = (d.rows + 63) & ~63;
    l.Cp = (d.cols + 63) & ~63;
    l.S = d.rows <= d.cols ? l.Rp : l.Cp;
    l.parts = (int)std::min<int64_t>(kParts, ((int64_t)d.rows * d.cols + 4095) / 4096);
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
    l.total = (at + 255) & ~255ll;
    return l;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <class C, int WHAT>
void launch(NsArgs p, const Muon &d, hipStream_t s) {
    p.tiles_m = ceil_div(p.M, C::BM);
    p.tiles_n = ceil_div(p.N, C::BN);
    const int tiles = WHAT == NS_GRAM || WHAT == NS_POLY ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
    hipLaunchKernelGGL((ns_product_kernel<C, WHAT>), dim3((unsigned)tiles, (unsigned)d.batch), dim3(C::NT), 0, s, p, d);
}

template <int TA, int TB, int WHAT>
void product(const NsArgs &p, const Muon &d, hipStream_t s) {
    const int64_t tiles = (int64_t)ceil_div(p.M, 256) * ceil_div(p.N, 256) * d.batch;
    if (tiles >= 128) launch<pg::Tile<256, 256, 4, 2, TA, TB, 2, 2, 2>, WHAT>(p, d, s);
    else launch<pg::Tile<128, 128, 2, 2, TA, TB, 2, 2, 2>, WHAT>(p, d, s);
}

}  // namespace

int64_t muon_workspace(const Muon &d) { return layout(d).total; }

hipError_t muon(const Muon &d, void *wsp, hipStream_t s) {
    const Layout l = layout(d);
    char *ws = (char *)wsp;
    double *part = (double *)(ws + l.part);
    half_t *X = (half_t *)(ws + l.X0), *Xn = (half_t *)(ws + l.X1), *A = (half_t *)(ws + l.A), *B = (half_t *)(ws + l.B);
    const bool wide = d.rows <= d.cols;
    hipLaunchKernelGGL(muon_norm_kernel, dim3((unsigned)l.parts, (unsigned)d.batch), dim3(256), 0, s, d, part);
    hipLaunchKernelGGL(muon_pack_kernel, dim3((unsigned)std::min(l.Rp, 2048), (unsigned)d.batch), dim3(256), 0, s, d, part, l.parts, X, l.Rp, l.Cp);
    const long ldx = 2l * l.Cp, lds = 2l * l.S, sx = (long)l.Rp * l.Cp * 4, ss = (long)l.S * l.S * 4;
    for (int k = 0; k < d.steps; k++) {
        NsArgs g{};   // A = X X^T or X^T X
        g.M = g.N = l.S;
        g.out = A;
        g.so = ss / 2;
        g.ldo = lds;
        g.sA = g.sB = sx;
        g.A = g.B = pg::Operand{(const char *)X, ldx, l.S, wide ? l.Cp : l.Rp};
        g.nk = (wide ? l.Cp : l.Rp) / 32;
        if (wide) product<0, 0, NS_GRAM>(g, d, s);
        else product<1, 1, NS_GRAM>(g, d, s);

        NsArgs q = g;   // B = a I + b A + c A A
        q.Q = A;
        q.sQ = ss / 2;
        q.out = B;
        q.sA = q.sB = ss;
        q.A = q.B = pg::Operand{(const char *)A, lds, l.S, l.S};
        q.nk = l.S / 32;
        product<0, 0, NS_POLY>(q, d, s);

        NsArgs n{};   // B X or X B (B is symmetric: its rows serve as columns)
        n.M = l.Rp;
        n.N = l.Cp;
        n.out = Xn;
        n.so = sx / 2;
        n.ldo = ldx;
        const pg::Operand b{(const char *)B, lds, l.S, l.S};
        if (wide) {
            n.A = b;
            n.sA = ss;
            n.B = pg::Operand{(const char *)X, ldx, l.Cp, l.Rp};
            n.sB = sx;
        } else {
            n.A = pg::Operand{(const char *)X, ldx, l.Rp, l.Cp};
            n.sA = sx;
            n.B = b;
            n.sB = ss;
        }
        n.nk = l.S / 32;
        const bool last = k + 1 == d.steps;
        if (wide) last ? product<0, 1, NS_LAST>(n, d, s) : product<0, 1, NS_NEXT>(n, d, s);
        else last ? product<0, 0, NS_LAST>(n, d, s) : product<0, 0, NS_NEXT>(n, d, s);
        std::swap(X, Xn);
    }
    return hipGetLastError();
}

}  // namespace ah
