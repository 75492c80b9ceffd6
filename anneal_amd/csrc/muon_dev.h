// muon_dev.h — device code shared by the two forms of the orthogonalisation (muon.hip, muon_small.hip).
#pragma once
#include <algorithm>
#include <cmath>

#include "muon.h"
#include "plane_gemm.h"

namespace ah {
namespace ns {

using pg::h4;
using pg::load4;
using pg::store4;

constexpr int kSX = 12;   // power of two of X's planes; of the short side's matrices: Scales

__device__ __forceinline__ floatx4 load_g(const Muon &d, long z, int r, int c) {
    const long at = z * d.sg + r * d.ldg;
    return d.f16 ? load4((const half_t *)d.G + at, c, d.cols) : load4((const float *)d.G + at, c, d.cols);
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

// Four values of the update, at column c of row r of matrix z, times inv, which may pass f32's range; zeros past the matrix.
__device__ __forceinline__ floatx4 scaled_update(const Muon &d, long z, int r, int c, double inv) {
    floatx4 v = {};
    if (r < d.rows && c < d.cols) {
        v = load_g(d, z, r, c);
        if (d.W) v = update_of(d, v, load4(d.M_out + z * d.sw + r * d.ldw, c, d.cols));
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)((double)v[k] * inv);
    }
    return v;
}

// 2^kSX / (|U| + eps), or 0 for a zero matrix, from the blocks' sums of squares; red: NT / 64 doubles of LDS. All NT threads of a workgroup.
template <int NT>
__device__ __forceinline__ double inverse_norm(const Muon &d, const double *part, int parts, long z, double *red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += NT) s += part[z * parts + i];
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = red[0];
    for (int w = 1; w < NT / 64; w++) s += red[w];
    return s == 0.0 ? 0.0 : (double)(1 << kSX) / (sqrt(s) + (double)d.eps);
}

// Four values of the last iterate (without the planes' scale) at column c of row r: into O, or into the weights.
__device__ __forceinline__ void store_result(const Muon &d, long z, int r, int c, floatx4 v) {
    if (r >= d.rows || c >= d.cols) return;
    const float keep = 1.0f - d.lr * d.decay, step = d.lr * d.scale;
    if (d.W) {
        const long w0 = z * d.sw + (long)r * d.ldw;
        const floatx4 w = load4(d.W + w0, c, d.cols);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = keep * w[k] - step * v[k];
        store4(d.W_out + w0, c, d.cols, v);
        if (d.W16_out) store4((half_t *)d.W16_out + w0, c, d.cols, v);
    } else {
        const long o0 = z * d.so + (long)r * d.ldo;
        if (d.out16) store4((half_t *)d.O + o0, c, d.cols, v);
        else store4((float *)d.O + o0, c, d.cols, v);
    }
}

}  // namespace ns

// How large the polynomial's matrices become: over squared singular values x that the iterates before the last reach (1 at the start; the
// caller keeps them to 16), the largest x, |a + b x + c x^2|, |b x + c x^2| and |a + b x + c x^2| x, from samples, with 2% for what lies
// between them.
struct Reach {
    double x, step, b, ba;
};
inline Reach reach(const Muon &d) {
    constexpr int n = 128;
    const auto poly = [&](double x) { return d.a + d.b * x + d.c * x * x; };
    double top = 1.0;
    for (int k = 1; k < d.steps && top < 4.0; k++) {
        double next = 0.0;
        for (int i = 1; i <= n; i++) {
            const double s = top * i / n;
            next = std::max(next, 1.02 * std::fabs(s * poly(s * s)));
        }
        if (next <= top) break;
        top = std::min(next, 4.0);
    }
    Reach r{top * top, 0, 0, 0};
    for (int i = 0; i <= n; i++) {
        const double x = r.x * i / n;
        r.step = std::max(r.step, 1.02 * std::fabs(poly(x)));
        r.b = std::max(r.b, 1.02 * std::fabs(d.b * x + d.c * x * x));
        r.ba = std::max(r.ba, 1.02 * std::fabs(poly(x) * x));
    }
    return r;
}

// Powers of two of the planes of A, B, (a I + B) A and of the polynomials of groups of two and three steps (less their multiple of I). No
// entry passes f16's largest value: an entry is at most the largest eigenvalue. The caps are what a polynomial that keeps the singular
// values to 1.2 takes.
struct Scales {
    int A, B, BA, Q2, Q3;
};
inline Scales scales(const Muon &d) {
    const Reach r = reach(d);
    const auto most = [](double top, int cap) { return top * std::ldexp(1.0, cap) <= 65504.0 ? cap : (int)std::floor(std::log2(65504.0 / top)); };
    const double a = std::fabs(d.a);
    return {most(r.x, 13), most(r.b, 11), most(r.ba, 12), most(r.step * r.step + a * a, 11), most(r.step * r.step * r.step + a * a * a, 9)};
}

// Steps of the longest group: the largest |a + b x + c x^2| bounds a step's growth. A short side under 256 starts with larger singular values of X and has less to average
// over: three steps at once cost it more than 32-bit products lose (16 x 64: 7 times the error of step by step), and under 32 two at
// once do (8 x 8: 1.3e-6 off, step by step 0.7e-6, 32-bit products 0.6e-6).
inline int longest_group(const Muon &d) {
    double grow = 0;
    const double top = std::max(1.5, reach(d).x);
    for (int i = 0; i <= 60; i++) {
        const double x = i * top / 60;
        grow = std::max(grow, std::fabs(d.a + d.b * x + d.c * x * x));
    }
    const int side = std::min(d.rows, d.cols);
    return grow <= 3.5 && side >= 256 ? 3 : grow <= 5.0 && side >= 32 ? 2 : 1;
}
// Steps of group `index` with `left` to go: 3, 2, 1, 1, .. or 2, 1, 1, .. Of the ways to cut five steps in 32-bit products these
// stay nearest to step by step over short sides of 8 to 512 and flat and steep spectra (1.1 to 1.7 times its error at 3, 2 from 256
// on, 1.0 to 1.3 at 2, 1, 1, 1 from 32 to there; pairs throughout 1.2 to 2.8, other cuts 4 to 40). Step by step in planes has 0.6 (s = 4096) to
// 1.5 times (s = 8) the error of 32-bit products.
inline int group_size(int longest, int index, int left) { return std::min(std::max(1, longest - index), left); }

// The form for a short side of at most kSmallSide (muon_small.hip).
constexpr int kSmallSide = 128;
int64_t muon_small_workspace(const Muon &d);
void muon_small(const Muon &d, const double *part, int parts, void *ws, hipStream_t s);

}  // namespace ah
