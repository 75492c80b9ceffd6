// muon_small.hip — orthogonalisation with a short side of at most 128: one launch for a group of steps.
//
// Products of this size are all launch, first load and join (the general form takes 117 us for five steps of 128 x 784, of which
// the arithmetic is 2). Here a group of steps is one kernel. The long side is cut into slices of 128; a workgroup holds the short side's
// matrices and one slice at a time in LDS:
//   A = the sum of all workgroups' parts of the Gram matrix (each workgroup forms it for itself, in a fixed order);
//   Q of a group of steps;  for each of its slices: X <- qi X + Q X, and X X^T of the new slice onto its part for the next group.
// What bounds it is the reading of the parts (workgroups * 4 S^2 bytes each, at what one CU draws) against the slices a workgroup
// goes through, about 3 us each: the number of workgroups balances the two. Groups (muon.hip) spare the parts' way to memory, most
// of a step's time: they are always as long as the polynomial and the precision admit.
//
// LDS holds stage images as plane_gemm.h reads them: 32 k of R rows in two planes are R * 128 bytes.
#include <algorithm>
#include <cmath>

#include "muon_dev.h"

namespace ah {
namespace {

using namespace ns;
using pg::h8;

constexpr int kSlice = 128;

struct SmallArgs {
    half_t *X;             // planes in panels, slices updated in place
    long sx;               // halves from matrix to matrix
    int Rp, Cp;            // padded sides
    int slices, groups;    // of the long side; workgroups a matrix
    const float *in;       // Gram parts of the step before: [matrix][group][S * S] in accumulator order
    float *out;
    const double *part;    // first kernel: sums of squares
    int parts;
    int steps;             // of the group, 1 or 2
    float qi;              // the group's polynomial is qi I + Q
    float ga;              // A's planes from the Gram matrix of X's
    float b2, b1;          // c A A and b A in B's planes
    float p2, p1;          // B A and a A in those of (a I + B) A
    float a2, a1;          // times B, and times a, in A's
    float q2, q1, qs;      // B Q and a Q + a B in those of a group of two; what its planes are scaled by
};

// Byte offsets in an image of R rows: four values at row r, k c (T = 0), or at k r, row c (T = 1). The lo plane is at the offset xor 64.
template <int R>
__device__ __forceinline__ int image0(int r, int c) { return (c >> 5) * (R * 128) + g16::koff<64>(r, (c & 31) >> 3) + (c & 7) * 2; }
template <int R>
__device__ __forceinline__ int image1(int r, int c) { return (r >> 5) * (R * 128) + g16::mnoff<2 * R>(r & 31, (c >> 5) * 64 + (c & 31)); }

__device__ __forceinline__ void image_store(char *img, int off, floatx4 v) {
    h4 hi, lo;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        hi[k] = (half_t)v[k];
        lo[k] = (half_t)(v[k] - (float)hi[k]);
    }
    *(h4 *)(img + off) = hi;
    *(h4 *)(img + (off ^ 64)) = lo;
}
__device__ __forceinline__ floatx4 image_load(const char *img, int off) {
    const h4 hi = *(const h4 *)(img + off), lo = *(const h4 *)(img + (off ^ 64));
    floatx4 v;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = (float)hi[k] + (float)lo[k];
    return v;
}

// acc += the products of nst stages of two images; a, b: LDS addresses of the wave's first fragments. The small products come first, so
// that a sum of 32 is rounded once at its full size. NP = 4: lo lo is one of them, which sums as short as a side under 64 show (0.85 of
// the error of an 8 x 25 without; at 128 it would take 95 us, not 90, for 128 x 784 and show nothing).
template <int NP, int RA, int TA, int RB, int TB, int FA, int FB>
__device__ __forceinline__ void multiply(uint32_t a, uint32_t b, int nst, floatx4 (&acc)[FA][FB]) {
    using A = pg::PFrag<RA, TA, 2, 32>;
    using B = pg::PFrag<RB, TB, 2, 32>;
    for (int q = 0; q < nst; q++, a += RA * 128, b += RB * 128) {
        uint32_t av = a, bv = b;
        asm volatile("" : "+v"(av), "+v"(bv));
        h8 x[2][FA], y[2][FB];
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int i = 0; i < FA; i++) x[s][i] = A::read(av, i, s);
#pragma unroll
            for (int j = 0; j < FB; j++) y[s][j] = B::read(bv, j, s);
        }
#pragma unroll
        for (int p = 4 - NP; p < 4; p++)   // lo lo, lo hi, hi lo, hi hi
#pragma unroll
            for (int i = 0; i < FA; i++)
#pragma unroll
                for (int j = 0; j < FB; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[p == 0 || p == 2][j], x[p < 2][i], acc[i][j], 0, 0, 0);
    }
}

template <int FA, int FB>
__device__ __forceinline__ void clear(floatx4 (&v)[FA][FB]) {
#pragma unroll
    for (int i = 0; i < FA; i++)
#pragma unroll
        for (int j = 0; j < FB; j++) v[i][j] = (floatx4){};
}

enum { FIRST = 0, STEP = 1, LAST = 2 };

// S: the padded short side, 64 or 128. WIDE: the matrix has S rows, else S columns. The waves, S / 32 x S / 32 over every product,
// hold 32 x 32 of a square each: at S = 128 four on a SIMD, which cover each other's LDS reads and conversions (with one of
// 64 x 64 a step of 128 x 784 took 20 us, not 16).
template <int S, bool WIDE, int WHAT>
__global__ __launch_bounds__(S / 32 * (S / 32) * 64, 1) void muon_small_kernel(SmallArgs p, Muon d) {
    constexpr int WV = S / 32, NT = WV * WV * 64, NP = S == 64 ? 4 : 3;   // (NP: products of planes)
    constexpr int FQ = 2;                                               // 16-row blocks a wave holds of a side of S
    constexpr int XM = WIDE ? S : kSlice, XN = WIDE ? kSlice : S;       // a slice of X
    constexpr int FM = XM / WV / 16, FN = XN / WV / 16;
    __shared__ __attribute__((aligned(1024))) char slice_img[S * kSlice * 4];   // a slice, before that A
    __shared__ __attribute__((aligned(1024))) char square_img[S * S * 4];       // B
    __shared__ double red[WV * WV];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wr = wave / WV, wc = wave % WV;
    const uint32_t slice_lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)slice_img;
    const uint32_t square_lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)square_img;
    const long z = blockIdx.y;
    half_t *X = p.X + z * p.sx;
    const int rows = p.Rp;   // of the panels
    // the wave's place in a square of S and in a slice
    const int qm = wr * (S / WV) + (lane & 15), qn = wc * (S / WV) + 4 * (lane >> 4);
    const int xm = wr * (XM / WV) + (lane & 15), xn = wc * (XN / WV) + 4 * (lane >> 4);
    floatx4 gram[FQ][FQ];
    clear(gram);

    // X X^T (X^T X) of the slice image onto the part
    const auto add_gram = [&]() {
        if constexpr (WIDE) {
            pg::PFrag<S, 0, 2, 32> f;
            f.init(slice_lds, wr * (S / WV), lane);
            const uint32_t a = f.first;
            f.init(slice_lds, wc * (S / WV), lane);
            multiply<NP, S, 0, S, 0>(a, f.first, kSlice / 32, gram);
        } else {
            pg::PFrag<S, 1, 2, 32> f;
            f.init(slice_lds, wr * (S / WV), lane);
            const uint32_t a = f.first;
            f.init(slice_lds, wc * (S / WV), lane);
            multiply<NP, S, 1, S, 1>(a, f.first, kSlice / 32, gram);
        }
    };
    const auto slice_at = [&](int m, int n) { return WIDE ? image0<S>(m, n) : image1<S>(m, n); };   // of the image that add_gram reads

    if constexpr (WHAT == FIRST) {
        const double inv = inverse_norm<NT>(d, p.part, p.parts, z, red);
        for (int sl = blockIdx.x; sl < p.slices; sl += p.groups) {
            const int m0 = WIDE ? 0 : sl * kSlice, n0 = WIDE ? sl * kSlice : 0;
            __syncthreads();
            for (int q = tid; q < XM * XN / 4; q += NT) {
                const int m = q / (XN / 4), n = q % (XN / 4) * 4;
                const floatx4 v = scaled_update(d, z, m0 + m, n0 + n, inv);
                image_store(slice_img, slice_at(m, n), v);
                if (m0 + m < p.Rp && n0 + n < p.Cp) pg::plane_store(X + pg::panel_at<2>(rows, m0 + m, n0 + n), v);
            }
            __syncthreads();
            add_gram();
        }
    } else {
        {   // A, then the group's Q, by the products that muon.hip describes
            typedef floatx4 Square[FQ][FQ];
            // v = k (image 0 or 1 times image 0 or 1) + k1 p + k2 q
            uint32_t row[2], col[2];
            pg::PFrag<S, 0, 2, 32> f;
            for (int i = 0; i < 2; i++) {
                f.init(i ? square_lds : slice_lds, wr * (S / WV), lane);
                row[i] = f.first;
                f.init(i ? square_lds : slice_lds, wc * (S / WV), lane);
                col[i] = f.first;
            }
            const auto product = [&](int left, int right, float k, Square &p1, float k1, Square &p2, float k2, Square &v) {
                Square t;
                clear(t);
                multiply<NP, S, 0, S, 0>(row[left], col[right], S / 32, t);
#pragma unroll
                for (int i = 0; i < FQ; i++)
#pragma unroll
                    for (int j = 0; j < FQ; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) v[i][j][r] = k * t[i][j][r] + k1 * p1[i][j][r] + k2 * p2[i][j][r];
            };
            const auto put = [&](char *img, Square &v) {
#pragma unroll
                for (int i = 0; i < FQ; i++)
#pragma unroll
                    for (int j = 0; j < FQ; j++) image_store(img, image0<S>(qm + 16 * i, qn + 16 * j), v[i][j]);
            };
            Square A, B, Q;
            clear(A);
            const floatx4 *in = (const floatx4 *)p.in + z * p.groups * (S * S / 4) + tid;
            constexpr int U = S == 128 ? 2 : 8;   // parts whose loads are in flight together
            for (int g = 0; g < p.groups; g += U) {
                floatx4 v[U][FQ][FQ];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < FQ; i++)
#pragma unroll
                        for (int j = 0; j < FQ; j++)
                            v[u][i][j] = g + u < p.groups ? in[(long)(g + u) * (S * S / 4) + (i * FQ + j) * NT] : (floatx4){};
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < FQ; i++)
#pragma unroll
                        for (int j = 0; j < FQ; j++) A[i][j] += v[u][i][j];
            }
#pragma unroll
            for (int i = 0; i < FQ; i++)
#pragma unroll
                for (int j = 0; j < FQ; j++) A[i][j] *= p.ga;
            put(slice_img, A);
            __syncthreads();
            product(0, 0, p.b2, A, p.b1, A, 0.0f, B);
#pragma unroll
            for (int i = 0; i < FQ; i++)
#pragma unroll
                for (int j = 0; j < FQ; j++) Q[i][j] = B[i][j];
            if (p.steps == 2) {
                Square P;
                put(square_img, B);   // nothing reads image 1 here
                __syncthreads();
                product(1, 0, p.p2, A, p.p1, A, 0.0f, P);   // (a I + B) A
                __syncthreads();
                put(slice_img, P);
                __syncthreads();
                product(0, 1, p.a2, P, p.a1, P, 0.0f, A);   // (a I + B) A (a I + B)
                __syncthreads();
                put(slice_img, A);
                __syncthreads();
                product(0, 0, p.b2, A, p.b1, A, 0.0f, B);
                __syncthreads();
                put(slice_img, Q);
                put(square_img, B);
                __syncthreads();
                product(1, 0, p.q2, Q, p.q1, B, p.q1, Q);
            }
            __syncthreads();
            put(square_img, Q);
        }
        const float qi = p.qi, qs = p.qs;
        for (int sl = blockIdx.x; sl < p.slices; sl += p.groups) {
            const int m0 = WIDE ? 0 : sl * kSlice, n0 = WIDE ? sl * kSlice : 0;
            __syncthreads();   // B is there; the slice image has been read
            {   // the slice as the product's operand: S k-rows of 128 columns, or 128 rows of S k
                pg::PFetch<kSlice, WIDE ? 1 : 0, 2, 32, WV * WV> fetch;
                const long ps = (long)rows * 128;
                fetch.init(64, ps, sl * kSlice, WIDE ? p.Cp : p.Rp, wave, lane);
                const char *base = (const char *)X + (WIDE ? (long)sl * (kSlice * 2 / 64) * ps : (long)sl * kSlice * 128);
                const int wave_u = __builtin_amdgcn_readfirstlane(wave);
                for (int q = 0; q < S / 32; q++)
#pragma unroll
                    for (int f = 0; f < fetch.PER; f++)
                        fetch.issue(f, base + q * (WIDE ? 32l * 128 : ps), 64, 32, slice_lds + q * (kSlice * 128), wave_u, lane);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            __syncthreads();
            floatx4 x[FM][FN];
            clear(x);
            if constexpr (WIDE) {
                pg::PFrag<S, 0, 2, 32> fb;
                pg::PFrag<kSlice, 1, 2, 32> fx;
                fb.init(square_lds, wr * (S / WV), lane);
                fx.init(slice_lds, wc * (kSlice / WV), lane);
                multiply<NP, S, 0, kSlice, 1>(fb.first, fx.first, S / 32, x);
            } else {
                pg::PFrag<kSlice, 0, 2, 32> fx;
                pg::PFrag<S, 0, 2, 32> fb;
                fx.init(slice_lds, wr * (kSlice / WV), lane);
                fb.init(square_lds, wc * (S / WV), lane);
                multiply<NP, kSlice, 0, S, 0>(fx.first, fb.first, S / 32, x);
            }
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    const int m = xm + 16 * i, n = xn + 16 * j;
                    const floatx4 old = image_load(slice_img, WIDE ? image1<kSlice>(m, n) : image0<kSlice>(m, n));
                    const bool in = m0 + m < p.Rp && n0 + n < p.Cp;   // past them the fetch repeated the last values
#pragma unroll
                    for (int r = 0; r < 4; r++) x[i][j][r] = in ? qi * old[r] + x[i][j][r] * qs : 0.0f;
                }
            __syncthreads();   // all waves have read the old slice
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) {
                    const int m = xm + 16 * i, n = xn + 16 * j;
                    if constexpr (WHAT == LAST) {
                        floatx4 v = x[i][j];
#pragma unroll
                        for (int r = 0; r < 4; r++) v[r] *= 1.0f / (1 << kSX);
                        store_result(d, z, m0 + m, n0 + n, v);
                    } else {
                        image_store(slice_img, slice_at(m, n), x[i][j]);
                        if (m0 + m < p.Rp && n0 + n < p.Cp) pg::plane_store(X + pg::panel_at<2>(rows, m0 + m, n0 + n), x[i][j]);
                    }
                }
            if constexpr (WHAT != LAST) {
                __syncthreads();
                add_gram();
            }
        }
    }
    if constexpr (WHAT != LAST) {
        floatx4 *out = (floatx4 *)p.out + (z * p.groups + blockIdx.x) * (S * S / 4) + tid;
#pragma unroll
        for (int i = 0; i < FQ; i++)
#pragma unroll
            for (int j = 0; j < FQ; j++) out[(i * FQ + j) * NT] = gram[i][j];
    }
}

struct SmallLayout {
    int Rp, Cp, S, slices, groups;
    bool wide;
    int64_t X, part[2], total;
};

SmallLayout small_layout(const Muon &d) {
    SmallLayout l{};
    l.Rp = (d.rows + 63) & ~63;
    l.Cp = (d.cols + 63) & ~63;
    l.wide = d.rows <= d.cols;
    l.S = std::min(l.Rp, l.Cp);
    l.slices = (std::max(l.Rp, l.Cp) + kSlice - 1) / kSlice;
    // reading a part costs 0.3 us (S = 128) or 0.08 (64), a slice 3 or 2
    double best = 1e30;
    for (int g = 1; g <= l.slices && g <= 64; g++) {
        const double us = (l.S == 128 ? 0.3 : 0.08) * g + (l.S == 128 ? 3.0 : 2.0) * ((l.slices + g - 1) / g);
        if (us < best) {
            best = us;
            l.groups = g;
        }
    }
    const auto up = [](int64_t n) { return (n + 255) & ~255ll; };
    const int64_t part = up((int64_t)d.batch * l.groups * l.S * l.S * 4);
    l.X = 0;
    l.part[0] = up((int64_t)d.batch * l.Rp * l.Cp * 4);
    l.part[1] = l.part[0] + part;
    l.total = l.part[1] + part;
    return l;
}

template <int S, bool WIDE>
void run(const Muon &d, SmallArgs a, float *const (&parts)[2], hipStream_t s) {
    const dim3 grid((unsigned)a.groups, (unsigned)d.batch);
    const Scales c = scales(d);
    const int longest = longest_group(d);
    const auto p2 = [](double v, int e) { return (float)std::ldexp(v, e); };
    a.ga = p2(1, c.A - 2 * kSX);
    a.b2 = p2(d.c, c.B - 2 * c.A);
    a.b1 = p2(d.b, c.B - c.A);
    a.p2 = p2(1, c.BA - c.A - c.B);
    a.p1 = p2(d.a, c.BA - c.A);
    a.a2 = p2(1, c.A - c.B - c.BA);
    a.a1 = p2(d.a, c.A - c.BA);
    a.q2 = p2(1, c.Q2 - 2 * c.B);
    a.q1 = p2(d.a, c.Q2 - c.B);
    a.out = parts[0];
    hipLaunchKernelGGL((muon_small_kernel<S, WIDE, FIRST>), grid, dim3(S / 32 * (S / 32) * 64), 0, s, a, d);
    for (int left = d.steps, k = 0; left > 0; k++) {
        a.steps = group_size(longest, k, left);
        left -= a.steps;
        a.qi = (float)std::pow((double)d.a, a.steps);
        a.qs = p2(1, a.steps == 2 ? -c.Q2 : -c.B);
        a.in = parts[k & 1];
        a.out = parts[(k + 1) & 1];
        if (left) hipLaunchKernelGGL((muon_small_kernel<S, WIDE, STEP>), grid, dim3(S / 32 * (S / 32) * 64), 0, s, a, d);
        else hipLaunchKernelGGL((muon_small_kernel<S, WIDE, LAST>), grid, dim3(S / 32 * (S / 32) * 64), 0, s, a, d);
    }
}

}  // namespace

int64_t muon_small_workspace(const Muon &d) { return small_layout(d).total; }

void muon_small(const Muon &d, const double *part, int nparts, void *ws, hipStream_t s) {
    const SmallLayout l = small_layout(d);
    SmallArgs a{};
    a.X = (half_t *)((char *)ws + l.X);
    a.sx = (long)l.Rp * l.Cp * 2;
    a.Rp = l.Rp;
    a.Cp = l.Cp;
    a.slices = l.slices;
    a.groups = l.groups;
    a.part = part;
    a.parts = nparts;
    float *const parts[2] = {(float *)((char *)ws + l.part[0]), (float *)((char *)ws + l.part[1])};
    if (l.S == 64) l.wide ? run<64, true>(d, a, parts, s) : run<64, false>(d, a, parts, s);
    else l.wide ? run<128, true>(d, a, parts, s) : run<128, false>(d, a, parts, s);
}

}  // namespace ah
