// linear_ce.hip — loss and gradients of softmax cross-entropy over a linear head's logits, of which a piece of rows is in memory at a time.
//
//   z = X W^T + b,  lse_n = log sum_v exp z_nv,  l_n = lse_n - z_n,y(n),  P = exp(z - lse) - onehot(y)
//   dX = s P W,  dW = s P^T X,  db = s sum_n P        (s: the gradient's scale, divided by the number of counted rows for a mean)
//
// The counted rows of X are gathered first (rows whose label is outside [0, V) cost nothing after that, and whatever they hold
// stays out of the products), then worked on in pieces of rows. Per piece: the logits' product, whose epilogue keeps each row's
// maximum and sum of exponentials per wave tile of the vocabulary and writes the piece's logits; one pass that joins the statistics of
// a row; one pass that turns the piece into P in place; the two gradient products. Keeping a logit moves 14 (f16 gradients) or 20
// bytes, computing it again would cost a third product, 2 D operations: at 5 TB/s and 1 PFLOP/s the two are even at D = 1400 and 2000, but
// only 8 of the bytes stand outside a product that hides them (at 4096 x 4096 x 131072 P's pass is 4% of the time).
//
// Precision. f16 operands are exact in the products; f32 operands are carried as two f16 planes scaled by a power of two taken
// from their largest magnitude (plane_gemm.h). P is formed in f32 and goes into the gradient products as 2^15 P in one f16 plane for f16
// gradients (one rounding, 2^-11 of |P| above 2^-29 at most, 2^-40 below; what it leaves at the label, mostly the largest entry, is added apart:
// add_label_rows, add_labelled) and in two for f32 gradients (2^-22 above 2^-18, 2^-40 below).
// Statistics, losses and sums are f32; sums over rows and pieces run in a fixed order, so results repeat bit for bit.
#include "linear_ce.h"

#include <algorithm>

#include "act.h"
#include "linear_ce_few.h"
#include "plane_gemm.h"

namespace ah {
namespace {

using pg::h4;
using pg::h8;
using pg::magnitude;
using pg::pack_row;
using pg::plane_exp;
typedef half_t h2 __attribute__((ext_vector_type(2)));

constexpr int kPScale = 15;   // P is carried as 2^15 P: |P| <= 1, so the largest value is 2^15

// Device scalars at the workspace's start.
struct Scalars {
    int count;                // counted rows
    unsigned xmax, wmax;      // bits of the largest magnitudes (f32 operands)
    int pad;
};

__device__ __forceinline__ int chunk_rows(const int *count, int row0, int rows) { return max(0, min(rows, *count - row0)); }

// ── rows that count ────────────────────────────────────────────────────────────

constexpr int kMaxBlocks = 1024;  // workgroups that look for the largest magnitudes, at most

struct ScanArgs {
    const int *labels;
    int N, V, D, Wrows;    // Wrows: V, or 0 where W need not be looked at
    int *rowmap, *pos, *lab;
    Scalars *sc;
    const float *X, *W;    // f32 operands
    long ldx, ldw;
    uint2 *maxes;          // [workgroup] bits of the largest magnitudes of X's counted rows and of W
};

// Workgroup 0: the counted rows in order (rowmap), each row's place among them or -1 (pos), their labels. 16 rows a thread at a
// time, so that their labels are loaded together.
__device__ __forceinline__ void index_rows(const ScanArgs &a) {
    __shared__ int sums[4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int done = 0;
    for (int r0 = 0; r0 < a.N; r0 += 4096) {
        typedef int i4 __attribute__((ext_vector_type(4), aligned(4)));
        const int first = r0 + t * 16;
        int y[16], c = 0;
        if (first + 15 < a.N) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const i4 v = *(const i4 *)(a.labels + first + i);
#pragma unroll
                for (int k = 0; k < 4; k++) y[i + k] = v[k];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = first + i < a.N ? a.labels[first + i] : -1;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) c += (unsigned)y[i] < (unsigned)a.V;
        int inc = c;
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(inc, o, 64);
            if (lane >= o) inc += u;
        }
        __syncthreads();
        if (lane == 63) sums[wave] = inc;
        __syncthreads();
        int at = done + inc - c;
        for (int w = 0; w < 4; w++) {
            if (w < wave) at += sums[w];
            done += sums[w];
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = first + i;
            const bool ok = (unsigned)y[i] < (unsigned)a.V;
            if (r < a.N) a.pos[r] = ok ? at : -1;
            if (ok) {
                a.rowmap[at] = r;
                a.lab[at++] = y[i];
            }
        }
    }
    if (t == 0) a.sc->count = done;
}

// Workgroup 0 indexes the rows; the others (f32 operands) find the largest magnitudes of W and of the counted rows of X, a wave per
// stretch of 2048 values of a row. The bits of non-negative floats order as integers. Infinities and NaN are passed over: they make their
// own row's logits NaN under any scale, and the other rows' scale is not theirs.
__global__ __launch_bounds__(256) void lce_scan_kernel(ScanArgs a) {
    if (blockIdx.x == 0) {
        index_rows(a);
        return;
    }
    __shared__ unsigned red[2][4];
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, segs = (a.D + 2047) / 2048;
    unsigned mx = 0, mw = 0;
    for (long q = (long)(blockIdx.x - 1) * 4 + wave; q < ((long)a.N + a.Wrows) * segs; q += (long)(gridDim.x - 1) * 4) {
        const long r = q / segs;
        const int c0 = (int)(q - r * segs) * 2048 + lane * 4, end = min(a.D, c0 - lane * 4 + 2048);
        const bool x = r < a.N;
        if (x && (unsigned)a.labels[r] >= (unsigned)a.V) continue;
        const uint32_t *p = (const uint32_t *)(x ? a.X + r * a.ldx : a.W + (r - a.N) * a.ldw);
        unsigned m = 0;
#pragma unroll
        for (int k = 0; k < 2048; k += 256) {
            const int c = c0 + k;
            if (c + 3 < end) {
                const u4 v = *(const u4 *)(p + c);
                m = max(m, max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3]))));
            } else {
                for (int u = c; u < end; u++) m = max(m, magnitude(p[u]));
            }
        }
        if (x) mx = max(mx, m);
        else mw = max(mw, m);
    }
    for (int o = 32; o >= 1; o >>= 1) {
        mx = max(mx, (unsigned)__shfl_xor((int)mx, o, 64));
        mw = max(mw, (unsigned)__shfl_xor((int)mw, o, 64));
    }
    if (lane == 0) {
        red[0][wave] = mx;
        red[1][wave] = mw;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        a.maxes[blockIdx.x - 1] = make_uint2(max(max(red[0][0], red[0][1]), max(red[0][2], red[0][3])), max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3])));
}

// The workgroups' largest magnitudes joined; all 256 threads of a workgroup.
__device__ __forceinline__ uint2 join_maxes(const uint2 *maxes, int n) {
    __shared__ uint2 red[4];
    uint2 m = make_uint2(0, 0);
    for (int i = threadIdx.x; i < n; i += 256) m = make_uint2(max(m.x, maxes[i].x), max(m.y, maxes[i].y));
    for (int o = 32; o >= 1; o >>= 1)
        m = make_uint2(max(m.x, (unsigned)__shfl_xor((int)m.x, o, 64)), max(m.y, (unsigned)__shfl_xor((int)m.y, o, 64)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    return make_uint2(max(max(red[0].x, red[1].x), max(red[2].x, red[3].x)), max(max(red[0].y, red[1].y), max(red[2].y, red[3].y)));
}

// A wave a row. Of the first N + 64, row r of X goes to its place among the counted rows, or its dX and outputs are cleared; the last
// 64 clear the packed rows that fill up the last stage of the dW product. The others pack W.
struct PackArgs {
    half_t *X, *W;         // W: null where it is read as it lies
    int Np, Dp, piece;     // padded rows and features; rows of a piece: each piece has panels of its own
    int wshift, wstored;   // log2 of the rows of a block of W, and the rows that its panels are apart
};
template <int P>
__global__ __launch_bounds__(256) void lce_pack_kernel(LinearCe d, PackArgs a, const int *pos, Scalars *sc, const uint2 *maxes, int blocks) {
    int ex = 0, ew = 0;
    if constexpr (P == 2) {
        const uint2 top = join_maxes(maxes, blocks);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            sc->xmax = top.x;
            sc->wmax = top.y;
        }
        ex = plane_exp(top.x);
        ew = plane_exp(top.y);
    }
    constexpr int ESZ = P == 1 ? 2 : 4;
    const int lane = threadIdx.x & 63, count = sc->count, Dp = a.Dp;
    const long total = (long)d.N + 64 + (a.W ? d.V : 0);
    const auto xrow = [&](auto planes, int q, const void *in, int D, int width, int e) {   // row q of the counted ones
        const int first = q / a.piece * a.piece;
        pack_row<decltype(planes)::value>(a.X + (long)first * Dp * P, min(a.piece, a.Np - first), q - first, in, D, width, e);
    };
    for (long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6); r < total; r += (long)gridDim.x * 4) {
        if (r < d.N) {
            const int q = pos[r];
            if (q >= 0) {
                xrow(std::integral_constant<int, P>(), q, (const char *)d.X + r * d.ldx * ESZ, d.D, Dp, ex);
                continue;
            }
            if (d.dX)
                for (int i = lane * 4; i < d.D; i += 256) {
                    if (d.g16) pg::store4((half_t *)d.dX + r * d.lddx, i, d.D, (floatx4){});
                    else pg::store4((float *)d.dX + r * d.lddx, i, d.D, (floatx4){});
                }
            if (lane == 0) {
                if (d.rowloss) d.rowloss[r] = 0.0f;
                if (d.lse) d.lse[r] = 0.0f;
            }
        } else if (r < d.N + 64) {
            const int q = count + (int)(r - d.N);
            if (q < ((count + 63) & ~63)) xrow(std::integral_constant<int, 1>(), q, nullptr, 0, Dp * P, 0);
        } else {
            const int v = (int)(r - d.N - 64);
            pack_row<P>(a.W + (long)(v >> a.wshift) * a.wstored * Dp * P, a.wstored, v & (int)((1u << a.wshift) - 1), (const char *)d.W + (long)v * d.ldw * ESZ, d.D, Dp, ew);
        }
    }
}

// ── the logits' product ────────────────────────────────────────────────────────

enum { KEEP_NONE = 0, KEEP_Z = 1 };

struct LogitArgs {
    pg::Operand X, W;
    int V, nk, tiles_m;
    pg::Work w;
    const Scalars *sc;
    int row0, rows;       // the piece
    int planes;           // operands are scaled planes
    const void *bias;
    int bias16;
    const int *lab;       // of the piece's rows
    float *zt;            // each row's logit of its label
    float2 *stats;        // [rows][T]: maximum and sum of exponentials of each wave tile's columns
    int T;
    char *E;              // the piece's logits in panels of 128 bytes, 32 columns each
    int Vp;
};

// Bytes to a logit of the piece: 32 columns fill a panel's row, as the two planes that replace them do (one plane of 64 columns fills
// every other panel).
__device__ __forceinline__ long z_at(long rows, long r, long c) { return ((c >> 5) * rows + r) * 128 + (c & 31) * 4; }

// Tiles are walked down the rows first: the tiles of one run share their columns of W, the larger operand.
template <class C>
__device__ __forceinline__ void logits_tile(const LogitArgs &a, int tile, int &m0, int &n0) {
    m0 = tile % a.tiles_m * C::BM;
    n0 = tile / a.tiles_m * C::BN;
}

// What follows the product, for NR accumulator rows from row i0. What the rows share (biases, where the columns lie in E) is
// formed once; their labels are loaded together.
template <class C, int KEEP, int NR>
__device__ __forceinline__ void logits_rows(const LogitArgs &a, int M, int m0, int n0, int i0, floatx4 (&z)[NR][C::FB]) {
    const pg::Place<C> at(m0, n0);
    const int tcol = n0 / C::WN + at.wave % C::WVN, m1 = at.m + 16 * i0;
    const int e = a.planes ? -(plane_exp(a.sc->xmax) + plane_exp(a.sc->wmax)) : 0;
    const float ninf = -__builtin_inff();
    const bool whole = n0 + C::BN <= a.V;
    int y[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) y[i] = m1 + 16 * i < M ? a.lab[m1 + 16 * i] - at.n : -1;
    floatx4 bias[C::FB];   // -inf past the last class
#pragma unroll
    for (int j = 0; j < C::FB; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int n = at.n + 16 * j + r;
            bias[j][r] = n >= a.V ? ninf : !a.bias ? 0.0f : a.bias16 ? (float)((const half_t *)a.bias)[n] : ((const float *)a.bias)[n];
        }
    // this lane's first column in E; 16 j columns on are 64 (j & 1) bytes further in the panel and j / 2 panels on
    const int nw = n0 + (at.wave % C::WVN) * C::WN;
    char *const tile = KEEP == KEEP_NONE ? nullptr : a.E + z_at(a.rows, m0, nw);
    const uint32_t panel = (uint32_t)a.rows * 128;
#pragma unroll
    for (int i = 0; i < NR; i++) {
        __builtin_amdgcn_sched_barrier(0);   // one row at a time: together they spill
        int m = m1 + 16 * i;
        asm volatile("" : "+v"(m));
        float mx = ninf;
#pragma unroll
        for (int j = 0; j < C::FB; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                z[i][j][r] = ldexpf(z[i][j][r], e) + bias[j][r];
                mx = fmaxf(mx, z[i][j][r]);
            }
        if ((unsigned)y[i] < (unsigned)(16 * C::FB) && (y[i] & 15) < 4) {   // the label's column is this lane's
            float zt = 0.0f;
#pragma unroll
            for (int j = 0; j < C::FB; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) zt = y[i] == 16 * j + r ? z[i][j][r] : zt;
            a.zt[m] = zt;
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ref = mx == ninf ? 0.0f : mx;   // columns that are all -inf (a bias that rules them out) add nothing
        float sum = 0.0f;
        const uint32_t off = (uint32_t)(m - m0) * 128 + (at.lane >> 4) * 16;
#pragma unroll
        for (int j = 0; j < C::FB; j++) {
#pragma unroll
            for (int r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f((z[i][j][r] - ref) * kLog2e);
            if (KEEP != KEEP_NONE && m < M && (whole || at.n + 16 * j < a.Vp))
                *(floatx4 *)(tile + (off + (uint32_t)(j / 2) * panel) + (j & 1) * 64) = z[i][j];
        }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (at.lane < 16 && m < M) a.stats[(long)m * a.T + tcol] = make_float2(mx, sum);
    }
}

template <class C, int KEEP>
__global__ __launch_bounds__(C::NT, 2) void lce_logits_kernel(LogitArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows);
    int tile, slot, first, count, m0, n0;
    pg::pick(a.w, blockIdx.x, a.nk, tile, slot, first, count);
    logits_tile<C>(a, tile, m0, n0);
    if (m0 >= M) return;
    floatx4 acc[C::FA][C::FB];
    pg::contract<C, true>(a.X, a.W, m0, n0, first, count, smem, acc);
    if (slot >= 0) {
        pg::store_partials<C>(a.w.part, slot, acc);
        return;
    }
    logits_rows<C, KEEP, C::FA>(a, M, m0, n0, 0, acc);
}

// The same from X and W as they lie, for few rows.
struct FewArgs {
    const void *X, *W;
    long ldx, ldw;
    const int *rowmap;
    int D, Vp;
};
template <class C, int KEEP, bool F16>
__device__ __forceinline__ void few_logits(const LogitArgs &a, const FewArgs &f, int M, char *smem) {
    int tile, slot, first, count, m0, n0;
    pg::pick(a.w, blockIdx.x, a.nk, tile, slot, first, count);
    logits_tile<C>(a, tile, m0, n0);
    floatx4 acc[C::FA][C::FB];
    few::contract_along<C, F16>(f.X, f.ldx, f.rowmap, M, f.W, f.ldw, a.V, f.D, n0, first, count, smem, acc);
    if (slot >= 0) pg::store_partials<C>(a.w.part, slot, acc);
    else logits_rows<C, KEEP, C::FA>(a, M, m0, n0, 0, acc);
}
// Room for 16 FA rows; the rows that count may be fewer, and then the tile is.
template <int FA, int KEEP, bool F16>
__global__ __launch_bounds__(256, 2) void lce_few_logits_kernel(LogitArgs a, FewArgs f) {
    __shared__ __attribute__((aligned(16))) char smem[few::smem_bytes<few::Tile<FA, 2>>()];
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows);
    if (M == 0) return;
    few::with_rows<FA>(M, [&](auto fa) { few_logits<few::Tile<fa, 2>, KEEP, F16>(a, f, M, smem); });
}
template <int FA, int KEEP>
__global__ __launch_bounds__(256) void lce_few_logits_join_kernel(LogitArgs a) {
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows);
    if (16 * (int)blockIdx.y >= M) return;
    few::with_rows<FA>(M, [&](auto fa) {
        typedef few::Tile<fa, 2> C;
        int m0, n0;
        logits_tile<C>(a, a.w.whole + blockIdx.x, m0, n0);
        floatx4 z[1][C::FB];
        pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, z[0]);
        logits_rows<C, KEEP, 1>(a, M, m0, n0, blockIdx.y, z);
    });
}

template <class C, int KEEP>
__global__ __launch_bounds__(C::NT) void lce_logits_join_kernel(LogitArgs a) {
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows);
    int m0, n0;
    logits_tile<C>(a, a.w.whole + blockIdx.x, m0, n0);
    if (m0 >= M) return;
    floatx4 z[1][C::FB];
    pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, z[0]);
    logits_rows<C, KEEP, 1>(a, M, m0, n0, blockIdx.y, z);
}

// ── a row's statistics ─────────────────────────────────────────────────────────

// One wave per row joins the T tiles' (maximum, sum) pairs.
__global__ __launch_bounds__(256) void lce_rows_kernel(const Scalars *sc, int row0, int rows, const float2 *stats, int T, const float *zt,
                                                       const int *rowmap, float *lse_c, float *loss_c, float *rowloss, float *lse_out) {
    const int M = chunk_rows(&sc->count, row0, rows), lane = threadIdx.x & 63;
    const int m = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= M) return;
    const float2 *p = stats + (long)m * T;
    float mx = -__builtin_inff();
    bool nan = false;
#pragma unroll 8
    for (int t = lane; t < T; t += 64) {
        mx = fmaxf(mx, p[t].x);
        nan |= p[t].y != p[t].y;
    }
    mx = wave_max(mx);
    const float ref = mx == -__builtin_inff() ? 0.0f : mx;
    float s = 0.0f;
#pragma unroll 8
    for (int t = lane; t < T; t += 64) {
        const float2 v = p[t];
        if (v.y > 0.0f) s += v.y * __builtin_amdgcn_exp2f((v.x - ref) * kLog2e);
    }
    s = wave_sum(s);
    if (__ballot(nan)) s = __builtin_nanf("");   // a NaN logit, which the maximum passes over
    if (lane == 0) {
        const float lse = mx + logf(s), l = lse - zt[m];
        lse_c[m] = lse;
        loss_c[m] = l;
        const int r = rowmap[m];
        if (rowloss) rowloss[r] = l;
        if (lse_out) lse_out[r] = lse;
    }
}

// ── P, in place of what the product kept ───────────────────────────────────────

struct GradArgs {
    const Scalars *sc;
    int row0, rows, V, Vp;
    const float *lse, *zt;
    const int *lab;
    char *E;                        // the logits, then P
    float *res;                     // one plane: what its rounding leaves of each row's P at its label
    float *dbpart;                  // [row block of the piece][V] column sums of P, or null
};

constexpr int kGradRows = 64;       // rows of a block; also the k of a one-plane stage, up to which rows are cleared

// A thread owns 4 columns, 8 threads a panel's 128 bytes of a row, and walks down kGradRows / 4 rows. The change in place is sound
// because the 128 bytes of planes, or the 256 of 64 columns that one plane takes half of, belong to one wave, whose loads return before
// it stores.
template <int PLANES>
__global__ __launch_bounds__(256) void lce_grad_kernel(GradArgs a) {
    constexpr int NC = 4;
    __shared__ float red[3][64][NC];
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows), Mp = (M + 63) & ~63;
    const int n = (blockIdx.x * 64 + (threadIdx.x & 63)) * NC, w = threadIdx.x >> 6;
    const int r0 = blockIdx.y * kGradRows;
    if (r0 >= Mp) return;
    float col[NC] = {};
    if (n < a.Vp) {
        for (int k = w; k < kGradRows; k += 4) {
            const int m = r0 + k;
            floatx4 p = {};
            char *at = a.E + z_at(a.rows, m, n);
            if (m < M) {
                const float lse = a.lse[m];
                const int y = a.lab[m] - n;
                const floatx4 z = *(const floatx4 *)at;
#pragma unroll
                for (int c = 0; c < NC; c++) p[c] = exp_of(z[c] - lse) * (float)(1 << kPScale);
                if ((unsigned)y < (unsigned)NC) {
                    const float q = expm1f(a.zt[m] - lse) * (float)(1 << kPScale);
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        if (c == y) p[c] = q;
                    if constexpr (PLANES == 1) a.res[m] = q - (float)(half_t)q;
                }
            }
#pragma unroll
            for (int c = 0; c < NC; c++) col[c] += p[c];
            if constexpr (PLANES == 1) {
                h4 h;
#pragma unroll
                for (int c = 0; c < NC; c++) h[c] = (half_t)p[c];
                *(h4 *)((half_t *)a.E + pg::panel_at<1>(2l * a.rows, m, n)) = h;
            } else {
                pg::plane_store((half_t *)a.E + pg::panel_at<2>(a.rows, m, n), p);
            }
        }
    }
    if (!a.dbpart) return;
    if (w > 0)
#pragma unroll
        for (int c = 0; c < NC; c++) red[w - 1][threadIdx.x & 63][c] = col[c];
    __syncthreads();
    if (w == 0)
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (n + c < a.V)
                a.dbpart[(long)blockIdx.y * a.V + n + c] =
                    col[c] + red[0][threadIdx.x][c] + red[1][threadIdx.x][c] + red[2][threadIdx.x][c];
}

__device__ __forceinline__ float grad_mult(const Scalars *sc, float grad_scale, int mean) {
    return mean ? grad_scale / (float)max(1, sc->count) : grad_scale;
}

// db's sum of P over the rows to the end of the piece [row0, row0 + rows): what the pieces before left in dbias, then the piece's row
// blocks in order.
__device__ __forceinline__ float db_sum(const Scalars *sc, int row0, int rows, const float *part, int V, const float *dbias, int n) {
    const int blocks = (chunk_rows(&sc->count, row0, rows) + kGradRows - 1) / kGradRows;
    float s = row0 ? dbias[n] : 0.0f;
    for (int b = 0; b < blocks; b++) s += part[(long)b * V + n];
    return s;
}
// After a piece that others follow.
__global__ __launch_bounds__(256) void lce_db_kernel(const Scalars *sc, int row0, int rows, const float *part, int V, float *dbias) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n < V) dbias[n] = db_sum(sc, row0, rows, part, V, dbias, n);
}

// Workgroup 0: the loss, in f64. The others: db, after the last piece.
__global__ __launch_bounds__(256) void lce_finish_kernel(const Scalars *sc, const float *loss_c, int mean, float *loss, int row0, int rows,
                                                         const float *part, int V, float grad_scale, float *dbias) {
    const int c = sc->count, t = threadIdx.x;
    if (blockIdx.x > 0) {
        const int n = (blockIdx.x - 1) * 256 + t;
        if (n < V) dbias[n] = ldexpf(db_sum(sc, row0, rows, part, V, dbias, n), -kPScale) * grad_mult(sc, grad_scale, mean);
        return;
    }
    __shared__ double red[4];
    double s = 0.0;
    for (int i = t; i < c; i += 256) s += (double)loss_c[i];
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((t & 63) == 0) red[t >> 6] = s;
    __syncthreads();
    if (t == 0) {
        s = red[0] + red[1] + red[2] + red[3];
        *loss = (float)(mean && c > 0 ? s / c : s);
    }
}

// ── the gradient products ──────────────────────────────────────────────────────

struct ProductArgs {
    pg::Operand A, B;
    int M, N, tiles_m, tiles_n;
    pg::Work w;
    int cap;               // partial tiles that there is room for
    const Scalars *sc;
    int row0, rows;
    int rows_are;          // 0: C's rows are the piece's (dX); 1: k runs over them (dW)
    int k;                 // k of dX
    const int *rowmap;     // dX: where C's rows go
    const unsigned *bmax;  // largest magnitude of the other operand (planes), or null
    float grad_scale;
    int mean;
    void *C;
    long ldc;
    int out16;             // C is f16
    const float *acc_in;   // dW: the earlier pieces' sum, or null
    float *acc_out;        // dW: the sum goes there in f32 and C is left, or null
    long ldacc;
    // P in one plane: what its rounding left of each of the piece's rows at its label, the labels, and W as it lies
    const float *res;
    const int *lab;
    const half_t *W;
    long ldw;
};

__device__ __forceinline__ int product_size(const ProductArgs &a, int &nk, int BK) {
    const int rows = chunk_rows(&a.sc->count, a.row0, a.rows);
    nk = ((a.rows_are == 0 ? a.k : (rows + 63) & ~63) + BK - 1) / BK;
    return a.rows_are == 0 ? rows : a.M;
}

// The work that is there: the host plans for rows that all count; where fewer do, dX has fewer tiles, and its workgroups are dealt
// to those (8192 rows of 2048 features over 32000 classes of which three quarters count are 192 tiles of 256: 1.5 ms in one piece
// each, 1.25 in four, and 0.05 for the join).
template <class C>
__device__ __forceinline__ pg::Work product_work(const ProductArgs &a, int M, int nk, int &tiles_m) {
    tiles_m = a.rows_are == 0 ? (M + C::BM - 1) / C::BM : a.tiles_m;
    if (a.rows_are == 1 || tiles_m == a.tiles_m) return a.w;
    return pg::deal(tiles_m * a.tiles_n, nk, C::BM == 256 ? 256 : 512, a.cap, C::BM == 256 ? 0.07f : C::BM == 128 ? 0.03f : 0.02f, a.w.part);
}

template <class C>
__device__ __forceinline__ void product_tile(const ProductArgs &a, int tile, int tiles_m, int &m0, int &n0) {
    int tr, tc;
    pg::grouped_tile(tile, tiles_m, a.tiles_n, tr, tc);
    m0 = tr * C::BM;
    n0 = tc * C::BN;
}

// What follows the product, for accumulator row i: row m of C, which is row `row` of the output.
template <class C>
__device__ __forceinline__ void product_row(const ProductArgs &a, int m, long row, int n0, float mult, int e, const floatx4 (&acc)[C::FB]) {
    const pg::Place<C> at(0, n0);
#pragma unroll
    for (int j = 0; j < C::FB; j++) {
        const int n = at.n + 16 * j;
        if (n >= a.N) continue;
        floatx4 v;
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = ldexpf(acc[j][r], e) * mult;
        if (a.acc_in) v += pg::load4(a.acc_in + (long)m * a.ldacc, n, a.N);
        if (a.acc_out) pg::store4(a.acc_out + (long)m * a.ldacc, n, a.N, v);
        else if (a.out16) pg::store4((half_t *)a.C + row * a.ldc, n, a.N, v);
        else pg::store4((float *)a.C + row * a.ldc, n, a.N, v);
    }
}

// NR accumulator rows from row i0; their places are loaded together.
template <class C, int NR>
__device__ __forceinline__ void product_rows(const ProductArgs &a, int M, int m0, int n0, int i0, const floatx4 (&acc)[NR][C::FB]) {
    const pg::Place<C> at(m0, n0);
    const int m1 = at.m + 16 * i0, e = -kPScale - (a.bmax ? plane_exp(*a.bmax) : 0);
    const float mult = grad_mult(a.sc, a.grad_scale, a.mean);
    int row[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) row[i] = m1 + 16 * i >= M ? -1 : a.rowmap ? a.rowmap[m1 + 16 * i] : m1 + 16 * i;
#pragma unroll
    for (int i = 0; i < NR; i++)
        if (row[i] >= 0) product_row<C>(a, m1 + 16 * i, row[i], n0, mult, e, acc[i]);
}

// P at the label is near -1 in most rows while the others are small, so in one plane its rounding (2^-11 of it at most) is most of what a
// gradient is off by: 1.4e-4 beside the 2.1e-4 of an f16 output's own rounding. What is left of it there, res, is added to the products.
// dX: row m gets res times the label's row of W, from the workgroup that has that class in its k range [k0, k1).
template <class C>
__device__ __forceinline__ void add_label_rows(const ProductArgs &a, int M, int m0, int n0, int k0, int k1, floatx4 (&acc)[C::FA][C::FB]) {
    const pg::Place<C> at(m0, n0);
    int y[C::FA];
    float res[C::FA];
#pragma unroll
    for (int i = 0; i < C::FA; i++) {   // all together, for one wait
        const int m = min(at.m + 16 * i, M - 1);
        y[i] = a.lab[m];
        res[i] = a.res[m];
    }
#pragma unroll
    for (int i = 0; i < C::FA; i++) {
        __builtin_amdgcn_sched_barrier(0);
        if (at.m + 16 * i >= M || y[i] < k0 || y[i] >= k1) continue;
        const half_t *w = a.W + (long)y[i] * a.ldw;
#pragma unroll
        for (int j = 0; j < C::FB; j++) acc[i][j] += res[i] * pg::load4(w, at.n + 16 * j, a.N);
    }
}

// dW: row v gets the sum of res times X over the rows n in [k0, k1) whose label it is. The workgroup looks through 512 labels a wave at a
// time and lists those of each row of waves, in a fixed order; a wave adds its row's 32 at a time by one more product: A is res at
// (label, entry), B the listed rows of X. (Every wave through all labels for itself took 11 us a tile of 4096 rows.)
template <class C>
__device__ __forceinline__ void add_labelled(const ProductArgs &a, int m0, int n0, int k0, int k1, char *smem, floatx4 (&acc)[C::FA][C::FB]) {
    constexpr int G = C::WVM, R = C::NW * 512;
    static_assert((G * R + C::NW * G) * 4 <= C::SMEM && R <= 1 << 16, "the lists fit the stages' buffers, an entry 16 + 16 bits");
    uint32_t *const list = (uint32_t *)smem;   // [row of waves][R]: row of X from the chunk's first, the label's place in the waves' rows
    int *const counts = (int *)smem + G * R;   // [wave][row of waves]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, nw = n0 + wave % C::WVN * C::WN;
    for (int c0 = k0; c0 < k1; c0 += R) {
        typedef int i4 __attribute__((ext_vector_type(4)));
        const int n = c0 + wave * 512 + lane * 8;
        int y[8], at[G];
#pragma unroll
        for (int q = 0; q < 8; q += 4) {
            i4 l = {};
            if (n + q < k1) l = *(const i4 *)(a.lab + n + q);
#pragma unroll
            for (int r = 0; r < 4; r++) y[q + r] = n + q + r < k1 ? l[r] - m0 : -1;
        }
        const auto hit = [&](int q, int g) { return (unsigned)(y[q] - g * C::WM) < (unsigned)C::WM; };
#pragma unroll
        for (int g = 0; g < G; g++) {
            at[g] = 0;
#pragma unroll
            for (int q = 0; q < 8; q++) at[g] += __popcll(__ballot(hit(q, g)));
            if (lane == 0) counts[wave * G + g] = at[g];
        }
        __syncthreads();
        int mine = 0;   // entries of this wave's row
#pragma unroll
        for (int g = 0; g < G; g++) {
            at[g] = 0;
#pragma unroll
            for (int w = 0; w < C::NW; w++) {
                const int c = counts[w * G + g];
                if (w < wave) at[g] += c;
                if (g == wave / C::WVN) mine += c;
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const uint64_t hits = __ballot(hit(q, g));
                if (hit(q, g)) list[g * R + at[g] + __popcll(hits & ((1ull << lane) - 1))] = (uint32_t)(n + q - c0) | (uint32_t)(y[q] - g * C::WM) << 16;
                at[g] += __popcll(hits);
            }
        __syncthreads();
        const uint32_t *const own = list + wave / C::WVN * R;
        for (int first = 0; first < mine; first += 32) {
            uint32_t v[8];
            const char *row[8];
            float res[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = own[min(first + 8 * (lane >> 4) + k, mine - 1)];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                row[k] = a.B.p + (long)(c0 + (int)(v[k] & 0xffff)) * 128 + col * 2;
                res[k] = a.res[c0 + (int)(v[k] & 0xffff)];
            }
            h8 x[C::FA];
            constexpr int H = C::FB > 4 ? C::FB / 2 : C::FB;   // columns whose loads are in flight together
#pragma unroll
            for (int j0 = 0; j0 < C::FB; j0 += H) {
                h8 b[H];
#pragma unroll
                for (int j = 0; j < H; j++) {
                    const int c = min(nw + 16 * (j0 + j), a.B.rows - 16);   // past the last feature: those columns are not stored
                    const long X = (long)(c >> 6) * a.B.ps + (c & 63) * 2;
#pragma unroll
                    for (int k = 0; k < 8; k++) b[j][k] = *(const half_t *)(row[k] + X);
                }
                if (j0 == 0)
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const half_t r = (half_t)res[k];
#pragma unroll
                        for (int i = 0; i < C::FA; i++)
                            x[i][k] = first + 8 * (lane >> 4) + k < mine && (int)(v[k] >> 16) == 16 * i + col ? r : (half_t)0;
                    }
#pragma unroll
                for (int j = 0; j < H; j++)
#pragma unroll
                    for (int i = 0; i < C::FA; i++) acc[i][j0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[j], x[i], acc[i][j0 + j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();   // the lists have been read
    }
}

template <class C>
__global__ __launch_bounds__(C::NT, 2) void lce_product_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
    int nk, tiles_m, tile, slot, first, count, m0, n0;
    const int M = product_size(a, nk, C::BK);
    const pg::Work w = product_work<C>(a, M, nk, tiles_m);
    if ((int)blockIdx.x >= w.blocks()) return;
    pg::pick(w, blockIdx.x, nk, tile, slot, first, count);
    product_tile<C>(a, tile, tiles_m, m0, n0);
    floatx4 acc[C::FA][C::FB];
    pg::contract<C, C::TA == 0>(a.A, a.B, m0, n0, first, count, smem, acc);   // B is W for dX
    if constexpr (C::PA == 1) {
        if constexpr (C::TA == 0) {
            add_label_rows<C>(a, M, m0, n0, first * C::BK, (first + count) * C::BK, acc);
        } else {
            __syncthreads();   // the stages' buffers are free
            const int rows = chunk_rows(&a.sc->count, a.row0, a.rows);
            add_labelled<C>(a, m0, n0, first * C::BK, min(rows, (first + count) * C::BK), smem, acc);
        }
    }
    if (slot >= 0) {
        pg::store_partials<C>(w.part, slot, acc);
        return;
    }
    product_rows<C, C::FA>(a, M, m0, n0, 0, acc);
}

// dX from W as it lies, for few rows: one row of tiles.
template <class C, int PP, bool F16>
__device__ __forceinline__ void few_dx(const ProductArgs &a, const FewArgs &f, const char *P, int M, char *smem) {
    int tile, slot, first, count;
    pg::pick(a.w, blockIdx.x, (a.k + few::across_v(PP) - 1) / few::across_v(PP), tile, slot, first, count);
    floatx4 acc[C::FA][C::FB];
    few::contract_across<C, PP, F16>(P, PP == 1 ? 2l * a.rows : a.rows, f.Vp, f.W, f.ldw, a.k, a.N, tile * C::BN, first, count, smem, acc);
    if constexpr (PP == 1) add_label_rows<C>(a, M, 0, tile * C::BN, first * few::across_v(PP), (first + count) * few::across_v(PP), acc);
    if (slot >= 0) pg::store_partials<C>(a.w.part, slot, acc);
    else product_rows<C, C::FA>(a, M, 0, tile * C::BN, 0, acc);
}
template <int FA, int PP, bool F16>
__global__ __launch_bounds__(256, 2) void lce_few_dx_kernel(ProductArgs a, FewArgs f, const char *P) {
    __shared__ __attribute__((aligned(16))) char smem[few::smem_bytes<few::Tile<FA, 4>>()];
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows);
    if (M == 0) return;
    few::with_rows<FA>(M, [&](auto fa) { few_dx<few::Tile<fa, 4>, PP, F16>(a, f, P, M, smem); });
}
template <int FA>
__global__ __launch_bounds__(256) void lce_few_dx_join_kernel(ProductArgs a) {
    const int M = chunk_rows(&a.sc->count, a.row0, a.rows);
    if (16 * (int)blockIdx.y >= M) return;
    few::with_rows<FA>(M, [&](auto fa) {
        typedef few::Tile<fa, 4> C;
        floatx4 v[1][C::FB];
        pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, v[0]);
        product_rows<C, 1>(a, M, 0, (a.w.whole + blockIdx.x) * C::BN, blockIdx.y, v);
    });
}

template <class C>
__global__ __launch_bounds__(C::NT) void lce_product_join_kernel(ProductArgs a) {
    int nk, tiles_m, m0, n0;
    const int M = product_size(a, nk, C::BK);
    const pg::Work w = product_work<C>(a, M, nk, tiles_m);
    if ((int)blockIdx.x >= w.rest || w.splits == 1) return;
    product_tile<C>(a, w.whole + blockIdx.x, tiles_m, m0, n0);
    floatx4 v[1][C::FB];
    pg::sum_partials<C>(w, blockIdx.x, blockIdx.y, v[0]);
    product_rows<C, 1>(a, M, m0, n0, blockIdx.y, v);
}

// ── host ───────────────────────────────────────────────────────────────────────

constexpr int kPieceMb = 2048;   // MiB of kept logits: one piece holds 4096 rows of 131072 classes
constexpr int kMaxPieceRows = 1 << 20;          // a tile's offsets over its panels stay within 32 bits (pg::kMaxPanelRows)
constexpr int kBlockRowsLog = 17;               // rows of a block of packed W, where it has too many for one
// Rows up to which a W that would have to be packed is read as it lies. 4096 features, 32000 classes in f32, with gradients, packed and as
// it lies: 16 rows 731 and 438 us, 128 rows 823 and 850; the loss alone 433 and 139 us at 16 rows, 545 and 367 at 121 (2944 x 51416).
constexpr int kFewRows = 128;

struct Layout {
    int Dp, Vp, P;             // padded widths; planes of X and W
    int PP;                    // planes of P, which takes the logits' place
    int rows, pieces;          // rows of a piece
    bool pack_w, grad;
    int wshift, wstored;       // of packed W: PackArgs
    int few;                   // 16-row tiles of the form for few rows, or 0
    int64_t maxes, rowmap, pos, lab, zt, lse, loss, stats, Xp, Wp, E, res, dbpart, dwacc, sums, total;
};

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

pg::Plan plan_of(int64_t M, int64_t N, int64_t k, int pa, int pb, bool narrow) {
    return pg::plan([&](int w) { return (long)ceil_div(M, w) * ceil_div(N, w); }, k, pa, pb, narrow);
}
pg::Plan logits_plan(const Layout &l, int V, int rows) { return plan_of(rows, V, l.Dp, l.P, l.P, true); }
// Statistics of a row: one for each wave tile of the logits' product.
int stat_tiles(const Layout &l, int V, int rows) { return l.few ? ceil_div(V, 128) * 4 : ceil_div(V, logits_plan(l, V, rows).width) * 2; }
// (64-wide tiles of one plane have no layout for operands along k)
pg::Plan dx_plan(const Layout &l, const LinearCe &d, int rows) { return plan_of(rows, d.D, d.V, l.PP, l.P, l.P == 2); }
// Room for partial tiles: four rounds of them where half a round to two rounds of tiles may turn out to be fewer (below that, what
// the plan has fills a round with any number of tiles; above, rounds are short against the whole).
int dx_cap(const pg::Plan &p) {
    const int slots = p.width == 256 ? 256 : 512, planned = p.w.splits > 1 ? p.w.rest * p.w.splits : 0;
    return p.w.tiles() > slots / 2 && p.w.tiles() <= 2 * slots ? std::max(planned, 4 * slots) : planned;
}
// The form for few rows: tiles of 128 classes, 1.75 us a stage at the rate of memory, 3.4 at the f32 matrix rate for 128 rows; tiles of
// 256 features, twice that.
double few_stage(const Layout &l, const LinearCe &d) { return std::max(1.75, d.f16 ? 0.0 : 0.43 * l.few); }
pg::Work few_logits_work(const Layout &l, const LinearCe &d) {
    return few::work(ceil_div(d.V, 128), ceil_div(d.D, few::along_k(d.f16)), few_stage(l, d), l.few * 16l * 128 * 4);
}
pg::Work few_dx_work(const Layout &l, const LinearCe &d) {
    return few::work(ceil_div(d.D, 256), ceil_div(d.V, few::across_v(l.PP)), 2 * few_stage(l, d), l.few * 16l * 256 * 4);
}
int64_t few_part_bytes(const Layout &l, const pg::Work &w, int columns) { return w.splits > 1 ? (int64_t)w.rest * w.splits * l.few * 16 * columns * 4 : 0; }
pg::Plan dw_plan(const Layout &l, const LinearCe &d, int rows) { return plan_of(d.V, d.D, rows, l.PP, l.P, l.P == 2); }

Layout layout(const LinearCe &d) {
    Layout l{};
    l.Dp = (d.D + 63) & ~63;
    l.Vp = (d.V + 63) & ~63;
    l.P = d.f16 ? 1 : 2;
    l.grad = d.dX || d.dW || d.dbias;
    l.PP = d.g16 ? 1 : 2;
    l.pack_w = !d.f16 || d.D % 8 || d.ldw % 8 || ((uintptr_t)d.W & 15) || d.ldw > 1 << 22;
    if (l.pack_w && d.N <= kFewRows && d.D >= 8) {
        l.pack_w = false;
        l.few = d.N <= 16 ? 1 : d.N <= 64 ? 4 : 8;
    }
    const int64_t Np = ((int64_t)d.N + 63) & ~63ll;
    const int64_t piece = (int64_t)(d.piece_mb ? d.piece_mb : kPieceMb) << 20;
    int64_t rows = Np;
    if (l.grad) {
        rows = std::min({rows, (int64_t)kMaxPieceRows, std::max<int64_t>(256, piece / ((int64_t)l.Vp * 4) / 256 * 256)});
    } else {   // without gradients the statistics are what a piece keeps
        rows = std::min<int64_t>(rows, 16384);
        while (rows > 256 && rows * stat_tiles(l, d.V, (int)rows) * 8 > piece) rows = (rows / 2 + 255) / 256 * 256;
    }
    l.pieces = (int)((Np + rows - 1) / rows);
    if (l.pieces > 1) rows = ((Np + l.pieces - 1) / l.pieces + 255) / 256 * 256;
    l.rows = (int)rows;
    l.pieces = (int)((Np + rows - 1) / rows);
    int64_t at = sizeof(Scalars);
    auto take = [&](int64_t bytes) {
        at = (at + 255) & ~255ll;
        const int64_t o = at;
        at += bytes;
        return o;
    };
    l.maxes = take(kMaxBlocks * sizeof(uint2));
    l.rowmap = take(Np * 4);
    l.pos = take(Np * 4);
    l.lab = take(Np * 4);
    l.zt = take(Np * 4);
    l.lse = take(Np * 4);
    l.loss = take(Np * 4);
    const int64_t last = Np - (l.pieces - 1) * rows;   // the last piece has fewer rows, and its own plan
    l.stats = take(std::max(rows * stat_tiles(l, d.V, (int)rows), last * stat_tiles(l, d.V, (int)last)) * 8);
    l.Xp = take(Np * l.Dp * 2 * l.P);
    l.wshift = d.V <= pg::kMaxPanelRows ? 31 : kBlockRowsLog;
    l.wstored = l.wshift == 31 ? d.V : 1 << kBlockRowsLog;
    if (l.pack_w) l.Wp = take((((int64_t)d.V - 1 >> l.wshift) + 1) * l.wstored * l.Dp * 2 * l.P);
    if (l.grad) l.E = take(rows * l.Vp * 4);
    if (l.PP == 1) l.res = take(rows * 4);
    if (d.dbias) l.dbpart = take(rows / kGradRows * d.V * 4);
    if (d.dW && d.g16 && l.pieces > 1) l.dwacc = take((int64_t)d.V * d.D * 4);
    int64_t sums = 0;
    for (const int64_t r : {rows, last}) {
        sums = std::max(sums, l.few ? few_part_bytes(l, few_logits_work(l, d), 128) : (int64_t)logits_plan(l, d.V, (int)r).part_bytes());
        if (d.dX && l.few) sums = std::max(sums, few_part_bytes(l, few_dx_work(l, d), 256));
        else if (d.dX) {
            const pg::Plan p = dx_plan(l, d, (int)r);
            sums = std::max(sums, (int64_t)dx_cap(p) * p.width * p.width * 4);
        }
        if (d.dW) sums = std::max(sums, (int64_t)dw_plan(l, d, (int)r).part_bytes());
    }
    l.sums = take(sums);
    l.total = (at + 255) & ~255ll;
    return l;
}

template <class C, int KEEP>
void launch_logits(LogitArgs a, hipStream_t s) {
    a.tiles_m = ceil_div(a.rows, C::BM);
    hipLaunchKernelGGL((lce_logits_kernel<C, KEEP>), dim3((unsigned)a.w.blocks()), dim3(C::NT), 0, s, a);
    if (a.w.splits > 1) hipLaunchKernelGGL((lce_logits_join_kernel<C, KEEP>), dim3((unsigned)a.w.rest, C::FA), dim3(C::NT), 0, s, a);
}

template <class C>
void logits(const LogitArgs &a, bool keep, hipStream_t s) {
    keep ? launch_logits<C, KEEP_Z>(a, s) : launch_logits<C, KEEP_NONE>(a, s);
}

template <int FA, bool F16, int KEEP>
void launch_few_logits(LogitArgs a, const FewArgs &f, hipStream_t s) {
    a.tiles_m = 1;
    hipLaunchKernelGGL((lce_few_logits_kernel<FA, KEEP, F16>), dim3((unsigned)a.w.blocks()), dim3(256), 0, s, a, f);
    if (a.w.splits > 1) hipLaunchKernelGGL((lce_few_logits_join_kernel<FA, KEEP>), dim3((unsigned)a.w.rest, FA), dim3(256), 0, s, a);
}
template <int FA>
void launch_few_logits(const LogitArgs &a, const FewArgs &f, const LinearCe &d, bool keep, hipStream_t s) {
    if (d.f16) keep ? launch_few_logits<FA, true, KEEP_Z>(a, f, s) : launch_few_logits<FA, true, KEEP_NONE>(a, f, s);
    else keep ? launch_few_logits<FA, false, KEEP_Z>(a, f, s) : launch_few_logits<FA, false, KEEP_NONE>(a, f, s);
}

template <int PP, bool F16, int FA>
void launch_few_dx(const ProductArgs &a, const FewArgs &f, const char *P, hipStream_t s) {
    hipLaunchKernelGGL((lce_few_dx_kernel<FA, PP, F16>), dim3((unsigned)a.w.blocks()), dim3(256), 0, s, a, f, P);
    if (a.w.splits > 1) hipLaunchKernelGGL((lce_few_dx_join_kernel<FA>), dim3((unsigned)a.w.rest, FA), dim3(256), 0, s, a);
}

template <class C>
void launch_product(ProductArgs a, hipStream_t s) {
    a.tiles_m = ceil_div(a.rows_are == 0 ? a.rows : a.M, C::BM);
    a.tiles_n = ceil_div(a.N, C::BN);
    hipLaunchKernelGGL((lce_product_kernel<C>), dim3((unsigned)std::max(a.w.blocks(), a.cap)), dim3(C::NT), 0, s, a);
    const int joins = std::max(a.w.splits > 1 ? a.w.rest : 0, std::min(a.cap / 2, a.tiles_m * a.tiles_n));
    if (joins) hipLaunchKernelGGL((lce_product_join_kernel<C>), dim3((unsigned)joins, C::FA), dim3(C::NT), 0, s, a);
}

template <int TA, int TB, int PA, int PB>
void launch_product(const ProductArgs &a, int width, hipStream_t s) {
    if (width == 256) launch_product<pg::Tile256<TA, TB, PA, PB>>(a, s);
    else if (width == 128) launch_product<pg::Tile128<TA, TB, PA, PB>>(a, s);
    else if constexpr (PB == 2) launch_product<pg::Tile64<TA, TB, PA, PB>>(a, s);
}

template <int PP, int PO>
void gradients(const LinearCe &d, const Layout &l, ProductArgs a, const pg::Operand &W, const pg::Operand &X, int piece, char *ws, hipStream_t s) {
    const Scalars *sc = (const Scalars *)ws;
    const char *P = ws + l.E;
    const int prows = PP == 1 ? 2 * a.rows : a.rows;   // rows that P's panels are apart
    if (d.dX) {
        ProductArgs b = a;
        b.N = d.D;
        b.k = d.V;
        b.rows_are = 0;
        b.rowmap = (const int *)(ws + l.rowmap) + a.row0;
        b.C = d.dX;
        b.ldc = d.lddx;
        if (l.few) {
            const FewArgs f{d.X, d.W, d.ldx, d.ldw, b.rowmap, d.D, l.Vp};
            b.w = few_dx_work(l, d);
            b.w.part = (float *)(ws + l.sums);
            if (l.few == 1) launch_few_dx<PP, PO == 1, 1>(b, f, P, s);
            else if (l.few == 4) launch_few_dx<PP, PO == 1, 4>(b, f, P, s);
            else launch_few_dx<PP, PO == 1, 8>(b, f, P, s);
        } else {
            const pg::Plan plan = dx_plan(l, d, a.rows);
            b.w = plan.w;
            b.w.part = (float *)(ws + l.sums);
            b.cap = dx_cap(plan);
            b.A = pg::panels(P, prows, a.rows, a.rows);
            b.B = W;
            b.B.rows = l.pack_w ? l.Dp : d.D;
            b.B.k = d.V;
            b.bmax = PO == 2 ? &sc->wmax : nullptr;
            launch_product<0, 1, PP, PO>(b, plan.width, s);
        }
    }
    if (d.dW) {
        ProductArgs b = a;
        const pg::Plan plan = dw_plan(l, d, a.rows);
        b.w = plan.w;
        b.w.part = (float *)(ws + l.sums);
        b.A = pg::panels(P, prows, l.Vp, a.rows);
        b.B = X;
        b.B.rows = l.Dp;
        b.B.k = a.rows;
        b.M = d.V;
        b.N = d.D;
        b.rows_are = 1;
        b.bmax = PO == 2 ? &sc->xmax : nullptr;
        b.C = d.dW;
        b.ldc = d.lddw;
        if (l.pieces > 1) {
            float *acc = (float *)(ws + l.dwacc);
            if (!d.g16) {   // an f32 dW adds up in place
                b.acc_in = piece ? (const float *)d.dW : nullptr;
                b.ldacc = d.lddw;
            } else {
                b.ldacc = d.D;
                b.acc_in = piece ? acc : nullptr;
                b.acc_out = piece + 1 < l.pieces ? acc : nullptr;
            }
        }
        launch_product<1, 1, PP, PO>(b, plan.width, s);
    }
}

}  // namespace

int64_t linear_ce_workspace(const LinearCe &d) { return layout(d).total; }

hipError_t linear_ce(const LinearCe &d, void *wsp, hipStream_t s) {
    const Layout l = layout(d);
    char *ws = (char *)wsp;
    Scalars *sc = (Scalars *)ws;
    int *rowmap = (int *)(ws + l.rowmap), *pos = (int *)(ws + l.pos), *lab = (int *)(ws + l.lab);
    float *zt = (float *)(ws + l.zt), *lse = (float *)(ws + l.lse), *loss = (float *)(ws + l.loss);
    float2 *stats = (float2 *)(ws + l.stats);
    half_t *Xp = (half_t *)(ws + l.Xp), *Wp = l.pack_w ? (half_t *)(ws + l.Wp) : nullptr;

    uint2 *maxes = (uint2 *)(ws + l.maxes);
    const int Wrows = l.few ? 0 : d.V, scans = d.f16 ? 0 : (int)std::min<int64_t>(((int64_t)d.N + Wrows) * ceil_div(d.D, 2048) / 4 + 1, kMaxBlocks);
    const ScanArgs scan{d.labels, d.N, d.V, d.D, Wrows, rowmap, pos, lab, sc, (const float *)d.X, (const float *)d.W, d.ldx, d.ldw, maxes};
    hipLaunchKernelGGL(lce_scan_kernel, dim3((unsigned)(1 + scans)), dim3(256), 0, s, scan);
    const dim3 pgrid((unsigned)std::min<int64_t>(((int64_t)d.N + 64 + (l.pack_w ? d.V : 0) + 3) / 4, 4096));
    const int Np = (d.N + 63) & ~63;
    const PackArgs pack{Xp, Wp, Np, l.Dp, l.rows, l.wshift, l.wstored};
    if (d.f16) hipLaunchKernelGGL(lce_pack_kernel<1>, pgrid, dim3(256), 0, s, d, pack, pos, sc, maxes, scans);
    else hipLaunchKernelGGL(lce_pack_kernel<2>, pgrid, dim3(256), 0, s, d, pack, pos, sc, maxes, scans);

    pg::Operand W = l.pack_w ? pg::panels(Wp, l.wstored, d.V, l.Dp) : pg::row_major(d.W, d.ldw, d.V, d.D);
    if (l.pack_w && l.wshift < 31) W.shift = l.wshift, W.block = (long)l.wstored * l.Dp * 2 * l.P;
    for (int piece = 0; piece < l.pieces; piece++) {
        const int row0 = piece * l.rows, rows = std::min(l.rows, Np - row0);
        const pg::Operand X = pg::panels(Xp + (long)row0 * l.Dp * l.P, rows, rows, l.Dp);
        const pg::Plan plan = logits_plan(l, d.V, rows);
        LogitArgs a{};
        a.X = X;
        a.W = W;
        a.V = d.V;
        a.nk = l.few ? ceil_div(d.D, few::along_k(d.f16)) : l.Dp / (l.P == 1 ? 64 : 32);
        a.w = l.few ? few_logits_work(l, d) : plan.w;
        a.w.part = (float *)(ws + l.sums);
        a.sc = sc;
        a.row0 = row0;
        a.rows = rows;
        a.planes = l.P == 2 && !l.few;
        a.bias = d.bias;
        a.bias16 = d.f16;
        a.lab = lab + row0;
        a.zt = zt + row0;
        a.stats = stats;
        a.T = stat_tiles(l, d.V, rows);
        a.E = ws + l.E;
        a.Vp = l.Vp;
        if (l.few) {
            const FewArgs f{d.X, d.W, d.ldx, d.ldw, rowmap, d.D, l.Vp};
            if (l.few == 1) launch_few_logits<1>(a, f, d, l.grad, s);
            else if (l.few == 4) launch_few_logits<4>(a, f, d, l.grad, s);
            else launch_few_logits<8>(a, f, d, l.grad, s);
        } else if (l.P == 1) {
            if (plan.width == 256) logits<pg::Tile256<0, 0, 1, 1>>(a, l.grad, s);
            else if (plan.width == 128) logits<pg::Tile128<0, 0, 1, 1>>(a, l.grad, s);
            else logits<pg::Tile64<0, 0, 1, 1>>(a, l.grad, s);
        } else {
            if (plan.width == 256) logits<pg::Tile256<0, 0, 2, 2>>(a, l.grad, s);
            else if (plan.width == 128) logits<pg::Tile128<0, 0, 2, 2>>(a, l.grad, s);
            else logits<pg::Tile64<0, 0, 2, 2>>(a, l.grad, s);
        }
        hipLaunchKernelGGL(lce_rows_kernel, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, s, sc, row0, rows, stats, a.T, zt + row0, rowmap + row0,
                           lse + row0, loss + row0, d.rowloss, d.lse);
        if (!l.grad) continue;
        const GradArgs g{sc, row0, rows, d.V, l.Vp, lse + row0, zt + row0, lab + row0, ws + l.E, (float *)(ws + l.res), d.dbias ? (float *)(ws + l.dbpart) : nullptr};
        const dim3 ggrid((unsigned)ceil_div(l.Vp, 256), (unsigned)ceil_div(rows, kGradRows));
        if (l.PP == 1) hipLaunchKernelGGL(lce_grad_kernel<1>, ggrid, dim3(256), 0, s, g);
        else hipLaunchKernelGGL(lce_grad_kernel<2>, ggrid, dim3(256), 0, s, g);
        if (d.dbias && piece + 1 < l.pieces)
            hipLaunchKernelGGL(lce_db_kernel, dim3((unsigned)ceil_div(d.V, 256)), dim3(256), 0, s, sc, row0, rows, g.dbpart, d.V, d.dbias);
        ProductArgs p{};
        p.sc = sc;
        p.row0 = row0;
        p.rows = rows;
        p.grad_scale = d.grad_scale;
        p.mean = d.mean;
        p.out16 = d.g16;
        p.res = (const float *)(ws + l.res);
        p.lab = lab + row0;
        p.W = (const half_t *)d.W;
        p.ldw = d.ldw;
        if (l.PP == 1) gradients<1, 1>(d, l, p, W, X, piece, ws, s);
        else if (d.f16) gradients<2, 1>(d, l, p, W, X, piece, ws, s);
        else gradients<2, 2>(d, l, p, W, X, piece, ws, s);
    }
    const int last = (l.pieces - 1) * l.rows;
    hipLaunchKernelGGL(lce_finish_kernel, dim3((unsigned)(1 + (d.dbias ? ceil_div(d.V, 256) : 0))), dim3(256), 0, s, sc, loss, d.mean, d.loss, last,
                       Np - last, (const float *)(ws + l.dbpart), d.V, d.grad_scale, d.dbias);
    return hipGetLastError();
}

}  // namespace ah
