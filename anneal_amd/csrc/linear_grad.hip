// linear_grad.hip — gradients of a linear layer with bias, activation, factor and residual.
//
//   dZ = s dY U act'(Z),  dX = dZ W,  dW = dZ^T X,  db = sum_n dZ,  dU = s dY act(Z)
//
// A first pass finds dZ's largest magnitude, which sets the power of two that its planes are scaled by; a second one stores it as
// one f16 plane (f16 gradients) or two (f32 ones), which both products then read (plane_gemm.h), also writes dU and
// leaves db's sums of up to 64 rows. Where dZ is large the first pass reads neither Z nor evaluates an activation: it bounds dZ by |s dY U| times
// the largest slope. What is large where the activation is off makes that bound as loose as it likes, so the second pass finds
// the true magnitude, and where the bound has cost the planes bits a third launch stores them again (else it returns at once: 4 us, where reading Z
// for the bound as well took 20 of 588 and 28 of 332). f32 X and W are scanned with it and packed as two planes; f16 ones are read as they lie where their
// rows are aligned. Up to 128 rows (64 in f16) dX reads W once, as it lies (linear_ce_few.h). Sums run in a fixed order. Bound by the
// matrix cores: two products of 2 N D F operations; dZ's passes move 10 (f16) to 28 (f32) bytes an element.
//
// f16 gradients of 8192 x 2048 -> 8192 with a factor: 587 us. (The profiler, which adds to each launch: the scan 58, dZ and dU 133, products 489, the third
// launch 5.) dZ in one plane has the 11 bits that a program's own f16 dZ has (off by 2.9e-4 of the norm, 2.1e-4 of it the output's rounding); two planes, as
// for f32 gradients, 1004 us.
#include "linear.h"

#include <string.h>

#include <algorithm>

#include "act.h"
#include "linear_ce_few.h"
#include "tile_out.h"

namespace ah {
namespace {

constexpr int kScans = 1024;   // workgroups that look for an array's largest magnitude, at most
constexpr int kTops = 256, kTopStep = 16;   // places, 64 bytes apart, for dZ's: at one place 2304 waves took 14 us
// Rows of a block of dZ: 64, or fewer where those blocks would not fill the chip (300 x 1024 -> 1024 in 8 rather than 32: 29 -> 23 us).
int block_rows(int Np, int Fp) {
    const int64_t blocks = (int64_t)(Np / 64) * ((Fp + 511) / 512);
    return blocks >= 512 ? 64 : blocks >= 128 ? 32 : 8;
}

struct GradIn {
    int N, D, F, act;
    float scale;
    const void *dY, *Z, *U;
    long lddy, ldz, ldu;
    const void *X, *W;
    long ldx, ldw;
};

// What a row's eight columns of dZ are made of, as it lies.
template <class T>
struct Line {
    typename Raw8<T>::type dy, z, u;
};
template <class T>
__device__ __forceinline__ Line<T> load_line(const GradIn &g, long n, int c) {
    Line<T> l = {};
    l.dy = load_raw8((const T *)g.dY + n * g.lddy, c, g.F);
    if (g.Z) l.z = load_raw8((const T *)g.Z + n * g.ldz, c, g.F);
    if (g.U) l.u = load_raw8((const T *)g.U + n * g.ldu, c, g.F);
    return l;
}
// dZ and dU; P: planes of dZ. One plane takes the activations' FAST forms: its dZ is rounded to f16 (db's terms with them: off by 2^-20, where
// dY itself has f16's 2^-12).
template <class T, int P>
__device__ __forceinline__ f8 dz_of(const GradIn &g, const Line<T> &l, f8 &du) {
    f8 v;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        float slope;
        const float y = act_slope<P == 1>(g.act, (float)l.z[k], slope), t = g.scale * (float)l.dy[k];
        v.v[k] = g.U ? t * slope * (float)l.u[k] : t * slope;
        du.v[k] = t * y;
    }
    return v;
}

// ── largest magnitudes ─────────────────────────────────────────────────────────

struct ScanArgs {
    int zblocks, xblocks, wblocks;   // workgroups of each array, in this order
    unsigned *maxes;                 // [3][kScans]
    unsigned *tops;                  // [kTops * kTopStep]: bits of dZ's largest magnitudes, for the second pass to raise
};
template <class T>
__device__ __forceinline__ unsigned max8(unsigned m, const T &v) {
#pragma unroll
    for (int k = 0; k < 8; k++) m = max(m, pg::magnitude(__float_as_uint((float)v[k])));
    return m;
}
// The larger of m and |v|; infinities and NaN are passed over: v + 0 v is NaN then, which fmaxf drops.
__device__ __forceinline__ float max_finite(float m, float v) { return fmaxf(m, fabsf(fmaf(v, 0.0f, v))); }

// A wave a stretch of 2048 values of a row, or, P > 0, of 512 for dZ's own magnitudes in place of bounds (P: planes of dZ).
template <class T, int P>
__global__ __launch_bounds__(256) void linear_grad_scan_kernel(GradIn g, ScanArgs a) {
    __shared__ unsigned red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = (int)blockIdx.x < a.zblocks ? 0 : (int)blockIdx.x < a.zblocks + a.xblocks ? 1 : 2;
    const int b = blockIdx.x - (which == 0 ? 0 : which == 1 ? a.zblocks : a.zblocks + a.xblocks), blocks = which == 0 ? a.zblocks : which == 1 ? a.xblocks : a.wblocks;
    const int width = which == 0 ? g.F : g.D, stretch = which == 0 && P ? 512 : 2048, segs = (width + stretch - 1) / stretch;
    const long rows = which == 2 ? g.F : g.N;
    if (blockIdx.x == 0 && threadIdx.x < kTops) a.tops[threadIdx.x * kTopStep] = 0;
    unsigned m = 0;
    for (long q = (long)b * 4 + wave; q < rows * segs; q += (long)blocks * 4) {
        const long r = q / segs;
        const int c0 = (int)(q - r * segs) * stretch + lane * 8;
        if (which == 0) {
            if constexpr (P > 0) {
                if (c0 >= width) continue;
                f8 du;
                m = max8(m, dz_of<T, P>(g, load_line<T>(g, r, c0), du).v);
            } else {
                typename Raw8<T>::type dy[4] = {}, u[4] = {};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (c0 + k * 512 >= width) continue;
                    dy[k] = load_raw8((const T *)g.dY + r * g.lddy, c0 + k * 512, width);
                    if (g.U) u[k] = load_raw8((const T *)g.U + r * g.ldu, c0 + k * 512, width);
                }
                const float s = g.scale * slope_bound(g.act);
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float v = s * (float)dy[k][e] * (g.U ? (float)u[k][e] : 1.0f);
                        top = g.act == AH_ACT_NONE ? max_finite(top, v) : fmaxf(top, fabsf(v));   // (without an activation it is dZ)
                    }
                // a bound past f32's range counts as its largest value: dZ may be finite, and the second pass will tell
                m = max(m, __float_as_uint(fminf(top, 0x1.fffffep127f)));
            }
        } else {
            const float *p = which == 1 ? (const float *)g.X + r * g.ldx : (const float *)g.W + r * g.ldw;
            raw8_f32 v[4] = {};
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (c0 + k * 512 < width) v[k] = load_raw8(p, c0 + k * 512, width);
#pragma unroll
            for (int k = 0; k < 4; k++) m = max8(m, v[k]);
        }
    }
    for (int o = 32; o >= 1; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    if (lane == 0) red[wave] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.maxes[which * kScans + b] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// The largest of n values `step` apart; all 256 threads of a workgroup.
__device__ __forceinline__ unsigned join_maxes(const unsigned *maxes, int n, int step = 1) {
    __shared__ unsigned red[4];
    unsigned m = 0;
    for (int i = threadIdx.x; i < n; i += 256) m = max(m, maxes[i * step]);
    for (int o = 32; o >= 1; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    return max(max(red[0], red[1]), max(red[2], red[3]));
}

// ── dZ, dU, db's parts, and the packed operands ────────────────────────────────

struct PackArgs {
    half_t *dZ, *Xp, *Wp;      // null: not packed
    void *dU;
    long lddu;
    float *dbpart;             // [row block][F] or null
    int Np, Fp, Dp;
    int zblocks, zcols, zrows, rest;  // workgroups for dZ (zcols a block of zrows rows), and for X's and W's rows
    int *exps;                 // [4]: exponents of dZ, X and W; dZ's from the bound
    bool track;                // dZ's exponent is from a bound: its largest magnitude is wanted
};
// Binades by which dZ's largest magnitude may lie below 2^14: two planes hold 22 bits down to 2^-3, and they are to do so down to 2^-14 of the
// largest. A bound over many entries is within two binades where their slopes differ, as the slopes of a layer's features do.
constexpr int kSlack = 3;

// dZ's block zb: zrows rows by 512 columns, a thread eight columns of every fourth row. AGAIN: dZ alone. Returns this thread's largest magnitude.
template <class T, int P, bool AGAIN>
__device__ __forceinline__ float pack_dz(const GradIn &g, const PackArgs &a, int zb, int e) {
    __shared__ float red[3][64][8];
    const int rb = zb / a.zcols, n = (zb - rb * a.zcols) * 512 + (threadIdx.x & 63) * 8, w = threadIdx.x >> 6;
    constexpr int B = sizeof(T) == 2 ? 4 : 2;   // rows whose loads are in flight together
    f8 col = {};
    float top = 0.0f;
    if (n < a.Fp) {
        for (int k0 = w; k0 < a.zrows; k0 += 4 * B) {
            Line<T> line[B] = {};
#pragma unroll
            for (int b = 0; b < B; b++) {
                const int m = rb * a.zrows + k0 + 4 * b;
                if (k0 + 4 * b < a.zrows && m < g.N && n < g.F) line[b] = load_line<T>(g, m, n);
            }
#pragma unroll
            for (int b = 0; b < B; b++) {
                if (k0 + 4 * b >= a.zrows) break;
                const int m = rb * a.zrows + k0 + 4 * b;
                f8 v = {}, du;
                if (m < g.N && n < g.F) {
                    v = dz_of<T, P>(g, line[b], du);
                    if (!AGAIN && a.dU) store8((T *)a.dU + (long)m * a.lddu, n, g.F, du);
#pragma unroll
                    for (int c = 0; c < 8; c++) col.v[c] += v.v[c];
                    if (!AGAIN && a.track)
#pragma unroll
                        for (int c = 0; c < 8; c++) top = max_finite(top, v.v[c]);
                }
                if (!a.dZ) continue;
#pragma unroll
                for (int c = 0; c < 8; c++) v.v[c] = n + c < g.F ? ldexpf(v.v[c], e) : 0.0f;
                plane_store8<P>(a.dZ + pg::panel_at<P>(a.Np, m, n), v);
            }
        }
    }
    if (AGAIN || !a.dbpart) return top;
    if (w > 0)
#pragma unroll
        for (int c = 0; c < 8; c++) red[w - 1][threadIdx.x & 63][c] = col.v[c];
    __syncthreads();
    if (w == 0)
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (n + c < g.F) a.dbpart[(long)rb * g.F + n + c] = col.v[c] + red[0][threadIdx.x][c] + red[1][threadIdx.x][c] + red[2][threadIdx.x][c];
    return top;
}

// P: planes of dZ; PO: of X and W.
template <class T, int P, int PO>
__global__ __launch_bounds__(256) void linear_grad_pack_kernel(GradIn g, PackArgs a, ScanArgs s) {
    int e[3] = {};
    if (s.zblocks) e[0] = pg::plane_exp(join_maxes(s.maxes, s.zblocks));
    if (s.xblocks) e[1] = pg::plane_exp(join_maxes(s.maxes + kScans, s.xblocks));
    if (s.wblocks) e[2] = pg::plane_exp(join_maxes(s.maxes + 2 * kScans, s.wblocks));
    if (blockIdx.x == 0 && threadIdx.x < 4) a.exps[threadIdx.x] = threadIdx.x % 3 == 0 ? e[0] : threadIdx.x == 1 ? e[1] : e[2];
    if ((int)blockIdx.x < a.zblocks) {
        // the last rows first, which the scan has left in the caches (16384 x 1024 -> 4096, both passes and the products: 420 -> 414 us)
        unsigned top = __float_as_uint(pack_dz<T, P, false>(g, a, a.zblocks - 1 - (int)blockIdx.x, e[0]));
        if (!a.track) return;
        for (int o = 32; o >= 1; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
        if ((threadIdx.x & 63) == 0) atomicMax(s.tops + (blockIdx.x * 4 + (threadIdx.x >> 6)) % kTops * kTopStep, top);   // in any order the same
        return;
    }
    constexpr int ESZ = PO == 1 ? 2 : 4;
    const long xrows = a.Xp ? g.N : 0, rows = xrows + (a.Wp ? g.F : 0);
    for (long q = (long)(blockIdx.x - a.zblocks) * 4 + (threadIdx.x >> 6); q < rows; q += (long)a.rest * 4) {
        if (q < xrows) pg::pack_row<PO>(a.Xp, g.N, q, (const char *)g.X + q * g.ldx * ESZ, g.D, a.Dp, e[1]);
        else pg::pack_row<PO>(a.Wp, g.F, q - xrows, (const char *)g.W + (q - xrows) * g.ldw * ESZ, g.D, a.Dp, e[2]);
    }
}

// dZ's planes again, by its own magnitude, where the bound's exponent has cost them bits.
template <class T, int P>
__global__ __launch_bounds__(256) void linear_grad_again_kernel(GradIn g, PackArgs a, const unsigned *tops) {
    const unsigned top = join_maxes(tops, kTops, kTopStep);
    const int e = pg::plane_exp(top);
    if (top == 0 || e <= a.exps[3] + kSlack) return;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.exps[0] = e;
    for (int zb = blockIdx.x; zb < a.zblocks; zb += gridDim.x) pack_dz<T, P, true>(g, a, zb, e);
}

// ── the products ───────────────────────────────────────────────────────────────
// dX and dW go in one launch (and what was split of them is joined in one), dX's workgroups first: what one leaves idle in its last round the
// other fills (1999 x 776 x 3104 in f32: 49 and 50 us one after the other, 73 together). db's workgroups follow.

struct ProductArgs {
    pg::Operand A, B;
    int M, N, nk, tiles_m, tiles_n;   // C is [M, N]
    pg::Work w;
    const int *ea, *eb;    // the operands' exponents; eb null: none
    void *C;
    long ldc;
    int out16;
};
struct PairArgs {
    ProductArgs x, w;      // dX, dW
    int xblocks, wblocks;  // workgroups; dX's a multiple of 8, some of which may have nothing to do
    const float *dbpart;
    int dbrows, F;
    float *db;
};

// db: the row blocks' sums in order, 64 columns a workgroup and NT / 64 runs of blocks.
template <int NT>
__device__ __forceinline__ void sum_db(const PairArgs &a, int block, char *smem) {
    float(*red)[64] = (float(*)[64])smem;
    const int c = block * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6, each = (a.dbrows + NT / 64 - 1) / (NT / 64);
    float s = 0.0f;
    if (c < a.F)
#pragma unroll 8
        for (int b = k * each; b < min(a.dbrows, (k + 1) * each); b++) s += a.dbpart[(long)b * a.F + c];
    red[k][threadIdx.x & 63] = s;
    __syncthreads();
    if (k || c >= a.F) return;
    for (int r = 1; r < NT / 64; r++) s += red[r][threadIdx.x];
    a.db[c] = s;
}

template <class C>
__device__ __forceinline__ void tile_at(const ProductArgs &a, int tile, int &m0, int &n0) {
    int tr, tc;
    pg::grouped_tile(tile, a.tiles_m, a.tiles_n, tr, tc);
    m0 = tr * C::BM;
    n0 = tc * C::BN;
}

template <class C>
__device__ __forceinline__ void product_rows(const ProductArgs &a, int m0, int n0, int i, const floatx4 (&acc)[C::FB], char *smem) {
    TileOut<C> out(smem, m0, n0, i);
    asm volatile("" : "+v"(out.m), "+v"(out.n));
    const int e = -(*a.ea + (a.eb ? *a.eb : 0));
    out.put(acc);
    if (out.n >= a.N) return;
#pragma unroll
    for (int p = 0; p < TileOut<C>::kParts; p++) {
        const long m = out.m + p * TileOut<C>::kStep;
        if (m >= a.M) continue;
        f8 v = out.get(p);
#pragma unroll
        for (int k = 0; k < 8; k++) v.v[k] = ldexpf(v.v[k], e);
        if (a.out16) store8((half_t *)a.C + m * a.ldc, out.n, a.N, v);
        else store8((float *)a.C + m * a.ldc, out.n, a.N, v);
    }
}

template <class C>
__device__ __forceinline__ void product(const ProductArgs &a, int block, char *smem) {
    static_assert(tile_out_bytes<C>() <= C::SMEM, "the tile leaves through the stages' buffers");
    int tile, slot, first, count, m0, n0;
    pg::pick(a.w, block, a.nk, tile, slot, first, count);
    tile_at<C>(a, tile, m0, n0);
    floatx4 acc[C::FA][C::FB];
    pg::contract<C>(a.A, a.B, m0, n0, first, count, smem, acc);
    if (slot >= 0) {
        pg::store_partials<C>(a.w.part, slot, acc);
        return;
    }
    g16::lds_barrier();   // the last stage has been read
#pragma unroll
    for (int i = 0; i < C::FA; i++) {
        __builtin_amdgcn_sched_barrier(0);
        product_rows<C>(a, m0, n0, i, acc[i], smem);
    }
}
template <class C>
__device__ __forceinline__ void join(const ProductArgs &a, int tile, int row, char *smem) {
    int m0, n0;
    tile_at<C>(a, a.w.whole + tile, m0, n0);
    floatx4 v[C::FB];
    pg::sum_partials<C>(a.w, tile, row, v);
    product_rows<C>(a, m0, n0, row, v, smem);
}

template <class X, class W>
__global__ __launch_bounds__(X::NT, 2) void linear_grad_kernel(PairArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[std::max(X::SMEM, W::SMEM)];
    static_assert(X::NT == W::NT, "one launch");
    const int b = blockIdx.x;
    if (b < a.xblocks) {
        if (b < a.x.w.blocks()) product<X>(a.x, b, smem);
    } else if (b < a.xblocks + a.wblocks) {
        product<W>(a.w, b - a.xblocks, smem);
    } else {
        sum_db<X::NT>(a, b - a.xblocks - a.wblocks, smem);
    }
}
// A workgroup for each 16 rows of a tile's waves; xblocks, wblocks count those.
template <class X, class W>
__global__ __launch_bounds__(X::NT) void linear_grad_join_kernel(PairArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[std::max(tile_out_bytes<X>(), tile_out_bytes<W>())];
    const int b = blockIdx.x;
    if (b < a.xblocks) join<X>(a.x, b / X::FA, b % X::FA, smem);
    else join<W>(a.w, (b - a.xblocks) / W::FA, (b - a.xblocks) % W::FA, smem);
}

// dX from W as it lies, for few rows: one row of tiles.
struct FewArgs {
    const char *P;      // dZ's panels, of prows rows
    long prows;
    int Fp, F;
    const void *W;
    long ldw;
};
template <int FA, int PP, bool F16, class W>
__global__ __launch_bounds__(256, 2) void linear_grad_few_kernel(PairArgs a, FewArgs f) {
    __shared__ __attribute__((aligned(1024))) char smem[std::max({few::smem_bytes<few::Tile<FA, 4>>(), tile_out_bytes<few::Tile<FA, 4>>(), W::SMEM})];
    static_assert(W::NT == 256, "one launch");
    const int b = blockIdx.x;
    if (b >= a.xblocks + a.wblocks) {
        sum_db<256>(a, b - a.xblocks - a.wblocks, smem);
    } else if (b >= a.xblocks) {
        product<W>(a.w, b - a.xblocks, smem);
    } else if (b < a.x.w.blocks()) {
        few::with_rows<FA>(a.x.M, [&](auto fa) {
            typedef few::Tile<fa, 4> C;
            int tile, slot, first, count;
            pg::pick(a.x.w, b, a.x.nk, tile, slot, first, count);
            floatx4 acc[C::FA][C::FB];
            few::contract_across<C, PP, F16>(f.P, f.prows, f.Fp, f.W, f.ldw, f.F, a.x.N, tile * C::BN, first, count, smem, acc);
            if (slot >= 0) {
                pg::store_partials<C>(a.x.w.part, slot, acc);
                return;
            }
            few::sync();
#pragma unroll
            for (int i = 0; i < C::FA; i++) product_rows<C>(a.x, 0, tile * C::BN, i, acc[i], smem);
        });
    }
}
template <int FA>
__global__ __launch_bounds__(256) void linear_grad_few_join_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[tile_out_bytes<few::Tile<FA, 4>>()];
    few::with_rows<FA>(a.M, [&](auto fa) {
        typedef few::Tile<fa, 4> C;
        if ((int)blockIdx.y >= C::FA) return;
        floatx4 v[C::FB];
        pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, v);
        product_rows<C>(a, 0, (a.w.whole + blockIdx.x) * C::BN, blockIdx.y, v, smem);
    });
}

// ── host ───────────────────────────────────────────────────────────────────────

constexpr int kFewF32 = 128, kFewF16 = 64;   // rows up to which dX reads W as it lies

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

bool rows_aligned(const void *p, int64_t ld, int D) { return D % 8 == 0 && ld % 8 == 0 && ((uintptr_t)p & 15) == 0 && ld <= 1 << 22; }

// How the two products are cut: widths of the tiles and splits of K, by a model of the time they take together. Stage times are those of
// pg::plan; tiles of 256 go with each other, and narrower ones, which have half the threads. (64-wide tiles of one plane have no
// layout along k.)
struct Cut {
    int width;
    pg::Work w;
    long part_bytes() const { return w.splits > 1 ? (long)w.rest * w.splits * width * width * 4 : 0; }
};
struct Cuts {
    Cut x, w;
};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};

// n jobs of p us and then m of q on `slots` machines: when the last is done.
double makespan(long n, double p, long m, double q, long slots) {
    const long a = n / slots, r = n % slots;   // r machines have a + 1 of the first, the others a
    if (m == 0) return (a + (r > 0)) * p;
    double t = (n * p + m * q) / slots;
    for (int i = 0; i < 64; i++) {
        const auto fit = [&](double from) { return t <= from ? 0l : (long)((t - from) / q + 1e-6); };
        const long can = r * fit((a + 1) * p) + (slots - r) * fit(a * p);
        if (can >= m) break;
        t += std::max(q * (m - can) / slots, q / 64);
    }
    return std::max(t, (a + (r > 0)) * p);
}

Cuts cuts_of(int N, int D, int F, int P, int PO, bool with_x) {
    struct Key {
        int v[6];
    };
    const Key key{{N, D, F, P, PO, with_x}};
    static thread_local Key last_key{};
    static thread_local Cuts last{};
    if (!memcmp(&key, &last_key, sizeof key)) return last;   // of the call's own workspace query, or the step before
    const int row = P == 1 ? 0 : PO == 1 ? 1 : 2;
    // us a stage of 256, 128 and 64, with one workgroup on each CU (of 256: one alone on the chip) and with as many as there is room for
    constexpr double kFirst[3][3] = {{1.22, 0.72, 0}, {1.18, 0.61, 0}, {1.53, 0.68, 0.26}}, kFull[3][3] = {{1.77, 1.15, 0}, {1.73, 0.97, 0}, {2.30, 1.33, 0.41}};
    const int bk = row == 0 ? 64 : 32;
    const long nx = ceil_div(F, bk), nw = ceil_div(N, bk);
    double best = 1e30;
    Cuts c{};
    for (int kind = 0; kind < 2; kind++) {
        const long slots = kind == 0 ? 256 : 512;
        for (int ix = kind; ix <= (kind && PO == 2 ? 2 : kind); ix++)
            for (int iw = kind; iw <= (kind && PO == 2 ? 2 : kind); iw++) {
                const int wx = 256 >> ix, ww = 256 >> iw;
                const long tx = with_x ? (long)ceil_div(N, wx) * ceil_div(D, wx) : 0, tw = (long)ceil_div(F, ww) * ceil_div(D, ww);
                for (const int sx : kSplits) {
                    if (sx > 1 && (!with_x || nx < 2 * sx || tx * sx > 4 * slots)) break;
                    for (const int sw : kSplits) {
                        if (sw > 1 && (nw < 2 * sw || tw * sw > 4 * slots)) break;
                        const double busy = (double)std::min(slots, tx * sx + tw * sw) / 256, fixed = kind == 0 ? 7.0 : 5.0;
                        const double load = kind == 0 ? busy : std::max(0.0, busy - 1.0);
                        const auto stage = [&](int i) { return kFirst[row][i] + (kFull[row][i] - kFirst[row][i]) * load; };
                        const double px = (nx + sx - 1) / sx * stage(ix) + fixed, pw = (nw + sw - 1) / sw * stage(iw) + fixed;
                        double us = makespan(tx * sx, px, tw * sw, pw, slots);
                        if (sx > 1 || sw > 1) us += 4.0 + ((sx > 1 ? (double)tx * sx * wx * wx : 0.0) + (sw > 1 ? (double)tw * sw * ww * ww : 0.0)) * 8 / 4e6;
                        if (us < best) {
                            best = us;
                            c.x = {wx, sx > 1 ? pg::Work{0, (int)tx, sx, nullptr} : pg::Work{(int)tx, 0, 1, nullptr}};
                            c.w = {ww, sw > 1 ? pg::Work{0, (int)tw, sw, nullptr} : pg::Work{(int)tw, 0, 1, nullptr}};
                        }
                    }
                }
            }
    }
    last_key = key;
    last = c;
    return c;
}
struct Layout {
    int P, PO;                 // planes of dZ; of X and W
    int Np, Fp, Dp, few, zrows;
    bool products, pack_x, pack_w;
    bool exact, track;         // dZ's magnitudes are scanned for, or bounded and found by the second pass
    Cuts cuts;
    int64_t exps, tops, maxes, dbpart, dZ, Xp, Wp, sums, wsums, total;
};

pg::Work few_work(const ah_linear_grad_desc &d, const Layout &l) {
    return few::work(ceil_div(d.D, 256), ceil_div(d.F, few::across_v(l.P)), 2 * std::max(1.75, d.dtype == AH_F16 ? 0.0 : 0.43 * l.few), l.few * 16l * 256 * 4);
}

Layout layout(const ah_linear_grad_desc &d) {
    Layout l{};
    const bool f16 = d.dtype == AH_F16;
    l.P = d.grad_dtype == AH_F16 ? 1 : 2;
    l.PO = f16 ? 1 : 2;
    l.Np = (d.N + 63) & ~63;
    l.Fp = (d.F + 63) & ~63;
    l.Dp = (d.D + 63) & ~63;
    l.products = d.dX || d.dW;
    l.zrows = block_rows(l.Np, l.Fp);
    // dZ itself is looked through where a wave has one stretch of it, or two whose slopes cost little (the third launch | that: f32, tanh GELU's and GELU's
    // slopes in full, 1900 x 512 -> 2048 47.5 | 48.8 and 63.4 | 66.7 us; f16 SiLU 1100 rows 37.9 | 36.2). Without an activation the bound is exact.
    const bool cheap = l.P == 1 || d.act == AH_ACT_RELU;
    l.exact = d.act != AH_ACT_NONE && (int64_t)d.N * ((d.F + 511) / 512) <= (cheap ? 8 : 4) * kScans;
    l.track = l.products && d.act != AH_ACT_NONE && !l.exact;
    if (d.dX && d.N <= (f16 ? kFewF16 : kFewF32) && d.D >= 8) l.few = d.N <= 16 ? 1 : d.N <= 64 ? 4 : 8;
    l.pack_x = d.dW && (!f16 || !rows_aligned(d.X, d.ldx, d.D));
    l.pack_w = d.dX && !l.few && (!f16 || !rows_aligned(d.W, d.ldw, d.D));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at = (at + bytes + 255) & ~255ll;
        return o;
    };
    l.exps = take(16);
    l.tops = take(kTops * kTopStep * 4);
    l.maxes = take(3 * kScans * 4);
    if (d.dbias) l.dbpart = take((int64_t)(l.Np / l.zrows) * d.F * 4);
    if (l.products) l.dZ = take((int64_t)l.Np * l.Fp * 2 * l.P);
    if (l.pack_x) l.Xp = take((int64_t)d.N * l.Dp * 2 * l.PO);
    if (l.pack_w) l.Wp = take((int64_t)d.F * l.Dp * 2 * l.PO);
    const bool few = d.N <= (f16 ? kFewF16 : kFewF32) && d.D >= 8;
    if (l.products) l.cuts = cuts_of(d.N, d.D, d.F, l.P, l.PO, !few);   // of both products, whichever are asked for: the same bits
    if (l.few) {
        const pg::Work w = few_work(d, l);
        l.sums = take(w.splits > 1 ? (int64_t)w.rest * w.splits * l.few * 16 * 256 * 4 : 0);
    } else if (d.dX) {
        l.sums = take(l.cuts.x.part_bytes());
    }
    if (d.dW) l.wsums = take(l.cuts.w.part_bytes());
    l.total = at;
    return l;
}

template <class X, class W>
void launch(PairArgs a, bool x, bool w, hipStream_t s) {
    a.x.tiles_m = ceil_div(a.x.M, X::BM);
    a.x.tiles_n = ceil_div(a.x.N, X::BN);
    a.w.tiles_m = ceil_div(a.w.M, W::BM);
    a.w.tiles_n = ceil_div(a.w.N, W::BN);
    a.xblocks = x ? (a.x.w.blocks() + 7) & ~7 : 0;
    a.wblocks = w ? a.w.w.blocks() : 0;
    hipLaunchKernelGGL((linear_grad_kernel<X, W>), dim3((unsigned)(a.xblocks + a.wblocks + (a.db ? ceil_div(a.F, 64) : 0))), dim3(X::NT), 0, s, a);
    a.xblocks = x && a.x.w.splits > 1 ? a.x.w.rest * X::FA : 0;
    a.wblocks = w && a.w.w.splits > 1 ? a.w.w.rest * W::FA : 0;
    if (a.xblocks + a.wblocks) hipLaunchKernelGGL((linear_grad_join_kernel<X, W>), dim3((unsigned)(a.xblocks + a.wblocks)), dim3(X::NT), 0, s, a);
}
template <int PA, int PB>
void launch(const PairArgs &a, const Cuts &c, bool x, bool w, hipStream_t s) {
    typedef pg::Tile128<0, 1, PA, PB> X128;
    typedef pg::Tile128<1, 1, PA, PB> W128;
    if (c.w.width == 256) {
        launch<pg::Tile256<0, 1, PA, PB>, pg::Tile256<1, 1, PA, PB>>(a, x, w, s);
        return;
    }
    if constexpr (PB == 2) {
        typedef pg::Tile64<0, 1, PA, PB> X64;
        typedef pg::Tile64<1, 1, PA, PB> W64;
        if (c.x.width == 64 && c.w.width == 64) return launch<X64, W64>(a, x, w, s);
        if (c.x.width == 64) return launch<X64, W128>(a, x, w, s);
        if (c.w.width == 64) return launch<X128, W64>(a, x, w, s);
    }
    launch<X128, W128>(a, x, w, s);
}

template <int P, bool F16, int FA, class W>
void launch_few(PairArgs a, const FewArgs &f, bool w, hipStream_t s) {
    a.w.tiles_m = ceil_div(a.w.M, W::BM);
    a.w.tiles_n = ceil_div(a.w.N, W::BN);
    a.xblocks = (a.x.w.blocks() + 7) & ~7;
    a.wblocks = w ? a.w.w.blocks() : 0;
    hipLaunchKernelGGL((linear_grad_few_kernel<FA, P, F16, W>), dim3((unsigned)(a.xblocks + a.wblocks + (a.db ? ceil_div(a.F, 64) : 0))), dim3(256), 0, s, a, f);
    if (a.x.w.splits > 1) hipLaunchKernelGGL((linear_grad_few_join_kernel<FA>), dim3((unsigned)a.x.w.rest, FA), dim3(256), 0, s, a.x);
    if (w && a.w.w.splits > 1) {
        a.xblocks = 0;
        a.wblocks = a.w.w.rest * W::FA;
        hipLaunchKernelGGL((linear_grad_join_kernel<W, W>), dim3((unsigned)a.wblocks), dim3(256), 0, s, a);
    }
}
// dX of few rows, and in its launch dW and db where their tiles have as many threads (7 x 1024 -> 4096 f16: 27.6 -> 22 us for all four).
template <int P, int PO, int FA>
void launch_few(const PairArgs &a, const FewArgs &f, int width, bool w, hipStream_t s) {
    constexpr bool F16 = PO == 1;
    if constexpr (PO == 2) {
        if (width == 64) return launch_few<P, F16, FA, pg::Tile64<1, 1, P, PO>>(a, f, w, s);
    }
    launch_few<P, F16, FA, pg::Tile128<1, 1, P, PO>>(a, f, w, s);
}

template <class T, int P, int PO>
void run(const ah_linear_grad_desc &d, const Layout &l, hipStream_t s) {
    char *ws = (char *)d.ws;
    const GradIn g{d.N, d.D, d.F, d.act, d.scale, d.dY, d.Z, d.U, d.lddy, d.ldz, d.ldu, d.X, d.W, d.ldx, d.ldw};
    const auto scans = [](int64_t rows, int64_t width, int stretch = 2048) { return (int)std::min<int64_t>((rows * ((width + stretch - 1) / stretch) + 3) / 4, kScans); };
    ScanArgs sc{};
    sc.zblocks = l.products ? scans(d.N, d.F, l.exact ? 512 : 2048) : 0;
    sc.xblocks = l.pack_x && PO == 2 ? scans(d.N, d.D) : 0;
    sc.wblocks = l.pack_w && PO == 2 ? scans(d.F, d.D) : 0;
    sc.maxes = (unsigned *)(ws + l.maxes);
    sc.tops = (unsigned *)(ws + l.tops);
    if (l.products) {
        const dim3 grid((unsigned)(sc.zblocks + sc.xblocks + sc.wblocks));
        if (l.exact) hipLaunchKernelGGL((linear_grad_scan_kernel<T, P>), grid, dim3(256), 0, s, g, sc);
        else hipLaunchKernelGGL((linear_grad_scan_kernel<T, 0>), grid, dim3(256), 0, s, g, sc);
    }

    PackArgs p{};
    if (l.products) p.dZ = (half_t *)(ws + l.dZ);
    if (l.pack_x) p.Xp = (half_t *)(ws + l.Xp);
    if (l.pack_w) p.Wp = (half_t *)(ws + l.Wp);
    p.dU = d.dU;
    p.lddu = d.lddu;
    if (d.dbias) p.dbpart = (float *)(ws + l.dbpart);
    p.Np = l.Np;
    p.Fp = l.Fp;
    p.Dp = l.Dp;
    p.zcols = ceil_div(l.Fp, 512);
    p.zrows = l.zrows;
    p.zblocks = l.Np / l.zrows * p.zcols;
    p.rest = (int)std::min<int64_t>(((l.pack_x ? d.N : 0) + (int64_t)(l.pack_w ? d.F : 0) + 3) / 4, 4096);
    p.exps = (int *)(ws + l.exps);
    p.track = l.track;
    hipLaunchKernelGGL((linear_grad_pack_kernel<T, P, PO>), dim3((unsigned)(p.zblocks + p.rest)), dim3(256), 0, s, g, p, sc);
    if (l.track) hipLaunchKernelGGL((linear_grad_again_kernel<T, P>), dim3((unsigned)std::min(p.zblocks, 1024)), dim3(256), 0, s, g, p, sc.tops);
    PairArgs a{};
    a.x.ea = a.w.ea = p.exps;
    a.x.out16 = a.w.out16 = d.grad_dtype == AH_F16;
    a.x.N = a.w.N = d.D;
    a.x.M = d.N;
    a.x.C = d.dX;
    a.x.ldc = d.lddx;
    a.w.M = d.F;
    a.w.C = d.dW;
    a.w.ldc = d.lddw;
    a.db = d.dbias;
    a.dbpart = p.dbpart;
    a.dbrows = l.Np / l.zrows;
    a.F = d.F;
    const bool x = d.dX && !l.few;
    if (!d.dX && !d.dW && !d.dbias) return;
    constexpr int BK = P == 1 ? 64 : 32;   // every stage begins at a row of W or X that there is
    if (x) {
        a.x.w = l.cuts.x.w;
        a.x.w.part = (float *)(ws + l.sums);
        a.x.A = pg::panels(p.dZ, l.Np, l.Np, l.Fp);
        a.x.B = l.pack_w ? pg::panels(p.Wp, d.F, l.Dp, d.F) : pg::row_major(d.W, d.ldw, d.D, d.F);
        a.x.nk = ceil_div(d.F, BK);
        a.x.eb = PO == 2 ? p.exps + 2 : nullptr;
    }
    if (d.dW) {
        a.w.w = l.cuts.w.w;
        a.w.w.part = (float *)(ws + l.wsums);
        a.w.A = pg::panels(p.dZ, l.Np, l.Fp, l.Np);
        a.w.B = l.pack_x ? pg::panels(p.Xp, d.N, l.Dp, d.N) : pg::row_major(d.X, d.ldx, d.D, d.N);
        a.w.nk = ceil_div(d.N, BK);
        a.w.eb = PO == 2 ? p.exps + 1 : nullptr;
    }
    if (l.few) {
        const FewArgs f{ws + l.dZ, l.Np, l.Fp, d.F, d.W, d.ldw};
        const bool with_w = d.dW && l.cuts.w.width < 256;
        PairArgs b = a;
        b.x.nk = ceil_div(d.F, few::across_v(P));
        b.x.w = few_work(d, l);
        b.x.w.part = (float *)(ws + l.sums);
        if (!with_w && d.dW) b.db = nullptr;   // db goes with dW
        if (l.few == 1) launch_few<P, PO, 1>(b, f, l.cuts.w.width, with_w, s);
        else if (l.few == 4) launch_few<P, PO, 4>(b, f, l.cuts.w.width, with_w, s);
        else if constexpr (PO == 2) launch_few<P, PO, 8>(b, f, l.cuts.w.width, with_w, s);
        if (with_w || !d.dW) return;
    }
    launch<P, PO>(a, l.cuts, x, d.dW != nullptr, s);
}

}  // namespace

int64_t linear_grad_workspace(const ah_linear_grad_desc &d) { return layout(d).total; }

hipError_t linear_grad(const ah_linear_grad_desc &d, hipStream_t s) {
    const Layout l = layout(d);
    if (d.dtype == AH_F32) run<float, 2, 2>(d, l, s);
    else if (d.grad_dtype == AH_F32) run<half_t, 2, 1>(d, l, s);
    else run<half_t, 1, 1>(d, l, s);
    return hipGetLastError();
}

}  // namespace ah
