// linear_grad.hip — gradients of a linear layer with bias, activation, factor and residual.
//
//   dZ = s dY U act'(Z),  dX = dZ W,  dW = dZ^T X,  db = sum_n dZ,  dU = s dY act(Z)
//
// dZ is formed twice: once for its largest magnitude, which sets the power of two that its planes are scaled by, and once to be stored as
// one f16 plane (f16 gradients) or two (f32 ones), which both products then read (plane_gemm.h); the second pass also writes dU and
// leaves db's sums of 64 rows. f32 X and W are scanned with it and packed as two planes; f16 ones are read as they lie where their
// rows are aligned. Up to 128 rows (64 in f16) dX reads W once, as it lies (linear_ce_few.h). Sums run in a fixed order. Bound by the
// matrix cores: two products of 2 N D F operations; dZ's passes move 10 (f16) to 28 (f32) bytes an element.
#include "linear.h"

#include <algorithm>

#include "act.h"
#include "linear_ce_few.h"
#include "tile_out.h"

namespace ah {
namespace {

constexpr int kScans = 1024;   // workgroups that look for an array's largest magnitude, at most
constexpr int kRows = 64;      // rows of a block of dZ; also the k of a one-plane stage, up to which rows are cleared

struct GradIn {
    int N, D, F, act;
    float scale;
    const void *dY, *Z, *U;
    long lddy, ldz, ldu;
    const void *X, *W;
    long ldx, ldw;
};

// dZ and dU at row n, columns c .. c+3.
template <class T>
__device__ __forceinline__ floatx4 dz_at(const GradIn &g, long n, int c, floatx4 &du) {
    const floatx4 dy = pg::load4((const T *)g.dY + n * g.lddy, c, g.F);
    floatx4 z = {}, u = {1.0f, 1.0f, 1.0f, 1.0f}, v;
    if (g.Z) z = pg::load4((const T *)g.Z + n * g.ldz, c, g.F);
    if (g.U) u = pg::load4((const T *)g.U + n * g.ldu, c, g.F);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        float slope;
        const float y = act_slope<sizeof(T) == 2>(g.act, z[k], slope), t = g.scale * dy[k];
        v[k] = t * slope * u[k];
        du[k] = t * y;
    }
    return v;
}

// ── largest magnitudes ─────────────────────────────────────────────────────────

struct ScanArgs {
    int zblocks, xblocks, wblocks;   // workgroups of each array, in this order
    unsigned *maxes;                 // [3][kScans]
};
__device__ __forceinline__ unsigned max4(unsigned m, floatx4 v) {
#pragma unroll
    for (int k = 0; k < 4; k++) m = max(m, pg::magnitude(__float_as_uint(v[k])));
    return m;
}
// A wave a stretch of 1024 values of a row.
template <class T>
__global__ __launch_bounds__(256) void linear_grad_scan_kernel(GradIn g, ScanArgs a) {
    __shared__ unsigned red[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = (int)blockIdx.x < a.zblocks ? 0 : (int)blockIdx.x < a.zblocks + a.xblocks ? 1 : 2;
    const int b = blockIdx.x - (which == 0 ? 0 : which == 1 ? a.zblocks : a.zblocks + a.xblocks), blocks = which == 0 ? a.zblocks : which == 1 ? a.xblocks : a.wblocks;
    const int width = which == 0 ? g.F : g.D, segs = (width + 1023) / 1024;
    const long rows = which == 2 ? g.F : g.N;
    unsigned m = 0;
    for (long q = (long)b * 4 + wave; q < rows * segs; q += (long)blocks * 4) {
        const long r = q / segs;
        const int c0 = (int)(q - r * segs) * 1024 + lane * 4;
#pragma unroll
        for (int k = 0; k < 1024; k += 256) {
            if (c0 + k >= width) continue;
            floatx4 unused;
            if (which == 0) m = max4(m, dz_at<T>(g, r, c0 + k, unused));
            else m = max4(m, pg::load4(which == 1 ? (const float *)g.X + r * g.ldx : (const float *)g.W + r * g.ldw, c0 + k, width));
        }
    }
    for (int o = 32; o >= 1; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    if (lane == 0) red[wave] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.maxes[which * kScans + b] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// The largest of n workgroups' values; all 256 threads of a workgroup.
__device__ __forceinline__ unsigned join_maxes(const unsigned *maxes, int n) {
    __shared__ unsigned red[4];
    unsigned m = 0;
    for (int i = threadIdx.x; i < n; i += 256) m = max(m, maxes[i]);
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
    int zblocks, zcols, rest;  // workgroups for dZ (zcols a row block), and for X's and W's rows
    int *exps;                 // [3]: exponents of dZ, X and W
};
// P: planes of dZ; PO: of X and W.
template <class T, int P, int PO>
__global__ __launch_bounds__(256) void linear_grad_pack_kernel(GradIn g, PackArgs a, ScanArgs s) {
    __shared__ float red[3][64][4];
    int e[3] = {};
    if (s.zblocks) e[0] = pg::plane_exp(join_maxes(s.maxes, s.zblocks));
    if (s.xblocks) e[1] = pg::plane_exp(join_maxes(s.maxes + kScans, s.xblocks));
    if (s.wblocks) e[2] = pg::plane_exp(join_maxes(s.maxes + 2 * kScans, s.wblocks));
    if (blockIdx.x == 0 && threadIdx.x < 3) a.exps[threadIdx.x] = threadIdx.x == 0 ? e[0] : threadIdx.x == 1 ? e[1] : e[2];
    if ((int)blockIdx.x < a.zblocks) {   // 64 rows by 256 columns: a thread has four columns of every fourth row
        const int rb = blockIdx.x / a.zcols, n = ((int)blockIdx.x - rb * a.zcols) * 256 + (threadIdx.x & 63) * 4, w = threadIdx.x >> 6;
        floatx4 col = {};
        if (n < a.Fp) {
#pragma unroll 4
            for (int k = w; k < kRows; k += 4) {
                const int m = rb * kRows + k;
                floatx4 v = {}, du;
                if (m < g.N && n < g.F) {
                    v = dz_at<T>(g, m, n, du);
                    if (a.dU) pg::store4((T *)a.dU + (long)m * a.lddu, n, g.F, du);
                    col += v;
                }
                if (!a.dZ) continue;
#pragma unroll
                for (int c = 0; c < 4; c++) v[c] = n + c < g.F ? ldexpf(v[c], e[0]) : 0.0f;
                if constexpr (P == 1) {
                    pg::h4 h;
#pragma unroll
                    for (int c = 0; c < 4; c++) h[c] = (half_t)v[c];
                    *(pg::h4 *)(a.dZ + pg::panel_at<1>(a.Np, m, n)) = h;
                } else {
                    pg::plane_store(a.dZ + pg::panel_at<2>(a.Np, m, n), v);
                }
            }
        }
        if (!a.dbpart) return;
        if (w > 0)
#pragma unroll
            for (int c = 0; c < 4; c++) red[w - 1][threadIdx.x & 63][c] = col[c];
        __syncthreads();
        if (w == 0)
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (n + c < g.F) a.dbpart[(long)rb * g.F + n + c] = col[c] + red[0][threadIdx.x][c] + red[1][threadIdx.x][c] + red[2][threadIdx.x][c];
        return;
    }
    constexpr int ESZ = PO == 1 ? 2 : 4;
    const long xrows = a.Xp ? g.N : 0, rows = xrows + (a.Wp ? g.F : 0);
    for (long q = (long)(blockIdx.x - a.zblocks) * 4 + (threadIdx.x >> 6); q < rows; q += (long)a.rest * 4) {
        if (q < xrows) pg::pack_row<PO>(a.Xp, g.N, q, (const char *)g.X + q * g.ldx * ESZ, g.D, a.Dp, e[1]);
        else pg::pack_row<PO>(a.Wp, g.F, q - xrows, (const char *)g.W + (q - xrows) * g.ldw * ESZ, g.D, a.Dp, e[2]);
    }
}

// db: the row blocks' sums in order, 64 columns a workgroup and 16 runs of blocks.
__global__ __launch_bounds__(1024) void linear_grad_db_kernel(const float *part, int blocks, int F, float *db) {
    __shared__ float red[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6, each = (blocks + 15) / 16;
    float s = 0.0f;
    if (c < F)
#pragma unroll 8
        for (int b = k * each; b < min(blocks, (k + 1) * each); b++) s += part[(long)b * F + c];
    red[k][threadIdx.x & 63] = s;
    __syncthreads();
    if (k || c >= F) return;
    for (int r = 1; r < 16; r++) s += red[r][threadIdx.x];
    db[c] = s;
}

// ── the products ───────────────────────────────────────────────────────────────

struct ProductArgs {
    pg::Operand A, B;
    int M, N, nk, tiles_m, tiles_n;   // C is [M, N]
    pg::Work w;
    const int *ea, *eb;    // the operands' exponents; eb null: none
    void *C;
    long ldc;
    int out16;
};

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
        if (a.out16) store_f8((half_t *)a.C + m * a.ldc, out.n, a.N, v);
        else store_f8((float *)a.C + m * a.ldc, out.n, a.N, v);
    }
}

template <class C>
__global__ __launch_bounds__(C::NT, 2) void linear_grad_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
    static_assert(tile_out_bytes<C>() <= C::SMEM, "the tile leaves through the stages' buffers");
    int tile, slot, first, count, m0, n0;
    pg::pick(a.w, blockIdx.x, a.nk, tile, slot, first, count);
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
__global__ __launch_bounds__(C::NT) void linear_grad_join_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[tile_out_bytes<C>()];
    int m0, n0;
    tile_at<C>(a, a.w.whole + blockIdx.x, m0, n0);
    floatx4 v[C::FB];
    pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, v);
    product_rows<C>(a, m0, n0, blockIdx.y, v, smem);
}

// dX from W as it lies, for few rows: one row of tiles.
struct FewArgs {
    const char *P;      // dZ's panels, of prows rows
    long prows;
    int Fp, F;
    const void *W;
    long ldw;
};
template <int FA, int PP, bool F16>
__global__ __launch_bounds__(256, 2) void linear_grad_few_kernel(ProductArgs a, FewArgs f) {
    __shared__ __attribute__((aligned(16))) char smem[std::max(few::smem_bytes<few::Tile<FA, 4>>(), tile_out_bytes<few::Tile<FA, 4>>())];
    few::with_rows<FA>(a.M, [&](auto fa) {
        typedef few::Tile<fa, 4> C;
        int tile, slot, first, count;
        pg::pick(a.w, blockIdx.x, a.nk, tile, slot, first, count);
        floatx4 acc[C::FA][C::FB];
        few::contract_across<C, PP, F16>(f.P, f.prows, f.Fp, f.W, f.ldw, f.F, a.N, tile * C::BN, first, count, smem, acc);
        if (slot >= 0) {
            pg::store_partials<C>(a.w.part, slot, acc);
            return;
        }
        few::sync();
#pragma unroll
        for (int i = 0; i < C::FA; i++) product_rows<C>(a, 0, tile * C::BN, i, acc[i], smem);
    });
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

struct Layout {
    int P, PO;                 // planes of dZ; of X and W
    int Np, Fp, Dp, few;
    bool products, pack_x, pack_w;
    int64_t exps, maxes, dbpart, dZ, Xp, Wp, sums, total;
};

pg::Plan dx_plan(const ah_linear_grad_desc &d, const Layout &l) {
    return pg::plan([&](int w) { return (long)ceil_div(d.N, w) * ceil_div(d.D, w); }, d.F, l.P, l.PO, l.PO == 2);   // (64-wide tiles of one plane
}
pg::Plan dw_plan(const ah_linear_grad_desc &d, const Layout &l) {
    return pg::plan([&](int w) { return (long)ceil_div(d.F, w) * ceil_div(d.D, w); }, d.N, l.P, l.PO, l.PO == 2);   // have no layout along k)
}
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
    l.maxes = take(3 * kScans * 4);
    if (d.dbias) l.dbpart = take((int64_t)(l.Np / kRows) * d.F * 4);
    if (l.products) l.dZ = take((int64_t)l.Np * l.Fp * 2 * l.P);
    if (l.pack_x) l.Xp = take((int64_t)d.N * l.Dp * 2 * l.PO);
    if (l.pack_w) l.Wp = take((int64_t)d.F * l.Dp * 2 * l.PO);
    int64_t sums = 0;
    if (l.few) {
        const pg::Work w = few_work(d, l);
        sums = w.splits > 1 ? (int64_t)w.rest * w.splits * l.few * 16 * 256 * 4 : 0;
    } else if (d.dX) {
        sums = dx_plan(d, l).part_bytes();
    }
    if (d.dW) sums = std::max<int64_t>(sums, dw_plan(d, l).part_bytes());
    l.sums = take(sums);
    l.total = at;
    return l;
}

template <class C>
void launch(ProductArgs a, hipStream_t s) {
    a.tiles_m = ceil_div(a.M, C::BM);
    a.tiles_n = ceil_div(a.N, C::BN);
    hipLaunchKernelGGL((linear_grad_kernel<C>), dim3((unsigned)a.w.blocks()), dim3(C::NT), 0, s, a);
    if (a.w.splits > 1) hipLaunchKernelGGL((linear_grad_join_kernel<C>), dim3((unsigned)a.w.rest, C::FA), dim3(C::NT), 0, s, a);
}
template <int TA, int TB, int PA, int PB>
void launch(const ProductArgs &a, int width, hipStream_t s) {
    if (width == 256) launch<pg::Tile256<TA, TB, PA, PB>>(a, s);
    else if (width == 128) launch<pg::Tile128<TA, TB, PA, PB>>(a, s);
    else if constexpr (PB == 2) launch<pg::Tile64<TA, TB, PA, PB>>(a, s);
}

template <int P, bool F16, int FA>
void launch_few(const ProductArgs &a, const FewArgs &f, hipStream_t s) {
    hipLaunchKernelGGL((linear_grad_few_kernel<FA, P, F16>), dim3((unsigned)a.w.blocks()), dim3(256), 0, s, a, f);
    if (a.w.splits > 1) hipLaunchKernelGGL((linear_grad_few_join_kernel<FA>), dim3((unsigned)a.w.rest, FA), dim3(256), 0, s, a);
}

template <class T, int P, int PO>
void run(const ah_linear_grad_desc &d, const Layout &l, hipStream_t s) {
    char *ws = (char *)d.ws;
    const GradIn g{d.N, d.D, d.F, d.act, d.scale, d.dY, d.Z, d.U, d.lddy, d.ldz, d.ldu, d.X, d.W, d.ldx, d.ldw};
    const auto scans = [](int64_t rows, int64_t width) { return (int)std::min<int64_t>((rows * ((width + 1023) / 1024) + 3) / 4, kScans); };
    ScanArgs sc{};
    sc.zblocks = l.products ? scans(d.N, d.F) : 0;
    sc.xblocks = l.pack_x && PO == 2 ? scans(d.N, d.D) : 0;
    sc.wblocks = l.pack_w && PO == 2 ? scans(d.F, d.D) : 0;
    sc.maxes = (unsigned *)(ws + l.maxes);
    if (l.products) hipLaunchKernelGGL(linear_grad_scan_kernel<T>, dim3((unsigned)(sc.zblocks + sc.xblocks + sc.wblocks)), dim3(256), 0, s, g, sc);

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
    p.zcols = ceil_div(l.Fp, 256);
    p.zblocks = l.Np / kRows * p.zcols;
    p.rest = (int)std::min<int64_t>(((l.pack_x ? d.N : 0) + (int64_t)(l.pack_w ? d.F : 0) + 3) / 4, 4096);
    p.exps = (int *)(ws + l.exps);
    hipLaunchKernelGGL((linear_grad_pack_kernel<T, P, PO>), dim3((unsigned)(p.zblocks + p.rest)), dim3(256), 0, s, g, p, sc);
    if (d.dbias) hipLaunchKernelGGL(linear_grad_db_kernel, dim3((unsigned)ceil_div(d.F, 64)), dim3(1024), 0, s, p.dbpart, l.Np / kRows, d.F, d.dbias);

    ProductArgs a{};
    a.ea = p.exps;
    a.out16 = d.grad_dtype == AH_F16;
    a.N = d.D;
    if (d.dX) {
        ProductArgs b = a;
        b.M = d.N;
        b.C = d.dX;
        b.ldc = d.lddx;
        if (l.few) {
            const FewArgs f{ws + l.dZ, l.Np, l.Fp, d.F, d.W, d.ldw};
            b.nk = ceil_div(d.F, few::across_v(P));
            b.w = few_work(d, l);
            b.w.part = (float *)(ws + l.sums);
            if (l.few == 1) launch_few<P, PO == 1, 1>(b, f, s);
            else if (l.few == 4) launch_few<P, PO == 1, 4>(b, f, s);
            else if constexpr (PO == 2) launch_few<P, PO == 1, 8>(b, f, s);
        } else {
            const pg::Plan plan = dx_plan(d, l);
            b.w = plan.w;
            b.w.part = (float *)(ws + l.sums);
            b.A = pg::panels(p.dZ, l.Np, l.Np, l.Fp);
            b.B = l.pack_w ? pg::panels(p.Wp, d.F, l.Dp, d.F) : pg::row_major(d.W, d.ldw, d.D, d.F);
            b.nk = ceil_div(d.F, P == 1 ? 64 : 32);   // every stage begins at a row of W that there is
            b.eb = PO == 2 ? p.exps + 2 : nullptr;
            launch<0, 1, P, PO>(b, plan.width, s);
        }
    }
    if (d.dW) {
        ProductArgs b = a;
        const pg::Plan plan = dw_plan(d, l);
        b.M = d.F;
        b.C = d.dW;
        b.ldc = d.lddw;
        b.w = plan.w;
        b.w.part = (float *)(ws + l.sums);
        b.A = pg::panels(p.dZ, l.Np, l.Fp, l.Np);
        b.B = l.pack_x ? pg::panels(p.Xp, d.N, l.Dp, d.N) : pg::row_major(d.X, d.ldx, d.D, d.N);
        b.nk = ceil_div(d.N, P == 1 ? 64 : 32);
        b.eb = PO == 2 ? p.exps + 1 : nullptr;
        launch<1, 1, P, PO>(b, plan.width, s);
    }
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
