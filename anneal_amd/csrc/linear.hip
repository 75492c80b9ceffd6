// linear.hip — a linear layer with bias, activation, factor and residual in its product's epilogue.
//
//   Z = X W^T + b,  Y = R + s act(Z) U
//
// Many rows: the tile loops of plane_gemm.h. f16 operands go there as they lie where their rows are aligned (X also needs D to be a multiple
// of a stage's 64), others packed into panels. f32 operands are packed as two f16 planes, each row scaled by a power of two of its own
// that brings its largest magnitude to 2^15: the row's exponent leaves the product in the epilogue, so nothing but the row itself has
// to be read before it is packed, and a row keeps 22 bits whatever the others hold. Few rows: linear_ce_few.h, which reads W once, as it
// lies (f32 on the f32 matrix instruction, all 24 bits), or K over the waves of small workgroups where one launch is worth more.
//
// The epilogue takes Z from the accumulators in f32 through LDS (tile_out.h), eight columns of a row to a lane, so that U, R, Z and Y are
// read and written in 16 bytes; the loads of 16 rows are in flight together. Bound by the matrix cores for many rows, by W's bytes for few.
// f16 8192 x 4096 -> 16384 with bias, GELU and Z: 960-980 us (1135 TFLOP/s), 60 of them the epilogue; 1 x 4096 -> 16384 with a factor 26 (5.2 TB/s);
// 48 x 8192 -> 2048 14; f32 777 x 1001 -> 2003 29.
#include "linear.h"

#include <algorithm>

#include "act.h"
#include "linear_ce_few.h"
#include "tile_out.h"

namespace ah {
namespace {

struct Layer {
    int N, F, act;
    float scale;
    const void *bias, *U, *R;
    void *Y, *Z;
    long ldu, ldr, ldy, ldz;
    const int *ex, *ew;   // exponents of the planes' rows, or null
};

struct ProductArgs {
    pg::Operand X, W;
    int nk, tiles_m, tiles_n;
    pg::Work w;
    Layer l;
};

template <class C>
__device__ __forceinline__ void tile_at(const ProductArgs &a, int tile, int &m0, int &n0) {
    int tr, tc;
    pg::grouped_tile(tile, a.tiles_m, a.tiles_n, tr, tc);
    m0 = tr * C::BM;
    n0 = tc * C::BN;
}

// What follows the product for accumulator row i of the tile at (m0, n0).
template <class C, class T>
__device__ __forceinline__ void layer_rows(const Layer &l, int m0, int n0, int i, const floatx4 (&acc)[C::FB], char *smem) {
    typedef typename Raw8<T>::type raw;
    TileOut<C> out(smem, m0, n0, i);
    asm volatile("" : "+v"(out.m), "+v"(out.n));   // addresses are formed anew for each accumulator row: kept for all, they spill
    constexpr int P = TileOut<C>::kParts;
    const bool in = out.n < l.F;
    raw u[P], r[P];
    const auto row = [&](int p) { return out.m + p * TileOut<C>::kStep; };
#pragma unroll
    for (int p = 0; p < P; p++) {
        u[p] = r[p] = (raw){};
        if (!in || row(p) >= l.N) continue;
        if (l.U) u[p] = load_raw8((const T *)l.U + row(p) * l.ldu, out.n, l.F);
        if (l.R) r[p] = load_raw8((const T *)l.R + row(p) * l.ldr, out.n, l.F);
    }
    raw b = {};
    if (l.bias && in) b = load_raw8((const T *)l.bias, out.n, l.F);
    typedef int i8 __attribute__((ext_vector_type(8), aligned(4)));
    i8 ew = {};
    if (l.ew && in) ew = *(const i8 *)(l.ew + out.n);   // (there is room behind the last)
    out.put(acc);
    if (!in) return;
#pragma unroll
    for (int p = 0; p < P; p++) {
        if (row(p) >= l.N) continue;
        f8 z = out.get(p);
        if (l.ew) {
            const int ex = l.ex[row(p)];
#pragma unroll
            for (int k = 0; k < 8; k++) z.v[k] = ldexpf(z.v[k], -(ex + ew[k]));
        }
#pragma unroll
        for (int k = 0; k < 8; k++) z.v[k] += (float)b[k];
        if (l.Z) store8((T *)l.Z + row(p) * l.ldz, out.n, l.F, z);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float y = l.scale * act_of<sizeof(T) == 2>(l.act, z.v[k]);
            if (l.U) y *= (float)u[p][k];
            if (l.R) y += (float)r[p][k];
            z.v[k] = y;
        }
        store8((T *)l.Y + row(p) * l.ldy, out.n, l.F, z);
    }
}

template <class C, class T>
__global__ __launch_bounds__(C::NT, 2) void linear_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
    static_assert(tile_out_bytes<C>() <= C::SMEM, "the tile leaves through the stages' buffers");
    int tile, slot, first, count, m0, n0;
    pg::pick(a.w, blockIdx.x, a.nk, tile, slot, first, count);
    tile_at<C>(a, tile, m0, n0);
    floatx4 acc[C::FA][C::FB];
    pg::contract<C>(a.X, a.W, m0, n0, first, count, smem, acc);
    if (slot >= 0) {
        pg::store_partials<C>(a.w.part, slot, acc);
        return;
    }
    g16::lds_barrier();   // the last stage has been read
#pragma unroll
    for (int i = 0; i < C::FA; i++) {
        __builtin_amdgcn_sched_barrier(0);
        layer_rows<C, T>(a.l, m0, n0, i, acc[i], smem);
    }
}
template <class C, class T>
__global__ __launch_bounds__(C::NT) void linear_join_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[tile_out_bytes<C>()];
    int m0, n0;
    tile_at<C>(a, a.w.whole + blockIdx.x, m0, n0);
    floatx4 z[C::FB];
    pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, z);
    layer_rows<C, T>(a.l, m0, n0, blockIdx.y, z, smem);
}

// ── few rows ───────────────────────────────────────────────────────────────────

struct FewArgs {
    const void *X, *W;
    long ldx, ldw;
    int D;
};

template <class C, class T>
__device__ __forceinline__ void few_rows(const ProductArgs &a, const FewArgs &f, char *smem) {
    int tile, slot, first, count;
    pg::pick(a.w, blockIdx.x, a.nk, tile, slot, first, count);
    floatx4 acc[C::FA][C::FB];
    few::contract_along<C, sizeof(T) == 2>(f.X, f.ldx, nullptr, a.l.N, f.W, f.ldw, a.l.F, f.D, tile * C::BN, first, count, smem, acc);
    if (slot >= 0) {
        pg::store_partials<C>(a.w.part, slot, acc);
        return;
    }
    few::sync();
#pragma unroll
    for (int i = 0; i < C::FA; i++) layer_rows<C, T>(a.l, 0, tile * C::BN, i, acc[i], smem);
}
// Room for 16 FA rows; there may be fewer, and then the tile is.
template <int FA, class T>
__global__ __launch_bounds__(256, 2) void linear_few_kernel(ProductArgs a, FewArgs f) {
    typedef few::Tile<FA, 2> C;
    __shared__ __attribute__((aligned(16))) char smem[std::max(few::smem_bytes<C>(), tile_out_bytes<C>())];
    few::with_rows<FA>(a.l.N, [&](auto fa) { few_rows<few::Tile<fa, 2>, T>(a, f, smem); });
}
template <int FA, class T>
__global__ __launch_bounds__(256) void linear_few_join_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(16))) char smem[tile_out_bytes<few::Tile<FA, 2>>()];
    few::with_rows<FA>(a.l.N, [&](auto fa) {
        typedef few::Tile<fa, 2> C;
        if ((int)blockIdx.y >= C::FA) return;
        floatx4 z[C::FB];
        pg::sum_partials<C>(a.w, blockIdx.x, blockIdx.y, z);
        layer_rows<C, T>(a.l, 0, (a.w.whole + blockIdx.x) * C::BN, blockIdx.y, z, smem);
    });
}

// ── few rows, K split over a workgroup's waves ─────────────────────────────────

// 16 columns a workgroup: its waves read their rows of W in turns of 128 bytes (two chunks of 64), each with the rows of X that go with
// them, and add their sums in LDS, in order. W goes from memory to registers once, all of its workgroups are at work from the start, and nothing
// has to be joined by another launch. Where a lane's 16 bytes end past D (D >= 8), it reads the row's last 16 and those that were there before
// are zeros.
struct RowArgs {
    FewArgs f;
    Layer l;
};
template <int FA, class T>
__global__ __launch_bounds__(1024) void linear_rows_kernel(RowArgs a) {
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int E = 16 / sizeof(T), K = 4 * E, U = F16 && FA == 1 ? 8 : 4;   // k of a lane's load, of a chunk; chunks in flight
    typedef T vec __attribute__((ext_vector_type(E)));
    typedef T vec_any __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    __shared__ floatx4 red[16][FA][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, row = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, D = a.f.D, nc = (D + K - 1) / K;
    const T *w = (const T *)a.f.W + (long)min(n0 + row, a.l.F - 1) * a.f.ldw, *x[FA];
#pragma unroll
    for (int i = 0; i < FA; i++) x[i] = (const T *)a.f.X + (long)min(16 * i + row, a.l.N - 1) * a.f.ldx;
    floatx4 acc[FA];
#pragma unroll
    for (int i = 0; i < FA; i++) acc[i] = (floatx4){};
    const auto chunk = [&](int c) { return (c >> 1) * 2 * waves + 2 * wave + (c & 1); };   // this wave's c-th
    for (int c0 = 0; chunk(c0) < nc; c0 += U) {
        vec wv[U], xv[U][FA];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = min(chunk(c0 + u) * K + g * E, D - E);
            wv[u] = *(const vec_any *)(w + at);
#pragma unroll
            for (int i = 0; i < FA; i++) xv[u][i] = *(const vec_any *)(x[i] + at);
        }
        if (chunk(c0 + U - 1) * K + K > D)
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = chunk(c0 + u) * K + g * E, at = min(k, D - E);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const bool again = at + e < k;
                    wv[u][e] = again ? (T)0 : wv[u][e];
#pragma unroll
                    for (int i = 0; i < FA; i++) xv[u][i][e] = again ? (T)0 : xv[u][i][e];
                }
            }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < FA; i++) {
                if constexpr (F16) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wv[u], xv[u][i], acc[i], 0, 0, 0);
                else
#pragma unroll
                    for (int e = 0; e < E; e++) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[u][e], xv[u][i][e], acc[i], 0, 0, 0);
            }
    }
#pragma unroll
    for (int i = 0; i < FA; i++) red[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < FA; i += waves) {   // a wave 16 rows: a lane one of them and four columns
        floatx4 z = red[0][i][lane];
        for (int v = 1; v < waves; v++) z += red[v][i][lane];
        const Layer &l = a.l;
        const long m = 16 * i + row;
        const int n = n0 + 4 * g;
        if (m >= l.N || n >= l.F) continue;
        if (l.bias) z += pg::load4((const T *)l.bias, n, l.F);
        if (l.Z) pg::store4((T *)l.Z + m * l.ldz, n, l.F, z);
        floatx4 u = {1.0f, 1.0f, 1.0f, 1.0f}, r = {};
        if (l.U) u = pg::load4((const T *)l.U + m * l.ldu, n, l.F);
        if (l.R) r = pg::load4((const T *)l.R + m * l.ldr, n, l.F);
#pragma unroll
        for (int k = 0; k < 4; k++) z[k] = r[k] + l.scale * act_of<F16>(l.act, z[k]) * u[k];
        pg::store4((T *)l.Y + m * l.ldy, n, l.F, z);
    }
}

// ── packing ────────────────────────────────────────────────────────────────────

struct PackArgs {
    const void *X, *W;       // null: not packed
    long ldx, ldw;
    int N, F, D, Dp;
    half_t *Xp, *Wp;
    int *ex, *ew;
};
// A wave a row, of X and then of W. f32: the row's largest magnitude first, then its planes; a longer row's second reading comes from the caches.
template <int P>
__global__ __launch_bounds__(256) void linear_pack_kernel(PackArgs a) {
    constexpr int E = P == 1 ? 2 : 4;
    const int lane = threadIdx.x & 63;
    const long xrows = a.X ? a.N : 0, rows = xrows + (a.W ? a.F : 0);
    for (long q = (long)blockIdx.x * 4 + (threadIdx.x >> 6); q < rows; q += (long)gridDim.x * 4) {
        const bool x = q < xrows;
        const long r = x ? q : q - xrows;
        const char *in = x ? (const char *)a.X + r * a.ldx * E : (const char *)a.W + r * a.ldw * E;
        int e = 0;
        if constexpr (P == 2) {
            constexpr int HELD = 8;   // 256 columns each: longer rows that a wave's registers hold are read once
            floatx4 v[HELD];
            // 200 x 2048 -> 8192 71 -> 64 us, 777 x 1001 -> 2003 31.6 -> 30.2; shorter rows are no faster from registers (4000 x 768 -> 3000 118 | 121)
            const bool held = a.D > 768 && a.D <= 256 * HELD;
            unsigned m = 0;
            const auto most = [&](floatx4 y) {
#pragma unroll
                for (int k = 0; k < 4; k++) m = max(m, pg::magnitude(__float_as_uint(y[k])));
            };
            if (held) {
#pragma unroll
                for (int j = 0; j < HELD; j++) v[j] = j * 256 < a.D ? pg::load4((const float *)in, lane * 4 + 256 * j, a.D) : (floatx4){};
#pragma unroll
                for (int j = 0; j < HELD; j++) most(v[j]);
            } else {
#pragma unroll 4
                for (int c = lane * 4; c < a.D; c += 256) most(pg::load4((const float *)in, c, a.D));
            }
            for (int o = 32; o >= 1; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
            e = pg::plane_exp(m);
            if (lane == 0) (x ? a.ex : a.ew)[r] = e;
            if (held) {
#pragma unroll
                for (int j = 0; j < HELD; j++) {
                    const int c = lane * 4 + 256 * j;
                    if (c >= a.Dp) continue;
#pragma unroll
                    for (int k = 0; k < 4; k++) v[j][k] = ldexpf(v[j][k], e);
                    pg::plane_store((x ? a.Xp : a.Wp) + pg::panel_at<2>(x ? a.N : a.F, r, c), v[j]);
                }
                continue;
            }
        }
        pg::pack_row<P>(x ? a.Xp : a.Wp, x ? a.N : a.F, r, in, a.D, a.Dp, e);
    }
}

// ── host ───────────────────────────────────────────────────────────────────────

constexpr int kFewF32 = 128, kFewF16 = 64;   // rows up to which W is read as it lies

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct Layout {
    int P, Dp, few;          // planes; padded D; 16-row tiles of the forms for few rows, or 0
    bool rows, pack_x, pack_w;   // rows: K over a workgroup's waves
    int64_t Xp, Wp, ex, ew, sums, total;
};

bool rows_aligned(const void *p, int64_t ld, int D) { return D % 8 == 0 && ld % 8 == 0 && ((uintptr_t)p & 15) == 0 && ld <= 1 << 22; }

pg::Plan plan_of(const ah_linear_desc &d, const Layout &l) {
    return pg::plan([&](int w) { return (long)ceil_div(d.N, w) * ceil_div(d.F, w); }, l.Dp, l.P, l.P, true);
}
// The form for few rows: tiles of 128 columns, 1.75 us a stage at the rate of memory, 3.4 at the f32 matrix rate for 128 rows.
pg::Work few_work(const ah_linear_desc &d, const Layout &l) {
    const bool f16 = d.dtype == AH_F16;
    return few::work(ceil_div(d.F, 128), ceil_div(d.D, few::along_k(f16)), std::max(1.75, f16 ? 0.0 : 0.43 * l.few), l.few * 16l * 128 * 4);
}

// Which form for few rows. K over the waves reads all of X beside every 16 rows of W, at 33 GB/s a CU of both; tiles of 128 columns read W at 6.6
// (f16) or 5 TB/s, and then 3.5 us go into a second launch. Measured, K over the waves | tiles: f16 1 x 4096 -> 16384 25.7 | 28.5 us,
// 8 x 2048 -> 8192 9.6 | 13.5, 16 x 8192 -> 2048 17.3 | 15.8, 64 x 1024 -> 1024 7.6 | 8.9, 64 x 4096 -> 16384 82 | 38; f32 1 x 4096 -> 16384 58 | 70,
// 16 x 4096 -> 1024 17.1 | 12.6.
bool over_waves(const ah_linear_desc &d) {
    if (d.N > 64) return false;
    const bool f16 = d.dtype == AH_F16;
    const double tiles = ceil_div(d.F, 16), row = (double)d.D * (f16 ? 2 : 4), bytes = row * d.F;
    const double both = tiles * row * (16 + d.N) / (33e3 * std::min(256.0, tiles));
    return std::max(both, bytes / 5.3e6) <= 6.0 + bytes / (f16 ? 6.6e6 : 5e6);
}

Layout layout(const ah_linear_desc &d) {
    Layout l{};
    const bool f16 = d.dtype == AH_F16;
    l.P = f16 ? 1 : 2;
    l.Dp = (d.D + 63) & ~63;
    if (d.N <= (f16 ? kFewF16 : kFewF32) && d.D >= 8) l.few = d.N <= 16 ? 1 : d.N <= 64 ? 4 : 8;
    l.rows = l.few && over_waves(d);
    l.pack_x = !l.few && (!f16 || d.D % 64 || !rows_aligned(d.X, d.ldx, d.D));
    l.pack_w = !l.few && (!f16 || !rows_aligned(d.W, d.ldw, d.D));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at = (at + bytes + 255) & ~255ll;
        return o;
    };
    if (l.pack_x) l.Xp = take((int64_t)d.N * l.Dp * 2 * l.P);
    if (l.pack_w) l.Wp = take((int64_t)d.F * l.Dp * 2 * l.P);
    if (!f16 && !l.few) {
        l.ex = take((int64_t)d.N * 4);
        l.ew = take(((int64_t)d.F + 7) * 4);
    }
    if (l.few && !l.rows) {
        const pg::Work w = few_work(d, l);
        l.sums = take(w.splits > 1 ? (int64_t)w.rest * w.splits * l.few * 16 * 128 * 4 : 0);
    } else if (!l.few) {
        l.sums = take(plan_of(d, l).part_bytes());
    }
    l.total = std::max<int64_t>(at, 16);
    return l;
}

template <class C, class T>
void launch(ProductArgs a, hipStream_t s) {
    a.tiles_m = ceil_div(a.l.N, C::BM);
    a.tiles_n = ceil_div(a.l.F, C::BN);
    hipLaunchKernelGGL((linear_kernel<C, T>), dim3((unsigned)a.w.blocks()), dim3(C::NT), 0, s, a);
    if (a.w.splits > 1) hipLaunchKernelGGL((linear_join_kernel<C, T>), dim3((unsigned)a.w.rest, C::FA), dim3(C::NT), 0, s, a);
}
template <int P, class T>
void launch(const ProductArgs &a, int width, hipStream_t s) {
    if (width == 256) launch<pg::Tile256<0, 0, P, P>, T>(a, s);
    else if (width == 128) launch<pg::Tile128<0, 0, P, P>, T>(a, s);
    else launch<pg::Tile64<0, 0, P, P>, T>(a, s);
}
void launch_rows(const ah_linear_desc &d, const RowArgs &r, hipStream_t s) {
    const bool f16 = d.dtype == AH_F16;
    const int tiles = ceil_div(d.F, 16), chunks = ceil_div(d.D, f16 ? 32 : 16);
    int waves = 4;   // up to 16 on each CU, of four pairs of chunks or more
    while (waves < 16 && tiles * waves < 4096 && chunks >= waves * 8) waves *= 2;
    const auto go = [&](auto fa) {
        if (f16) hipLaunchKernelGGL((linear_rows_kernel<fa, half_t>), dim3((unsigned)tiles), dim3(64 * waves), 0, s, r);
        else hipLaunchKernelGGL((linear_rows_kernel<fa, float>), dim3((unsigned)tiles), dim3(64 * waves), 0, s, r);
    };
    if (d.N <= 16) go(std::integral_constant<int, 1>());
    else if (d.N <= 32) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
}
template <int FA, class T>
void launch_few(const ProductArgs &a, const FewArgs &f, hipStream_t s) {
    hipLaunchKernelGGL((linear_few_kernel<FA, T>), dim3((unsigned)a.w.blocks()), dim3(256), 0, s, a, f);
    if (a.w.splits > 1) hipLaunchKernelGGL((linear_few_join_kernel<FA, T>), dim3((unsigned)a.w.rest, FA), dim3(256), 0, s, a);
}
template <class T>
void launch_few(const ProductArgs &a, const FewArgs &f, int few, hipStream_t s) {
    if (few == 1) launch_few<1, T>(a, f, s);
    else if (few == 4) launch_few<4, T>(a, f, s);
    else if constexpr (sizeof(T) == 4) launch_few<8, T>(a, f, s);   // (f16 stops at 64 rows)
}

}  // namespace

int64_t linear_workspace(const ah_linear_desc &d) { return layout(d).total; }

hipError_t linear(const ah_linear_desc &d, hipStream_t s) {
    const Layout l = layout(d);
    char *ws = (char *)d.ws;
    const bool f16 = d.dtype == AH_F16;
    ProductArgs a{};
    a.l = {d.N, d.F, d.act, d.scale, d.bias, d.U, d.R, d.Y, d.Z, d.ldu, d.ldr, d.ldy, d.ldz, nullptr, nullptr};
    if (l.few) {
        const FewArgs f{d.X, d.W, d.ldx, d.ldw, d.D};
        if (l.rows) {
            launch_rows(d, RowArgs{f, a.l}, s);
            return hipGetLastError();
        }
        a.nk = ceil_div(d.D, few::along_k(f16));
        a.w = few_work(d, l);
        a.w.part = (float *)(ws + l.sums);
        if (f16) launch_few<half_t>(a, f, l.few, s);
        else launch_few<float>(a, f, l.few, s);
        return hipGetLastError();
    }
    const PackArgs p{l.pack_x ? d.X : nullptr, l.pack_w ? d.W : nullptr, d.ldx, d.ldw, d.N, d.F, d.D, l.Dp, (half_t *)(ws + l.Xp), (half_t *)(ws + l.Wp),
                     (int *)(ws + l.ex), (int *)(ws + l.ew)};
    const int64_t rows = (l.pack_x ? d.N : 0) + (int64_t)(l.pack_w ? d.F : 0);
    if (rows) {
        const dim3 grid((unsigned)std::min<int64_t>((rows + 3) / 4, 4096));
        if (f16) hipLaunchKernelGGL(linear_pack_kernel<1>, grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL(linear_pack_kernel<2>, grid, dim3(256), 0, s, p);
    }
    const pg::Plan plan = plan_of(d, l);
    a.X = l.pack_x ? pg::panels(p.Xp, d.N, d.N, l.Dp) : pg::row_major(d.X, d.ldx, d.N, d.D);
    a.W = l.pack_w ? pg::panels(p.Wp, d.F, d.F, l.Dp) : pg::row_major(d.W, d.ldw, d.F, d.D);
    a.nk = l.Dp / (f16 ? 64 : 32);
    a.w = plan.w;
    a.w.part = (float *)(ws + l.sums);
    if (f16) {
        launch<1, half_t>(a, plan.width, s);
    } else {
        a.l.ex = p.ex;
        a.l.ew = p.ew;
        launch<2, float>(a, plan.width, s);
    }
    return hipGetLastError();
}

}  // namespace ah
