// linear_ce_few.h — the head's products with W for few rows (at most 128), where W is read once, as it lies, straight into registers.
//
// Packing W for the tile loops of plane_gemm.h reads it twice and writes it, which many rows pay for and few do not: at 121 rows, 2944
// features and 51416 classes in f32 scan and packing were 400 of 545 us. Here every wave owns columns of the result for all rows and
// reads W from memory itself, because no other wave wants the same values; what the waves share (the rows) goes through LDS. f32 operands go to the f32 matrix instruction, unaligned f16 ones to the f16 one. A lane's 16-byte load
// holds neighbouring k of one row: which of them an instruction calls its k-th is open as long as both operands agree, so the
// loads need no reordering. Bounds: W's bytes up to 32 rows in f32 (4.8 TB/s), then the f32 matrix rate, 256 operations a cycle and CU.
#pragma once
#include "plane_gemm.h"

namespace ah {
namespace few {

using pg::h4;
using pg::h8;

// 16 FA rows by 4 waves of 16 FB columns each; the accumulators' order is that of pg::contract.
template <int FA_, int FB_>
struct Tile {
    static constexpr int FA = FA_, FB = FB_, WVM = 1, WVN = 4, NT = 256, WM = 16 * FA, WN = 16 * FB, BM = WM, BN = 4 * WN;
};

// Calls f with the constant for the smallest of 1, 2, 4, 6 and 8 tiles of 16 rows that hold M, of at most FA.
template <int FA, class F>
__device__ __forceinline__ void with_rows(int M, F f) {
    if constexpr (FA == 1) f(std::integral_constant<int, 1>());
    else if (M <= 16) f(std::integral_constant<int, 1>());
    else if (M <= 32) f(std::integral_constant<int, 2>());
    else if constexpr (FA == 4) f(std::integral_constant<int, 4>());
    else if (M <= 64) f(std::integral_constant<int, 4>());
    else if (M <= 96) f(std::integral_constant<int, 6>());
    else f(std::integral_constant<int, 8>());
}

// The rows' side of a stage: 256 bytes of each row in LDS, shared by the waves (each wave fetching its own copy through the caches took
// 984 us, not 432, at 64 rows of 4001 f16 features over 131072 classes). 16-byte pieces are swizzled by the row, so that a fragment's
// 16 rows lie in different banks. Two buffers, one barrier a stage.
template <class C>
constexpr int smem_bytes() { return 2 * C::BM * 256; }
__device__ __forceinline__ const char *piece_at(const char *buf, int m, int piece) { return buf + m * 256 + ((piece ^ (m & 15)) * 16); }

// Waits for this wave's LDS accesses, not for its loads from memory, which run on across the barrier.
__device__ __forceinline__ void sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Stages [first, first + count) of NCH chunks. fetch(stage, r): this thread's piece (threadIdx & 15) of rows threadIdx / 16 + 16 i;
// load(slot, chunk): a chunk of W into a slot of registers, PF chunks ahead; use(buf, c, slot): the products of the stage's chunk c.
template <class C, int NCH, int PF, class Fetch, class Load, class Use>
__device__ __forceinline__ void stages(int first, int count, char *smem, Fetch fetch, Load load, Use use) {
    static_assert(NCH % PF == 0, "a stage ends where it began in the slots");
    if (count <= 0) return;
    const int row = threadIdx.x >> 4, last = (first + count) * NCH - 1;
    u4 r[C::FA];
    const auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < C::FA; i++) *(u4 *)piece_at(smem + buf * C::BM * 256, 16 * i + row, threadIdx.x & 15) = r[i];
    };
    fetch(first, r);
#pragma unroll
    for (int p = 0; p < PF; p++) load(p, first * NCH + p);
    put(0);
    sync();
    for (int s = 0; s < count; s++) {
        if (s + 1 < count) fetch(first + s + 1, r);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            use(smem + (s & 1) * C::BM * 256, c, c % PF);
            if (c & 1) {   // two chunks at a time: the halves of one cache line
                load((c - 1) % PF, min((first + s) * NCH + c - 1 + PF, last));
                load(c % PF, min((first + s) * NCH + c + PF, last));
            }
            __builtin_amdgcn_sched_barrier(0);   // loads stay where they are: sunk to the body's end, they would be waited for there
        }
        if (s + 1 < count) put((s + 1) & 1);
        sync();
    }
}

// k of a stage of the logits' product: 256 bytes of a row.
constexpr int along_k(bool f16) { return f16 ? 128 : 64; }

// acc[i][j] += X(m, k) W(n, k) over stages [first, first + count) of k, four chunks of 64 bytes each. Rows m of X are rowmap[m], the
// last of M for those past it; past the last class the last row of W is read (the epilogue leaves those columns out). Where a lane's
// 16 bytes end past D (D >= 8), both operands read the row's last 16, and the rows' side has zeros for the k that were there before.
template <class C, bool F16>
__device__ __forceinline__ void contract_along(const void *X, long ldx, const int *rowmap, int M, const void *W, long ldw, int V, int D, int n0,
                                               int first, int count, char *smem, floatx4 (&acc)[C::FA][C::FB]) {
    typedef typename std::conditional<F16, half_t, float>::type T;
    constexpr int E = F16 ? 8 : 4, NCH = 4, K = 4 * E;
    typedef T vec __attribute__((ext_vector_type(E)));
    typedef T vec_any __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
    const T *xp[C::FA], *wp[C::FB];
#pragma unroll
    for (int i = 0; i < C::FA; i++) xp[i] = (const T *)X + (long)rowmap[min(16 * i + (int)(threadIdx.x >> 4), M - 1)] * ldx;
#pragma unroll
    for (int j = 0; j < C::FB; j++) wp[j] = (const T *)W + (long)min(n0 + wave * C::WN + 16 * j + row, V - 1) * ldw;
#pragma unroll
    for (int i = 0; i < C::FA; i++)
#pragma unroll
        for (int j = 0; j < C::FB; j++) acc[i][j] = (floatx4){};
    vec w[NCH][C::FB];
    stages<C, NCH, NCH>(first, count, smem, [&](int stage, u4 (&r)[C::FA]) {
        const int k = stage * NCH * K + (threadIdx.x & 15) * E, at = min(k, D - E);
#pragma unroll
        for (int i = 0; i < C::FA; i++) {
            vec v = *(const vec_any *)(xp[i] + at);
            if ((stage + 1) * NCH * K > D)
#pragma unroll
                for (int e = 0; e < E; e++) v[e] = at + e < k ? (T)0 : v[e];
            r[i] = __builtin_bit_cast(u4, v);
        }
    }, [&](int p, int c) {
#pragma unroll
        for (int j = 0; j < C::FB; j++) w[p][j] = *(const vec_any *)(wp[j] + min(c * K + g * E, D - E));
    }, [&](const char *buf, int c, int p) {
#pragma unroll
        for (int i = 0; i < C::FA; i++) {
            const vec x = *(const vec *)piece_at(buf, 16 * i + row, 4 * c + g);
#pragma unroll
            for (int j = 0; j < C::FB; j++) {
                if constexpr (F16) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[p][j], x, acc[i][j], 0, 0, 0);
                else
#pragma unroll
                    for (int e = 0; e < E; e++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[p][j][e], x[e], acc[i][j], 0, 0, 0);
            }
        }
    });
}

// v of a stage of the dX product: two panels of P.
constexpr int across_v(int pp) { return pp == 2 ? 64 : 128; }

// out[i][j] += P(m, v) W(v, n) over stages [first, first + count) of v, chunks of 16; P in panels of `prows` rows and PP planes, Vp wide,
// zeros past V. A lane reads four columns of rows v: those are 16-column tiles j's row `lane % 16`, and the columns are dealt to
// lanes so that result lane g, tile r, element j is column 16 r + 4 g + j of the wave's 64: as in pg::contract, after swapping r and j.
// Lanes whose columns end past D (D >= 8) read the last four, and the result is shifted into place.
template <class C, int PP, bool F16>
__device__ __forceinline__ void contract_across(const char *P, long prows, int Vp, const void *W, long ldw, int V, int D, int n0, int first, int count,
                                                char *smem, floatx4 (&out)[C::FA][C::FB]) {
    static_assert(C::FB == 4, "four columns a lane");
    typedef typename std::conditional<F16, half_t, float>::type T;
    typedef T vec __attribute__((ext_vector_type(4)));
    typedef T vec_any __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    constexpr int NCH = across_v(PP) / 16, PF = C::FA == 8 || (C::FA == 6 && !F16) ? 2 : 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, row = lane & 15;
    const int nw = n0 + wave * C::WN, panels = Vp / (across_v(PP) / 2);
    const T *wp = (const T *)W + min(nw + 4 * (4 * (row & 3) + (row >> 2)), D - 4);
    floatx4 acc[C::FA][4];
#pragma unroll
    for (int i = 0; i < C::FA; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = (floatx4){};
    vec w[PF][4];
    stages<C, NCH, PF>(first, count, smem, [&](int stage, u4 (&r)[C::FA]) {
        const int q = 2 * stage + ((threadIdx.x & 15) >> 3);
        const char *p = P + ((long)min(q, panels - 1) * prows + (threadIdx.x >> 4)) * 128 + (threadIdx.x & 7) * 16;
#pragma unroll
        for (int i = 0; i < C::FA; i++) {
            r[i] = *(const u4 *)(p + 2048 * i);
            if (q >= panels) r[i] = (u4){};
        }
    }, [&](int p, int c) {
#pragma unroll
        for (int t = 0; t < 4; t++) w[p][t] = *(const vec_any *)(wp + (long)min(16 * c + 4 * g + t, V - 1) * ldw);
    }, [&](const char *buf, int c, int p) {
        h4 k[4];
        if constexpr (F16)
#pragma unroll
            for (int j = 0; j < 4; j++) k[j] = (h4){w[p][0][j], w[p][1][j], w[p][2][j], w[p][3][j]};
#pragma unroll
        for (int i = 0; i < C::FA; i++) {
            const int piece = PP == 2 ? 8 * (c >> 1) + 2 * (c & 1) + (g >> 1) : 8 * (c >> 2) + 2 * (c & 3) + (g >> 1);
            const h4 hi = *(const h4 *)(piece_at(buf, 16 * i + row, piece) + 8 * (g & 1));
            h4 lo = {};
            if constexpr (PP == 2) lo = *(const h4 *)(piece_at(buf, 16 * i + row, piece + 4) + 8 * (g & 1));
            if constexpr (F16) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x16f16(k[j], hi, acc[i][j], 0, 0, 0);
                    if constexpr (PP == 2) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x16f16(k[j], lo, acc[i][j], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[p][t][j], (float)hi[t] + (float)lo[t], acc[i][j], 0, 0, 0);
            }
        }
    });
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int n = nw + 16 * r + 4 * g, shift = max(0, n - (D - 4));   // 4 and more: past D, never stored
#pragma unroll
        for (int i = 0; i < C::FA; i++) {
            floatx4 v = {acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
            if (shift == 1) v = __builtin_shufflevector(v, v, 1, 2, 3, 3);
            else if (shift == 2) v = __builtin_shufflevector(v, v, 2, 3, 3, 3);
            else if (shift == 3) v = __builtin_shufflevector(v, v, 3, 3, 3, 3);
            out[i][r] = v;
        }
    }
}

// `tiles` tiles of nk stages that take `us` each with a tile on every CU: what does not fill the CUs evenly is split over k, by the time
// that leaves, with at least two workgroups a CU where there are stages enough. 402 tiles of 128 rows over 2944 features in one piece
// each leave 110 CUs idle half the time: 421 us, and 372 with 146 of them in 7 pieces.
inline pg::Work work(int tiles, int nk, double us, long tile_bytes) {
    pg::Work best{tiles, 0, 1, nullptr};
    double best_us = 1e30;
    for (const int whole : {tiles / 256 * 256, 0})
        for (int s = 1; s <= 64 && (s == 1 || nk >= 2 * s); s++) {
            const long rest = tiles - whole, blocks = whole + rest * s;
            if (rest * s > 4096 && s > 1) break;
            const double t = (whole / 256 + (double)((rest * s + 255) / 256) / s) * nk * us * (blocks < 512 ? 1.25 : 1.0) +
                             (s > 1 ? 4.0 + 2e-6 / 4.8 * (double)(rest * s * tile_bytes) : 0.0);
            if (t < best_us) {
                best_us = t;
                best = s == 1 ? pg::Work{tiles, 0, 1, nullptr} : pg::Work{whole, (int)rest, s, nullptr};
            }
            if (!rest) break;
        }
    return best;
}

}  // namespace few
}  // namespace ah
