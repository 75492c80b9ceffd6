// plane_gemm.h — contractions of matrices held as one or two f16 planes, for the operators whose products must keep more
// than f16's 11 bits or whose epilogue is their own (linear_ce.hip, muon.hip).
//
//   C[m,n] = epi( sum_k A(m,k) B(n,k) )
//
// An f32 matrix x is carried as hi = f16(2^s x), lo = f16(2^s x - hi): 22 bits of each value whose magnitude is within 2^14 of
// 2^15, with an absolute floor of 2^-24 (an f16 subnormal) below that. A product of two such matrices is three f16 products,
// hi*hi + lo*hi + hi*lo (lo*lo is below the rounding of the sum), accumulated in one f32 accumulator; every f16 product is exact
// in f32. Three f16 MFMAs do the work of one f32 MFMA of the same shape in 3/16 of its time.
//
// Layout of a two-plane matrix: each stored row holds groups of 32 hi values and then their 32 lo values (128 bytes, one cache
// line). To the staging code it is an f16 matrix of twice the width, so both planes of a tile arrive with the one set of
// global->LDS loads, and a stage of 32 k in two planes has the LDS image of a stage of 64 k in one.
//   T = 0: rows of the operand are stored rows, k runs along them;  T = 1: stored rows are k, the operand's rows run along them.
//
// Per stage a wave reads each fragment once: hi*hi and lo*hi share B's hi, hi*hi and hi*lo share A's hi. So two planes take 2/3
// of the LDS reads per MFMA that one plane takes, and a 256x256 tile of 8 waves is bound by MFMA issue, not by LDS.
#pragma once
#include "ah_common.h"
#include "gemm16_kernel.h"

namespace ah {
namespace pg {

using g16::h8;
using g16::lds_s4;
using g16::s4;

typedef half_t h4 __attribute__((ext_vector_type(4)));

// Halves from the start of a stored row to the hi value of column c (lo: 32 further) in a matrix of P planes.
template <int P>
__host__ __device__ __forceinline__ long plane_col(long c) {
    return P == 1 ? c : (c >> 5) * 64 + (c & 31);
}

// Splits 4 values into the two planes at p (hi) and p + 32 (lo).
__device__ __forceinline__ void plane_store(half_t *p, floatx4 v) {
    h4 hi, lo;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        hi[r] = (half_t)v[r];
        lo[r] = (half_t)(v[r] - (float)hi[r]);
    }
    *(h4 *)p = hi;
    *(h4 *)(p + 32) = lo;
}

// One stage's 1 KiB blocks that a wave fetches: R operand rows x BK k in P planes. Offsets are relative to the tile's corner.
template <int R, int T, int P, int BK, int NW>
struct PFetch {
    static constexpr int W = T == 0 ? BK * P : R * P;   // halves of a stored row in the stage
    static constexpr int NB = R * BK * P * 2 / 1024, PER = NB / NW;
    static constexpr int ROWS = 512 / W;                // T = 1: stored rows in a block
    static_assert(PER * NW == NB, "a stage's blocks split evenly over the waves");
    static_assert(T == 0 || W >= 128, "the T = 1 swizzle spans eight 16-column segments");
    uint32_t off[PER];
    // rmax: rows of the operand (a multiple of 8 for T = 1); a row past it reads the last one
    __device__ __forceinline__ void init(long ld, int r0, int rmax, int wave, int lane) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int b = wave * PER + j;
            if constexpr (T == 0) {
                constexpr int CH = W / 8, SR = 16 / CH;   // chunks per row, rows per 256-byte super-row (koff)
                const int q = 4 * b + (lane >> 4), x = (lane & 15) ^ (q & 15);
                const int row = min(q * SR + x / CH, rmax - 1 - r0);
                off[j] = (uint32_t)((long)row * ld * 2 + (x % CH) * 16);
            } else {
                const int kk = b * ROWS + (16 * lane) / (2 * W), pos = (16 * lane) % (2 * W) / 16;
                const int m = min(((pos >> 1) ^ g16::mn_swz(kk)) * 16 + (pos & 1) * 8, (rmax - r0) * P - 8);
                off[j] = (uint32_t)((long)kk * ld * 2 + m * 2);
            }
        }
    }
    // krem: k-rows of the operand from the stage's first on; one past them (T = 1) reads the last
    __device__ __forceinline__ void issue(int j, const char *base, long ld, int krem, uint32_t lds, int wave_u, int lane) const {
        uint32_t o = off[j];
        if (T == 1 && krem < BK) {
            const int kk = (wave_u * PER + j) * ROWS + (16 * lane) / (2 * W);
            if (kk >= krem) o -= (uint32_t)((long)(kk - (krem - 1)) * ld * 2);
        }
        g16::dma16(o, base, lds + (uint32_t)((wave_u * PER + j) * 1024));
    }
};

// Fragment of 16 operand rows from row r, 32 k: lane l holds row r + l%16, k 8*(l/16) .. +7. s: the k-step of a one-plane stage
// of 64 k, or the plane of a two-plane one.
template <int R, int T, int P, int BK>
__device__ __forceinline__ h8 pfrag(const char *tile, int r, int s, int lane) {
    if constexpr (T == 0) {
        return *(const h8 *)(tile + g16::koff<BK * P>(r + (lane & 15), 4 * s + (lane >> 4)));
    } else {
        const int g = lane >> 4, j = lane & 15;
        const int c = P == 2 ? (r >> 5) * 64 + s * 32 + (r & 31) : r;
        const int m = c + 4 * (j & 3), k = (P == 2 ? 0 : 32 * s) + 8 * g + (j >> 2);
        s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(tile + g16::mnoff<R * P>(k, m)));
        s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(tile + g16::mnoff<R * P>(k + 4, m)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(h8, (s8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// BM x BN tile shared by WVM x WVN waves; NS stages of BK k in LDS.
template <int BM_, int BN_, int WVM_, int WVN_, int TA_, int TB_, int PA_, int PB_, int NS_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WVM = WVM_, WVN = WVN_, TA = TA_, TB = TB_, PA = PA_, PB = PB_, NS = NS_;
    static constexpr int NW = WVM * WVN, NT = 64 * NW, WM = BM / WVM, WN = BN / WVN, FA = WM / 16, FB = WN / 16;
    static constexpr int BK = PA == 1 && PB == 1 ? 64 : 32;
    static constexpr int ABYTES = BM * BK * PA * 2, STAGE = ABYTES + BN * BK * PB * 2, SMEM = NS * STAGE;
    using FetchA = PFetch<BM, TA, PA, BK, NW>;
    using FetchB = PFetch<BN, TB, PB, BK, NW>;
    static_assert(PA >= PB, "a two-plane B takes a two-plane A");
    static_assert(SMEM <= 160 * 1024, "stages exceed the LDS");
};

struct Operand {
    const char *p;   // the array
    long ld;         // halves from a stored row to the next
    int rows;        // operand rows
    int k;           // T = 1: stored rows that exist (stages past them read the last one)
};

// acc[i][j] += the tile's products over stages kt0 .. kt0 + nk - 1. The first MFMA operand is B's fragment, so a lane ends up
// with one row m = 16 i + lane%16 of C and four neighbouring columns n = 16 j + 4 (lane/16) + r: rows leave as 16-byte stores and
// a row's statistics take two shuffles.
//
// The stage pipeline: NS buffers; the wait and barrier for stage t+1 stand before the last MFMA group of stage t, so that its
// first fragments arrive during that group, and the refill of stage t's buffer goes out between that group's MFMAs.
template <class C>
__device__ __forceinline__ void contract(const Operand &A, const Operand &B, int m0, int n0, int kt0, int nk, char *smem,
                                         floatx4 (&acc)[C::FA][C::FB]) {
    constexpr int FA = C::FA, FB = C::FB, BK = C::BK, NS = C::NS, STAGE = C::STAGE, ABYTES = C::ABYTES;
    constexpr int PERA = C::FetchA::PER, PERS = PERA + C::FetchB::PER;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wave_u = __builtin_amdgcn_readfirstlane(wave);
    const int wm0 = (wave / C::WVN) * C::WM, wn0 = (wave % C::WVN) * C::WN;
    const uint32_t lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)smem;
#pragma unroll
    for (int i = 0; i < FA; i++)
#pragma unroll
        for (int j = 0; j < FB; j++) acc[i][j] = (floatx4){};
    if (nk <= 0) return;

    typename C::FetchA fa;
    typename C::FetchB fb;
    fa.init(A.ld, m0, A.rows, wave, lane);
    fb.init(B.ld, n0, B.rows, wave, lane);
    const char *Ab = A.p + (C::TA == 0 ? (long)m0 * A.ld * 2 : (long)m0 * C::PA * 2);
    const char *Bb = B.p + (C::TB == 0 ? (long)n0 * B.ld * 2 : (long)n0 * C::PB * 2);
    auto issue_one = [&](int f, int t, int buf) {   // load f of stage t into buffer buf
        const long k = (long)(kt0 + t) * BK;
        if (f < PERA) fa.issue(f, Ab + (C::TA == 0 ? k * C::PA * 2 : k * A.ld * 2), A.ld, BK, lds + buf * STAGE, wave_u, lane);
        else fb.issue(f - PERA, Bb + (C::TB == 0 ? k * C::PB * 2 : k * B.ld * 2), B.ld, C::TB == 1 ? (int)(B.k - k) : BK,
                      lds + buf * STAGE + ABYTES, wave_u, lane);
    };
    auto fragA = [&](h8 (&v)[FA], int buf, int s) {
#pragma unroll
        for (int i = 0; i < FA; i++) v[i] = pfrag<C::BM, C::TA, C::PA, BK>(smem + buf * STAGE, wm0 + 16 * i, s, lane);
    };
    auto fragB = [&](h8 (&v)[FB], int buf, int s) {
#pragma unroll
        for (int j = 0; j < FB; j++) v[j] = pfrag<C::BN, C::TB, C::PB, BK>(smem + buf * STAGE + ABYTES, wn0 + 16 * j, s, lane);
    };
    auto mma = [&](h8 (&a)[FA], h8 (&b)[FB]) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FA; i++)
#pragma unroll
            for (int j = 0; j < FB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[j], a[i], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // the last group of stage t, with the refill of its buffer spread between the MFMAs (the tail re-fetches the last stage into
    // idle buffers, so that the number of loads in flight stays the same)
    auto mma_refill = [&](h8 (&a)[FA], h8 (&b)[FB], int t, int buf) {
        constexpr int NM = FA * FB, STEP = NM >= PERS ? NM / PERS : 1, EACH = NM >= PERS ? 1 : (PERS + NM - 1) / NM;
        const int tr = min(t + NS, nk - 1);
        __builtin_amdgcn_sched_barrier(0);
        int f = 0;
#pragma unroll
        for (int q = 0; q < NM; q++) {
            acc[q / FB][q % FB] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[q % FB], a[q / FB], acc[q / FB][q % FB], 0, 0, 0);
            if (q % STEP == STEP - 1) {
#pragma unroll
                for (int e = 0; e < EACH; e++)
                    if (f < PERS) issue_one(f++, tr, buf);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        static_assert((NM / STEP) * EACH >= PERS, "every load of the stage is issued");
        __builtin_amdgcn_sched_barrier(0);
    };
    // stage t+1 has landed (its loads are older than the NS - 2 youngest stages'), and every wave has read stage t
    auto open_next = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"((NS - 2) * PERS) : "memory");
        g16::lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    g16::lds_barrier();   // the LDS may still be read by a caller's earlier tile
#pragma unroll
    for (int p = 0; p < NS; p++)
#pragma unroll
        for (int f = 0; f < PERS; f++) issue_one(f, min(p, nk - 1), p);
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"((NS - 1) * PERS) : "memory");
    g16::lds_barrier();

    h8 a0[FA], a1[FA], b0[FB], b1[FB];
    fragA(a0, 0, 0);
    fragB(b0, 0, 0);
    // One stage. On entry a and b hold its first fragments; on exit `an` and `bn` those of the next stage.
    if constexpr (C::PB == 2) {
        auto stage = [&](int t, int buf, h8 (&a)[FA], h8 (&an)[FA]) {
            const int nbuf = buf + 1 == NS ? 0 : buf + 1;
            fragA(an, buf, 1);   // lo
            mma(a, b0);
            fragB(b1, buf, 1);   // lo
            mma(an, b0);
            open_next();
            fragA(an, nbuf, 0);
            fragB(b0, nbuf, 0);
            mma_refill(a, b1, t, buf);
        };
        int buf = 0;
        for (int t = 0; t < nk; t += 2) {
            stage(t, buf, a0, a1);
            buf = buf + 1 == NS ? 0 : buf + 1;
            if (t + 1 < nk) {
                stage(t + 1, buf, a1, a0);
                buf = buf + 1 == NS ? 0 : buf + 1;
            }
        }
    } else if constexpr (C::PA == 2) {
        auto stage = [&](int t, int buf, h8 (&b)[FB], h8 (&bn)[FB]) {
            const int nbuf = buf + 1 == NS ? 0 : buf + 1;
            fragA(a1, buf, 1);   // lo
            mma(a0, b);
            open_next();
            fragA(a0, nbuf, 0);
            fragB(bn, nbuf, 0);
            mma_refill(a1, b, t, buf);
        };
        int buf = 0;
        for (int t = 0; t < nk; t += 2) {
            stage(t, buf, b0, b1);
            buf = buf + 1 == NS ? 0 : buf + 1;
            if (t + 1 < nk) {
                stage(t + 1, buf, b1, b0);
                buf = buf + 1 == NS ? 0 : buf + 1;
            }
        }
    } else {
        int buf = 0;
        for (int t = 0; t < nk; t++) {
            const int nbuf = buf + 1 == NS ? 0 : buf + 1;
            fragA(a1, buf, 1);   // second k-step
            fragB(b1, buf, 1);
            mma(a0, b0);
            open_next();
            fragA(a0, nbuf, 0);
            fragB(b0, nbuf, 0);
            mma_refill(a1, b1, t, buf);
            buf = nbuf;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the tail's re-fetches land before the LDS is given up
}

// Runs of neighbouring tiles on one XCD (workgroups go to the XCDs in turn): workgroup L of n takes tile xcd_tile(L, n).
__device__ __forceinline__ int xcd_tile(int L, int n) {
    const int x = L & 7, i = L >> 3, q = n >> 3, r = n & 7;
    return x * q + min(x, r) + i;
}

// Tile t of the upper triangle (row <= column) of a square of n tiles a side, walked by columns.
__device__ __forceinline__ void tri_tile(int t, int &row, int &col) {
    col = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((col + 1) * (col + 2) / 2 <= t) col++;
    while (col * (col + 1) / 2 > t) col--;
    row = t - col * (col + 1) / 2;
}

}  // namespace pg
}  // namespace ah
