// plane_gemm.h — contractions of matrices held as one or two f16 planes, for the operators whose products must keep more
// than f16's 11 bits or whose epilogue is their own (linear_ce.hip, muon.hip).
//
//   C[m,n] = epi( sum_k A(m,k) B(n,k) )
//
// An f32 matrix x is carried as hi = f16(2^s x), lo = f16(2^s x - hi): 22 bits of each value whose magnitude is within 2^14 of
// 2^15, with an absolute floor of 2^-24 (an f16 subnormal) below that. A product of two such matrices is three f16 products,
// hi*hi + lo*hi + hi*lo (lo*lo, at most 2^-22 of the product, is left out: as much as the operands' own planes lose, and shows in sums as
// short as muon_small.hip has them alone), accumulated in one f32 accumulator; every f16 product is exact
// in f32. Three f16 MFMAs do the work of one f32 MFMA of the same shape in 3/16 of its time.
//
// Layout of a two-plane matrix: each stored row holds groups of 32 hi values and then their 32 lo values (128 bytes, one cache
// line). To the staging code it is an f16 matrix of twice the width, so both planes of a tile arrive with the one set of
// global->LDS loads, and a stage of 32 k in two planes has the LDS image of a stage of 64 k in one.
//   T = 0: rows of the operand are stored rows, k runs along them;  T = 1: stored rows are k, the operand's rows run along them.
// Matrices that only these kernels read are stored in panels of 128-byte columns: all rows' first 128 bytes, then all rows' next.
// A stage of 256 rows is then one run of 32 KiB, whatever the matrix's width.
//
// Per stage a wave reads each fragment once: hi*hi and lo*hi share B's hi, hi*hi and hi*lo share A's hi. So two planes take 2/3
// of the LDS reads per MFMA that one plane takes, and a 256x256 tile of 8 waves is bound by MFMA issue, not by LDS.
#pragma once
#include <algorithm>

#include "ah_common.h"
#include "gemm16_kernel.h"

namespace ah {
namespace pg {

using g16::h8;
using g16::lds_s4;
using g16::s4;

typedef half_t h4 __attribute__((ext_vector_type(4)));
// The same vectors where nothing but their elements' alignment is known: callers' rows. (Such an access costs no more than the
// cache lines that it touches; element by element, the product that ends in a 32003 x 1001 f16 gradient took 84 us, not 50.)
typedef half_t h4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef half_t h8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));

// Four values at column c of a row of `cols`: zeros past its end, nothing stored there.
template <class T>
struct Any4;
template <>
struct Any4<float> {
    typedef f4_any type;
};
template <>
struct Any4<half_t> {
    typedef h4_any type;
};
template <class T>
__device__ __forceinline__ floatx4 load4(const T *row, int c, int cols) {
    floatx4 v = {};
    if (c + 3 < cols) {
        const typename Any4<T>::type x = *(const typename Any4<T>::type *)(row + c);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (float)x[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (c + k < cols) v[k] = (float)row[c + k];
    }
    return v;
}
template <class T>
__device__ __forceinline__ void store4(T *row, int c, int cols, floatx4 v) {
    if (c + 3 < cols) {
        typename Any4<T>::type x;
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = (T)v[k];
        *(typename Any4<T>::type *)(row + c) = x;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (c + k < cols) row[c + k] = (T)v[k];
    }
}

// Halves from the start of a matrix of P planes in panels of `rows` rows to the (hi) value of row r, column c (lo: 32 further).
template <int P>
__host__ __device__ __forceinline__ long panel_at(long rows, long r, long c) {
    return P == 1 ? ((c >> 6) * rows + r) * 64 + (c & 63) : ((c >> 5) * rows + r) * 64 + (c & 31);
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
    __device__ __forceinline__ void init(long ld, long ps, int r0, int rmax, int wave, int lane) {
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
                off[j] = (uint32_t)((long)kk * ld * 2 + (m >> 6) * ps + (m & 63) * 2);
            }
        }
    }
    // krem: k of the operand from the stage's first on. Past them T = 1 reads the last k-row and T = 0 the stage's first chunk of the
    // row (krem is then a multiple of a chunk's 8): the other operand is 0 there, and nothing behind the array is read.
    __device__ __forceinline__ void issue(int j, const char *base, long ld, int krem, uint32_t lds, int wave_u, int lane) const {
        uint32_t o = off[j];
        if (krem < BK) {
            if constexpr (T == 1) {
                const int kk = (wave_u * PER + j) * ROWS + (16 * lane) / (2 * W);
                if (kk >= krem) o -= (uint32_t)((long)(kk - (krem - 1)) * ld * 2);
            } else if constexpr (P == 1) {
                const int q = 4 * (wave_u * PER + j) + (lane >> 4), c = ((lane & 15) ^ (q & 15)) % (W / 8);
                if (c * 8 >= krem) o -= (uint32_t)(c * 16);
            }
        }
        g16::dma16(o, base, lds + (uint32_t)((wave_u * PER + j) * 1024));
    }
};

// Fragments of 16 operand rows and 32 k: lane l holds row l%16, k 8*(l/16) .. +7. s: the k-step of a one-plane stage of 64 k, or
// the plane of a two-plane one. A fragment's LDS address is the wave's first one with a constant xored into bits 5 to 7 (the
// swizzle) and a constant added, so one register per operand addresses all of them; a stage's base is added per stage.
template <int R, int T, int P, int BK>
struct PFrag {
    static constexpr int W = T == 0 ? BK * P : R * P;
    static_assert(T == 1 || W == 64, "stored rows of 128 bytes");
    uint32_t first;
    __device__ __forceinline__ void init(uint32_t lds, int r, int lane) {   // lds: of the operand in buffer 0; r: the wave's first row
        const int g = lane >> 4, j = lane & 15;
        if constexpr (T == 0) first = lds + g16::koff<W>(r + j, g);
        else first = lds + g16::mnoff<W>(8 * g + (j >> 2), r * P + 4 * (j & 3));
    }
    // fragment i; stage = first + the buffer's offset, opaque to the compiler, which would otherwise keep every address it finds
    static __device__ __forceinline__ h8 read(uint32_t stage, int i, int s) {
        typedef const __attribute__((address_space(3))) char *ptr;
        if constexpr (T == 0) {
            return *(const __attribute__((address_space(3))) h8 *)((ptr)(stage ^ (uint32_t)(((i & 1) << 7) | (s << 6))) + 2048 * i);
        } else {
            // 16-column segments: a plane's 32 columns are two, the planes of 32 columns four
            const int seg = P == 2 ? (i >> 1) * 4 + s * 2 + (i & 1) : i, k = P == 2 ? 0 : 32 * s;
            const ptr p = (ptr)(stage ^ (uint32_t)((seg & 7) << 5)) + (seg >> 3) * 256 + k * (W * 2);
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 4 * (W * 2)));
            typedef short s8 __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(h8, (s8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// BM x BN tile shared by WVM x WVN waves; NS stages of BK k in LDS.
template <int BM_, int BN_, int WVM_, int WVN_, int TA_, int TB_, int PA_, int PB_, int NS_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WVM = WVM_, WVN = WVN_, TA = TA_, TB = TB_, PA = PA_, PB = PB_, NS = NS_;
    static constexpr int NW = WVM * WVN, NT = 64 * NW, WM = BM / WVM, WN = BN / WVN, FA = WM / 16, FB = WN / 16;
    static constexpr int BK = PA == 1 && PB == 1 ? 64 : 32;
    static constexpr int ABYTES = BM * BK * PA * 2, STAGE = ABYTES + BN * BK * PB * 2, SMEM = NS * STAGE;
    using FetchA = PFetch<BM, TA, PA, BK, NW>;
    using FetchB = PFetch<BN, TB, PB, BK, NW>;
    using FragA = PFrag<BM, TA, PA, BK>;
    using FragB = PFrag<BN, TB, PB, BK>;
    static_assert((TA == 0 || WM * PA == 64 || WM * PA % 128 == 0) && (TB == 0 || WN * PB == 64 || WN * PB % 128 == 0),
                  "a fragment's segment is the wave's first one xor a constant");
    static_assert(PA >= PB, "a two-plane B takes a two-plane A");
    static_assert(SMEM <= 160 * 1024, "stages exceed the LDS");
};

struct Operand {
    const char *p;   // the array
    long ld;         // halves from a stored row to the next
    long ps;         // bytes from 64 halves of a row to the next 64
    int rows;        // operand rows
    int k;           // k that there are (B's may end inside a stage: PFetch::issue)
    // B of contract<C, true>: stored rows come in blocks of 2^shift, a multiple of a tile's and a stage's, each `block` bytes on with panels of its own
    int shift = 31;
    long block = 0;
};

// A lane's offset from its tile's corner is 32 bits wide and spans up to 8 panels (T = 1: 256 operand rows of two planes), so panels may
// not be further apart than this many stored rows; more of them go in blocks.
constexpr int kMaxPanelRows = 1 << 22;
static_assert(7l * kMaxPanelRows * 128 + 64 * 128 < 1l << 32, "the last panel's rows are in reach");

// `stored` rows in panels; rows of the operand, k as above.
inline Operand panels(const void *p, long stored, int rows, int k) { return {(const char *)p, 64, stored * 128, rows, k}; }
// Rows one after the other.
inline Operand row_major(const void *p, long ld, int rows, int k) { return {(const char *)p, ld, 128, rows, k}; }

// acc[i][j] += the tile's products over stages kt0 .. kt0 + nk - 1. The first MFMA operand is B's fragment, so a lane ends up
// with one row m = 16 i + lane%16 of C and four neighbouring columns n = 16 j + 4 (lane/16) + r: rows leave as 16-byte stores and
// a row's statistics take two shuffles.
//
// The stage pipeline: NS buffers; the wait and barrier for stage t+1 stand before the last MFMA group of stage t, so that its
// first fragments arrive during that group, and the refill of stage t's buffer goes out between that group's MFMAs.
// BLOCKS: B's stored rows may lie in blocks (always reckoned with, it costs the orthogonalisation of 4096 x 1024 2%).
template <class C, bool BLOCKS = false>
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
    // a tile's rows start a multiple of 64 halves into a stored row (T = 1), and a stage of k fills 64 halves (T = 0)
    static_assert(C::TA == 1 || BK * C::PA == 64, "a stage of A is one panel");
    static_assert(C::TB == 1 || BK * C::PB == 64, "a stage of B is one panel");
    fa.init(A.ld, A.ps, m0, A.rows, wave, lane);
    fb.init(B.ld, B.ps, n0, B.rows, wave, lane);
    const char *Ab = A.p + (C::TA == 0 ? (long)m0 * A.ld * 2 : (long)(m0 * C::PA / 64) * A.ps);
    const auto stored = [&](int r) {   // B's row r
        return BLOCKS ? (long)(r >> B.shift) * B.block + (long)(r & (int)((1u << B.shift) - 1)) * B.ld * 2 : (long)r * B.ld * 2;
    };
    const char *Bb = B.p + (C::TB == 0 ? stored(n0) : (long)(n0 * C::PB / 64) * B.ps);
    const long da = C::TA == 0 ? A.ps : (long)BK * A.ld * 2, db = C::TB == 0 ? B.ps : (long)BK * B.ld * 2;   // bytes a stage
    auto issue_one = [&](int f, int t, int buf) {   // load f of stage t into buffer buf
        if (f < PERA) fa.issue(f, Ab + (kt0 + t) * da, A.ld, BK, lds + buf * STAGE, wave_u, lane);
        else fb.issue(f - PERA, Bb + (BLOCKS && C::TB == 1 ? stored((kt0 + t) * BK) : (kt0 + t) * db), B.ld, C::TB == 1 || C::PB == 1 ? B.k - (kt0 + t) * BK : BK, lds + buf * STAGE + ABYTES, wave_u, lane);
    };
    typename C::FragA ra;
    typename C::FragB rb;
    ra.init(lds, wm0, lane);
    rb.init(lds + ABYTES, wn0, lane);
    auto fragA = [&](h8 (&v)[FA], int buf, int s) {
        uint32_t at = ra.first + buf * STAGE;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int i = 0; i < FA; i++) v[i] = C::FragA::read(at, i, s);
    };
    auto fragB = [&](h8 (&v)[FB], int buf, int s) {
        uint32_t at = rb.first + buf * STAGE;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int j = 0; j < FB; j++) v[j] = C::FragB::read(at, j, s);
    };
    // a group of MFMAs, with the NR LDS reads that stand before it spread between them
    auto mma = [&](h8 (&a)[FA], h8 (&b)[FB], auto nr) {
        constexpr int NM = FA * FB, NR = decltype(nr)::value, PER = NM >= NR ? NM / NR : 1, EACH = NM >= NR ? 1 : (NR + NM - 1) / NM;
#pragma unroll
        for (int i = 0; i < FA; i++)
#pragma unroll
            for (int j = 0; j < FB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[j], a[i], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < NR / EACH; q++) {
            __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);    // MFMAs
            __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);   // LDS reads
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, FA *(C::TA ? 2 : 1)> NRA{};                                // LDS reads of A's fragments,
    constexpr std::integral_constant<int, FB *(C::TB ? 2 : 1)> NRB{};                                // of B's,
    constexpr std::integral_constant<int, decltype(NRA)::value + decltype(NRB)::value> NRAB{};       // of both
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
            mma(a, b0, NRA);
            fragB(b1, buf, 1);   // lo
            mma(an, b0, NRB);
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
            mma(a0, b, NRA);
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
            mma(a0, b0, NRAB);
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

// Tile t of tiles_m x tiles_n: rows in groups of 4, walked by columns within a group, so that the tiles at work on one XCD
// share operand panels in its L2.
__device__ __forceinline__ void grouped_tile(int t, int tiles_m, int tiles_n, int &row, int &col) {
    const int g = t / (4 * tiles_n) * 4, rem = t - g * tiles_n, size = min(4, tiles_m - g);
    row = g + rem % size;
    col = rem / size;
}

// Tile t of the upper triangle (row <= column) of a square of n tiles a side: rows in groups of 4, walked by columns within a
// group, as above.
__device__ __forceinline__ void tri_tile(int t, int n, int &row, int &col) {
    int g = 0;
    for (;; g += 4) {   // a group's four rows hold n - g, n - g - 1, ... tiles
        const int rows = min(4, n - g), count = rows * (n - g) - rows * (rows - 1) / 2;
        if (t < count) break;
        t -= count;
    }
    const int rows = min(4, n - g);
    // the columns of the group's corner hold 1, 2, .. tiles, the others `rows`
    int c = 0;
    while (c < rows - 1 && t > c) t -= ++c;
    if (c == rows - 1) {
        c += t / rows;
        t %= rows;
    }
    row = g + t;
    col = g + c;
}

// ── tiles, and K split over workgroups ─────────────────────────────────────────
// Tiles are worked on in rounds of as many as the chip takes at once. What does not fill a round (all of them, where there are few)
// is split over K: `splits` workgroups share a tile's stages and leave their accumulators in the workspace, and a second kernel
// adds them in order (results repeat bit for bit) and runs the epilogue, one workgroup for each 16 rows of a tile's waves.
struct Work {
    int whole, rest, splits;   // tiles 0 .. whole-1 in one piece each, then `rest` tiles of `splits` pieces
    float *part;               // [split][rest] partial tiles
    __host__ __device__ int tiles() const { return whole + rest; }
    __host__ __device__ int blocks() const { return whole + rest * splits; }
};

// Workgroup b's tile and its stages [first, first + count) of nk; slot: where its partial sums go, -1 for a whole tile.
__device__ __forceinline__ void pick(const Work &w, int b, int nk, int &tile, int &slot, int &first, int &count) {
    slot = -1;
    first = 0;
    count = nk;
    if (b < w.whole) {
        tile = xcd_tile(b, w.whole);
        return;
    }
    const int r = xcd_tile(b - w.whole, w.rest * w.splits), split = r / w.rest;
    tile = w.whole + r - split * w.rest;
    if (w.splits == 1) return;
    const int q = (nk + w.splits - 1) / w.splits;
    first = min(nk, split * q);
    count = min(nk, first + q) - first;
    slot = r;
}

// `tiles` tiles of nk stages on a chip that takes `slots` at once, with room for `cap` partial tiles: how a kernel deals out work whose
// size the host did not know. Costs in stages: three for a round's start and end, `join` for a partial tile's way to memory and back.
__device__ __forceinline__ Work deal(int tiles, int nk, int slots, int cap, float join, float *part) {
    int best = 1;
    float best_cost = 1e30f;
    for (int s = 1; s <= 16 && (s == 1 || (tiles * s <= cap && nk >= 2 * s)); s++) {
        const float cost = (float)((tiles * s + slots - 1) / slots * ((nk + s - 1) / s + 3)) + (s > 1 ? 4.0f + join * (float)(tiles * s) : 0.0f);
        if (cost < best_cost) {
            best_cost = cost;
            best = s;
        }
    }
    return best == 1 ? Work{tiles, 0, 1, part} : Work{0, tiles, best, part};
}

// Partial sums of accumulator row i: [slot][i][j][thread] of four floats.
template <class C>
__device__ __forceinline__ floatx4 *partial(float *part, long slot, int i) {
    return (floatx4 *)part + (slot * C::FA + i) * C::FB * C::NT + threadIdx.x;
}
template <class C>
__device__ __forceinline__ void store_partials(float *part, long slot, const floatx4 (&acc)[C::FA][C::FB]) {
#pragma unroll
    for (int i = 0; i < C::FA; i++)
#pragma unroll
        for (int j = 0; j < C::FB; j++) partial<C>(part, slot, i)[j * C::NT] = acc[i][j];
}
template <class C>
__device__ __forceinline__ void sum_partials(const Work &w, int r, int i, floatx4 (&v)[C::FB]) {
#pragma unroll
    for (int j = 0; j < C::FB; j++) v[j] = (floatx4){};
    constexpr int B = C::FB == 8 ? 4 : 8;   // splits whose loads are in flight together
    for (int s = 0; s < w.splits; s += B) {
        floatx4 x[B][C::FB];
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int j = 0; j < C::FB; j++)
                x[b][j] = s + b < w.splits ? partial<C>(w.part, (long)(s + b) * w.rest + r, i)[j * C::NT] : (floatx4){};
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int j = 0; j < C::FB; j++) v[j] += x[b][j];
    }
}

// A wave's place in a tile: the row of C that this lane holds of accumulator row 0, and its first column.
template <class C>
struct Place {
    int m, n, lane, wave;
    // Opaque, so that an epilogue that runs row after row forms its addresses anew for each: kept for all rows, they spill.
    __device__ __forceinline__ Place(int m0, int n0) {
        lane = threadIdx.x & 63;
        wave = threadIdx.x >> 6;
        m = m0 + (wave / C::WVN) * C::WM + (lane & 15);
        n = n0 + (wave % C::WVN) * C::WN + 4 * (lane >> 4);
        asm volatile("" : "+v"(m), "+v"(n));
    }
};

// Tile width and splits of a product, by a model of the time it takes.
struct Plan {
    int width;   // of the tiles: 256 (8 waves, one workgroup a CU), 128 (4 waves, two a CU) or 64 (4 waves, two a CU, four stages)
    Work w;
    double us;
    long part_bytes() const { return w.splits > 1 ? (long)w.rest * w.splits * width * width * 4 : 0; }
};
template <int TA, int TB, int PA, int PB>
using Tile256 = Tile<256, 256, 4, 2, TA, TB, PA, PB, 2>;
template <int TA, int TB, int PA, int PB>
using Tile128 = Tile<128, 128, 2, 2, TA, TB, PA, PB, 2>;
template <int TA, int TB, int PA, int PB>
using Tile64 = Tile<64, 64, 2, 2, TA, TB, PA, PB, 4>;

// tiles(width): number of tiles at a width; k: the summed length; pa, pb: planes; narrow: 64-wide tiles may be taken. Microseconds
// a stage of the tile loops on this chip, measured over k = 1024 to 4096 with operands in panels (a stage is 64 k of one plane, 32
// of two), by workgroups:
//                  256 wide: 32 / 256      128 wide: to 256 / 512      64 wide: to 256 / 512
//   planes 1 x 1      1.28 / 1.77             0.72 / 1.15                 0.22 / 0.36
//   planes 2 x 1      1.23 / 1.58             0.61 / 0.97                   -
//   planes 2 x 2      1.62 / 2.30             0.68 / 1.33                 0.26 / 0.41
// (many CUs at once run slower than few: the clock gives way). Splitting adds a launch and the partial sums' way to memory and
// back; no piece is longer than `piece`. 1024 x 1024 over k = 1024 in two planes, measured: 15 us in 256 tiles of 64, 24 in 64 of 128.
template <class Tiles>
Plan plan(Tiles tiles, long k, int pa, int pb, bool narrow, long piece = 1l << 40) {
    const int row = pa == 1 ? 0 : pb == 1 ? 1 : 2;
    constexpr double kFew[3] = {1.22, 1.18, 1.53}, kMore[3] = {0.55, 0.40, 0.77};
    constexpr double k128[3][2] = {{0.72, 1.15}, {0.61, 0.97}, {0.68, 1.33}}, k64[2][2] = {{0.22, 0.36}, {0.26, 0.41}};
    const long nk = (k + (row == 0 ? 63 : 31)) / (row == 0 ? 64 : 32);
    Plan best{};
    double best_us = 1e30;
    for (const int width : {256, 128, 64}) {
        if (width == 64 && !narrow) break;
        const long n = tiles(width), slots = width == 256 ? 256 : 512;
        const auto stage = [&](long wg) {
            return width == 256 ? kFew[row] + kMore[row] * (double)wg / 256 : width == 128 ? k128[row][wg > 256] : k64[row / 2][wg > 256];   // (not with planes 2 x 1)
        };
        const double fixed = width == 256 ? 7.0 : 5.0;   // launch, first loads, the epilogue
        const long least = (nk * (row == 0 ? 64 : 32) + piece - 1) / piece;
        const long rest = least > 1 ? n : n % slots, rounds = least > 1 ? 0 : n / slots;
        for (long s = std::max(1l, least); s <= std::max(32l, least) && (s <= least || (rest * s <= 4 * slots && nk >= 2 * s)); s++) {
            const double joined = (double)rest * s * width * width * 8 / 4e6;   // us at 4 TB/s
            const long turns = (rest * s + slots - 1) / slots;
            const double us = rounds * (nk * stage(slots) + fixed) + turns * ((double)((nk + s - 1) / s) * stage(std::min(slots, rest * s)) + fixed) +
                              (s > 1 ? 4.0 + joined : 0);
            if (us < best_us) {
                best_us = us;
                best.us = us;
                best.width = width;
                best.w = s == 1 ? Work{(int)n, 0, 1, nullptr} : Work{(int)(rounds * slots), (int)rest, (int)s, nullptr};
            }
            if (!rest) break;
        }
    }
    return best;
}

}  // namespace pg
}  // namespace ah
