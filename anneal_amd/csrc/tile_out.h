// tile_out.h — the way of a product tile's accumulators to memory: through LDS, so that a lane has eight neighbouring columns of a row.
//
// A lane of the product (plane_gemm.h) holds four columns of one row, 16 rows a wave: 8-byte accesses in f16, in 32-byte pieces of 16
// rows. Each wave turns 16 rows at a time over in LDS of its own, padded by 16 bytes a row (no bank is met twice by the eight lanes that
// store or load together): then 4 to 16 lanes share a row's 16-byte accesses.
#pragma once
#include "plane_gemm.h"
#include "vec8.h"

namespace ah {

// Columns c .. c+7 of a row of D, zeros past its end. (The last columns one by one: in flight together with others, as here, they cost less than
// moving them as vec8.h does, 31.0 against 32.5 us at 777 x 1001 -> 2003.)
template <class T>
__device__ __forceinline__ typename Raw8<T>::type load_raw8(const T *row, int c, int D) {
    typename Raw8<T>::type x = {};
    if (c + 8 <= D) {
        x = *(const typename Raw8<T>::type *)(row + c);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (c + k < D) x[k] = row[c + k];
    }
    return x;
}

// The two planes of eight values at p (hi) and p + 32 (lo), or one.
template <int P>
__device__ __forceinline__ void plane_store8(half_t *p, const f8 &v) {
    pg::h8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        hi[k] = (half_t)v.v[k];
        lo[k] = (half_t)(v.v[k] - (float)hi[k]);
    }
    *(pg::h8 *)p = hi;
    if constexpr (P == 2) *(pg::h8 *)(p + 32) = lo;
}

template <class C>
constexpr int tile_out_bytes() {
    return C::NT / 64 * 16 * (C::WN + 4) * 4;
}

// Where a wave's 16 rows of accumulator row i go. Lane's part p of kParts: row m + p * kStep, columns n .. n+7.
template <class C>
struct TileOut {
    static constexpr int LANES = C::WN / 8, kStep = 64 / LANES, kParts = 16 / kStep;   // lanes a row
    char *base;
    int m, n, lane;
    __device__ __forceinline__ TileOut(char *smem, int m0, int n0, int i) {
        const int wave = threadIdx.x >> 6;
        lane = threadIdx.x & 63;
        base = smem + wave * 16 * (C::WN + 4) * 4;
        m = m0 + wave / C::WVN * C::WM + 16 * i + lane / LANES;
        n = n0 + wave % C::WVN * C::WN + lane % LANES * 8;
    }
    // Wave-wide: a wave's LDS accesses keep their order; the fences keep the compiler from moving them across.
    __device__ __forceinline__ void put(const floatx4 (&acc)[C::FB]) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
        for (int j = 0; j < C::FB; j++) *(floatx4 *)(base + (lane & 15) * (C::WN + 4) * 4 + (16 * j + 4 * (lane >> 4)) * 4) = acc[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    }
    __device__ __forceinline__ f8 get(int p) const {
        f8 r;
        const char *q = base + (lane / LANES + p * kStep) * (C::WN + 4) * 4 + lane % LANES * 32;
        const floatx4 a = *(const floatx4 *)q, b = *(const floatx4 *)(q + 16);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            r.v[k] = a[k];
            r.v[k + 4] = b[k];
        }
        return r;
    }
};

}  // namespace ah
