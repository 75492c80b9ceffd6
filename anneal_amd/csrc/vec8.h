// vec8.h — neighbouring columns of a row, eight (or four) to a lane, as it loads and stores them.
#pragma once
#include "ah_common.h"

namespace ah {

template <int N>
struct fN {
    float v[N];
};
typedef fN<8> f8;

template <class T, int N>
struct RawN;   // N values as they lie; rows may start anywhere
template <int N>
struct RawN<half_t, N> {
    typedef half_t type __attribute__((ext_vector_type(N), aligned(2)));
};
template <int N>
struct RawN<float, N> {
    typedef float type __attribute__((ext_vector_type(N), aligned(4)));
};
template <class T>
using Raw8 = RawN<T, 8>;
typedef Raw8<float>::type raw8_f32;

// Columns c .. c+N-1 (c < D) of a row of D. Those that end past D are its last N, for settle to move: one load, and no branch that waits for it
// (norms' gradients of 1999 x 1001 f32: 23.5 us, 28.2 with the last columns loaded one by one). A row of fewer than N (NARROW: there may be) has
// zeros behind its end.
template <class T, int N, bool NARROW = true>
__device__ __forceinline__ typename RawN<T, N>::type load_raw(const T *row, int c, int D) {
    typename RawN<T, N>::type x = {};
    if (!NARROW || D >= N) {
        x = *(const typename RawN<T, N>::type *)(row + min(c, D - N));
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (c + k < D) x[k] = row[c + k];
    }
    return x;
}
// What load_raw has loaded, each column in its place: zeros past the row's end.
template <class T, int N, bool NARROW = true>
__device__ __forceinline__ typename RawN<T, N>::type settle(typename RawN<T, N>::type x, int c, int D) {
    const int past = c + N - D;
    if (past > 0 && (!NARROW || D >= N)) {
        constexpr int W = N * sizeof(T) / 4;
        typedef uint32_t words __attribute__((ext_vector_type(W)));
        words u = __builtin_bit_cast(words, x);
        const int bits = sizeof(T) == 2 ? past >> 1 : past;   // whole words
#pragma unroll
        for (int s = W / 2; s >= 1; s /= 2)
#pragma unroll
            for (int k = 0; k < W; k++) u[k] = bits & s ? (k + s < W ? u[k + s < W ? k + s : 0] : 0u) : u[k];
        if (sizeof(T) == 2 && (past & 1))
#pragma unroll
            for (int k = 0; k < W; k++) u[k] = (u[k] >> 16) | (k + 1 < W ? u[k + 1 < W ? k + 1 : 0] << 16 : 0u);
        x = __builtin_bit_cast(typename RawN<T, N>::type, u);
    }
    return x;
}
template <int N, class V>
__device__ __forceinline__ fN<N> widen(V x) {
    fN<N> r;
#pragma unroll
    for (int k = 0; k < N; k++) r.v[k] = (float)x[k];
    return r;
}
template <int N>
__device__ __forceinline__ fN<N> all_of(float x) {
    fN<N> r;
#pragma unroll
    for (int k = 0; k < N; k++) r.v[k] = x;
    return r;
}
// Nothing is stored past D.
template <class T, int N>
__device__ __forceinline__ void store_cols(T *row, int c, int D, const fN<N> &v) {
    typename RawN<T, N>::type x;
#pragma unroll
    for (int k = 0; k < N; k++) x[k] = (T)v.v[k];
    if (c + N <= D) {
        *(typename RawN<T, N>::type *)(row + c) = x;
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (c + k < D) row[c + k] = x[k];
    }
}

template <class T>
__device__ __forceinline__ f8 load8(const T *row, int c, int D) {
    return widen<8>(settle<T, 8>(load_raw<T, 8>(row, c, D), c, D));
}
template <class T>
__device__ __forceinline__ void store8(T *row, int c, int D, const f8 &v) {
    store_cols<T, 8>(row, c, D, v);
}

}  // namespace ah
