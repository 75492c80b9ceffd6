// clip.hip — the global norm of many tensors, and clipping by it.
//
//   norm = unscale sqrt(sum g^2);  c = min(1, max_norm / (norm + eps));  dst = unscale c src
//
// Two launches, whatever the tensors: one leaves a sum of squares a workgroup, one joins those (every workgroup for itself, in the same
// order: 16 KB from the L2) and scales. Tensors are cut into chunks of 2048 elements that are numbered through; a workgroup takes a run of
// neighbouring chunks, so it looks for its first tensor once (a binary search) and then walks on. The table of tensors travels with the
// launch where it fits there, else small launches lay it down in the workspace first: no host memory has to outlive the call, and
// a graph holds the table itself. The second launch goes through a workgroup's run from its end, which the first has left in the caches.
//
// Bound by memory: every entry is read twice and written once (354 million f32: 823 us, 5.2 TB/s). Squares go to f64 at once (f32 squares of entries under 2^-63 would vanish
// and of those over 2^64 be infinite); squares of f16 are exact in f32 and are summed there eight at a time.
#include "clip.h"

#include <algorithm>

#include "ah_common.h"

namespace ah {
namespace {

constexpr long kChunk = 2048;    // elements
constexpr int kBlocks = 2048;    // workgroups, at most
constexpr int kInline = 90;      // tensors whose table travels with a launch (4 KB of arguments)

struct Entry {
    const void *src;
    void *dst;
    long count;
    long first;      // chunks before it
    int half, half_out;
};
struct Args {
    const Entry *table;
    int n, blocks;
    long chunks;
    double *part;    // [blocks]
    float max_norm, eps, unscale;
    float *norm, *coef;
};
struct Inline {
    Entry e[kInline];
};
static_assert(sizeof(Args) + sizeof(Inline) <= 4096, "the arguments of a launch");

int64_t chunks_of(int64_t count) { return (count + kChunk - 1) / kChunk; }

// f(entry, from, to) for each stretch of a tensor among this workgroup's chunks, from the first to the last or (BACK) the other way; at(i):
// entry i.
template <bool BACK, class At, class F>
__device__ __forceinline__ void walk(const Args &a, At at, F f) {
    const long begin = a.chunks * blockIdx.x / a.blocks, end = a.chunks * (blockIdx.x + 1) / a.blocks;
    if (begin >= end) return;
    long c = BACK ? end - 1 : begin;
    int t = 0;
    for (int hi = a.n - 1; t < hi;) {   // the last tensor that starts at or before c (empty ones start where the next does)
        const int mid = (t + hi + 1) / 2;
        if (at(mid).first <= c) t = mid;
        else hi = mid - 1;
    }
    if constexpr (BACK) {
        for (c = end; c > begin; t--) {
            const Entry e = at(t);
            const long start = max(begin, e.first);
            f(e, (start - e.first) * kChunk, min(e.count, (c - e.first) * kChunk));
            c = start;
        }
    } else {
        for (; c < end; t++) {
            const Entry e = at(t);
            const long stop = min(end, e.first + (e.count + kChunk - 1) / kChunk);
            f(e, (c - e.first) * kChunk, min(e.count, (stop - e.first) * kChunk));
            c = stop;
        }
    }
}

template <class T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));   // tensors may start anywhere
};

template <class T>
__device__ __forceinline__ double squares(typename Vec<T>::type v) {
    if constexpr (sizeof(T) == 2) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < Vec<T>::N; k++) s = fmaf((float)v[k], (float)v[k], s);
        return (double)s;
    } else {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < Vec<T>::N; k++) s = fma((double)v[k], (double)v[k], s);
        return s;
    }
}

constexpr int kAhead = 4;   // 16-byte loads a thread has in flight

template <class T>
__device__ __forceinline__ double sum_squares(const T *p, long from, long to) {
    typedef Vec<T> V;
    double s[kAhead] = {};
    long i = from + threadIdx.x * V::N;
    for (; i - threadIdx.x * V::N + 256 * V::N * kAhead <= to; i += 256 * V::N * kAhead) {
        typename V::type v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u] = *(const typename V::type *)(p + i + u * 256 * V::N);
#pragma unroll
        for (int u = 0; u < kAhead; u++) s[u] += squares<T>(v[u]);
    }
    for (; i < to; i += 256 * V::N) {
        if (i + V::N <= to) {
            s[0] += squares<T>(*(const typename V::type *)(p + i));
        } else {
            for (long k = i; k < to; k++) s[0] += (double)p[k] * (double)p[k];
        }
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// The sum over 256 threads, in every one of them.
__device__ __forceinline__ double block_sum(double s) {
    __shared__ double red[4];
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class At>
__device__ __forceinline__ void norm_part(const Args &a, At at) {
    double s = 0.0;
    walk<false>(a, at, [&](const Entry &e, long from, long to) {
        s += e.half ? sum_squares((const half_t *)e.src, from, to) : sum_squares((const float *)e.src, from, to);
    });
    s = block_sum(s);
    if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

// A value times unscale c, which is an f32 but where a norm near f32's end makes it less than f32's normal numbers: products in f64 have all of
// f32's bits then.
struct Single {
    float f;
    __device__ __forceinline__ float of(float v) const { return v * f; }
};
struct Double {
    double f;
    __device__ __forceinline__ float of(float v) const { return (float)((double)v * f); }
};
struct Zero {   // what is not finite is 0 too
    __device__ __forceinline__ float of(float) const { return 0.0f; }
};

template <class T, class O, class Factor>
__device__ __forceinline__ void scale_range(const T *p, O *q, long from, long to, Factor f) {
    typedef Vec<T> V;
    typedef O out __attribute__((ext_vector_type(V::N), aligned(sizeof(O))));
    const auto put = [&](long i, typename V::type v) {
        out o;
#pragma unroll
        for (int k = 0; k < V::N; k++) o[k] = (O)f.of((float)v[k]);
        *(out *)(q + i) = o;
    };
    constexpr long step = 256 * V::N * kAhead;
    const long whole = (to - from) / step;
    for (long i = from + whole * step + threadIdx.x * V::N; i < to; i += 256 * V::N) {
        if (i + V::N <= to) {
            put(i, *(const typename V::type *)(p + i));
        } else {
            for (long k = i; k < to; k++) q[k] = (O)f.of((float)p[k]);
        }
    }
    for (long s = whole - 1; s >= 0; s--) {
        const long i = from + s * step + threadIdx.x * V::N;
        typename V::type v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u] = *(const typename V::type *)(p + i + u * 256 * V::N);
#pragma unroll
        for (int u = 0; u < kAhead; u++) put(i + u * 256 * V::N, v[u]);
    }
}

template <class At>
__device__ __forceinline__ void scale_part(const Args &a, At at) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kBlocks; k += 256) s += k + (int)threadIdx.x < a.blocks ? a.part[k + threadIdx.x] : 0.0;
    s = block_sum(s);
    const double norm = (double)a.unscale * sqrt(s), under = norm + (double)a.eps;
    const bool bad = !(s < __builtin_inf());
    const double c = bad ? 0.0 : (double)a.max_norm < under ? (double)a.max_norm / under : 1.0;
    const double f = c * (double)a.unscale;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (a.norm) *a.norm = (float)norm;
        if (a.coef) *a.coef = (float)c;
    }
    const auto scale = [&](auto factor, bool one) {
        walk<true>(a, at, [&](const Entry &e, long from, long to) {
            if (!e.dst || (e.dst == e.src && one)) return;
            if (!e.half) scale_range((const float *)e.src, (float *)e.dst, from, to, factor);
            else if (e.half_out) scale_range((const half_t *)e.src, (half_t *)e.dst, from, to, factor);
            else scale_range((const half_t *)e.src, (float *)e.dst, from, to, factor);
        });
    };
    if (bad) scale(Zero{}, false);
    else if (f < 0x1p-126) scale(Double{f}, false);
    else scale(Single{(float)f}, (float)f == 1.0f);
}

__global__ __launch_bounds__(256) void clip_norm_kernel(Args a) {
    norm_part(a, [&](int i) { return a.table[i]; });
}
__global__ __launch_bounds__(256) void clip_norm_inline_kernel(Args a, Inline t) {
    norm_part(a, [&](int i) { return t.e[i]; });
}
__global__ __launch_bounds__(256) void clip_scale_kernel(Args a) {
    scale_part(a, [&](int i) { return a.table[i]; });
}
__global__ __launch_bounds__(256) void clip_scale_inline_kernel(Args a, Inline t) {
    scale_part(a, [&](int i) { return t.e[i]; });
}

__global__ __launch_bounds__(128) void clip_table_kernel(Inline t, int n, Entry *table) {
    if ((int)threadIdx.x < n) table[threadIdx.x] = t.e[threadIdx.x];
}

constexpr int64_t kPartBytes = kBlocks * sizeof(double);

}  // namespace

int64_t clip_workspace(const ah_clip_desc &d) { return kPartBytes + (d.n > kInline ? (int64_t)d.n * sizeof(Entry) : 0); }

hipError_t clip_norm(const ah_clip_desc &d, hipStream_t s) {
    Args a{};
    Inline t{};
    a.table = (const Entry *)((char *)d.ws + kPartBytes);
    a.n = d.n;
    a.part = (double *)d.ws;
    a.max_norm = d.max_norm;
    a.eps = d.eps;
    a.unscale = d.unscale;
    a.norm = d.norm;
    a.coef = d.coef;
    for (int i = 0; i < d.n; i++) {
        const ah_tensor &v = d.tensors[i];
        t.e[i % kInline] = {v.src, v.dst, (long)v.count, a.chunks, v.dtype == AH_F16, v.out_dtype == AH_F16};
        a.chunks += chunks_of(v.count);
        if (d.n > kInline && (i % kInline == kInline - 1 || i == d.n - 1))
            hipLaunchKernelGGL(clip_table_kernel, dim3(1), dim3(128), 0, s, t, i % kInline + 1, (Entry *)a.table + i / kInline * kInline);
    }
    a.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(a.chunks, kBlocks));
    bool scaled = d.norm || d.coef;
    for (int i = 0; i < d.n && !scaled; i++) scaled = d.tensors[i].dst != nullptr;
    if (d.n > kInline) {
        hipLaunchKernelGGL(clip_norm_kernel, dim3((unsigned)a.blocks), dim3(256), 0, s, a);
        if (scaled) hipLaunchKernelGGL(clip_scale_kernel, dim3((unsigned)a.blocks), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL(clip_norm_inline_kernel, dim3((unsigned)a.blocks), dim3(256), 0, s, a, t);
        if (scaled) hipLaunchKernelGGL(clip_scale_inline_kernel, dim3((unsigned)a.blocks), dim3(256), 0, s, a, t);
    }
    return hipGetLastError();
}

}  // namespace ah
