// lm_args.h — argument checks that the C entries of the language model's operators share (lmops.cpp, blockops.cpp).
#pragma once
#include "ah_internal.h"

namespace ah {

// Makes the handle's device current for the launches of a call, and the caller's again after it.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const ah_device *d) {
        if (hipGetDevice(&before) != hipSuccess || before == d->ordinal) before = -1;
        else hipSetDevice(d->ordinal);
    }
    ~OnDevice() {
        if (before >= 0) hipSetDevice(before);
    }
};

constexpr int64_t kMaxSide = 1 << 20, kMaxRows = 1 << 27, kMaxStride = 1ll << 40, kMaxElems = 1ll << 40;
constexpr int64_t kMaxSpan = 1ll << 48;   // elements from a strided array's first to its last: their bytes stay within 64 bits

// A block of device memory: rows of `width` bytes, `ld` bytes apart.
struct Span {
    const char *name;
    const char *p;
    int64_t bytes;
};

inline Span span(const char *name, const void *p, int64_t rows, int64_t ld, int64_t cols, int64_t esz) {
    return {name, (const char *)p, p ? ((rows - 1) * ld + cols) * esz : 0};
}

inline bool overlap(const Span &a, const Span &b) { return a.p && b.p && a.p < b.p + b.bytes && b.p < a.p + a.bytes; }

// Each of the first n_out spans against all others.
inline int check_overlap(const char *fn, const Span *s, int n, int n_out) {
    for (int i = 0; i < n_out; i++)
        for (int j = i + 1; j < n; j++)
            if (overlap(s[i], s[j])) return set_error(AH_ERR_INVALID, "%s: %s overlaps %s", fn, s[i].name, s[j].name);
    return AH_OK;
}

inline int check_ws(const char *fn, const void *ws, int64_t have, int64_t need) {
    if (!ws || ((uintptr_t)ws & 15)) return set_error(AH_ERR_INVALID, "%s: the workspace is null or not 16-byte aligned", fn);
    if (have < need) return set_error(AH_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", fn, (long long)have, (long long)need);
    return AH_OK;
}

inline int aligned(const char *fn, const char *name, const void *p, int64_t esz) {
    return (uintptr_t)p % (uintptr_t)esz ? set_error(AH_ERR_INVALID, "%s: %s is not aligned to its %d-byte elements", fn, name, (int)esz) : AH_OK;
}

inline int esize(int32_t dtype) { return dtype == AH_F16 ? 2 : 4; }

}  // namespace ah
