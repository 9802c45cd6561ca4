// paged_attn.h -- arguments and index rules of attention over paged caches,
// shared by its kernels (paged_attn*.cu).
#pragma once

#include "common.cuh"
#include "internal.h"

namespace bc {

struct PagedArgs {
    const void* q = nullptr;  // [T][H][D]
    const void* ck = nullptr;  // [pages][page_size][Hkv][D]
    const void* cv = nullptr;
    void* out = nullptr;      // [T][H][D]
    const int32_t* table = nullptr;    // [B][max_pages]
    const int32_t* lens = nullptr;     // [B]
    const int32_t* qstarts = nullptr;  // [B + 1]; null: row b is sequence b's only query
    const int32_t* gstarts = nullptr;  // [groups + 1]; null: no prefixes
    const int32_t* prefix = nullptr;   // [groups]
    int64_t pages = 0;
    int T = 0, B = 0, H = 0, Hkv = 0, G = 0, D = 0, groups = 0;  // G = H / Hkv
    int max_pages = 0, page_size = 0;
    float scale = 0.0f;
    int* err = nullptr;
};

// A start array entry kept inside [0, n] (callers hold it in a device tensor).
__device__ __forceinline__ int start_at(const int32_t* s, int i, int n, int* err) {
    const int v = s[i];
    if (v >= 0 && v <= n) return v;
    *err = kErrIndex;
    return v < 0 ? 0 : n;
}

// The i with starts[i] <= x < starts[i + 1] of an ascending array of n + 1
// entries; -1 if there is none.
__device__ __forceinline__ int span_of(const int32_t* starts, int n, int x) {
    int lo = 0, hi = n;  // the last i with starts[i] <= x lies in [lo, hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= x) lo = mid;
        else hi = mid;
    }
    return n > 0 && starts[lo] <= x && x < starts[lo + 1] ? lo : -1;
}

// Rows that sequence b holds, its queries and the prefix it shares.
struct SeqInfo {
    int len = 0;          // cached rows, within the table's capacity
    int q0 = 0, nq = 0;   // query rows [q0, q0 + nq)
    int prefix = 0;       // keys [0, prefix) are read through sequence `first`
    int first = 0;
};

__device__ __forceinline__ int kv_len(const PagedArgs& a, int b) {
    const int len = a.lens[b];
    const long long cap = (long long)a.max_pages * a.page_size;
    if (len >= 0 && len <= cap) return len;
    *a.err = kErrIndex;
    return len < 0 ? 0 : (int)cap;
}

__device__ __forceinline__ int prefix_len(const PagedArgs& a, int g) {
    const int p = a.prefix[g];
    const long long cap = (long long)a.max_pages * a.page_size;
    if (p >= 0 && p <= cap) return p;
    *a.err = kErrIndex;
    return p < 0 ? 0 : (int)cap;
}

__device__ __forceinline__ SeqInfo seq_info(const PagedArgs& a, int b) {
    SeqInfo s;
    s.len = kv_len(a, b);
    if (a.qstarts) {
        s.q0 = start_at(a.qstarts, b, a.T, a.err);
        s.nq = start_at(a.qstarts, b + 1, a.T, a.err) - s.q0;
        if (s.nq < 0) {
            *a.err = kErrIndex;
            s.nq = 0;
        }
    } else {
        s.q0 = b;
        s.nq = 1;
    }
    s.first = b;
    if (a.gstarts) {
        const int g = span_of(a.gstarts, a.groups, b);
        if (g >= 0) {
            s.prefix = prefix_len(a, g);
            s.first = start_at(a.gstarts, g, a.B, a.err);
            start_at(a.gstarts, g + 1, a.B, a.err);
            if (s.first >= a.B) s.first = b;  // cannot hold b
        }
    }
    return s;
}

// Cache row of position p < capacity through table row b; -1: bad page id.
__device__ __forceinline__ int64_t page_row(const PagedArgs& a, int b, int p) {
    const int64_t page = a.table[(int64_t)b * a.max_pages + p / a.page_size];
    if (page >= 0 && page < a.pages) return page * a.page_size + p % a.page_size;
    *a.err = kErrIndex;
    return -1;
}

}  // namespace bc
