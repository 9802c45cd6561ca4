// paged_attn.h -- arguments and index rules of attention over paged caches,
// shared by its kernels (paged_attn*.cu).
#pragma once

#include <cuda.h>

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
    int max_pages = 0, page_size = 0, page_shift = -1;  // page_shift: log2 of a power of two, else -1
    // 1: a sequence's queries take its prefix and its own keys together (they
    // fill row blocks by themselves); 0: prefixes are done for whole groups
    int merged = 0;
    // rows of one tensor copy of cache rows: the largest power of two, 8 to 128,
    // that divides the page size; 0: rows are copied one by one
    int box = 0;
    float scale = 0.0f;
    int* err = nullptr;
};

// Partial results. The keys of a query row fall into two parts, its group's
// prefix (kind 0) and its own sequence's rows behind it (kind 1). Each part is
// cut into key tiles; the tiles of all rows form one line that the CTAs of a
// launch share evenly, so a row's tiles may lie with several neighbouring
// CTAs. The CTA that has the first of them leaves (m, l, first CTA, last CTA)
// in `stat` and its sums in `head`; the CTAs after it, each of which has at
// most one such row block, leave theirs under their own number in `tail`.
// m is the largest score times log2(e), l the sum of 2^(score - m), and the
// sums are of 2^(score - m) v.
struct PartArgs {
    float4* stat = nullptr;   // [T * H]: m, l and, as integers, the CTAs
    float* head = nullptr;    // [T * H][D], or [ctas][slot_rows][D] when !by_row
    float2* tail_stat = nullptr;  // [ctas][slot_rows]
    float* tail = nullptr;        // [ctas][slot_rows][D]
    int by_row = 0;    // heads are kept per row: a row has both kinds
    int slot_rows = 0;  // rows of a row block
    int ctas = 0;
};

// CTAs that take part (each then has a tile, so those between two that share a
// row have a part of it), the share of CTA c of the line of `total` tiles, and
// the CTA that holds tile u.
__device__ __forceinline__ int sharers(long long total, int ctas) { return total < ctas ? (int)total : ctas; }
__device__ __forceinline__ long long share_begin(long long total, int ctas, int c) { return total * c / ctas; }
__device__ __forceinline__ int share_of(long long total, int ctas, long long u) {
    return (int)(((u + 1) * ctas - 1) / total);
}

// Launchers. `prefix`/`rest`: kinds 0 and 1.
constexpr int kDecodeMaxGroup = 16;  // query heads of one KV head that paged_decode_kernel holds
int paged_decode_ctas(const BeaconCudaContext* ctx, const PagedArgs& a, bool split);
void launch_paged_decode(const PagedArgs& a, const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s, bool pdl);
// Rows of a block and CTAs of the tensor-core kernel (paged_tc.cu), for the
// prefixes and, when with_rest, the rest of every sequence.
struct PagedTcPlan {
    bool two = false;    // two row tiles of 128 share a CTA's keys
    bool rest = false;
    int slot_rows = 128;
    int ctas = 0;
};
PagedTcPlan plan_paged_tc(const BeaconCudaContext* ctx, const PagedArgs& a, bool split, bool with_rest);
struct CacheMaps {  // tensor maps of the caches (PagedArgs::box rows by 64 values of one head)
    CUtensorMap k, v;
};
void launch_paged_tc(const PagedTcPlan& plan, const PagedArgs& a, const CacheMaps& maps, const PartArgs& prefix,
                     const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s, bool pdl);
void launch_paged_combine(const PagedArgs& a, const PartArgs& prefix, const PartArgs& rest, int32_t tq, cudaStream_t s);

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
            s.first = start_at(a.gstarts, g, a.B, a.err);
            start_at(a.gstarts, g + 1, a.B, a.err);
            if (s.first >= a.B) s.first = b;  // cannot hold b
            s.prefix = min(prefix_len(a, g), kv_len(a, s.first));  // no row beyond what it holds is read
        }
    }
    return s;
}

// Cache row of position p < capacity through table row b, in two steps so that
// the table entry can be fetched ahead of its use; -1: bad page id.
__device__ __forceinline__ int page_index(const PagedArgs& a, int p) {
    return a.page_shift >= 0 ? p >> a.page_shift : p / a.page_size;
}
__device__ __forceinline__ int page_id(const PagedArgs& a, int b, int p) {
    return __ldg(a.table + (int64_t)b * a.max_pages + page_index(a, p));
}
__device__ __forceinline__ int64_t page_row(const PagedArgs& a, int page, int p) {
    if (page >= 0 && page < a.pages) return (int64_t)page * a.page_size + (p - page_index(a, p) * a.page_size);
    *a.err = kErrIndex;
    return -1;
}

}  // namespace bc
