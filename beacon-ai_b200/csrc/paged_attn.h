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
// CTAs. The CTA that has the first of them leaves m, l and where the parts are
// in `stat` and its sums in `head`; the CTAs after it, each of which has at
// most one such row block, leave theirs under their own number in `tail`.
// With scores times log2(e), m is the largest or a reference some powers of two
// off it (-inf: no score above -inf), l the sum of 2^(score - m), and the sums are
// of 2^(score - m) v. Every row has an entry of kind 1, also one that sees no key.
struct PartArgs {
    float4* stat = nullptr;   // [T * H]: m, l, PartPlace
    float* head = nullptr;    // [T * H][D], or [ctas][slot_rows][D] when !by_row
    float2* tail_stat = nullptr;  // [ctas][slot_rows]
    float* tail = nullptr;        // [ctas][slot_rows][D]
    // Of several rows of a sequence without prefixes only the row blocks that are
    // cut have to be joined: per CTA the one whose first part it has, as [8]: last CTA (-1: none), first
    // token, first row, rows of its sequence's queries, KV head.
    int* cuts = nullptr;
    int by_row = 0;    // heads are kept per row: a row has both kinds
    int slot_rows = 0;  // rows of a row block, at most 256
    int ctas = 0;       // at most 4096
};
// The CTAs [c0, c1] that have a row's parts, its row in their slots, and
// whether it has a part of kind 0 as well.
struct PartPlace {
    int c0, c1, row;
    bool prefix;
};
__device__ __forceinline__ float4 pack_stat(float m, float l, const PartPlace& p) {
    return make_float4(m, l, __int_as_float(p.c0 | p.row << 16), __int_as_float(p.c1 | (p.prefix ? 1 << 16 : 0)));
}
__device__ __forceinline__ PartPlace place_of(const float4& s) {
    const int a = __float_as_int(s.z), b = __float_as_int(s.w);
    return PartPlace{a & 0xFFFF, b & 0xFFFF, (a >> 16) & 0xFF, (b >> 16 & 1) != 0};
}

// Even shares of a line of `total` tiles: the first `more` CTAs have q + 1
// tiles, the others q. At most one CTA per tile takes part, so that every CTA
// between two that share a row has a part of it.
struct Shares {
    int ctas = 0, more = 0;
    long long q = 0;
    __device__ __forceinline__ Shares(long long total, int n) {
        ctas = total < n ? (int)total : n;
        if (ctas == 0) return;
        q = total >> 31 ? total / ctas : (long long)((uint32_t)total / (uint32_t)ctas);
        more = (int)(total - q * ctas);
    }
    __device__ __forceinline__ long long begin(int c) const { return q * c + min(c, more); }
    __device__ __forceinline__ int of(long long u) const {  // the CTA that has tile u
        const long long cut = (q + 1) * more;
        if (u < cut) return (u >> 31) | ((q + 1) >> 31) ? (int)(u / (q + 1)) : (int)((uint32_t)u / (uint32_t)(q + 1));
        u -= cut;
        return more + ((u >> 31) | (q >> 31) ? (int)(u / q) : (int)((uint32_t)u / (uint32_t)q));
    }
};

// Launchers. `prefix`/`rest`: kinds 0 and 1.
constexpr int kDecodeMaxGroup = 16;  // query heads of one KV head that paged_decode_kernel holds
struct CacheMaps {  // tensor maps of the caches: boxes of some rows by 64 values of one head
    CUtensorMap k, v;
};
constexpr int kDecodeBox = 16;  // most rows of a copy box of paged_decode_kernel
int paged_decode_ctas(const BeaconCudaContext* ctx, const PagedArgs& a);
// after_tc: the launch before it is paged_tc_kernel of the same call.
void launch_paged_decode(const BeaconCudaContext* ctx, const PagedArgs& a, const CacheMaps& maps, const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s,
                         bool pdl, bool after_tc);
// Rows of a block and CTAs of the tensor-core kernel (paged_tc.cu), for the
// prefixes and, when with_rest, the rest of every sequence.
struct PagedTcPlan {
    bool two = false;    // two row tiles of 128 share a CTA's keys
    bool rest = false;
    int slot_rows = 128;
    int ctas = 0;
};
PagedTcPlan plan_paged_tc(const BeaconCudaContext* ctx, const PagedArgs& a, bool split, bool with_rest);
void launch_paged_tc(const BeaconCudaContext* ctx, const PagedTcPlan& plan, const PagedArgs& a, const CacheMaps& maps, const PartArgs& prefix,
                     const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s, bool pdl);
void launch_paged_combine(const PagedArgs& a, const PartArgs& prefix, const PartArgs& rest, int32_t tq, cudaStream_t s);

// Values that callers hold in device tensors are kept inside their ranges; one
// outside marks the stream's error word. Loads come before the checks so that
// independent ones are in flight together.
__device__ __forceinline__ int keep_in(int v, long long most, bool& bad) {
    if (v >= 0 && v <= most) return v;
    bad = true;
    return v < 0 ? 0 : (int)most;
}
__device__ __forceinline__ long long capacity(const PagedArgs& a) { return (long long)a.max_pages * a.page_size; }

// The i with starts[i] <= x < starts[i + 1] of an ascending array of n + 1
// entries; -1 if there is none.
__device__ __forceinline__ int span_of(const int32_t* starts, int n, int x) {
    int lo = 0, hi = n;  // the last i with starts[i] <= x lies in [lo, hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(starts + mid) <= x) lo = mid;
        else hi = mid;
    }
    return n > 0 && __ldg(starts + lo) <= x && x < __ldg(starts + lo + 1) ? lo : -1;
}

// Rows that sequence b holds, its queries and the prefix it shares.
struct SeqInfo {
    int len = 0;          // cached rows, within the table's capacity
    int q0 = 0, nq = 0;   // query rows [q0, q0 + nq)
    int prefix = 0;       // keys [0, prefix) are read through sequence `first`
    int first = 0;
};

__device__ __forceinline__ SeqInfo seq_info(const PagedArgs& a, int b) {
    SeqInfo s;
    bool bad = false;
    const int len = __ldg(a.lens + b);
    int q0 = b, q1 = b + 1;
    if (a.qstarts) {
        q0 = __ldg(a.qstarts + b);
        q1 = __ldg(a.qstarts + b + 1);
    }
    s.first = b;
    if (a.gstarts) {
        const int g = span_of(a.gstarts, a.groups, b);
        if (g >= 0) {
            const int lo = __ldg(a.gstarts + g), hi = __ldg(a.gstarts + g + 1), p = __ldg(a.prefix + g);
            if (lo >= 0) s.first = lo;  // lo <= b
            bad |= lo < 0 || hi > a.B;
            // no row beyond what the first sequence holds is read
            s.prefix = min(keep_in(p, capacity(a), bad), keep_in(__ldg(a.lens + s.first), capacity(a), bad));
        }
    }
    s.len = keep_in(len, capacity(a), bad);
    s.q0 = keep_in(q0, a.T, bad);
    s.nq = keep_in(q1, a.T, bad) - s.q0;
    if (s.nq < 0) {
        bad = true;
        s.nq = 0;
    }
    if (bad) a.err[kErrWordIndex] = 1;
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
    a.err[kErrWordIndex] = 1;
    return -1;
}

}  // namespace bc
