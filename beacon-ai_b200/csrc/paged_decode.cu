// paged_decode.cu -- paged attention of single query rows (decode) and the
// join of partial results.
//
// o = sum_p 2^(t_p - m) v_p / sum_p 2^(t_p - m), t_p = scale log2(e) q . k_p,
// over the keys of a row behind its group's prefix. The G query heads of one
// KV head share its keys, so the bound is reading the cache once. A tile is 64
// keys, 16 for each of the 4 warps of a CTA: each brings its keys and values in
// through its own ring (tensor copies of 8 or 16 rows, no CTA barrier in the
// loop) and forms S^T = K Q^T (16 keys x 8 or 16 heads) and O^T += V^T P^T with
// m16n8k16 instructions, so that few heads waste little of them. Each warp
// keeps its own running maximum. The tiles of all sequences and KV heads form
// one line that the CTAs share evenly (PartArgs): a batch of uneven lengths
// loads every SM alike whatever the lengths are, and the lengths may change
// between replays of a captured call.
// Bound by the cache read where sequences are long (16 of 8192 keys ragged, f16,
// 32 heads on 8 of 128: 340 MB in 61.5 us with the join, 5.5 TB/s; tensor pipe 8%
// busy), by start and join where there are few keys (one sequence of 257 keys,
// 20 tiles: 7.8 us). Scores as K Q^T keep 8 or 16 heads of the 16 x 8 instruction
// busy; Q K^T with 4 heads on its 16 rows would waste three quarters.
// 32-bit queries are two f16 parts (products for both), and so are the
// weights; each tile's value sums are then added with rounding, because the
// instruction's own sums truncate and a long chain of them would drift.
#include <algorithm>
#include <cmath>

#include "internal.h"
#include "kernels.h"
#include "paged_attn.h"
#include "paged_mma.cuh"
#include "rotary.h"

namespace bc {
namespace {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16 * kDecWarps;  // keys of a tile
// Factor on the weights and their sums (kNarrowExponent): the largest weight is
// 2^15, so one of 2^-29 of it still has all 11 bits (22 in two parts down to
// 2^-18), and none is off by more than 2^-40 of the largest.
template <typename T>
constexpr float kWeightScale = kNarrowExponent<T> ? 32768.0f : 1.0f;

template <int DP, int NT, bool SPLIT>
struct DecodeSmem {
    static constexpr int stages = DP == 128 ? 2 : 4;
    static constexpr int part = 16 * DP * 2;        // 16 key (or value) rows: [64 values][row][128 bytes]
    static constexpr int ring = stages * 2 * part;  // of one warp
    static constexpr int rows = 8 * NT;             // heads, padded
    static constexpr int q = rows * DP * 2;         // one part of the queries
    // merge area: [warp][rows][DP] sums, then m and l [warp][rows], scales [rows]
    static constexpr int merge = kDecWarps * rows * DP * 4;
    static constexpr size_t bytes =
        (size_t)kDecWarps * ring + (SPLIT ? 2 : 1) * q + merge + (2 * kDecWarps + 1) * rows * 4 + 1024;
};

struct Span {  // keys [from, to) of one sequence, in tiles that begin at `base`
    int from = 0, to = 0, base = 0, tiles = 0;
};
__device__ __forceinline__ Span rest_of(const PagedArgs& a, int b) {
    Span s;
    if (b >= a.B) return s;
    const SeqInfo i = seq_info(a, b);
    s.from = i.prefix;
    s.to = i.len;
    s.base = a.box ? s.from & ~(min(a.box, kDecodeBox) - 1) : s.from;
    // a sequence without keys has a tile too: its rows are written by it
    s.tiles = s.to > s.from ? (s.to - s.base + kDecKeys - 1) / kDecKeys : 1;
    return s;
}

// Place in the line of tiles: sequence, KV head, tile.
struct Walk {
    int b = 0, kvh = 0, tile = 0;
    Span cur;
    __device__ __forceinline__ void step(const PagedArgs& a) {
        if (++tile < cur.tiles) return;
        tile = 0;
        if (++kvh < a.Hkv) return;
        kvh = 0;
        cur = rest_of(a, ++b);
    }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {  // 8x8 matrix of 16-bit values held by a warp
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <typename TQ, typename TK, int DP, int NT, bool SPLIT>
__global__ void __launch_bounds__(kDecThreads)
    paged_decode_kernel(const PagedArgs a, const __grid_constant__ CacheMaps maps, const PartArgs part, int after_tc) {
    using S = DecodeSmem<DP, NT, SPLIT>;
    constexpr int NS = S::stages;
    constexpr int KS = DP / 16;
    constexpr int CH = DP / 8;   // 16-byte chunks of a row
    constexpr int RPI = 32 / CH;  // rows that one copy instruction of a warp covers
    extern __shared__ uint8_t dec_smem_raw[];
    __shared__ __align__(8) uint64_t bars[kDecWarps][NS];
    __shared__ long long sums_s[kDecWarps];
    __shared__ int b_s;
    __shared__ long long before_s;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dec_smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = smem_u32(smem + warp * S::ring);
    const uint32_t q_at = smem_u32(smem + kDecWarps * S::ring);
    float* merge_o = reinterpret_cast<float*>(smem + kDecWarps * S::ring + (SPLIT ? 2 : 1) * S::q);  // [warp][rows][DP]
    float* merge_m = merge_o + kDecWarps * S::rows * DP;                                              // [warp][rows]
    float* merge_l = merge_m + kDecWarps * S::rows;
    float* scale_s = merge_l + kDecWarps * S::rows;                                                    // [rows]
    if (lane == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(&bars[warp][i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Behind the tensor-core kernel of the same call there is nothing to wait for.
    // That one let later kernels start only after its own wait, so all that came
    // before it is done, whatever another thread launched in between; and this one
    // writes only its rows of the result and the call's own scratch, which no
    // kernel but the call's touches.
    if (!after_tc) pdl_wait();

    // this CTA's share of the line
    const int chunk = (a.B + kDecThreads - 1) / kDecThreads;
    const int cb0 = min(a.B, tid * chunk), cb1 = min(a.B, cb0 + chunk);
    long long mine = 0;
    for (int b = cb0; b < cb1; ++b) mine += rest_of(a, b).tiles;
    long long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) sums_s[warp] = scan;
    __syncthreads();
    long long total = 0, before = scan - mine;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
        if (w < warp) before += sums_s[w];
        total += sums_s[w];
    }
    total *= a.Hkv;
    const int cta = blockIdx.x;
    const Shares shares(total, part.ctas);
    const long long u0 = cta < shares.ctas ? shares.begin(cta) : 0, u1 = cta < shares.ctas ? shares.begin(cta + 1) : 0;
    pdl_trigger();
    if (u0 < u1) {
        if (before * a.Hkv <= u0 && u0 < (before + mine) * a.Hkv) {
            int b = cb0;
            for (; b < cb1; ++b) {
                const int n = rest_of(a, b).tiles;
                if (u0 < (before + n) * a.Hkv) break;
                before += n;
            }
            b_s = b;
            before_s = before;
        }
        __syncthreads();
        Walk load;
        load.b = b_s;
        load.cur = rest_of(a, load.b);
        const long long off = u0 - before_s * a.Hkv;
        load.kvh = (int)(off / load.cur.tiles);
        load.tile = (int)(off - (long long)load.kvh * load.cur.tiles);
        Walk at = load;
        const int count = (int)(u1 - u0);
        const long long limit = g_wait_limit;
        bool failed = false;

        // --- copies: lanes below 16 / box (one by one: below 16) have a row each
        const int box = min(a.box, kDecodeBox);
        const int step = a.box ? box : 1;
        int page_next = 0;
        auto pos_of = [&](const Walk& w) { return w.cur.base + w.tile * kDecKeys + warp * 16 + lane * step; };
        auto fetch_page = [&](const Walk& w) {
            const int p = pos_of(w);
            return lane * step < 16 && p < w.cur.to ? page_id(a, w.b, p) : 0;
        };
        auto copy_tile = [&](int stage, const Walk& w, int page) {
            const int p = pos_of(w);
            const bool live = lane * step < 16 && p < w.cur.to && p + step > w.cur.from;
            const uint32_t dst = ring + stage * 2 * S::part;
            const int row = live ? (int)page_row(a, page, p) : -1;
            if (a.box) {
                const int n = __popc(__ballot_sync(0xffffffffu, live));
                if (lane == 0) mbar_expect_tx(&bars[warp][stage], (uint32_t)(n * box * DP * 4));
                __syncwarp();
                if (live) {
                    const int y = row >= 0 ? row : (int)(a.pages * a.page_size);  // a bad page: zeros
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h) {
                        const uint32_t d = dst + h * 2048 + lane * box * 128;
                        tma_rows(d, &maps.k, h * 64, w.kvh, y, &bars[warp][stage]);
                        tma_rows(d + S::part, &maps.v, h * 64, w.kvh, y, &bars[warp][stage]);
                    }
                }
            } else {
                const int c = lane % CH;
#pragma unroll
                for (int i = 0; i < 16 / RPI; ++i) {
                    const int r = i * RPI + lane / CH;
                    const int cr = __shfl_sync(0xffffffffu, row, r);
                    const bool on = cr >= 0 && c * 8 < a.D;
                    const int64_t src = on ? ((int64_t)cr * a.Hkv + w.kvh) * a.D + c * 8 : 0;
                    const uint32_t d = dst + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    cp_async16_zfill(d, static_cast<const TK*>(a.ck) + src, on);
                    cp_async16_zfill(d + S::part, static_cast<const TK*>(a.cv) + src, on);
                }
                cp_async_commit();
            }
        };
        // The queries of (b, kvh): thread i has 4 values of heads i / (DP / 4) + ...
        constexpr int QV = S::rows * (DP / 4) / kDecThreads;  // float4 per thread
        constexpr int QR = kDecThreads / (DP / 4);            // heads that the threads cover at a time
        const int qd = (tid % (DP / 4)) * 4;
        float4 qn[SPLIT ? QV : 1];
        uint2 qh[SPLIT ? 1 : QV];
        auto fetch_q = [&](int b, int kvh) {
#pragma unroll
            for (int i = 0; i < QV; ++i) {
                const int g = tid / (DP / 4) + i * QR;
                const bool on = g < a.G && qd < a.D && b < a.B;
                const TQ* q = static_cast<const TQ*>(a.q) + ((int64_t)b * a.H + kvh * a.G + g) * a.D + qd;
                if constexpr (SPLIT) qn[i] = on ? *reinterpret_cast<const float4*>(q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                else qh[i] = on ? *reinterpret_cast<const uint2*>(q) : make_uint2(0, 0);
            }
        };
        fetch_q(at.b, at.kvh);
        page_next = fetch_page(load);
#pragma unroll 1
        for (int i = 0; i < NS - 1; ++i) {
            if (i < count) {
                copy_tile(i, load, page_next);
                load.step(a);
                if (i + 1 < count) page_next = fetch_page(load);
            } else if (!a.box) {
                cp_async_commit();
            }
        }

        uint32_t qf[KS][2 * NT], ql[SPLIT ? KS : 1][2 * NT];
        float cs[NT][2], m[NT][2], l[NT][2], o[KS][NT][4];
        bool fresh = true;
        const int lr = lane & 7, mi = lane >> 3;
#pragma unroll 1
        for (int j = 0; j < count; ++j) {
            if (fresh) {
                // queries to shared memory as B operands (head rows, 16-byte chunks
                // in the order of chunk ^ row), then to registers
#pragma unroll
                for (int i = 0; i < QV; ++i) {
                    const int g = tid / (DP / 4) + i * QR;
                    const uint32_t d = q_at + g * (DP * 2) + ((((qd >> 3) ^ (g & 7)) << 4) | ((qd & 4) << 1));
                    if constexpr (SPLIT) {
                        float mx = fmaxf(fmaxf(fabsf(qn[i].x), fabsf(qn[i].y)), fmaxf(fabsf(qn[i].z), fabsf(qn[i].w)));
#pragma unroll
                        for (int s = DP / 8; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
                        float inv;
                        const float sc = query_scale(mx, inv);
                        uint2 h, lo;
                        split_f16(qn[i].x * sc, qn[i].y * sc, h.x, lo.x);
                        split_f16(qn[i].z * sc, qn[i].w * sc, h.y, lo.y);
                        asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(d), "r"(h.x), "r"(h.y) : "memory");
                        asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(d + S::q), "r"(lo.x), "r"(lo.y) : "memory");
                        if (qd == 0) scale_s[g] = a.scale * 1.4426950408889634f * inv;
                    } else {
                        asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(d), "r"(qh[i].x), "r"(qh[i].y) : "memory");
                    }
                }
                __syncthreads();
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {
                        const uint32_t src = q_at + (8 * n + lr) * (DP * 2) + (((2 * k + mi) ^ lr) << 4);
                        uint32_t b[4];
                        ldsm4(b, src);
                        qf[k][2 * n] = b[0];
                        qf[k][2 * n + 1] = b[1];
                        qf[k + 1][2 * n] = b[2];
                        qf[k + 1][2 * n + 1] = b[3];
                        if constexpr (SPLIT) {
                            ldsm4(b, src + S::q);
                            ql[k][2 * n] = b[0];
                            ql[k][2 * n + 1] = b[1];
                            ql[k + 1][2 * n] = b[2];
                            ql[k + 1][2 * n + 1] = b[3];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // above zero, so that a masked score (-inf) stays one
                        cs[n][e] = fmaxf(SPLIT ? scale_s[8 * n + 2 * (lane & 3) + e] : a.scale * 1.4426950408889634f, 1e-37f);
                        m[n][e] = -INFINITY;
                        l[n][e] = 0.0f;
                    }
                }
#pragma unroll
                for (int d = 0; d < KS; ++d)
#pragma unroll
                    for (int n = 0; n < NT; ++n) o[d][n][0] = o[d][n][1] = o[d][n][2] = o[d][n][3] = 0.0f;
                // the next head's are on their way meanwhile
                if (at.kvh + 1 < a.Hkv) fetch_q(at.b, at.kvh + 1);
                else fetch_q(at.b + 1, 0);
                fresh = false;
            }
            // the stage that was read last is filled again
            __syncwarp();
            if (j + NS - 1 < count && !failed) {
                copy_tile((j + NS - 1) % NS, load, page_next);
                load.step(a);
                if (j + NS < count) page_next = fetch_page(load);
            } else if (!a.box) {
                cp_async_commit();
            }
            const uint32_t ks = ring + (j % NS) * 2 * S::part, vs = ks + S::part;
            const int first = at.cur.base + at.tile * kDecKeys + warp * 16;
            if (a.box) {
                if (!failed && !wait_bar(&bars[warp][j % NS], (uint32_t)((j / NS) & 1), limit)) {
                    // reported; the ring stays in step as long as the copy comes at all
                    a.err[kErrWordWait] = 1;
                    failed = !mbar_drain(&bars[warp][j % NS], (uint32_t)((j / NS) & 1));
                }
                failed = __any_sync(0xffffffffu, failed);
                if (first < at.cur.from || first + 16 > at.cur.to) {
                    // value rows that are no keys: their weights are zero, but what the
                    // page holds there may be no number
                    const int lo = max(0, min(16, at.cur.from - first)), hi = max(lo, min(16, at.cur.to - first));
                    for (int i = lane; i < (lo + 16 - hi) * CH; i += 32) {
                        const int q = i / CH, r = q < lo ? q : hi + q - lo, c = i % CH;
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vs + (c >> 3) * 2048 + r * 128 + ((c & 7) << 4)), "r"(0) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a copy overwrites them
                }
            } else {
                cp_async_wait<NS - 1>();
            }
            __syncwarp();

            if (first < at.cur.to && first + 16 > at.cur.from) {
                float sc[NT][4] = {};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t ka[4];
                    const int r = lr + (mi & 1) * 8, c = 2 * k + (mi >> 1);
                    ldsm4(ka, ks + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816<TK>(sc[n], ka, qf[k][2 * n], qf[k][2 * n + 1]);
                        if constexpr (SPLIT) mma16816<TK>(sc[n], ka, ql[k][2 * n], ql[k][2 * n + 1]);
                    }
                }
                // keys first + lane / 4 (and + 8), heads 8 n + 2 (lane % 4) + e
                const int k0 = first + lane / 4;
                const bool on0 = k0 >= at.cur.from && k0 < at.cur.to, on1 = k0 + 8 >= at.cur.from && k0 + 8 < at.cur.to;
                uint32_t ph[NT][2], pl[SPLIT ? NT : 1][2];
                bool moved = false;
                float keep[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float ref[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sc[n][e] = on0 ? sc[n][e] * cs[n][e] : -INFINITY;
                        sc[n][2 + e] = on1 ? sc[n][2 + e] * cs[n][e] : -INFINITY;
                        float mx = fmaxf(sc[n][e], sc[n][2 + e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        mx = fmaxf(mx, m[n][e]);
                        keep[n][e] = m[n][e] == -INFINITY ? 1.0f : exp2_fast(m[n][e] - mx);  // nothing summed yet: nothing to scale
                        moved |= keep[n][e] != 1.0f;
                        m[n][e] = mx;
                        ref[e] = mx == -INFINITY ? 0.0f : mx;
                        sc[n][e] = exp2_fast(sc[n][e] - ref[e]) * kWeightScale<TK>;
                        sc[n][2 + e] = exp2_fast(sc[n][2 + e] - ref[e]) * kWeightScale<TK>;
                        l[n][e] = l[n][e] * keep[n][e] + (sc[n][e] + sc[n][2 + e]);
                    }
                    if constexpr (SPLIT) {
                        split_f16(sc[n][0], sc[n][1], ph[n][0], pl[n][0]);
                        split_f16(sc[n][2], sc[n][3], ph[n][1], pl[n][1]);
                        pl[n][0] = transpose8(pl[n][0]);
                        pl[n][1] = transpose8(pl[n][1]);
                    } else {
                        ph[n][0] = Half2Of<TK>::pack(sc[n][0], sc[n][1]);
                        ph[n][1] = Half2Of<TK>::pack(sc[n][2], sc[n][3]);
                    }
                    ph[n][0] = transpose8(ph[n][0]);
                    ph[n][1] = transpose8(ph[n][1]);
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int d = 0; d < KS; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[d][n][e] *= keep[n][e & 1];
                }
#pragma unroll
                for (int d = 0; d < KS; ++d) {
                    uint32_t va[4];
                    const int r = lr + (mi >> 1) * 8, c = 2 * d + (mi & 1);
                    ldsm4_t(va, vs + (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if constexpr (SPLIT) {
                            float t[4] = {};
                            mma16816<TK>(t, va, pl[n][0], pl[n][1]);  // small parts first: sums are cut to 24 bits
                            mma16816<TK>(t, va, ph[n][0], ph[n][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[d][n][e] += t[e];
                        } else {
                            mma16816<TK>(o[d][n], va, ph[n][0], ph[n][1]);
                        }
                    }
                }
            }

            if (at.tile + 1 == at.cur.tiles || j + 1 == count) {
                // join the warps' sums of (b, kvh)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = l[n][e];
                        x += __shfl_xor_sync(0xffffffffu, x, 4);
                        x += __shfl_xor_sync(0xffffffffu, x, 8);
                        x += __shfl_xor_sync(0xffffffffu, x, 16);
                        const int g = 8 * n + 2 * (lane & 3) + e;
                        if (lane < 4) {
                            merge_m[warp * S::rows + g] = m[n][e];
                            merge_l[warp * S::rows + g] = x;
                        }
                        float* mo = merge_o + (warp * S::rows + g) * DP + lane / 4;
                        if (g < a.G) {
#pragma unroll
                            for (int d = 0; d < KS; ++d) {
                                mo[16 * d] = o[d][n][e];
                                mo[16 * d + 8] = o[d][n][2 + e];
                            }
                        }
                    }
                __syncthreads();
                const long long tile0 = u0 + j - at.tile;  // of this head, in the line
                const int c0 = shares.of(tile0), c1 = shares.of(tile0 + at.cur.tiles - 1);
                const bool done = c0 == c1 && at.cur.from == 0;  // no other part anywhere
                for (int g = tid / (DP / 4); g < a.G; g += QR) {
                    float mw[kDecWarps], M = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kDecWarps; ++w) {
                        mw[w] = merge_m[w * S::rows + g];
                        M = fmaxf(M, mw[w]);
                    }
                    float sum = 0.0f;
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kDecWarps; ++w) {
                        const float wt = mw[w] == -INFINITY ? 0.0f : exp2_fast(mw[w] - M) * (1.0f / kWeightScale<TK>);
                        const float4 v = *reinterpret_cast<const float4*>(merge_o + (w * S::rows + g) * DP + qd);
                        acc.x = fmaf(v.x, wt, acc.x);
                        acc.y = fmaf(v.y, wt, acc.y);
                        acc.z = fmaf(v.z, wt, acc.z);
                        acc.w = fmaf(v.w, wt, acc.w);
                        sum = fmaf(merge_l[w * S::rows + g], wt, sum);
                    }
                    if (qd >= a.D) continue;
                    const int64_t row = (int64_t)at.b * a.H + at.kvh * a.G + g;
                    const int64_t slot = (int64_t)cta * part.slot_rows + g;
                    if (done) {
                        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                        TQ* dst = static_cast<TQ*>(a.out) + row * a.D + qd;
                        if constexpr (SPLIT)
                            *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                        else
                            *reinterpret_cast<uint2*>(dst) =
                                make_uint2(Half2Of<TK>::pack(acc.x * inv, acc.y * inv), Half2Of<TK>::pack(acc.z * inv, acc.w * inv));
                    } else {
                        float* dst = c0 == cta ? part.head + (part.by_row ? row : slot) * a.D : part.tail + slot * a.D;
                        *reinterpret_cast<float4*>(dst + qd) = acc;
                    }
                    if (qd == 0) {
                        if (c0 == cta) part.stat[row] = pack_stat(M, sum, PartPlace{c0, c1, g, at.cur.from > 0});
                        else part.tail_stat[slot] = make_float2(M, sum);
                    }
                }
                __syncthreads();  // the merge area and the queries are written again
                fresh = true;
            }
            at.step(a);
        }
        // Nothing lands after the CTA has ended: every copy was waited for above, and
        // when one did not come no more were requested.
        if (!a.box) cp_async_wait<0>();
    }
    // kernels launched after this one count on everything before it
    pdl_wait();
}

// The parts of the query rows where there are prefixes or single rows: kind 1,
// kind 0 where the row has it, each a first part and those of the CTAs after
// it. One warp per row. What is where stands in the row's entry, so nothing
// else has to be looked up first.
template <typename TQ, typename T16>
__global__ void __launch_bounds__(128) paged_join_rows_kernel(const PagedArgs a, const PartArgs prefix, const PartArgs rest) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    pdl_wait();
    if (row >= (int64_t)a.T * a.H) return;
    float4 st[2];
    st[1] = rest.stat[row];
    st[0] = rest.by_row ? prefix.stat[row] : st[1];
    if (a.qstarts) {  // rows of no sequence are not written
        const int t = (int)(row / a.H);
        if (t < __ldg(a.qstarts) || t >= __ldg(a.qstarts + a.B)) return;
    }
    const PartPlace place = place_of(st[1]);
    const bool both = rest.by_row && place.prefix;
    if (!both && place.c0 == place.c1) return;  // written by the CTA that had all of it
    // the parts in one line, a lane each
    const PartPlace pre = place_of(st[0]);
    const bool bad = place.c1 < place.c0 || place.c1 >= rest.ctas || place.row >= rest.slot_rows ||
                     (both && (pre.c1 < pre.c0 || pre.c1 >= prefix.ctas || pre.row >= prefix.slot_rows));
    if (bad) {  // start arrays that contradict each other: no CTA had the row
        a.err[kErrWordIndex] = 1;
        return;
    }
    const int n0 = both ? pre.c1 - pre.c0 + 1 : 0, n = n0 + place.c1 - place.c0 + 1;
    const bool live = lane * 4 < a.D;
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int base = 0; base < n; base += 32) {
        const int idx = base + lane;
        const bool zero = idx < n0;
        const PartArgs& p = zero ? prefix : rest;
        const PartPlace at = zero ? pre : place;
        const int c = at.c0 + (zero ? idx : idx - n0);
        const int64_t slot = (int64_t)c * p.slot_rows + at.row;
        float m = -INFINITY, l = 0.0f;
        const float* src = p.tail + slot * a.D;
        if (idx < n) {
            if (c == at.c0) {
                m = zero ? st[0].x : st[1].x;
                l = zero ? st[0].y : st[1].y;
                src = p.head + (p.by_row ? row : slot) * a.D;
            } else {
                const float2 v = p.tail_stat[slot];
                m = v.x;
                l = v.y;
            }
        }
        const float mx = fmaxf(M, warp_max(m));
        // parts without a key; a sum that is no number (of scores that are none,
        // which maxima leave out) is kept
        if (mx == -INFINITY && !__any_sync(0xffffffffu, l != 0.0f)) continue;
        const float keep = M == -INFINITY ? 0.0f : exp2_fast(M - mx);
        const float w = m == -INFINITY ? 0.0f : exp2_fast(m - mx);
        M = mx;
        L = L * keep + warp_sum(l * w);
        o.x *= keep;
        o.y *= keep;
        o.z *= keep;
        o.w *= keep;
        const int k = min(32, n - base);
        for (int i = 0; i < k; i += 8) {  // eight loads in flight
            float4 v[8];
            float wi[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                wi[q] = __shfl_sync(0xffffffffu, w, i + q);
                const float* s = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)src, i + q));
                v[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (live && i + q < k) v[q] = *reinterpret_cast<const float4*>(s + lane * 4);
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                o.x = fmaf(v[q].x, wi[q], o.x);
                o.y = fmaf(v[q].y, wi[q], o.y);
                o.z = fmaf(v[q].z, wi[q], o.z);
                o.w = fmaf(v[q].w, wi[q], o.w);
            }
        }
    }
    if (!live) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    TQ* dst = static_cast<TQ*>(a.out) + row * a.D + lane * 4;
    if constexpr (sizeof(TQ) == 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(Half2Of<T16>::pack(o.x * inv, o.y * inv), Half2Of<T16>::pack(o.z * inv, o.w * inv));
    }
}

// The same for several rows of a sequence without prefixes: only the row blocks that were cut have to be
// joined (grid: CTA, rows of its block); the blocks for other CTAs leave at
// once. A row has two or three parts mostly, so a warp has four rows, eight
// lanes for the parts of each, and sixteen loads in flight.
template <typename TQ, typename T16>
__global__ void __launch_bounds__(128) paged_join_cuts_kernel(const PagedArgs a, const PartArgs p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    const int c0 = blockIdx.x;
    const int4 rec = *reinterpret_cast<const int4*>(p.cuts + c0 * 8);
    if (rec.x < 0) return;
    const int kvh = p.cuts[c0 * 8 + 4];
    const int r = (blockIdx.y * 4 + warp) * 4 + lane / 8, br = rec.z + r;
    const bool on = r < p.slot_rows && br < rec.w;
    const int64_t row = (int64_t)(rec.y + br / a.G) * a.H + kvh * a.G + br % a.G;
    const int n = rec.x - c0 + 1;
    const bool live = lane * 4 < a.D;
    float M = -INFINITY, L = 0.0f;
    float4 o[4] = {};
    for (int base = 0; base < n; base += 8) {
        const int c = c0 + base + (lane & 7);
        const int64_t slot = (int64_t)c * p.slot_rows + r;
        float m = -INFINITY, l = 0.0f;
        if (on && c <= rec.x) {
            if (c == c0) {
                const float4 st = p.stat[row];
                m = st.x;
                l = st.y;
            } else {
                const float2 v = p.tail_stat[slot];
                m = v.x;
                l = v.y;
            }
        }
        float mx = m;
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        mx = fmaxf(mx, M);
        const float keep = M == -INFINITY ? 0.0f : exp2_fast(M - mx);
        const float w = m == -INFINITY ? 0.0f : exp2_fast(m - mx);
        float lw = l * w;
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) lw += __shfl_xor_sync(0xffffffffu, lw, k);
        M = mx;
        L = L * keep + lw;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float kq = __shfl_sync(0xffffffffu, keep, q * 8);
            o[q].x *= kq;
            o[q].y *= kq;
            o[q].z *= kq;
            o[q].w *= kq;
        }
        for (int i = 0; i < min(8, n - base); i += 4) {
            float4 v[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int cc = c0 + base + i + k;
                const float* src = (cc == c0 ? p.head : p.tail) + ((int64_t)cc * p.slot_rows + (blockIdx.y * 4 + warp) * 4) * a.D + lane * 4;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    v[k][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (cc <= rec.x && live && (blockIdx.y * 4 + warp) * 4 + q < p.slot_rows && br - lane / 8 + q < rec.w)
                        v[k][q] = *reinterpret_cast<const float4*>(src + q * a.D);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float wq = __shfl_sync(0xffffffffu, w, q * 8 + i + k);
                    o[q].x = fmaf(v[k][q].x, wq, o[q].x);
                    o[q].y = fmaf(v[k][q].y, wq, o[q].y);
                    o[q].z = fmaf(v[k][q].z, wq, o[q].z);
                    o[q].w = fmaf(v[k][q].w, wq, o[q].w);
                }
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float iq = __shfl_sync(0xffffffffu, inv, q * 8);
        const bool go = __shfl_sync(0xffffffffu, (int)on, q * 8) && live;
        const int64_t to = __shfl_sync(0xffffffffu, row, q * 8);
        if (!go) continue;
        TQ* dst = static_cast<TQ*>(a.out) + to * a.D + lane * 4;
        if constexpr (sizeof(TQ) == 4) {
            *reinterpret_cast<float4*>(dst) = make_float4(o[q].x * iq, o[q].y * iq, o[q].z * iq, o[q].w * iq);
        } else {
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(Half2Of<T16>::pack(o[q].x * iq, o[q].y * iq), Half2Of<T16>::pack(o[q].z * iq, o[q].w * iq));
        }
    }
}

template <typename TQ, typename TK, int DP, int NT, bool SPLIT>
void launch_decode_t(const BeaconCudaContext* ctx, const PagedArgs& a, const CacheMaps& maps, const PartArgs& rest, cudaStream_t s, bool pdl, bool after_tc) {
    auto kern = paged_decode_kernel<TQ, TK, DP, NT, SPLIT>;
    static std::atomic<uint64_t> allowed{0};
    allow_smem_once(kern, ctx, allowed);
    launch_kernel(kern, dim3((unsigned)rest.ctas), dim3(kDecThreads), DecodeSmem<DP, NT, SPLIT>::bytes, s, pdl, a, maps, rest,
                  (int)after_tc);
}

template <int DP, int NT>
void launch_decode_d(const BeaconCudaContext* ctx, const PagedArgs& a, const CacheMaps& maps, const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s,
                     bool pdl, bool after_tc) {
    using H = __half;
    using B = __nv_bfloat16;
    if (tq == BEACON_CUDA_DTYPE_F32) launch_decode_t<float, H, DP, NT, true>(ctx, a, maps, rest, s, pdl, after_tc);
    else if (tk == BEACON_CUDA_DTYPE_F16) launch_decode_t<H, H, DP, NT, false>(ctx, a, maps, rest, s, pdl, after_tc);
    else launch_decode_t<B, B, DP, NT, false>(ctx, a, maps, rest, s, pdl, after_tc);
}

}  // namespace

int paged_decode_ctas(const BeaconCudaContext* ctx, const PagedArgs& a) {
    (void)a;
    return 2 * ctx->sm_count;
}

void launch_paged_decode(const BeaconCudaContext* ctx, const PagedArgs& a, const CacheMaps& maps, const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s,
                         bool pdl, bool after_tc) {
    // up to 8 heads fit one column block of the matrix instructions
    if (a.D <= 64 && a.G <= 8) launch_decode_d<64, 1>(ctx, a, maps, rest, tq, tk, s, pdl, after_tc);
    else if (a.D <= 64) launch_decode_d<64, 2>(ctx, a, maps, rest, tq, tk, s, pdl, after_tc);
    else if (a.G <= 8) launch_decode_d<128, 1>(ctx, a, maps, rest, tq, tk, s, pdl, after_tc);
    else launch_decode_d<128, 2>(ctx, a, maps, rest, tq, tk, s, pdl, after_tc);
}

void launch_paged_combine(const PagedArgs& a, const PartArgs& prefix, const PartArgs& rest, int32_t tq, cudaStream_t s) {
    auto go = [&](auto rows, auto cuts) {
        if (rest.by_row || !a.qstarts)
            launch_kernel(rows, dim3((unsigned)(((int64_t)a.T * a.H + 3) / 4)), dim3(128), 0, s, true, a, prefix, rest);
        else
            launch_kernel(cuts, dim3((unsigned)rest.ctas, (unsigned)((rest.slot_rows + 15) / 16)), dim3(128), 0, s, true, a, rest);
    };
    if (tq == BEACON_CUDA_DTYPE_F32) go(paged_join_rows_kernel<float, __half>, paged_join_cuts_kernel<float, __half>);
    else if (tq == BEACON_CUDA_DTYPE_F16) go(paged_join_rows_kernel<__half, __half>, paged_join_cuts_kernel<__half, __half>);
    else go(paged_join_rows_kernel<__nv_bfloat16, __nv_bfloat16>, paged_join_cuts_kernel<__nv_bfloat16, __nv_bfloat16>);
}

}  // namespace bc
