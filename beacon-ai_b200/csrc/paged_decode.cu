// paged_decode.cu -- paged attention of single query rows (decode) and the
// join of partial results.
//
// o = sum_p 2^(t_p - m) v_p / sum_p 2^(t_p - m), t_p = scale log2(e) q . k_p,
// over the keys of a row behind its group's prefix. The G query heads of one
// KV head share its keys, so the bound is reading the cache once. A tile is 64
// keys, 16 for each of the 4 warps of a CTA, which brings them in with 16-byte
// asynchronous copies through its own ring (no CTA barrier in the loop), forms
// the scores and the value sums with m16n8k16 instructions (the G <= 16 heads
// as rows) and keeps its own running maximum. The tiles of all sequences and
// KV heads form one line that the CTAs share evenly (PartArgs): a batch of
// uneven lengths loads every SM alike whatever the lengths are, and the lengths
// may change between replays of a captured call.
#include <algorithm>
#include <cmath>

#include "internal.h"
#include "kernels.h"
#include "paged_attn.h"
#include "paged_mma.cuh"

namespace bc {
namespace {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16 * kDecWarps;  // keys of a tile

template <int DP>
struct DecodeSmem {
    static constexpr int stages = DP == 128 ? 3 : 4;
    static constexpr int sub = 16 * DP * 2;        // bytes of 16 key (or value) rows
    static constexpr int ring = stages * 2 * sub;  // of one warp
    // merge area: [warp][rows][DP] sums, then m and l
    static constexpr size_t bytes(int rows) { return (size_t)kDecWarps * (ring + rows * DP * 4 + 2 * rows * 4); }
};

struct Span {  // keys [from, to) of one sequence, in tiles
    int from = 0, to = 0, tiles = 0;
};
__device__ __forceinline__ Span rest_of(const PagedArgs& a, int b) {
    Span s;
    if (b >= a.B) return s;
    const SeqInfo i = seq_info(a, b);
    s.from = i.prefix;
    s.to = i.len;
    s.tiles = s.to > s.from ? (s.to - s.from + kDecKeys - 1) / kDecKeys : 0;
    return s;
}

// Place in the line of tiles: sequence, KV head, tile.
struct Walk {
    int b = 0, kvh = 0, tile = 0;
    Span cur, next;  // the sequence after b is fetched ahead of its use
    __device__ __forceinline__ void step(const PagedArgs& a) {
        if (++tile < cur.tiles) return;
        tile = 0;
        if (++kvh < a.Hkv) return;
        kvh = 0;
        do {
            ++b;
            cur = next;
            next = rest_of(a, b + 1);
        } while (b < a.B && cur.tiles == 0);
    }
};

template <typename TQ, typename TK, int DP, bool SPLIT>
__global__ void __launch_bounds__(kDecThreads) paged_decode_kernel(const PagedArgs a, const PartArgs part) {
    using S = DecodeSmem<DP>;
    constexpr int NS = S::stages;
    constexpr int KSTEPS = DP / 16;
    constexpr int CH = DP / 8;            // 16-byte chunks of a row
    constexpr int RPI = 32 / CH;          // rows that one copy instruction of a warp covers
    extern __shared__ __align__(128) uint8_t dec_smem[];
    __shared__ long long sums_s[kDecWarps];
    __shared__ int b_s;
    __shared__ long long before_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.G <= 8 ? 8 : 16;   // rows of the merge area
    uint8_t* ring = dec_smem + warp * S::ring;
    float* merge_o = reinterpret_cast<float*>(dec_smem + kDecWarps * S::ring);  // [warp][rows][DP]
    float* merge_m = merge_o + kDecWarps * rows * DP;                           // [warp][rows]
    float* merge_l = merge_m + kDecWarps * rows;
    pdl_wait();

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
    const int ctas = sharers(total, part.ctas);
    const long long u0 = cta < ctas ? share_begin(total, ctas, cta) : 0, u1 = cta < ctas ? share_begin(total, ctas, cta + 1) : 0;
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
        load.next = rest_of(a, load.b + 1);
        const long long off = u0 - before_s * a.Hkv;
        load.kvh = (int)(off / load.cur.tiles);
        load.tile = (int)(off - (long long)load.kvh * load.cur.tiles);
        Walk at = load;
        const int count = (int)(u1 - u0);
        const int rl = lane / CH, chunk16 = lane % CH;
        const bool chunk_live = chunk16 * 8 < a.D;

        // this lane's key of a tile and its page (fetched a tile ahead)
        struct Key {
            int pos, page;  // pos -1: no key
        };
        auto key_of = [&](const Walk& w) {
            const int p = w.cur.from + w.tile * kDecKeys + warp * 16 + (lane & 15);
            Key k{-1, 0};
            if (p < w.cur.to) k = Key{p, page_id(a, w.b, p)};
            return k;
        };
        auto copy_tile = [&](int stage, int kvh, Key k) {
            const int row = k.pos >= 0 ? (int)page_row(a, k.page, k.pos) : -1;
            const uint32_t dst = smem_u32(ring + stage * 2 * S::sub);
#pragma unroll
            for (int i = 0; i < 16 / RPI; ++i) {
                const int r = i * RPI + rl;
                const int cr = __shfl_sync(0xffffffffu, row, r);
                const bool live = cr >= 0 && chunk_live;
                const int64_t src = live ? ((int64_t)cr * a.Hkv + kvh) * a.D + chunk16 * 8 : 0;
                const uint32_t d = dst + r * (DP * 2) + ((chunk16 ^ (r & 7)) << 4);
                cp_async16_zfill(d, static_cast<const TK*>(a.ck) + src, live);
                cp_async16_zfill(d + S::sub, static_cast<const TK*>(a.cv) + src, live);
            }
        };
        Key key_next = key_of(load);
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) {
            if (i < count) {
                copy_tile(i, load.kvh, key_next);
                load.step(a);
                if (i + 1 < count) key_next = key_of(load);
            }
            cp_async_commit();
        }

        uint32_t qf[KSTEPS][4], ql[SPLIT ? KSTEPS : 1][4];
        float cs[2], m[2], l[2], o[DP / 8][4];
        long long u = u0;
        bool fresh = true;
        for (int j = 0; j < count; ++j, ++u) {
            if (fresh) {
                // the G query rows of (b, kvh) as A fragments (rows lane / 4 and + 8)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int g = lane / 4 + 8 * r;
                    const TQ* q = static_cast<const TQ*>(a.q) + ((int64_t)at.b * a.H + at.kvh * a.G + g) * a.D;
                    float v[KSTEPS][4];
                    float mx = 0.0f;
#pragma unroll
                    for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int d = k * 16 + h * 8 + (lane & 3) * 2;
                            const bool live = g < a.G && d < a.D;
                            if constexpr (SPLIT) {
                                const float2 x = live ? *reinterpret_cast<const float2*>(q + d) : make_float2(0.0f, 0.0f);
                                v[k][2 * h] = x.x;
                                v[k][2 * h + 1] = x.y;
                                mx = fmaxf(mx, fmaxf(fabsf(x.x), fabsf(x.y)));
                            } else {
                                qf[k][r + 2 * h] = live ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                            }
                        }
                    cs[r] = a.scale * 1.4426950408889634f;
                    if constexpr (SPLIT) {
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        float inv;
                        const float sc = query_scale(mx, inv);
                        cs[r] *= inv;
#pragma unroll
                        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                split_f16(v[k][2 * h] * sc, v[k][2 * h + 1] * sc, qf[k][r + 2 * h], ql[k][r + 2 * h]);
                    }
                    m[r] = -INFINITY;
                    l[r] = 0.0f;
                }
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
                fresh = false;
            }
            cp_async_wait<NS - 2>();
            __syncwarp();  // the tile has landed for every lane, and all have read the stage refilled next
            if (j + NS - 1 < count) {
                copy_tile((j + NS - 1) % NS, load.kvh, key_next);
                load.step(a);
                if (j + NS < count) key_next = key_of(load);
            }
            cp_async_commit();

            const int first = at.cur.from + at.tile * kDecKeys + warp * 16;
            if (first < at.cur.to) {
                const uint32_t ks = smem_u32(ring + (j % NS) * 2 * S::sub), vs = ks + S::sub;
                const int lr = lane & 7, mi = lane >> 3;
                float sc[2][4] = {};
#pragma unroll
                for (int k = 0; k < KSTEPS; ++k) {
                    uint32_t b[4];
                    const int r = lr + (mi & 2) * 4, c = 2 * k + (mi & 1);
                    ldsm4(b, ks + r * (DP * 2) + ((c ^ (r & 7)) << 4));
                    mma16816<TK>(sc[0], qf[k], b[0], b[1]);
                    mma16816<TK>(sc[1], qf[k], b[2], b[3]);
                    if constexpr (SPLIT) {
                        mma16816<TK>(sc[0], ql[k], b[0], b[1]);
                        mma16816<TK>(sc[1], ql[k], b[2], b[3]);
                    }
                }
                // scores of keys first + 8 n + 2 (lane % 4) + e, rows lane / 4 + 8 r
                float mx[2] = {m[0], m[1]};
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = first + 8 * n + 2 * (lane & 3) + (e & 1);
                        sc[n][e] = key < at.cur.to ? sc[n][e] * cs[e >> 1] : -INFINITY;
                        mx[e >> 1] = fmaxf(mx[e >> 1], sc[n][e]);
                    }
                float keep[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    keep[r] = m[r] == -INFINITY ? 1.0f : exp2_fast(m[r] - mx[r]);
                    m[r] = mx[r];
                    l[r] *= keep[r];
                }
                if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n) {
                        o[n][0] *= keep[0];
                        o[n][1] *= keep[0];
                        o[n][2] *= keep[1];
                        o[n][3] *= keep[1];
                    }
                }
                const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[n][e] = exp2_fast(sc[n][e] - ref[e >> 1]);
                        l[e >> 1] += sc[n][e];
                    }
                    if constexpr (SPLIT) {
                        split_f16(sc[n][0], sc[n][1], ph[2 * n], pl[2 * n]);
                        split_f16(sc[n][2], sc[n][3], ph[2 * n + 1], pl[2 * n + 1]);
                    } else {
                        ph[2 * n] = Half2Of<TK>::pack(sc[n][0], sc[n][1]);
                        ph[2 * n + 1] = Half2Of<TK>::pack(sc[n][2], sc[n][3]);
                    }
                }
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t b[4];
                    const int r = lr + (mi & 1) * 8, c = 2 * d + (mi >> 1);
                    ldsm4_t(b, vs + r * (DP * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (SPLIT) {
                            // the instruction's sums truncate: a long chain of them would
                            // drift, so each tile's is added with rounding
                            float t[4] = {};
                            mma16816<TK>(t, ph, b[2 * h], b[2 * h + 1]);
                            mma16816<TK>(t, pl, b[2 * h], b[2 * h + 1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[2 * d + h][e] += t[e];
                        } else {
                            mma16816<TK>(o[2 * d + h], ph, b[2 * h], b[2 * h + 1]);
                        }
                    }
                }
            }

            const bool last_of_head = at.tile + 1 == at.cur.tiles;
            if (last_of_head || j + 1 == count) {
                // join the warps' sums of (b, kvh)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                    const int g = lane / 4 + 8 * r;
                    if (g < a.G) {
                        if ((lane & 3) == 0) {
                            merge_m[warp * rows + g] = m[r];
                            merge_l[warp * rows + g] = l[r];
                        }
                        float* mo = merge_o + (warp * rows + g) * DP;
#pragma unroll
                        for (int n = 0; n < DP / 8; ++n)
                            *reinterpret_cast<float2*>(mo + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                    }
                }
                __syncthreads();
                const long long tile0 = u - at.tile;  // of this head, in the line
                const int c0 = share_of(total, ctas, tile0);
                const int c1 = share_of(total, ctas, tile0 + at.cur.tiles - 1);
                const bool done = c0 == c1 && at.cur.from == 0;  // no other part anywhere
                for (int i = tid; i < a.G * DP; i += kDecThreads) {
                    const int g = i / DP, d = i % DP;
                    float M = merge_m[g];
#pragma unroll
                    for (int w = 1; w < kDecWarps; ++w) M = fmaxf(M, merge_m[w * rows + g]);
                    float acc = 0.0f, sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < kDecWarps; ++w) {
                        const float mw = merge_m[w * rows + g];
                        const float wt = mw == -INFINITY ? 0.0f : exp2_fast(mw - M);
                        acc = fmaf(merge_o[(w * rows + g) * DP + d], wt, acc);
                        sum = fmaf(merge_l[w * rows + g], wt, sum);
                    }
                    if (d >= a.D) continue;
                    const int64_t row = (int64_t)at.b * a.H + at.kvh * a.G + g;
                    if (done) {
                        const float r = sum == 0.0f ? 0.0f : acc / sum;
                        TQ* dst = static_cast<TQ*>(a.out) + row * a.D + d;
                        if constexpr (sizeof(TQ) == 4) *dst = r;
                        else if constexpr (sizeof(TK) == 2) {
                            const uint32_t v = Half2Of<TK>::pack(r, 0.0f);
                            *reinterpret_cast<uint16_t*>(dst) = (uint16_t)v;
                        }
                    } else if (c0 == cta) {
                        const int64_t slot = part.by_row ? row : (int64_t)cta * part.slot_rows + g;
                        part.head[slot * a.D + d] = acc;
                    } else {
                        part.tail[((int64_t)cta * part.slot_rows + g) * a.D + d] = acc;
                    }
                    if (d == 0) {
                        if (c0 == cta) part.stat[row] = make_float4(M, sum, __int_as_float(c0), __int_as_float(c1));
                        else part.tail_stat[(int64_t)cta * part.slot_rows + g] = make_float2(M, sum);
                    }
                }
                __syncthreads();  // the merge area is written again by the next head
                fresh = true;
            }
            at.step(a);
        }
        cp_async_wait<0>();
    }
    // kernels launched after this one count on everything before it
    pdl_wait();
}

// The parts of the query rows of one token: both kinds, each a first part and
// those of the CTAs after it. A warp takes a head at a time; the token's place
// is worked out once for the block's heads.
template <typename TQ, typename T16>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedArgs a, const PartArgs prefix, const PartArgs rest, int heads) {
    const int lane = threadIdx.x & 31;
    pdl_wait();
    const int t = blockIdx.x;
    const int b = a.qstarts ? span_of(a.qstarts, a.B, t) : t;
    if (b < 0) return;
    const SeqInfo s = seq_info(a, b);
    const int limit = min(s.len, s.len - s.nq + (t - s.q0) + 1);
    const bool on[2] = {!a.merged && min(s.prefix, limit) > 0, limit > (a.merged ? 0 : s.prefix)};
    // first token of the row block that the prefix's CTAs share
    const int q0 = on[0] ? (a.qstarts ? start_at(a.qstarts, s.first, a.T, a.err) : s.first) : 0;
    const bool live = lane * 4 < a.D;
    const int h1 = min(a.H, (int)(blockIdx.y + 1) * heads);
    for (int h = blockIdx.y * heads + (threadIdx.x >> 5); h < h1; h += 4) {
        const int64_t row = (int64_t)t * a.H + h;
        float4 st[2];
        if (on[0]) st[0] = prefix.stat[row];
        if (on[1]) st[1] = rest.stat[row];
        float M = -INFINITY, L = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        bool written = false;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            if (!on[kind]) continue;
            const PartArgs& p = kind ? rest : prefix;
            const int c0 = __float_as_int(st[kind].z), c1 = __float_as_int(st[kind].w);
            if (c0 < 0 || c1 < c0 || c1 >= p.ctas) {  // start arrays that contradict each other: no CTA had the row
                *a.err = kErrIndex;
                continue;
            }
            if (kind == 1 && !on[0] && c0 == c1) {  // written by the CTA that had all of it
                written = true;
                continue;
            }
            const int r = (int)(((int64_t)max(0, t - (kind ? s.q0 : q0)) * a.G + h % a.G) % p.slot_rows);
            const float* first = p.head + (p.by_row ? row : (int64_t)c0 * p.slot_rows + r) * a.D;
            for (int base = c0; base <= c1; base += 32) {
                const int c = base + lane;
                float m = -INFINITY, l = 0.0f;
                if (c <= c1) {
                    if (c == c0) {
                        m = st[kind].x;
                        l = st[kind].y;
                    } else {
                        const float2 v = p.tail_stat[(int64_t)c * p.slot_rows + r];
                        m = v.x;
                        l = v.y;
                    }
                }
                const float mx = fmaxf(M, warp_max(m));
                if (mx == -INFINITY) continue;
                const float keep = M == -INFINITY ? 0.0f : exp2_fast(M - mx);
                const float w = m == -INFINITY ? 0.0f : exp2_fast(m - mx);
                M = mx;
                L = L * keep + warp_sum(l * w);
                o.x *= keep;
                o.y *= keep;
                o.z *= keep;
                o.w *= keep;
                const int n = min(32, c1 - base + 1);
#pragma unroll 8
                for (int i = 0; i < n; ++i) {
                    const float wi = __shfl_sync(0xffffffffu, w, i);
                    const float* src = base + i == c0 ? first : p.tail + ((int64_t)(base + i) * p.slot_rows + r) * a.D;
                    if (live) {
                        const float4 v = *reinterpret_cast<const float4*>(src + lane * 4);
                        o.x = fmaf(v.x, wi, o.x);
                        o.y = fmaf(v.y, wi, o.y);
                        o.z = fmaf(v.z, wi, o.z);
                        o.w = fmaf(v.w, wi, o.w);
                    }
                }
            }
        }
        if (!live || written) continue;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        TQ* dst = static_cast<TQ*>(a.out) + row * a.D + lane * 4;
        if constexpr (sizeof(TQ) == 4) {
            *reinterpret_cast<float4*>(dst) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
            *reinterpret_cast<uint2*>(dst) = make_uint2(Half2Of<T16>::pack(o.x * inv, o.y * inv), Half2Of<T16>::pack(o.z * inv, o.w * inv));
        }
    }
}

template <typename TQ, typename TK, int DP, bool SPLIT>
void launch_decode_t(const PagedArgs& a, const PartArgs& rest, cudaStream_t s, bool pdl) {
    auto kern = paged_decode_kernel<TQ, TK, DP, SPLIT>;
    allow_max_dynamic_smem(kern);
    launch_kernel(kern, dim3((unsigned)rest.ctas), dim3(kDecThreads), DecodeSmem<DP>::bytes(a.G <= 8 ? 8 : 16), s, pdl, a, rest);
}

template <int DP>
void launch_decode_d(const PagedArgs& a, const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s, bool pdl) {
    if (tq == BEACON_CUDA_DTYPE_F32) launch_decode_t<float, __half, DP, true>(a, rest, s, pdl);
    else if (tk == BEACON_CUDA_DTYPE_F16) launch_decode_t<__half, __half, DP, false>(a, rest, s, pdl);
    else launch_decode_t<__nv_bfloat16, __nv_bfloat16, DP, false>(a, rest, s, pdl);
}

}  // namespace

int paged_decode_ctas(const BeaconCudaContext* ctx, const PagedArgs& a, bool split) {
    (void)split;
    return 2 * ctx->sm_count;
}

void launch_paged_decode(const PagedArgs& a, const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s, bool pdl) {
    if (a.D <= 64) launch_decode_d<64>(a, rest, tq, tk, s, pdl);
    else launch_decode_d<128>(a, rest, tq, tk, s, pdl);
}

void launch_paged_combine(const PagedArgs& a, const PartArgs& prefix, const PartArgs& rest, int32_t tq, cudaStream_t s) {
    // four heads a block (one a warp) until the device is full, then more
    const int64_t blocks = (int64_t)a.T * ((a.H + 3) / 4);
    const int heads = (int)std::min<int64_t>((a.H + 3) / 4, std::max<int64_t>(1, blocks / 2048)) * 4;
    const dim3 grid((unsigned)a.T, (unsigned)((a.H + heads - 1) / heads));
    if (tq == BEACON_CUDA_DTYPE_F32) launch_kernel(paged_combine_kernel<float, __half>, grid, dim3(128), 0, s, true, a, prefix, rest, heads);
    else if (tq == BEACON_CUDA_DTYPE_F16) launch_kernel(paged_combine_kernel<__half, __half>, grid, dim3(128), 0, s, true, a, prefix, rest, heads);
    else launch_kernel(paged_combine_kernel<__nv_bfloat16, __nv_bfloat16>, grid, dim3(128), 0, s, true, a, prefix, rest, heads);
}

}  // namespace bc
