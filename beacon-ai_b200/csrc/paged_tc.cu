// paged_tc.cu -- paged attention of many query rows that share their keys
// (prefixes of a group of sequences, prompts) on the 5th-generation tensor
// cores.
//
// A row block is the query rows of one KV head that see the same keys: all
// sequences of a group against its prefix, or the rows of one sequence against
// its own keys (token-major, so row r is token r / G, head r % G). Per 128-key
// tile S = Q K^T and O += P V are chains of tcgen05.mma (M 128, K 16) with
// scores and sums in tensor memory. A CTA has two streams of them, each with
// its own 128 score and DP sum columns and its own 128 softmax threads (one
// row each), so that one stream's matrix products run under the other's
// exponentials:
//  * two row tiles (block of 256 rows) that share every key tile, or
//  * one row tile (128 rows) whose streams take the even and the odd key tiles
//    and are joined at the end. 32-bit queries come as two f16 parts (SPLIT):
//    two products for the scores, and two for the sums, whose weights are
//    split likewise.
// P replaces S in place, 32 keys at a time: the 16 columns of packed weights
// (then 16 of their remainders) lie where the 32 scores were, and are the A
// operand of O += P V from tensor memory; V is read N-major.
// Key and value rows come in page by page by tensor copies (TMA) of up to 128
// rows into a ring of tiles in the 128-byte swizzle, requested by four warps;
// rows of a value tile that are no keys of the block are zeroed there (their
// weights are zero, but what a page holds behind its last row may be no
// number). 16-byte asynchronous copies by the same warps, which zero-fill, serve
// page sizes that are no multiple of 8 (they reach 8 bytes a cycle and
// multiprocessor: the tensor copies are what feeds the matrix unit). One
// thread issues the products. The key tiles of all blocks form one line that the CTAs
// share evenly (PartArgs).
// The reference of the exponentials moves only when a tile exceeds it by some
// powers of two (kMost): the sums are rescaled in tensor memory then.
// Bounds, measured with both kernels around it (CUDA events): 4 prompts of 512
// rows over 4096 shared keys, bf16, 32 heads on 8 of 128: 163 us, 745 TFLOP/s of
// 1718, 39% tensor pipe. A pair of 128 x 128 tiles takes about 5,700 cycles, 2,048
// of them products; how the rest divides between the softmax threads and the
// hand-overs to them is not measured. 64 rows behind a prefix of 16384: 105 us of
// which 61 are here. 32 rows, 32-bit, behind 4096 keys: 49 us, of which 19 are here
// for 3.5 tiles a CTA: start, first use of the code and the first tile's latency.
// Every wait is bounded; one that runs out marks the stream's error word, and
// the CTA waits for what it issued and ends.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "internal.h"
#include "kernels.h"
#include "paged_attn.h"
#include "paged_mma.cuh"
#include "rotary.h"

namespace bc {
namespace {

constexpr int kTile = 128;              // rows of a row tile, keys of a key tile
constexpr int kSoftWarps = 8;
constexpr int kLoadWarp = 8, kLoadWarps = 4;
constexpr int kMmaWarp = 12;
constexpr int kTcThreads = 32 * (kMmaWarp + 1);
constexpr uint32_t kTmemCols = 512;     // S 2 x 128, O 2 x DP
// The weights are 2^(t - m) of scores t = scale log2(e) q . k and a reference m.
// A tile whose largest score comes to be kMost above m moves m up, to kLift
// below that score; the sums so far are rescaled then, which is rare. f16
// (kNarrowExponent): the largest weight is always between 2^11 and 2^15, so one
// of 2^-25 of it has all 11 bits and none is off by more than 2^-36 of the largest.
template <typename T>
constexpr float kMost = kNarrowExponent<T> ? 15.0f : 8.0f;
template <typename T>
constexpr float kLift = kNarrowExponent<T> ? 11.0f : 0.0f;
// The weights' fused operation does not round t, but m is made of a rounded one:
// for |t| from here on the difference, up to 2^-24 |t|, is taken care of.
constexpr float kFar = 0x1p18f;

template <int DP, bool SPLIT, bool TWO>
struct TcSmem {
    static constexpr int tile = kTile * DP * 2;
    static constexpr int q_tiles = TWO || SPLIT ? 2 : 1;
    static constexpr int stages = DP == 128 ? 6 - q_tiles : 8;
    static constexpr int stage_out = 32 * 64;  // per softmax warp: 64 bytes of each of its rows
    static constexpr size_t bytes = (size_t)(q_tiles + stages) * tile + kSoftWarps * stage_out + 1024;
};

// Shared-memory descriptors, 128-byte swizzle. K-major (queries, keys): 8-row
// atoms of 1024 bytes. N-major (values): 64 dims (128 bytes) of a key in a row,
// blocks of 64 dims 128 rows apart (leading offset), 8-key atoms 1024 bytes
// apart (stride offset).
__device__ __forceinline__ uint32_t desc_lo_k(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_n(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | ((uint32_t)((kTile * 128) >> 4) << 16); }
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
template <typename T>
constexpr uint32_t idesc(int n, bool b_n_major) {
    const uint32_t ty = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (ty << 7) | (ty << 10) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kTile >> 4) << 24);
}
// Products issued by the elected thread of a converged warp. The descriptors'
// upper halves are constants; only the address field (lower half) moves.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n}\n" ::"r"(d),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t on;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(on));
    return on != 0;
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// The rows that share keys: a group's queries against its prefix (kind 0), or a
// sequence's queries against its own keys (kind 1).
struct Block {
    int kind = 0;
    int b = 0;                   // page table row
    int cut = 0, first = 0;      // keys below cut are read through table row `first`
    int key0 = 0, key1 = 0;      // keys [key0, key1)
    int base = 0;                // where the first tile begins: key0, or the copy box that holds it
    int tok0 = 0, rows = 0;      // query rows tok0 * G ..
    int nq = 0, len = 0;         // kind 1: causal limits
};
__device__ __forceinline__ Block block_of(const PagedArgs& a, int e) {
    Block k;
    const int groups = a.merged ? 0 : a.groups;
    if (e < groups) {
        bool bad = false;
        int lo = __ldg(a.gstarts + e), hi = __ldg(a.gstarts + e + 1);
        const int p = __ldg(a.prefix + e);
        lo = keep_in(lo, a.B, bad);
        hi = keep_in(hi, a.B, bad);
        if (hi > lo) {
            const int len = __ldg(a.lens + lo);
            int t0 = lo, t1 = hi;
            if (a.qstarts) {
                t0 = __ldg(a.qstarts + lo);
                t1 = __ldg(a.qstarts + hi);
            }
            k.b = lo;
            k.key1 = min(keep_in(p, capacity(a), bad), keep_in(len, capacity(a), bad));
            k.tok0 = keep_in(t0, a.T, bad);
            k.rows = max(0, keep_in(t1, a.T, bad) - k.tok0) * a.G;
        }
        if (bad || hi < lo) a.err[kErrWordIndex] = 1;
        return k;
    }
    const SeqInfo s = seq_info(a, e - groups);
    k.kind = 1;
    k.b = e - groups;
    if (a.merged) {
        k.cut = s.prefix;
        k.first = s.first;
    } else {
        k.key0 = s.prefix;
    }
    k.base = a.box ? k.key0 & ~(a.box - 1) : k.key0;
    k.key1 = s.len;
    k.tok0 = s.q0;
    k.rows = s.nq * a.G;
    k.nq = s.nq;
    k.len = s.len;
    return k;
}
// Key tiles that row tile rt of a block needs (its last row sees the most keys);
// rows of a sequence have one at least, which then shows them nothing.
__device__ __forceinline__ int tiles_of(const PagedArgs& a, const Block& k, int rt, int block_rows) {
    int end = k.key1;
    if (k.kind) end = min(end, k.len - k.nq + (min((rt + 1) * block_rows, k.rows) - 1) / a.G + 1);
    return end > k.key0 ? (end - k.base + kTile - 1) / kTile : k.kind;
}
__device__ __forceinline__ int tiles_of_block(const PagedArgs& a, const Block& k, int block_rows) {
    const int n = (k.rows + block_rows - 1) / block_rows;
    if (k.kind == 0) return n * tiles_of(a, k, 0, block_rows);
    int sum = 0;
    for (int rt = 0; rt < n; ++rt) sum += tiles_of(a, k, rt, block_rows);
    return sum;
}

// Key tiles of a piece with 32-bit queries. The matrix unit cuts its sums to 24
// bits after every product, so a chain of n tiles shrinks them by about 1.7e-7 n
// of themselves; pieces are joined with rounding. 4 prompts of 1024 rows over
// 4096 keys, 32 heads on 8, D 128, off 64 bits and time: whole chains (16 tiles a
// stream) 3.4e-6, 383 us; 10 tiles (5 a stream) 1.7e-6, 463 us; 8 tiles 1.4e-6,
// 498 us; a plain form in 32 bits has 1.3e-6.
constexpr int kMostSplit = 10;

// A CTA's next piece of the line: key tiles [tile, tile + n) of row tile rt,
// at most MOST of them.
template <int MOST>
struct PieceOf {
    Block k;
    int e = 0, entries = 0, kvh = 0, rt = 0, tile = 0;
    int tiles = 0;     // of the row tile
    int n = 0;
    long long u = 0;   // place of `tile` in the line
    __device__ __forceinline__ void next(const PagedArgs& a, int block_rows, long long u1) {
        u += n;
        if (u >= u1) return;
        if (tile + n < tiles) {
            tile += n;
            n = (int)min((long long)min(tiles - tile, MOST), u1 - u);
            return;
        }
        tile = 0;
        for (;;) {
            ++rt;
            if ((long long)rt * block_rows >= k.rows) {
                rt = 0;
                if (++kvh == a.Hkv) {
                    kvh = 0;
                    if (++e >= entries) return;  // not reached while u < u1
                    k = block_of(a, e);
                }
                if (k.rows == 0) {
                    kvh = a.Hkv - 1;
                    rt = 0;
                    tiles = 0;
                    continue;
                }
            }
            tiles = tiles_of(a, k, rt, block_rows);
            if (tiles) break;
        }
        n = (int)min((long long)min(tiles, MOST), u1 - u);
    }
};

template <typename TQ, typename T16, int DP, bool SPLIT, bool TWO>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_tc_kernel(const PagedArgs a, const __grid_constant__ CacheMaps maps, const PartArgs prefix, const PartArgs rest, int entries,
                    int line_ctas, int least_tiles) {
    using SM = TcSmem<DP, SPLIT, TWO>;
    constexpr int NST = SM::stages;
    constexpr int LA = TWO ? 1 : 2;              // key tiles ahead of the value tile
    constexpr int BR = TWO ? 2 * kTile : kTile;  // rows of a block's row tile
    constexpr int CH = DP / 8;                   // 16-byte chunks of a row
    extern __shared__ uint8_t tc_smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[NST], empty_bar[NST], qfull_bar, qempty_bar, s_bar[2], p_bar[2], ofin_bar, join_bar,
        fix_bar, done_bar;
    __shared__ uint32_t tmem_s;
    __shared__ volatile int failed_s;
    __shared__ float qscale_s[2][kTile];   // SPLIT: what the scores are multiplied by
    __shared__ float2 join_s[2][kTile];    // !TWO: (m, l) of both streams
    __shared__ float2 so_far_s[2][kTile];  // SPLIT: (m, l) of the pieces of the row tile so far, each thread its own
    __shared__ long long sums_s[kTcThreads / 32];
    __shared__ long long before_s;
    __shared__ int entry_s;
    __shared__ int block_s[sizeof(Block) / sizeof(int)];
    uint8_t* q_smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = q_smem + SM::q_tiles * SM::tile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < NST; ++i) {
            mbar_init(&full_bar[i], a.box ? 1 : kLoadWarps * 32);
            mbar_init(&empty_bar[i], 1);
        }
        mbar_init(&qfull_bar, (SPLIT ? kSoftWarps : kLoadWarps) * 32);
        mbar_init(&qempty_bar, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_bar[i], 1);
            mbar_init(&p_bar[i], kTile);
        }
        mbar_init(&ofin_bar, 1);
        mbar_init(&join_bar, 2 * kTile);
        mbar_init(&fix_bar, 1);
        mbar_init(&done_bar, 1);
        failed_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();

    // this CTA's share of the line
    const int chunk = (entries + kTcThreads - 1) / kTcThreads;
    const int e0 = min(entries, tid * chunk), e1 = min(entries, e0 + chunk);
    long long mine = 0;
    Block own;  // the last of them
    for (int e = e0; e < e1; ++e) {
        own = block_of(a, e);
        mine += tiles_of_block(a, own, BR);
    }
    long long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) sums_s[warp] = scan;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_s;
    long long total = 0, before = scan - mine;
#pragma unroll
    for (int w = 0; w < kTcThreads / 32; ++w) {
        if (w < warp) before += sums_s[w];
        total += sums_s[w];
    }
    total *= a.Hkv;
    pdl_trigger();
    const int cta = blockIdx.x;
    // With single rows behind the prefixes the kernel of those starts on the SMs
    // that are free: few tiles go to half of them, four each (32 rows of a 4096-key
    // prefix: 55.4 -> 53.2 us with both kernels at once).
    const Shares shares(total, (int)min((long long)line_ctas, max((long long)line_ctas / 2, total / least_tiles)));
    const long long u0 = cta < shares.ctas ? shares.begin(cta) : 0, u1 = cta < shares.ctas ? shares.begin(cta + 1) : 0;
    if (u0 < u1 && before * a.Hkv <= u0 && u0 < (before + mine) * a.Hkv) {
        int e = e0;
        for (; e + 1 < e1; ++e) {
            const Block k = block_of(a, e);
            const int n = tiles_of_block(a, k, BR);
            if (u0 < (before + n) * a.Hkv) {
                own = k;
                break;
            }
            before += n;
        }
        entry_s = e;
        before_s = before;
        *reinterpret_cast<Block*>(block_s) = own;
    }
    __syncthreads();

    // no row block of this CTA is cut at its end, until one is
    if (tid == 0 && !rest.by_row) rest.cuts[cta * 8] = -1;
    using Piece = PieceOf<SPLIT ? kMostSplit : 0x7FFFFFFF>;
    Piece pc;
    if (u0 < u1) {
        pc.e = entry_s;
        pc.entries = entries;
        pc.k = *reinterpret_cast<const Block*>(block_s);
        const long long per = tiles_of_block(a, pc.k, BR), off = u0 - before_s * a.Hkv;
        pc.kvh = (int)(off / per);
        int at = (int)(off - pc.kvh * per);
        pc.tiles = tiles_of(a, pc.k, 0, BR);
        while (at >= pc.tiles) {
            at -= pc.tiles;
            pc.tiles = tiles_of(a, pc.k, ++pc.rt, BR);
        }
        pc.tile = at;
        pc.u = u0;
        pc.n = (int)min((long long)min(pc.tiles - at, SPLIT ? kMostSplit : 0x7FFFFFFF), u1 - u0);
    }
    const long long limit_cycles = g_wait_limit;
    auto give_up = [&]() {
        a.err[kErrWordWait] = 1;
        failed_s = 1;
    };

    if (warp >= kLoadWarp && warp < kLoadWarp + kLoadWarps) {
        // --- producers: queries, then key and value tiles in the order of their use
        const int pw = warp - kLoadWarp;
        const int64_t stride = (int64_t)a.Hkv * a.D * 2;  // bytes from one cache row to the next
        const int c = lane % CH;                          // this lane's chunk of the rows it copies
        const bool chunk_live = c * 8 < a.D;
        int it = 0, told = 0, nfix = 0;  // tiles requested, tiles announced
        bool ok = true;
        auto announce = [&](int upto) {  // tiles [told, upto) have landed
            if (told < upto) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            for (; told < upto; ++told) arrive(&full_bar[told % NST]);
        };
        constexpr int RPI = 32 / CH;  // rows that one copy instruction of a warp covers
        // The tiles of a piece in the order of their use: LA key tiles, then
        // value tile t and key tile t + LA in turn, then the last value tiles.
        auto key_tile = [&](const Piece& p, int f, bool& value) {
            const int la = min(LA, p.n), j = f - la, pairs = 2 * (p.n - la);
            value = j >= 0 && (j >= pairs || (j & 1) == 0);
            return j < 0 ? f : j >= pairs ? p.n - la + (j - pairs) : value ? j / 2 : j / 2 + la;
        };
        // Tensor copies, a box a lane: the lane's first key of a tile, its page, and
        // the cache row: -1 if there is none
        auto pos_of = [&](const Piece& p, int t) { return p.k.base + (p.tile + t) * kTile + lane * a.box; };
        auto page_of = [&](const Piece& p, int t) {
            const int pos = pos_of(p, t);
            if (!a.box || t >= p.n || pos >= p.k.key1 || lane * a.box >= kTile) return 0;
            return page_id(a, pos < p.k.cut ? p.k.first : p.k.b, pos);
        };
        auto row_of = [&](const Piece& p, int t, int page) {
            const int pos = pos_of(p, t);
            if (!a.box || pos >= p.k.key1 || lane * a.box >= kTile) return -1;
            const int row = (int)page_row(a, page, pos);
            return row < 0 ? (int)(a.pages * a.page_size) : row;  // a bad page: a box outside, zeros
        };
        auto room = [&]() {  // waits for the stage of tile `it`
            const uint32_t par = (uint32_t)((it / NST - 1) & 1);
            if (it >= NST && !mbar_test_wait(&empty_bar[it % NST], par)) {
                if (!a.box) {
                    cp_async_wait<0>();  // hand over all that is on its way before waiting
                    announce(it);
                }
                if (!wait_bar(&empty_bar[it % NST], par, limit_cycles) || failed_s) {
                    give_up();
                    ok = false;
                }
            }
            ok = __all_sync(0xffffffffu, ok);  // the lanes copy for each other: they go on or give up together
            return ok;
        };
        // Rows r0 .. r0 + 31 of a tile one by one, 16 bytes a lane (each lane looks one row up)
        auto copy_rows = [&](uint32_t dst, const Piece& p, const void* cache, int pos0, int r0) {
            const int q = pos0 + r0 + lane;
            const int row = q < p.k.key1 ? (int)page_row(a, page_id(a, q < p.k.cut ? p.k.first : p.k.b, q), q) : -1;
            dst += (c >> 3) * (kTile * 128);
            const uint8_t* src = static_cast<const uint8_t*>(cache) + (p.kvh * a.D + c * 8) * 2;
#pragma unroll 8
            for (int i = 0; i < 32 / RPI; ++i) {
                const int rr = i * RPI + lane / CH;
                const int cr = __shfl_sync(0xffffffffu, row, rr);
                const bool live = cr >= 0 && chunk_live;
                const int r = r0 + rr;
                cp_async16_zfill(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), live ? src + cr * stride : static_cast<const uint8_t*>(cache), live);
            }
        };
        auto load_tile = [&](const Piece& p, int t, bool value, int row) {
            if (!room()) return;
            const int pos0 = p.k.base + (p.tile + t) * kTile;
            const uint32_t dst = smem_u32(ring + (size_t)(it % NST) * SM::tile);
            if (!a.box) {
                for (int r0 = pw * 32; r0 < kTile; r0 += kLoadWarps * 32) copy_rows(dst, p, value ? a.cv : a.ck, pos0, r0);
                cp_async_commit();
                ++it;
                if (it - told > 2) {  // two tiles stay in flight
                    cp_async_wait<2>();
                    announce(it - 2);
                }
                return;
            }
            const int st = it++ % NST;
            const bool live = row >= 0;
            if (pos0 < p.k.cut && pos0 + kTile > p.k.cut && (p.k.cut & (a.box - 1))) {
                // a box whose rows lie in two tables: this tile row by row
                if (pw > 0) return;
                for (int r0 = 0; r0 < kTile; r0 += 32) copy_rows(dst, p, value ? a.cv : a.ck, pos0, r0);
                cp_async_commit();
                cp_async_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(&full_bar[st]);
                return;
            }
            // a value tile with rows that are no keys lands on fix_bar first
            const bool part = value && (pos0 < p.k.key0 || pos0 + kTile > p.k.key1);
            if (part && pw > 0) return;
            uint64_t* bar = part ? &fix_bar : &full_bar[st];
            const int boxes = __popc(__ballot_sync(0xffffffffu, live));
            // one arrival and all bytes from the first warp; the copies, whose
            // requests take a hundred cycles each, from all warps
            if (pw == 0 && lane == 0) mbar_expect_tx(bar, (uint32_t)(boxes * a.box * DP * 2));
            if (live && (part || lane % kLoadWarps == pw)) {
#pragma unroll
                for (int h = 0; h < DP / 64; ++h)
                    tma_rows(dst + h * (kTile * 128) + lane * a.box * 128, value ? &maps.v : &maps.k, h * 64, p.kvh, row, bar);
            }
            if (part) {
                if (!wait_bar(bar, (uint32_t)(nfix++ & 1), limit_cycles)) {
                    mbar_drain(bar, (uint32_t)((nfix - 1) & 1));
                    give_up();
                    ok = false;
                }
                const int lo = max(0, p.k.key0 - pos0), hi = max(lo, min(kTile, p.k.key1 - pos0));  // rows [lo, hi) are keys
                for (int i = lane; i < (lo + kTile - hi) * CH; i += 32) {
                    const int q = i / CH, r = q < lo ? q : hi + q - lo, cc = i % CH;
                    st_shared16(dst + (cc >> 3) * (kTile * 128) + r * 128 + ((cc & 7) << 4), 0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                ok = __all_sync(0xffffffffu, ok);
                if (lane == 0) arrive(&full_bar[st]);
            }
        };
        int seg = 0;
        for (Piece p = pc; ok && p.u < u1; p.next(a, BR, u1), ++seg) {
            // the first tiles are on their way while the queries are brought in
            // A key tile's pages are fetched when the one before it is requested, and
            // its rows kept for the value tile, up to LA of them.
            int f = 0, page = page_of(p, 0), rows[2] = {-1, -1}, kept = 0;
            auto load_next = [&]() {
                bool value;
                const int t = key_tile(p, f++, value);
                int row = rows[0];
                if (value) {
                    rows[0] = rows[1];
                    --kept;
                } else {
                    row = row_of(p, t, page);
                    page = page_of(p, t + 1);
                    if (kept == 0) rows[0] = row;
                    else rows[1] = row;
                    ++kept;
                }
                load_tile(p, t, value, row);
            };
            while (ok && f < min(3, 2 * p.n)) load_next();
            if (seg > 0 && !SPLIT) {
                if (!a.box) {
                    // the last products of the piece before need all of its tiles
                    cp_async_wait<0>();
                    announce(it);
                }
                if (!wait_bar(&qempty_bar, (uint32_t)((seg - 1) & 1), limit_cycles) || failed_s) {
                    give_up();
                    ok = false;
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if constexpr (!SPLIT) {
#pragma unroll 1
                for (int r0 = pw * 32; r0 < BR; r0 += kLoadWarps * 32) {
                    // this lane's query row, as a row of [T * H][D]; -1: behind the block
                    const int br = p.rt * BR + r0 + lane;
                    const int qrow = br < p.k.rows ? (p.k.tok0 + br / a.G) * a.H + p.kvh * a.G + br % a.G : -1;
                    const uint32_t dst = smem_u32(q_smem) + (r0 / kTile) * SM::tile + (c >> 3) * (kTile * 128);
#pragma unroll 8
                    for (int k = 0; k < 32 / RPI; ++k) {
                        const int rr = k * RPI + lane / CH;
                        const int qr = __shfl_sync(0xffffffffu, qrow, rr);
                        const bool live = qr >= 0 && chunk_live;
                        const int r = r0 % kTile + rr;
                        cp_async16_zfill(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                                         static_cast<const TQ*>(a.q) + (live ? (int64_t)qr * a.D + c * 8 : 0), live);
                    }
                }
            }
            if (!SPLIT) {
                cp_async_commit();
                cp_async_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(&qfull_bar);
            }
            while (ok && f < 2 * p.n) load_next();
        }
        // nothing may land after the CTA has ended
        cp_async_wait<0>();
        if (!a.box && ok) announce(it);
        // (after a wait that gave up some warp's part may not have been requested:
        // one limit for all stages, far beyond any copy's time)
        if (a.box && pw == 0) {
            const long long t0 = clock64();
            for (int i = max(0, it - NST); i < it; ++i)
                while (!mbar_try_wait(&full_bar[i % NST], (uint32_t)((i / NST) & 1)) && clock64() - t0 <= kBoundedWaitLimit) {
                }
        }
    } else if (warp >= kMmaWarp) {
        if (warp == kMmaWarp) {
            // the whole warp waits; its elected thread issues
            int it = 0, np[2] = {0, 0};
            bool ok = true;
            const uint32_t qa = smem_u32(q_smem), ra = smem_u32(ring);
            auto wait = [&](uint64_t* bar, uint32_t par) {
                if (ok && (!wait_bar(bar, par, limit_cycles) || failed_s)) {
                    give_up();
                    ok = false;
                }
                ok = __all_sync(0xffffffffu, ok);
                fence_after();
            };
            auto acquire = [&]() {
                wait(&full_bar[it % NST], (uint32_t)((it / NST) & 1));
                return it++ % NST;
            };
            constexpr int kParts = SPLIT ? 2 : 1;
            constexpr uint32_t id_qk = idesc<T16>(kTile, false), id_pv = idesc<T16>(DP, true);
            // S_s = Q K^T; then announces it and, if it was the tile's last use, frees the tile
            auto scores = [&](int s, int st, bool last) {
                if (elect_one()) {
                    const uint32_t d = tmem + s * kTile, b = desc_lo_k(ra + st * SM::tile);
                    // the small parts first: sums in the matrix unit are cut to 24 bits
                    // after every product, which costs nothing while they are small
#pragma unroll
                    for (int i = 0; i < kParts; ++i) {
                        const uint32_t q = desc_lo_k(qa + (TWO ? s : kParts - 1 - i) * SM::tile);
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k) {
                            const uint32_t off = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
                            mma_ss(d, q + off, kDescHi, b + off, kDescHi, id_qk, i + k > 0);
                        }
                    }
                    commit(&s_bar[s]);
                    if (last) commit(&empty_bar[st]);
                }
                __syncwarp();
            };
            // O_s += P V
            auto sums = [&](int s, int st, bool first, bool last) {
                wait(&p_bar[s], (uint32_t)(np[s]++ & 1));
                if (!ok) return;
                if (elect_one()) {
                    const uint32_t o = tmem + 2 * kTile + s * DP, p = tmem + s * kTile, b = desc_lo_n(ra + st * SM::tile);
#pragma unroll
                    for (int i = 0; i < kParts; ++i)
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)
                            mma_ts(o, p + (k >> 1) * 32 + (k & 1) * 8 + (kParts - 1 - i) * 16, b + k * (2048 >> 4), kDescHi, id_pv, i + k > 0 || !first);
                    if (last) commit(&empty_bar[st]);
                }
                __syncwarp();
            };
            int seg = 0;
            for (Piece p = pc; ok && p.u < u1; p.next(a, BR, u1), ++seg) {
                wait(&qfull_bar, (uint32_t)(seg & 1));
                for (int t = 0; ok && t < min(LA, p.n); ++t) {
                    const int st = acquire();
                    if (!ok) break;
                    scores(t, st, !TWO);
                    if (TWO) scores(1, st, true);
                }
                for (int t = 0; ok && t < p.n; ++t) {
                    const int sv = acquire();
                    if (!ok) break;
                    if (TWO) {
                        sums(0, sv, t == 0, false);
                        int sk = 0;
                        if (ok && t + 1 < p.n) {
                            sk = acquire();
                            if (ok) scores(0, sk, false);
                        }
                        if (ok) sums(1, sv, t == 0, true);
                        if (ok && t + 1 < p.n) scores(1, sk, true);
                    } else {
                        sums(t & 1, sv, t < 2, true);
                        if (ok && t + 2 < p.n) {
                            const int sk = acquire();
                            if (ok) scores(t & 1, sk, true);
                        }
                    }
                }
                if (!ok) break;
                if (elect_one()) {
                    commit(&qempty_bar);
                    commit(&ofin_bar);
                }
                __syncwarp();
            }
            if (elect_one()) commit(&done_bar);  // completes once every product issued above has
            __syncwarp();
        }
    } else {
        // --- softmax: stream s, row r of its tile
        const int s = warp >> 2, r = tid & (kTile - 1);
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + lane_at + s * kTile;
        int ns = 0, seg = 0, nj = 0;
        bool ok = true;
        int loads = 0;  // of queries (SPLIT)
        auto wait = [&](uint64_t* bar, uint32_t par) {
            if (ok && (!wait_bar(bar, par, limit_cycles) || failed_s)) {
                give_up();
                ok = false;
            }
            ok = __all_sync(0xffffffffu, ok);  // the warp's tensor memory accesses are collective
            fence_after();
        };
        for (Piece p = pc; ok && p.u < u1; p.next(a, BR, u1), ++seg) {
            const int row = p.rt * BR + (TWO ? s * kTile : 0) + r;  // of the block
            const bool live = row < p.k.rows;
            const int tok = p.k.tok0 + row / a.G;
            int limit = 0x7FFFFFFF;  // rows behind the block: whatever comes out is not written
            if (live) {
                if (p.k.kind) {
                    limit = min(p.k.len, p.k.len - p.k.nq + row / a.G + 1);
                } else if (!a.qstarts) {
                    limit = max(0, min(p.k.key1, __ldg(a.lens + tok)));
                } else {
                    const int b = span_of(a.qstarts, a.B, tok);
                    limit = 0;
                    if (b >= 0) {
                        const int len = max(0, (int)min((long long)__ldg(a.lens + b), capacity(a)));
                        limit = min(p.k.key1, len - __ldg(a.qstarts + b + 1) + tok + 1);
                    }
                }
            }
            const bool goes_on = SPLIT && seg > 0 && p.tile > 0;  // the row tile of the piece before
            if (SPLIT && !goes_on) {
                ++loads;
                // the block's queries as two f16 parts: 16 rows a warp, a row at a
                // time (each lane four values), eight on their way
                if (seg > 0) wait(&qempty_bar, (uint32_t)((seg - 1) & 1));
                if (!ok) break;
                const int mine = p.rt * BR + warp * 16 + (lane & 15);
                const int qrow = mine < p.k.rows ? (p.k.tok0 + mine / a.G) * a.H + p.kvh * a.G + mine % a.G : -1;
#pragma unroll 1
                for (int r0 = 0; r0 < 16; r0 += 8) {
                    float4 x[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int qr = __shfl_sync(0xffffffffu, qrow, r0 + k);
                        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (qr >= 0 && lane * 4 < a.D)
                            x[k] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + (int64_t)qr * a.D + lane * 4);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int qr = warp * 16 + r0 + k;
                        const float mx = warp_max(fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
                        float inv;
                        const float sc = query_scale(mx, inv);
                        if (lane == 0) qscale_s[loads & 1][qr] = a.scale * 1.4426950408889634f * inv;
                        if (lane * 4 < DP) {
                            uint2 h, l;
                            split_f16(x[k].x * sc, x[k].y * sc, h.x, l.x);
                            split_f16(x[k].z * sc, x[k].w * sc, h.y, l.y);
                            const int cc = lane >> 1;
                            const uint32_t at = smem_u32(q_smem) + (cc >> 3) * (kTile * 128) + qr * 128 + (((cc & 7) ^ (qr & 7)) << 4) + (lane & 1) * 8;
                            asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(at), "r"(h.x), "r"(h.y) : "memory");
                            asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(at + SM::tile), "r"(l.x), "r"(l.y) : "memory");
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(&qfull_bar);
            }
            wait(&qfull_bar, (uint32_t)(seg & 1));
            if (!ok) break;
            // above zero, so that a masked score (-inf) stays one
            const float cs = fmaxf(SPLIT ? qscale_s[loads & 1][r] : a.scale * 1.4426950408889634f, 1e-37f);
            const bool idle = __all_sync(0xffffffffu, !live);
            float m = -INFINITY, l = 0.0f;
            for (int t = TWO ? 0 : s; t < p.n; t += TWO ? 1 : 2) {
                wait(&s_bar[s], (uint32_t)(ns++ & 1));
                if (!ok) break;
                if (idle) {  // a warp without rows leaves its lanes as they are
                    fence_before();
                    arrive(&p_bar[s]);
                    continue;
                }
                const int key = p.k.base + (p.tile + t) * kTile;
                const int seen = limit - key, skip = p.k.key0 - key;  // columns [skip, seen) are visible
                if (!__all_sync(0xffffffffu, seen >= kTile && skip <= 0)) {
                    // a tile that not all rows see whole: the scores that are not seen
                    // become -inf where they lie
#pragma unroll 1
                    for (int c = 0; c < kTile; c += 16) {
                        float w[16];
                        uint32_t x[16];
                        tmem_ld16(s_col + c, w);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = c + i >= seen || c + i < skip ? 0xFF800000u : __float_as_uint(w[i]);
                        tmem_st16(s_col + c, x);
                    }
                    tmem_wait_st();
                }
                // Two buffers: the next 32 scores are on their way while these are
                // used. (They are read twice, maximum and weights: 128 registers for
                // them, or the maximum of 32 at a time, cost more.)
                float va[32], vb[32];
                auto top_of = [&](const float (&v)[32], float top) {
                    float x[4] = {top, v[0], v[1], v[2]};
#pragma unroll
                    for (int i = 3; i < 27; i += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = max3(x[k], v[i + k], v[i + 4 + k]);
                    return max3(max3(x[0], v[27], v[28]), max3(x[1], v[29], v[30]), max3(x[2], x[3], v[31]));
                };
                float top = -INFINITY;
                tmem_ld32(s_col, va);
#pragma unroll 1
                for (int c = 0; c < kTile; c += 64) {
                    tmem_wait_ld();
                    tmem_ld32(s_col + c + 32, vb);
                    top = top_of(va, top);
                    tmem_wait_ld();
                    tmem_ld32(s_col + ((c + 64) & (kTile - 1)), va);  // last: the first ones again
                    top = top_of(vb, top);
                }
                const float high = top * cs;
                const float up = fabsf(high) < 16.0f * kFar ? high - kLift<T16> : high;  // (no room for it in far ones)
                const bool move = m != -INFINITY && high - m > kMost<T16>;
                if (t >= (TWO ? 1 : 2) && __any_sync(0xffffffffu, move)) {
                    const float keep = move ? exp2_fast(m - up) : 1.0f;
                    l *= keep;
#pragma unroll 1
                    for (int c = 0; c < DP; c += 16) {
                        float w[16];
                        uint32_t x[16];
                        const uint32_t o_at = tmem + lane_at + 2 * kTile + s * DP + c;
                        tmem_ld16(o_at, w);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(w[i] * keep);
                        tmem_st16(o_at, x);
                    }
                }
                if (move || (m == -INFINITY && high != -INFINITY)) m = up;
                float ref = m == -INFINITY ? 0.0f : m, factor = cs;
                if (__any_sync(0xffffffffu, fabsf(high) >= kFar && high != -INFINITY)) {
                    // far scores: the exponents, from differences of scores, take their place
                    const float from = high == -INFINITY ? 0.0f : top, add = high == -INFINITY ? -ref : high - ref;
#pragma unroll 1
                    for (int c = 0; c < kTile; c += 16) {
                        float w[16];
                        uint32_t x[16];
                        tmem_ld16(s_col + c, w);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(fmaf(w[i] - from, cs, add));
                        tmem_st16(s_col + c, x);
                    }
                    tmem_wait_st();
                    tmem_ld32(s_col, va);
                    factor = 1.0f;
                    ref = 0.0f;
                }
                const float2 cs2 = make_float2(factor, factor), ref2 = make_float2(-ref, -ref);
                float2 sum[2] = {make_float2(l, 0.0f), make_float2(0.0f, 0.0f)};
                auto weights = [&](const float (&v)[32], int c) {
                    uint32_t w[16], w2[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 x = fma2(make_float2(v[2 * i], v[2 * i + 1]), cs2, ref2);
                        x.x = exp2_fast(x.x);
                        x.y = exp2_fast(x.y);
                        sum[i & 1] = add2(sum[i & 1], x);
                        if constexpr (SPLIT) split_f16(x.x, x.y, w[i], w2[i]);
                        else w[i] = Half2Of<T16>::pack(x.x, x.y);
                    }
                    tmem_st16(s_col + c, w);
                    if constexpr (SPLIT) tmem_st16(s_col + c + 16, w2);
                };
#pragma unroll 1
                for (int c = 0; c < kTile; c += 64) {
                    tmem_wait_ld();
                    tmem_ld32(s_col + c + 32, vb);
                    weights(va, c);
                    tmem_wait_ld();
                    if (c == 0) tmem_ld32(s_col + 64, va);
                    weights(vb, c + 32);
                }
                sum[0] = add2(sum[0], sum[1]);
                l = sum[0].x + sum[0].y;
                tmem_wait_st();
                fence_before();
                arrive(&p_bar[s]);
            }
            if (!ok) break;
            // more of this row tile: its next scores may be formed meanwhile
            const bool last = !SPLIT || p.tile + p.n == p.tiles || p.u + p.n >= u1;
            if (!last) arrive(&qfull_bar);
            const PartArgs& part = p.k.kind ? rest : prefix;
            const long long first = p.u - p.tile;
            const int c0 = shares.of(first), c1 = shares.of(first + p.tiles - 1);
            const bool whole = c0 == c1 && p.k.kind && p.k.key0 == 0;  // no other part anywhere
            wait(&ofin_bar, (uint32_t)(seg & 1));
            if (!ok) break;
            // --- results of the piece
            float w0 = 1.0f, w1 = 0.0f, M = m, L = l;
            if (!TWO) {
                join_s[s][r] = make_float2(m, l);
                arrive(&join_bar);
                wait(&join_bar, (uint32_t)(nj++ & 1));
                if (!ok) break;
                const float2 x = join_s[0][r], y = join_s[1][r];
                M = fmaxf(x.x, y.x);
                w0 = x.x == -INFINITY ? 0.0f : exp2_fast(x.x - M);
                w1 = y.x == -INFINITY ? 0.0f : exp2_fast(y.x - M);
                L = x.y * w0 + y.y * w1;
            }
            float kept = 0.0f;  // weight of the sums of the pieces before
            if (goes_on) {
                const float2 x = so_far_s[s][r];
                const float top = fmaxf(M, x.x), now = M == -INFINITY ? 0.0f : exp2_fast(M - top);
                kept = x.x == -INFINITY ? 0.0f : exp2_fast(x.x - top);
                w0 *= now;
                w1 *= now;
                L = L * now + x.y * kept;
                M = top;
            }
            if (!last) so_far_s[s][r] = make_float2(M, L);
            const bool done = whole && last;
            const int64_t orow = (int64_t)tok * a.H + p.kvh * a.G + row % a.G;
            const int slot_row = (TWO ? s * kTile : 0) + r;
            const int64_t slot = (int64_t)cta * part.slot_rows + slot_row;
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            // Each thread has a row; through 64 bytes of each row at a time in
            // shared memory the warp writes 8 rows by 64 bytes per instruction
            // (a thread writing its own row touches 32 lines at once: 14,000
            // cycles for 256 rows of 128 sums).
            if (c0 == cta && c1 > c0 && tid == 0 && !part.by_row) {  // the row block whose parts have to be joined
                int* rec = part.cuts + cta * 8;
                rec[0] = c1;
                rec[1] = p.k.tok0;
                rec[2] = p.rt * BR;
                rec[3] = p.k.rows;
                rec[4] = p.kvh;
            }
            const int64_t partial = !live ? -1 : (c0 == cta && part.by_row ? orow : slot) * a.D;
            const int64_t own = live && done ? orow * a.D : partial;
            int64_t to[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = __shfl_sync(0xffffffffu, own, i * 8 + lane / 4);
            const uint32_t st = smem_u32(ring + (size_t)NST * SM::tile) + warp * SM::stage_out;
            const uint32_t put = st + lane * 64, get = st + (lane / 4) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
            // one row tile: each stream's threads write half of the columns
            constexpr int CW = TWO ? DP : DP / 2;
            const bool both = !TWO && p.n > 1;  // the second stream had a tile
            auto sums_of = [&](int col, float (&v)[16]) {
                const uint32_t o_at = tmem + lane_at + 2 * kTile + col;
                tmem_ld16(o_at + (TWO ? s * DP : 0), v);
                tmem_wait_ld();
                if (!TWO) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] *= w0;
                    if (both) {
                        float y[16];
                        tmem_ld16(o_at + DP, y);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = fmaf(y[i], w1, v[i]);
                    }
                }
                if (done) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] *= inv;
                }
            };
            if (!done || sizeof(TQ) == 4) {
                float* parts = c0 == cta ? part.head : part.tail;
                float* base = done ? static_cast<float*>(a.out) : parts;
#pragma unroll 1
                for (int c = 0; c < CW; c += 16) {
                    const int col = (TWO ? 0 : s * CW) + c;
                    float v[16];
                    sums_of(col, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        st_shared16(put + ((i ^ ((lane >> 1) & 3)) << 4), __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                    __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
                    __syncwarp();
                    const int d = col + (lane & 3) * 4;
                    if (goes_on) {  // onto what the pieces before left there
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) {
                            const float w = __shfl_sync(0xffffffffu, done ? kept * inv : kept, i * 8 + lane / 4);
                            const int64_t from = __shfl_sync(0xffffffffu, partial, i * 8 + lane / 4);
                            const int64_t dst = __shfl_sync(0xffffffffu, own, i * 8 + lane / 4);
                            if (from < 0 || d >= a.D) continue;
                            const uint4 x = ld_shared16(get + i * 512);
                            const float4 y = *reinterpret_cast<const float4*>(parts + from + d);  // this lane's own
                            *reinterpret_cast<float4*>(base + dst + d) =
                                make_float4(fmaf(y.x, w, __uint_as_float(x.x)), fmaf(y.y, w, __uint_as_float(x.y)),
                                            fmaf(y.z, w, __uint_as_float(x.z)), fmaf(y.w, w, __uint_as_float(x.w)));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 x = ld_shared16(get + i * 512);
                            if (to[i] >= 0 && d < a.D) *reinterpret_cast<uint4*>(base + to[i] + d) = x;
                        }
                    }
                    __syncwarp();
                }
            } else if constexpr (sizeof(TQ) == 2) {
                TQ* base = static_cast<TQ*>(a.out);
#pragma unroll 1
                for (int c = 0; c < CW; c += 32) {
                    const int col = (TWO ? 0 : s * CW) + c;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[16];
                        sums_of(col + 16 * h, v);
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = Half2Of<T16>::pack(v[2 * i], v[2 * i + 1]);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            st_shared16(put + (((2 * h + i) ^ ((lane >> 1) & 3)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    }
                    __syncwarp();
                    const int d = col + (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 x = ld_shared16(get + i * 512);
                        if (to[i] >= 0 && d < a.D) *reinterpret_cast<uint4*>(base + to[i] + d) = x;
                    }
                    __syncwarp();
                }
            }
            if (live && last && (TWO || s == 0)) {
                if (c0 == cta) part.stat[orow] = pack_stat(M, L, PartPlace{c0, c1, slot_row, p.k.key0 > 0});
                else part.tail_stat[slot] = make_float2(M, L);
            }
            if (!TWO) {
                // the next piece's products overwrite sums that the other threads read
                fence_before();
                arrive(&join_bar);
                wait(&join_bar, (uint32_t)(nj++ & 1));
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        mbar_drain(&done_bar, 0);  // products still running use the memory that is freed here
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
    pdl_wait();
}

template <typename TQ, typename T16, int DP, bool SPLIT, bool TWO>
void launch_tc_t(const BeaconCudaContext* ctx, const PagedTcPlan& plan, const PagedArgs& a, const CacheMaps& maps, const PartArgs& prefix, const PartArgs& rest, cudaStream_t s, bool pdl) {
    auto kern = paged_tc_kernel<TQ, T16, DP, SPLIT, TWO>;
    static std::atomic<uint64_t> allowed{0};
    allow_smem_once(kern, ctx, allowed);
    const int entries = (a.merged ? 0 : a.groups) + (plan.rest ? a.B : 0);
    launch_kernel(kern, dim3((unsigned)plan.ctas), dim3(kTcThreads), TcSmem<DP, SPLIT, TWO>::bytes, s, pdl, a, maps, prefix, rest, entries,
                  plan.ctas, plan.rest ? 1 : 4);
}

template <int DP>
void launch_tc_d(const BeaconCudaContext* ctx, const PagedTcPlan& plan, const PagedArgs& a, const CacheMaps& maps, const PartArgs& prefix, const PartArgs& rest, int32_t tq, int32_t tk,
                 cudaStream_t s, bool pdl) {
    using H = __half;
    using B = __nv_bfloat16;
    if (tq == BEACON_CUDA_DTYPE_F32) launch_tc_t<float, H, DP, true, false>(ctx, plan, a, maps, prefix, rest, s, pdl);
    else if (tk == BEACON_CUDA_DTYPE_F16 && plan.two) launch_tc_t<H, H, DP, false, true>(ctx, plan, a, maps, prefix, rest, s, pdl);
    else if (tk == BEACON_CUDA_DTYPE_F16) launch_tc_t<H, H, DP, false, false>(ctx, plan, a, maps, prefix, rest, s, pdl);
    else if (plan.two) launch_tc_t<B, B, DP, false, true>(ctx, plan, a, maps, prefix, rest, s, pdl);
    else launch_tc_t<B, B, DP, false, false>(ctx, plan, a, maps, prefix, rest, s, pdl);
}

}  // namespace

PagedTcPlan plan_paged_tc(const BeaconCudaContext* ctx, const PagedArgs& a, bool split, bool with_rest) {
    PagedTcPlan p;
    // Blocks of more than 128 rows on average share each key tile between two row
    // tiles. (bf16, 32 heads on 8 of 128, one row tile and two: 16 sequences over 1024
    // keys, rows a sequence and KV head 64: 42 and 46 us, 128: 44 and 48, 160: 60 and 52,
    // 512: 89 and 81, 2048: 224 and 181; 4 over 2048, which leave CTAs idle: 256: 42 and
    // 44, 512: 50 and 52, 2048: 120 and 106.)
    p.two = !split && (int64_t)a.T * a.G > 128LL * (a.groups && !a.merged ? a.groups : a.B);
    p.rest = with_rest;
    p.slot_rows = p.two ? 2 * kTile : kTile;
    p.ctas = ctx->sm_count;
    return p;
}

void launch_paged_tc(const BeaconCudaContext* ctx, const PagedTcPlan& plan, const PagedArgs& a, const CacheMaps& maps, const PartArgs& prefix,
                     const PartArgs& rest, int32_t tq, int32_t tk, cudaStream_t s, bool pdl) {
    if (a.D <= 64) launch_tc_d<64>(ctx, plan, a, maps, prefix, rest, tq, tk, s, pdl);
    else launch_tc_d<128>(ctx, plan, a, maps, prefix, rest, tq, tk, s, pdl);
}

}  // namespace bc
