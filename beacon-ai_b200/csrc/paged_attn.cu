// paged_attn.cu -- causal attention over paged key/value caches with prefixes
// shared by groups of sequences (beacon_cuda_op_paged_attention): the argument
// checks and the kernel of any dtype and head size.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "internal.h"
#include "kernels.h"
#include "paged_attn.h"
#include "rotary.h"

namespace bc {
namespace {

constexpr int kAnyWarps = 4;
constexpr int kAnyMaxDim = 256;

template <typename T>
__device__ __forceinline__ float as_f32(T v);
template <>
__device__ __forceinline__ float as_f32(float v) { return v; }
template <>
__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// 32-bit caches, heads of more than 128 values, and caches without pages. One
// query row and head per block; each warp takes every fourth key, its lanes the
// head's values, with its own running maximum and sum; the warps' parts are
// joined at the end. f32 throughout. Every row reads its keys for itself: bound
// by L2, and a row's keys stay with one block (16 rows of 8192 keys each, 32 heads
// on 8 of 128 values: 4.8 ms; one row alone: 4.9 ms).
template <typename TQ, typename TK>
__global__ void __launch_bounds__(kAnyWarps * 32) paged_attn_any_kernel(const PagedArgs a) {
    constexpr int N = kAnyMaxDim / 32;
    __shared__ float m_s[kAnyWarps], l_s[kAnyWarps], o_s[kAnyWarps][kAnyMaxDim];
    const int t = blockIdx.x, h = blockIdx.y, kvh = h / a.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = a.qstarts ? span_of(a.qstarts, a.B, t) : t;
    if (b < 0) return;  // behind the last sequence
    const SeqInfo s = seq_info(a, b);
    const int limit = min(s.len, s.len - s.nq + (t - s.q0) + 1);
    const TQ* q = static_cast<const TQ*>(a.q) + ((int64_t)t * a.H + h) * a.D;
    float qv[N], o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int d = lane + 32 * i;
        qv[i] = d < a.D ? as_f32(q[d]) * a.scale : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int p = warp; p < limit; p += kAnyWarps) {
        const int64_t row = page_row(a, page_id(a, p < s.prefix ? s.first : b, p), p);
        if (row < 0) continue;
        const int64_t at = (row * a.Hkv + kvh) * a.D;
        const TK* k = static_cast<const TK*>(a.ck) + at;
        const TK* v = static_cast<const TK*>(a.cv) + at;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = lane + 32 * i;
            if (d < a.D) dot = fmaf(qv[i], as_f32(k[d]), dot);
        }
        dot = warp_sum(dot);
        const float mn = fmaxf(m, dot);
        // a row whose scores so far are all -inf keeps its empty sums; a score that
        // is no number is in them from the start (fmaxf leaves it out)
        const float keep = m == -INFINITY ? 1.0f : expf(m - mn);
        const float e = expf(dot - (mn == -INFINITY ? 0.0f : mn));
        m = mn;
        l = l * keep + e;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = lane + 32 * i;
            if (d < a.D) o[i] = fmaf(e, as_f32(v[d]), o[i] * keep);
        }
    }
    if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) o_s[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float mx = m_s[0];
    for (int w = 1; w < kAnyWarps; ++w) mx = fmaxf(mx, m_s[w]);
    float total = 0.0f, wt[kAnyWarps];
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) {
        wt[w] = m_s[w] == -INFINITY ? 0.0f : expf(m_s[w] - mx);
        total += l_s[w] * wt[w];
    }
    TQ* out = static_cast<TQ*>(a.out) + ((int64_t)t * a.H + h) * a.D;
    for (int d = threadIdx.x; d < a.D; d += kAnyWarps * 32) {
        float r = 0.0f;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) r = fmaf(o_s[w][d], wt[w], r);
        put(out + d, total == 0.0f ? 0.0f : r / total);
    }
}

// Scratch of one call: the stream's arena, which later calls on the stream use
// again in stream order (the caller holds the stream's launch_mu). A captured
// call gets memory of its graph instead, so graphs captured on one stream can
// replay at the same time.
class CallScratch {
   public:
    CallScratch(BeaconCudaStream* stream, size_t bytes) : s_(stream->s) {
        cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
        BC_CUDA(cudaStreamIsCapturing(s_, &st));
        if (st == cudaStreamCaptureStatusNone) {
            p_ = stream->arena.get(bytes, s_);
        } else {
            BC_CUDA(cudaMallocAsync(&p_, bytes, s_));
            graph_ = true;
        }
    }
    ~CallScratch() {
        if (graph_) cudaFreeAsync(p_, s_);
    }
    CallScratch(const CallScratch&) = delete;
    CallScratch& operator=(const CallScratch&) = delete;
    uint8_t* data() const { return static_cast<uint8_t*>(p_); }
    bool of_graph() const { return graph_; }

   private:
    cudaStream_t s_;
    void* p_ = nullptr;
    bool graph_ = false;
};

// Carves PartArgs out of one scratch region (base null: only counts the bytes).
class Carve {
   public:
    explicit Carve(uint8_t* base) : base_(base) {}
    template <typename T>
    T* take(int64_t n) {
        T* p = base_ ? reinterpret_cast<T*>(base_ + used_) : nullptr;
        used_ += (size_t)((n * (int64_t)sizeof(T) + 255) / 256 * 256);
        return p;
    }
    size_t used() const { return used_; }

   private:
    uint8_t* base_;
    size_t used_ = 0;
};

PartArgs carve_part(Carve& c, const PagedArgs& a, int ctas, int slot_rows, bool by_row) {
    PartArgs p;
    const int64_t rows = (int64_t)a.T * a.H, slots = (int64_t)ctas * slot_rows;
    p.stat = c.take<float4>(rows);
    p.head = c.take<float>((by_row ? rows : slots) * a.D);
    p.tail_stat = c.take<float2>(slots);
    p.tail = c.take<float>(slots * a.D);
    p.cuts = c.take<int>(8 * ctas);
    p.by_row = by_row;
    p.slot_rows = slot_rows;
    p.ctas = ctas;
    return p;
}

// [pages * page_size][Hkv][D] in boxes of box_rows rows by 64 values of one head,
// 128-byte swizzle; values past D and rows past the end arrive as zeros.
CUtensorMap cache_map(const PagedArgs& a, const void* cache, int32_t tk, int box_rows) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        BC_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !fn) fail(BEACON_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }();
    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.Hkv, (cuuint64_t)a.pages * (cuuint64_t)a.page_size};
    const cuuint64_t strides[2] = {(cuuint64_t)a.D * 2, (cuuint64_t)a.Hkv * (cuuint64_t)a.D * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows};
    const cuuint32_t es[3] = {1, 1, 1};
    const CUresult r = encode(&map, tk == BEACON_CUDA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                              const_cast<void*>(cache), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(BEACON_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled failed for a paged cache");
    return map;
}

void run_paged_attention(BeaconCudaContext* ctx, BeaconCudaStream* stream, PagedArgs a, int32_t tq, int32_t tk) {
    const int32_t F32 = BEACON_CUDA_DTYPE_F32, F16 = BEACON_CUDA_DTYPE_F16;
    if (tk != F32 && a.D <= 128 && a.pages > 0) {
        std::lock_guard<std::mutex> order(stream->launch_mu);
        // Single rows of few heads: paged_decode_kernel; prefixes, several rows of a
        // sequence or many heads: the tensor-core kernel, whose row block is 128.
        // (bf16, 8 KV heads of 128, either kernel: 16 rows of 8192 keys 110 and 122 us
        // with 2 heads a KV head, 114 and 122 with 16; 64 rows of 512 keys 42 and 63,
        // 48 and 63; 32-bit queries 112 and 175, 122 and 189; 44 and 85, 52 and 91.)
        const bool decode = !a.qstarts && a.G <= kDecodeMaxGroup, tc = a.gstarts || !decode;
        const bool split = tq == F32;
        // Sequences whose rows fill row blocks of 128 take prefix and rest together,
        // others share the prefix. (8 sequences behind 2048 keys with 128 each of their
        // own, 32 heads on 8 of 128, bf16, by rows a sequence and KV head, apart and
        // together: 16: 28 and 38 us, 64: 42 and 40, 128: 54 and 40, 512: 169 and 75. 63
        // single rows and one prompt of 512 rows: 120 and 159; of 2000 rows: 292 and 298.)
        a.merged = a.qstarts && (int64_t)a.T * a.G >= 128LL * a.B;
        const bool by_row = a.gstarts && !a.merged;
        const PagedTcPlan plan = tc ? plan_paged_tc(ctx, a, split, !decode) : PagedTcPlan{};
        const int dctas = decode ? paged_decode_ctas(ctx, a) : 0;
        PartArgs prefix, rest;
        auto carve = [&](uint8_t* base) {
            Carve c(base);
            if (tc && by_row) prefix = carve_part(c, a, plan.ctas, plan.slot_rows, by_row);
            rest = decode ? carve_part(c, a, dctas, a.G, by_row) : carve_part(c, a, plan.ctas, plan.slot_rows, by_row);
            return c.used();
        };
        CallScratch scratch(stream, carve(nullptr));
        carve(scratch.data());
        CacheMaps maps{}, dmaps{};
        if (a.page_size % 8 == 0) {
            a.box = 8;
            while (a.box < 128 && a.page_size % (2 * a.box) == 0) a.box *= 2;
            if (tc) maps = {cache_map(a, a.ck, tk, a.box), cache_map(a, a.cv, tk, a.box)};
            const int rows = std::min(a.box, kDecodeBox);
            if (decode) dmaps = {cache_map(a, a.ck, tk, rows), cache_map(a, a.cv, tk, rows)};
        }
        bool pdl = !scratch.of_graph();  // a graph's allocation comes first
        if (tc) {
            launch_paged_tc(ctx, plan, a, maps, prefix, rest, tq, tk, stream->s, pdl);
            pdl = true;
        }
        if (decode) launch_paged_decode(ctx, a, dmaps, rest, tq, tk, stream->s, pdl, tc);
        launch_paged_combine(a, prefix, rest, tq, stream->s);
        return;
    }
    const dim3 grid((unsigned)a.T, (unsigned)a.H);
    cudaStream_t s = stream->s;
    if (tq == F32 && tk == F32) paged_attn_any_kernel<float, float><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else if (tq == F32) paged_attn_any_kernel<float, __half><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else if (tq == F16) paged_attn_any_kernel<__half, __half><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else paged_attn_any_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, kAnyWarps * 32, 0, s>>>(a);
    BC_LAUNCHED("paged_attn_any_kernel");
}

void check_i32(const BeaconCudaContext* ctx, const BeaconCudaTensor* t, int64_t n, const char* what) {
    check_tensor(ctx, t, what);
    if (t->dtype != BEACON_CUDA_DTYPE_I32) fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, std::string(what) + " must be I32");
    if (n >= 0 && (t->shape.size() != 1 || t->numel() != n)) shape_err(std::string(what) + " has the wrong length");
}

}  // namespace
}  // namespace bc

using namespace bc;

extern "C" int32_t beacon_cuda_op_paged_attention(BeaconCudaContext* ctx, BeaconCudaStream* stream,
                                                  const BeaconCudaTensor* q, const BeaconCudaTensor* cache_k,
                                                  const BeaconCudaTensor* cache_v, const BeaconCudaTensor* page_table,
                                                  const BeaconCudaTensor* kv_lens, const BeaconCudaTensor* query_starts,
                                                  const BeaconCudaTensor* group_starts,
                                                  const BeaconCudaTensor* prefix_lens, float scale,
                                                  BeaconCudaTensor** inout_out) {
    return guard([&]() -> int32_t {
        require(ctx && stream && q && cache_k && cache_v && page_table && kv_lens && inout_out,
                "paged_attention: null argument");
        require((group_starts != nullptr) == (prefix_lens != nullptr),
                "paged_attention: group_starts and prefix_lens come together");
        check_stream(ctx, stream, "paged_attention");
        for (const BeaconCudaTensor* t : {q, cache_k, cache_v}) check_tensor(ctx, t, "paged_attention");
        const int32_t F32 = BEACON_CUDA_DTYPE_F32, F16 = BEACON_CUDA_DTYPE_F16, BF16 = BEACON_CUDA_DTYPE_BF16;
        const int32_t tq = q->dtype, tk = cache_k->dtype;
        if (cache_v->dtype != tk || !((tq == F32 && (tk == F16 || tk == F32)) || (tq == F16 && tk == F16) || (tq == BF16 && tk == BF16)))
            fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE,
                 "paged_attention: (q, caches) must be (F32, F16), (F16, F16), (BF16, BF16) or (F32, F32)");
        if (q->shape.size() != 3) shape_err("paged_attention: q must be [T, H, D]");
        if (cache_k->shape.size() != 4 || cache_v->shape != cache_k->shape)
            shape_err("paged_attention: caches must be alike, [pages, page_size, Hkv, D]");
        const int64_t T = q->shape[0], H = q->shape[1], D = q->shape[2], Hkv = cache_k->shape[2];
        if (cache_k->shape[3] != D) shape_err("paged_attention: q and the caches differ in head size");
        if (D < 8 || D > kAnyMaxDim || D % 8) shape_err("paged_attention: the head size must be a multiple of 8, 8 to 256");
        if (Hkv < 1 || H < 1 || H % Hkv || H > 65535) shape_err("paged_attention: H must be a multiple of Hkv, at most 65535");
        if (cache_k->shape[1] < 1 || cache_k->shape[1] > 0x7FFFFFFF) shape_err("paged_attention: empty pages");
        if (cache_k->shape[0] * cache_k->shape[1] > 0x7FFFFFFF) shape_err("paged_attention: more than 2^31 - 1 cache rows");
        check_i32(ctx, page_table, -1, "paged_attention: page_table");
        if (page_table->shape.size() != 2) shape_err("paged_attention: page_table must be [B, max_pages]");
        const int64_t B = page_table->shape[0], max_pages = page_table->shape[1];
        if (T > 0x3FFFFFFF || B > 0x3FFFFFFF || max_pages > 0x7FFFFFFF) shape_err("paged_attention: too many rows or pages");
        // positions and row numbers are 32-bit in the kernels, which step past them by a tile
        constexpr int64_t kMostIndex = 0x7FFFF000;
        if (T * H > kMostIndex) shape_err("paged_attention: more than 2^31 - 4096 query heads");
        if (max_pages * cache_k->shape[1] > kMostIndex)
            shape_err("paged_attention: page_table has room for more than 2^31 - 4096 positions of a sequence");
        check_i32(ctx, kv_lens, B, "paged_attention: kv_lens");
        if (query_starts) check_i32(ctx, query_starts, B + 1, "paged_attention: query_starts");
        else if (T != B) shape_err("paged_attention: without query_starts every sequence has one query row");
        int64_t groups = 0;
        if (group_starts) {
            groups = prefix_lens->numel();
            if (groups < 1 || groups > 0x3FFFFFFF) shape_err("paged_attention: no groups");
            check_i32(ctx, prefix_lens, groups, "paged_attention: prefix_lens");
            check_i32(ctx, group_starts, groups + 1, "paged_attention: group_starts");
        }
        if (!std::isfinite(scale) || scale < 0.0f) invalid("paged_attention: scale must be finite and not negative");
        for (const BeaconCudaTensor* t : {q, cache_k, cache_v})
            if (!aligned16(t->data())) invalid("paged_attention: tensors must be 16-byte aligned");
        DeviceScope dev(ctx);
        OutTensor out(ctx, inout_out, q->shape, tq, "paged_attention");
        if (!aligned16(out.data())) invalid("paged_attention: tensors must be 16-byte aligned");
        for (const BeaconCudaTensor* t : {q, cache_k, cache_v, page_table, kv_lens, query_starts, group_starts, prefix_lens})
            out.check_overlap(t, false, "paged_attention");
        PagedArgs a;
        a.q = q->data();
        a.ck = cache_k->data();
        a.cv = cache_v->data();
        a.out = out.data();
        a.table = static_cast<const int32_t*>(page_table->data());
        a.lens = static_cast<const int32_t*>(kv_lens->data());
        a.qstarts = query_starts ? static_cast<const int32_t*>(query_starts->data()) : nullptr;
        a.gstarts = group_starts ? static_cast<const int32_t*>(group_starts->data()) : nullptr;
        a.prefix = prefix_lens ? static_cast<const int32_t*>(prefix_lens->data()) : nullptr;
        a.pages = cache_k->shape[0];
        a.T = (int)T;
        a.B = (int)B;
        a.H = (int)H;
        a.Hkv = (int)Hkv;
        a.G = (int)(H / Hkv);
        a.D = (int)D;
        a.groups = (int)groups;
        a.max_pages = (int)max_pages;
        a.page_size = (int)cache_k->shape[1];
        for (int i = 0; i < 31; ++i)
            if (a.page_size == 1 << i) a.page_shift = i;
        a.scale = scale;
        a.err = stream_error_word(stream);
        if (T > 0 && B > 0) run_paged_attention(ctx, stream, a, tq, tk);
        out.release();
        return BEACON_CUDA_OK;
    });
}
