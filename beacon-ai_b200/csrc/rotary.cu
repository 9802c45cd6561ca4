// rotary.cu -- rotary positions of token-major rows (rope_scaled), head norms
// with the rotation (qk_norm_rope) and the cache append with the rotation
// (paged_append).
//
// All three are one pass over rows of `dim` values: read a head, optionally
// scale it by w / sqrt(mean(x^2) + eps), turn its first rotary_dim values, and
// write it to a dense row or to its cache page, so one kernel does them. It is
// bound by memory: 16-byte loads and stores, each value read and written once.
//
// A block takes a few tokens. A head is held by as many lanes as its 2 x
// 16-byte slots need, so a warp has several heads at a time, and the loads of
// its next two tokens (64 bytes a lane, 32 warps an SM) are always in flight. The sines and
// cosines of the block's tokens are computed once into shared memory while the
// first loads are on their way: the angle is a 64-bit product position * f_i /
// 2 pi reduced to one turn, then sincospif in 32 bits with the rest of the angle
// to first order, so position 10^6 is as exact as position 1. (Every warp computing its own: 1200 instructions a
// token and 60 us for 8192 x 32 heads of 128 bf16 values, 20 us of memory.)
// Measured, bf16, heads of 128: rotation of 8192 x 32 heads 27.1 us (4.95 TB/s),
// norms and rotation of 4099 x (64 + 8) heads 34.8 us (4.3 TB/s), append of about
// 8200 rows of 8 heads 16.4 us (4.1 TB/s); a handful of tokens costs the launch.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "internal.h"
#include "kernels.h"
#include "paged_mma.cuh"
#include "rotary.h"

namespace bc {

OutTensor::OutTensor(BeaconCudaContext* ctx, BeaconCudaTensor** inout, const std::vector<int64_t>& shape,
                     int32_t dtype, const char* what)
    : inout_(inout), t_(*inout) {
    if (t_) {
        check_tensor(ctx, t_, what);
        if (t_->shape != shape) shape_err(std::string(what) + ": the output tensor's shape is not the result's");
        if (t_->dtype != dtype)
            fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, std::string(what) + ": the output tensor's dtype is not the result's");
    } else {
        made_.reset(new_tensor(ctx, shape, dtype));
        t_ = made_.get();
    }
}

void OutTensor::check_overlap(const BeaconCudaTensor* x, bool in_place, const char* what) const {
    if (!x) return;
    const char *a = static_cast<const char*>(t_->data()), *b = static_cast<const char*>(x->data());
    const size_t an = t_->nbytes(), bn = x->nbytes();
    if (!an || !bn || a + an <= b || b + bn <= a) return;
    if (in_place && a == b && an == bn) return;
    invalid(std::string(what) + ": the output overlaps an input");
}

void check_tensor(const BeaconCudaContext* ctx, const BeaconCudaTensor* t, const char* what) {
    if (t->ctx != ctx) invalid(std::string(what) + ": a tensor belongs to another context");
}

void check_stream(const BeaconCudaContext* ctx, const BeaconCudaStream* stream, const char* what) {
    if (stream->ctx != ctx) invalid(std::string(what) + ": the stream belongs to another context");
}

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kMaxTokens = 32;  // of a block
constexpr int kMaxHeadDim = 512;
constexpr int kRowSteps = 2;  // tokens whose loads a lane has in flight: 64 bytes, four blocks an SM

struct RowSegment {                // heads of one input tensor
    const void* src = nullptr;     // [T][heads][dim]
    void* dst = nullptr;           // the same, or cache pages when RowArgs.table
    const void* weight = nullptr;  // norm weight [dim]; null: no norm
    int32_t weight_dtype = 0;
    int heads = 0;
    bool turn = false;
};

struct RowArgs {
    RowSegment seg[2];
    int64_t tokens = 0;
    int dim = 0, rotary = 0;
    float eps = 0.0f, inv_dim = 0.0f, amplitude = 1.0f;
    const int32_t* positions = nullptr;
    const double* turns = nullptr;  // [rotary / 2]
    // cache pages
    const int32_t* table = nullptr;  // [seqs][max_pages]; null: dense rows
    const int32_t* seq_ids = nullptr;
    int64_t seqs = 0, max_pages = 0, pages = 0, page_size = 0;
    int* err = nullptr;
    // launch shape
    int lanes = 1;         // of one head (power of two)
    int block_tokens = 1;  // tokens of a block
    int part_groups = 0;   // head groups (heads that a warp holds at a time) of a block, of each token
    int parts0 = 0;        // blocks (grid.y) that share the first segment's heads; the others have the second's
};

// 16 bytes of values as floats, and floats stored as values, two at a time: 16-bit
// values are never handled one by one.
template <typename T>
struct Slot;
template <>
struct Slot<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void unpack(const uint4& x, float* f) {
        f[0] = __uint_as_float(x.x), f[1] = __uint_as_float(x.y), f[2] = __uint_as_float(x.z), f[3] = __uint_as_float(x.w);
    }
};
template <typename T>
struct Slot16 {
    static constexpr int V = 8;
    static __device__ __forceinline__ void unpack(const uint4& x, float* f) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = Half2Of<T>::unpack(w[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
};
template <>
struct Slot<__half> : Slot16<__half> {};
template <>
struct Slot<__nv_bfloat16> : Slot16<__nv_bfloat16> {};

__device__ __forceinline__ float2 get2(const float* f) { return make_float2(f[0], f[1]); }
__device__ __forceinline__ void put2(float* f, float2 v) { f[0] = v.x, f[1] = v.y; }

template <typename T, int V>
__device__ __forceinline__ void store_slot(T* dst, const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else if constexpr (V == 4) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(Half2Of<T>::pack(f[0], f[1]), Half2Of<T>::pack(f[2], f[3]));
    } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(Half2Of<T>::pack(f[0], f[1]), Half2Of<T>::pack(f[2], f[3]),
                                                    Half2Of<T>::pack(f[4], f[5]), Half2Of<T>::pack(f[6], f[7]));
    }
}

__device__ __forceinline__ float load_weight(const void* w, int32_t dtype, int i) {
    return dtype == BEACON_CUDA_DTYPE_F16 ? __half2float(static_cast<const __half*>(w)[i])
                                          : static_cast<const float*>(w)[i];
}

// Row of the pages that token t's key and value go to; -1: skip.
__device__ __forceinline__ int64_t cache_row(const RowArgs& a, int64_t t) {
    const int64_t p = a.positions[t];
    if (p < 0) return -1;
    const int64_t b = a.seq_ids ? (int64_t)a.seq_ids[t] : t;
    if (b >= 0 && b < a.seqs && p < a.max_pages * a.page_size) {
        const int64_t page = a.table[b * a.max_pages + p / a.page_size];
        if (page >= 0 && page < a.pages) return page * a.page_size + p % a.page_size;
    }
    a.err[kErrWordIndex] = 1;
    return -1;
}

__device__ __forceinline__ float2 turn_at(const RowArgs& a, int position, int pair) {
    double turn = (double)position * __ldg(a.turns + pair);
    turn -= rint(turn);
    // sine and cosine at the turn's 32-bit value, then turned by what that left
    // (at most 2^-26 of a turn, so its square is nothing in 32 bits)
    const float near = (float)turn;
    const float left = (float)((turn - near) * 6.283185307179586);
    float s, c;
    sincospif(2.0f * near, &s, &c);
    return make_float2(fmaf(-s, left, c) * a.amplitude, fmaf(c, left, s) * a.amplitude);
}

// What a block computes before its heads: sines and cosines, norm weights in 32
// bits, cache rows.
struct RowTables {
    float* cos;      // [tokens][half_stride]: rotary / 2 entries, rows 16-byte aligned
    float* sin;      // the same
    float* weight;   // [dim]
    int64_t* rows;   // [tokens]
};
__host__ __device__ __forceinline__ int half_stride(const RowArgs& a) { return (a.rotary / 2 + 3) & ~3; }
__device__ __forceinline__ RowTables row_tables(const RowArgs& a, uint8_t* smem) {
    RowTables s;
    s.rows = reinterpret_cast<int64_t*>(smem);
    s.weight = reinterpret_cast<float*>(s.rows + kMaxTokens);
    s.cos = s.weight + ((a.dim + 3) & ~3);
    s.sin = s.cos + a.block_tokens * half_stride(a);
    return s;
}
inline size_t row_tables_bytes(const RowArgs& a) {
    return kMaxTokens * sizeof(int64_t) + ((a.dim + 3) & ~3) * sizeof(float) + 2 * (size_t)a.block_tokens * half_stride(a) * sizeof(float);
}
__device__ __forceinline__ void fill_tables(const RowArgs& a, const RowSegment& sg, const RowTables& s, int64_t t0, int nt) {
    const int half = a.rotary / 2;
    if (sg.turn)
        for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
            const int t = i / half;
            const int pair = i - t * half, at = t * half_stride(a) + pair;
            const float2 c = turn_at(a, a.positions[t0 + t], pair);
            s.cos[at] = c.x;
            s.sin[at] = c.y;
        }
    if (sg.weight)
        for (int i = threadIdx.x; i < a.dim; i += blockDim.x) s.weight[i] = load_weight(sg.weight, sg.weight_dtype, i);
    if (a.table)
        for (int t = threadIdx.x; t < nt; t += blockDim.x) s.rows[t] = cache_row(a, t0 + t);
}

// Each head is handled by `lanes` lanes, each with two slots of V values.
// HALF: slot 0 holds values of the first half of the rotated part and slot 1
// their partners; the lanes after those take the unrotated rest, two slots
// each. Interleaved: slots 2l and 2l + 1, whose pairs lie inside a slot. Either
// way lane l turns pairs l V .. l V + V - 1.
// A block has the tokens [t0, t0 + nt) and up to kRowWarps head groups (as many
// heads as a warp's lanes hold) of one segment; a warp goes through the tokens of
// one group, or shares them where there are fewer groups than warps.
template <typename TI, typename TO, bool HALF, bool NORM>
__global__ void __launch_bounds__(kRowThreads, 4) row_kernel(const __grid_constant__ RowArgs a) {
    constexpr int V = Slot<TI>::V;
    constexpr int U = kRowSteps;
    extern __shared__ __align__(16) uint8_t row_smem[];
    const RowTables tab = row_tables(a, row_smem);
    const int second = (int)blockIdx.y >= a.parts0, part = blockIdx.y - (second ? a.parts0 : 0);
    const RowSegment& sg = a.seg[second];
    const int64_t t0 = (int64_t)blockIdx.x * a.block_tokens;
    const int nt = (int)min((int64_t)a.block_tokens, a.tokens - t0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & (a.lanes - 1), groups = 32 / a.lanes;
    const int half = a.rotary / 2, hs = half_stride(a);
    // this lane's slots of every head
    int at0, at1;
    bool turn;
    if (HALF) {
        const int turning = half / V;
        turn = lane < turning;
        at0 = turn ? lane * V : a.rotary + (lane - turning) * 2 * V;
        at1 = turn ? at0 + half : at0 + V;
    } else {
        at0 = lane * 2 * V;
        at1 = at0 + V;
        turn = at0 < a.rotary;
    }
    turn = turn && sg.turn;
    const bool has1 = at1 < a.dim;
    // the block's head groups, and the warps that share one
    const int ng = (sg.heads + groups - 1) / groups, g0 = part * a.part_groups, n = min(ng, g0 + a.part_groups) - g0;
    const int share = kRowWarps / n;                     // n is at most kRowWarps
    const int first = warp / n < share ? warp / n : nt;  // first token of this warp; then every share-th
    const int stride = sg.heads * a.dim;                 // values from one token to the next
    const int h = (g0 + warp % n) * groups + (threadIdx.x & 31) / a.lanes;
    const TI* const src = static_cast<const TI*>(sg.src) + t0 * stride + (int64_t)h * a.dim + at0;
    const int to1 = at1 - at0;
    const bool live = h < sg.heads && at0 < a.dim;

    uint4 x0[U], x1[U];
    auto load = [&](int u, int t) {
        if (live && t < nt) {
            const TI* p = src + t * (int64_t)stride;
            x0[u] = *reinterpret_cast<const uint4*>(p);
            if (has1) x1[u] = *reinterpret_cast<const uint4*>(p + to1);
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(u, first + u * share);
    fill_tables(a, sg, tab, t0, nt);
    __syncthreads();
#pragma unroll 1
    for (int t = first; t < nt;) {
        int at = t * hs + lane * V;  // this lane's first pair in the tables
#pragma unroll
        for (int u = 0; u < U; ++u, t += share, at += share * hs) {
            if (t >= nt) break;  // the warp's lanes agree
            float f0[V], f1[V];
            Slot<TI>::unpack(x0[u], f0);
            Slot<TI>::unpack(x1[u], f1);
            load(u, t + U * share);
            if (NORM) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (live) ss = fmaf(f0[j], f0[j], ss);
                    if (live && has1) ss = fmaf(f1[j], f1[j], ss);
                }
                for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float inv = rsqrtf(fmaf(ss, a.inv_dim, a.eps));
                if (live) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const float2 in = make_float2(inv, inv);
                        const float4 p = *reinterpret_cast<const float4*>(tab.weight + at0 + j);
                        put2(f0 + j, mul2(get2(f0 + j), mul2(in, make_float2(p.x, p.y))));
                        put2(f0 + j + 2, mul2(get2(f0 + j + 2), mul2(in, make_float2(p.z, p.w))));
                        if (has1) {
                            const float4 q = *reinterpret_cast<const float4*>(tab.weight + at1 + j);
                            put2(f1 + j, mul2(get2(f1 + j), mul2(in, make_float2(q.x, q.y))));
                            put2(f1 + j + 2, mul2(get2(f1 + j + 2), mul2(in, make_float2(q.z, q.w))));
                        }
                    }
                }
            }
            if (turn) {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    // pairs lane V + j .. + 3 (the rotated part has a multiple of 4 values;
                    // entries of pairs that it does not have are not used)
                    if (!HALF && at0 + 2 * j >= a.rotary) continue;
                    const float4 c = *reinterpret_cast<const float4*>(tab.cos + at + j), s = *reinterpret_cast<const float4*>(tab.sin + at + j);
                    if (HALF) {
                        const float2 c2[2] = {make_float2(c.x, c.y), make_float2(c.z, c.w)}, s2[2] = {make_float2(s.x, s.y), make_float2(s.z, s.w)};
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float2 x = get2(f0 + j + 2 * i), y = get2(f1 + j + 2 * i);
                            put2(f0 + j + 2 * i, fma2(make_float2(-y.x, -y.y), s2[i], mul2(x, c2[i])));
                            put2(f1 + j + 2 * i, fma2(x, s2[i], mul2(y, c2[i])));
                        }
                    } else {
                        const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            // pair j + i of the lane's 2 V values
                            float* f = 2 * (j + i) < V ? f0 + 2 * (j + i) : f1 + 2 * (j + i) - V;
                            if (at0 + 2 * (j + i) >= a.rotary) continue;
                            const float x = f[0], y = f[1];
                            f[0] = x * cv[i] - y * sv[i];
                            f[1] = y * cv[i] + x * sv[i];
                        }
                    }
                }
            }
            const int64_t row = a.table ? tab.rows[t] : t0 + t;
            if (live && row >= 0) {
                TO* dst = static_cast<TO*>(sg.dst) + row * stride + (h * a.dim + at0);
                store_slot<TO, V>(dst, f0);
                if (has1) store_slot<TO, V>(dst + to1, f1);
            }
        }
    }
}

__device__ __forceinline__ float ld_value(const void* p, int32_t dtype, int64_t i) {
    switch (dtype) {
        case BEACON_CUDA_DTYPE_F16: return __half2float(static_cast<const __half*>(p)[i]);
        case BEACON_CUDA_DTYPE_BF16: return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
        default: return static_cast<const float*>(p)[i];
    }
}
__device__ __forceinline__ void st_value(void* p, int32_t dtype, int64_t i, float v) {
    switch (dtype) {
        case BEACON_CUDA_DTYPE_F16: static_cast<__half*>(p)[i] = __float2half_rn(v); break;
        case BEACON_CUDA_DTYPE_BF16: static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); break;
        default: static_cast<float*>(p)[i] = v;
    }
}

// The same for dims and addresses that 16-byte slots do not fit: a head at a
// time, a pair of values a lane (rotated pairs, then the rest two by two).
__global__ void __launch_bounds__(kRowThreads) row_scalar_kernel(const __grid_constant__ RowArgs a, int32_t ti, int32_t to, bool half_layout) {
    constexpr int N = kMaxHeadDim / 64;  // pairs of a lane
    extern __shared__ __align__(16) uint8_t row_smem[];
    const int second = (int)blockIdx.y >= a.parts0, part = blockIdx.y - (second ? a.parts0 : 0);
    const RowSegment& sg = a.seg[second];
    const bool norm = sg.weight != nullptr;
    const RowTables tab = row_tables(a, row_smem);
    const int64_t t0 = (int64_t)blockIdx.x * a.block_tokens;
    const int nt = (int)min((int64_t)a.block_tokens, a.tokens - t0);
    const int lane = threadIdx.x & 31;
    const int half = a.rotary / 2, pairs = half + (a.dim - a.rotary + 1) / 2;
    const int g0 = part * a.part_groups, n = min(sg.heads, g0 + a.part_groups) - g0;
    fill_tables(a, sg, tab, t0, nt);
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < nt * n; i += kRowWarps) {
        const int t = i / n, h = g0 + i % n;
        const int64_t row = a.table ? tab.rows[t] : t0 + t;
        const int64_t src = ((t0 + t) * sg.heads + h) * a.dim, dst = (row * sg.heads + h) * a.dim;
        const float* weight = tab.weight;
        float u[N], w[N];
        float ss = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int j = lane + 32 * k;
            const int i0 = j < half ? (half_layout ? j : 2 * j) : a.rotary + 2 * (j - half);
            const int i1 = j < half && half_layout ? j + half : i0 + 1;
            u[k] = j < pairs ? ld_value(sg.src, ti, src + i0) : 0.0f;
            w[k] = j < pairs && i1 < a.dim ? ld_value(sg.src, ti, src + i1) : 0.0f;
            ss = fmaf(u[k], u[k], fmaf(w[k], w[k], ss));
        }
        const float inv = norm ? rsqrtf(fmaf(warp_sum(ss), a.inv_dim, a.eps)) : 1.0f;
        if (row < 0) continue;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int j = lane + 32 * k;
            if (j >= pairs) continue;
            const int i0 = j < half ? (half_layout ? j : 2 * j) : a.rotary + 2 * (j - half);
            const int i1 = j < half && half_layout ? j + half : i0 + 1;
            float x = u[k], y = w[k];
            if (norm) {
                x *= inv * weight[i0];
                if (i1 < a.dim) y *= inv * weight[i1];
            }
            if (sg.turn && j < half) {
                const float2 c = make_float2(tab.cos[t * half_stride(a) + j], tab.sin[t * half_stride(a) + j]);
                const float x2 = x * c.x - y * c.y;
                y = y * c.x + x * c.y;
                x = x2;
            }
            st_value(sg.dst, to, dst + i0, x);
            if (i1 < a.dim) st_value(sg.dst, to, dst + i1, y);
        }
    }
}

template <typename TI, typename TO, bool NORM>
void launch_rows_t(const RowArgs& a, bool half_layout, dim3 grid, size_t smem, cudaStream_t s) {
    if (half_layout)
        row_kernel<TI, TO, true, NORM><<<grid, kRowThreads, smem, s>>>(a);
    else
        row_kernel<TI, TO, false, NORM><<<grid, kRowThreads, smem, s>>>(a);
}

template <typename TI>
void launch_rows_to(const RowArgs& a, int32_t to, bool half_layout, dim3 grid, size_t smem, cudaStream_t s) {
    if (a.seg[0].weight) launch_rows_t<TI, TI, true>(a, half_layout, grid, smem, s);  // norms keep the dtype
    else if (to == BEACON_CUDA_DTYPE_F32) launch_rows_t<TI, float, false>(a, half_layout, grid, smem, s);
    else if (to == BEACON_CUDA_DTYPE_F16) launch_rows_t<TI, __half, false>(a, half_layout, grid, smem, s);
    else launch_rows_t<TI, __nv_bfloat16, false>(a, half_layout, grid, smem, s);
}

void launch_rows(BeaconCudaContext* ctx, RowArgs a, int32_t ti, int32_t to, const BeaconCudaRope* rope, cudaStream_t s) {
    if (a.tokens == 0) return;
    a.inv_dim = 1.0f / (float)a.dim;
    const bool half_layout = rope && rope->layout == BEACON_CUDA_ROPE_HALF;
    if (rope) {
        a.rotary = rope->rotary_dim;
        a.amplitude = rope->amplitude;
        a.turns = static_cast<const double*>(rope->turns->ptr);
    }
    const int V = 16 / (int)plain_elem_bytes(ti);
    const int slots = half_layout ? a.rotary / 2 / V + (a.dim - a.rotary + 2 * V - 1) / (2 * V) : (a.dim + 2 * V - 1) / (2 * V);
    bool vec = a.dim % V == 0 && a.rotary % (half_layout ? 2 * V : V) == 0 && slots <= 32;
    for (const RowSegment& sg : a.seg)
        vec = vec && aligned16(sg.src) && reinterpret_cast<uintptr_t>(sg.dst) % (V * plain_elem_bytes(to)) == 0;
    a.lanes = 32;
    while (vec && a.lanes / 2 >= slots) a.lanes /= 2;
    const int hpg = vec ? 32 / a.lanes : 1;
    const int g0 = (a.seg[0].heads + hpg - 1) / hpg, g1 = (a.seg[1].heads + hpg - 1) / hpg;
    // As many blocks as run at once (four an SM), each with a warp per head
    // group and up to 32 tokens, so that the tables cost little; for fewer
    // tokens, blocks of one token and fewer groups.
    const int64_t want = 4 * ctx->sm_count;
    a.part_groups = (int)std::clamp<int64_t>((g0 + g1) * a.tokens / want, 1, kRowWarps);
    a.parts0 = (g0 + a.part_groups - 1) / a.part_groups;
    const int parts = a.parts0 + (g1 + a.part_groups - 1) / a.part_groups;
    int64_t tokens = kMaxTokens;
    if (a.rotary) tokens = std::clamp<int64_t>(6144 / a.rotary, 1, tokens);  // 24 KB of angles
    a.block_tokens = (int)std::clamp<int64_t>((a.tokens * parts + want - 1) / want, 1, tokens);
    const int64_t blocks = (a.tokens + a.block_tokens - 1) / a.block_tokens;
    if (blocks > 0x7FFFFFFF) shape_err("too many tokens");
    const dim3 grid((unsigned)blocks, (unsigned)parts);
    const size_t smem = row_tables_bytes(a);
    if (!vec) row_scalar_kernel<<<grid, kRowThreads, smem, s>>>(a, ti, to, half_layout);
    else if (ti == BEACON_CUDA_DTYPE_F32) launch_rows_to<float>(a, to, half_layout, grid, smem, s);
    else if (ti == BEACON_CUDA_DTYPE_F16) launch_rows_to<__half>(a, to, half_layout, grid, smem, s);
    else launch_rows_to<__nv_bfloat16>(a, to, half_layout, grid, smem, s);
    BC_LAUNCHED("row_kernel");
}

void check_rows(const BeaconCudaContext* ctx, const BeaconCudaTensor* x, const char* what) {
    check_tensor(ctx, x, what);
    if (x->dtype != BEACON_CUDA_DTYPE_F32 && x->dtype != BEACON_CUDA_DTYPE_F16 && x->dtype != BEACON_CUDA_DTYPE_BF16)
        fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, std::string(what) + ": rows must be F32, F16 or BF16");
    if (x->shape.size() != 3) shape_err(std::string(what) + ": rows must be [T, heads, dim]");
    if (x->shape[2] < 1 || x->shape[2] > kMaxHeadDim || x->shape[1] < 1 || x->shape[1] > 65535)
        shape_err(std::string(what) + ": 1 to 65535 heads of 1 to 512 values");
}

void check_ids(const BeaconCudaContext* ctx, const BeaconCudaTensor* t, int64_t n, const char* what) {
    check_tensor(ctx, t, what);
    if (t->dtype != BEACON_CUDA_DTYPE_I32) fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, std::string(what) + ": must be I32");
    if (t->numel() != n) shape_err(std::string(what) + ": one entry per row is needed");
}

void check_rope(const BeaconCudaContext* ctx, const BeaconCudaRope* rope, int64_t dim, const char* what) {
    if (!rope) return;
    if (rope->ctx != ctx) invalid(std::string(what) + ": the rotation belongs to another context");
    if (rope->rotary_dim > dim) shape_err(std::string(what) + ": the rotation is wider than the head");
}

}  // namespace
}  // namespace bc

using namespace bc;

extern "C" {

int32_t beacon_cuda_rope_create(BeaconCudaContext* ctx, const BeaconCudaRopeParams* params, const float* freq_factors,
                                BeaconCudaRope** out_rope) {
    return guard([&]() -> int32_t {
        require(ctx && params && out_rope, "rope_create: null argument");
        const BeaconCudaRopeParams& p = *params;
        if (p.rotary_dim < 2 || p.rotary_dim % 2 || p.rotary_dim > kMaxHeadDim)
            invalid("rope_create: rotary_dim must be even, 2 to 512");
        if (p.layout != BEACON_CUDA_ROPE_INTERLEAVED && p.layout != BEACON_CUDA_ROPE_HALF)
            invalid("rope_create: unknown layout");
        if (!(p.theta > 1.0f) || !std::isfinite(p.theta)) invalid("rope_create: theta must be above 1");
        if (p.scaling < BEACON_CUDA_ROPE_SCALING_NONE || p.scaling > BEACON_CUDA_ROPE_SCALING_BANDS)
            invalid("rope_create: unknown scaling");
        const bool scaled = p.scaling != BEACON_CUDA_ROPE_SCALING_NONE;
        if (scaled && (!(p.factor >= 1.0f) || !std::isfinite(p.factor))) invalid("rope_create: factor must be at least 1");
        if (!scaled && p.factor != 1.0f) invalid("rope_create: a factor needs a scaling");
        if (p.scaling >= BEACON_CUDA_ROPE_SCALING_YARN && p.original_context < 1)
            invalid("rope_create: the scaling needs the original context");
        if (!(p.attention_factor >= 0.0f) || !std::isfinite(p.attention_factor))
            invalid("rope_create: attention_factor must be finite and not negative");
        if (p.scaling == BEACON_CUDA_ROPE_SCALING_YARN &&
            (!(p.beta_slow > 0.0f) || !(p.beta_fast >= p.beta_slow) || !std::isfinite(p.beta_fast)))
            invalid("rope_create: yarn needs beta_fast >= beta_slow > 0");
        if (p.scaling == BEACON_CUDA_ROPE_SCALING_BANDS &&
            (!(p.low_freq_factor > 0.0f) || !(p.high_freq_factor > p.low_freq_factor) || !std::isfinite(p.high_freq_factor)))
            invalid("rope_create: bands need high_freq_factor > low_freq_factor > 0");
        const int half = p.rotary_dim / 2;
        const double pi2 = 6.283185307179586476925286766559, d = p.rotary_dim, c = p.original_context, s = p.factor;
        double lo = 0.0, hi = 0.0;
        if (p.scaling == BEACON_CUDA_ROPE_SCALING_YARN) {
            auto at = [&](double turns) { return d * std::log(c / (turns * pi2)) / (2.0 * std::log((double)p.theta)); };
            lo = std::max(0.0, std::floor(at(p.beta_fast)));
            hi = std::min(d - 1.0, std::ceil(at(p.beta_slow)));
        }
        std::vector<double> turns((size_t)half);
        for (int i = 0; i < half; ++i) {
            double f = std::pow((double)p.theta, -2.0 * i / d);
            if (p.scaling == BEACON_CUDA_ROPE_SCALING_LINEAR) {
                f /= s;
            } else if (p.scaling == BEACON_CUDA_ROPE_SCALING_YARN) {
                const double r = std::clamp((i - lo) / std::max(hi - lo, 0.001), 0.0, 1.0);
                f *= (1.0 - r) + r / s;
            } else if (p.scaling == BEACON_CUDA_ROPE_SCALING_BANDS) {
                const double m = std::clamp((c * f / pi2 - p.low_freq_factor) /
                                                ((double)p.high_freq_factor - p.low_freq_factor), 0.0, 1.0);
                f *= m + (1.0 - m) / s;
            }
            if (freq_factors) {
                if (!(freq_factors[i] > 0.0f) || !std::isfinite(freq_factors[i]))
                    invalid("rope_create: frequency factors must be positive");
                f /= freq_factors[i];
            }
            turns[(size_t)i] = f / pi2;
        }
        DeviceScope dev(ctx);
        auto r = std::make_unique<BeaconCudaRope>();
        r->ctx = ctx;
        r->rotary_dim = p.rotary_dim;
        r->layout = p.layout;
        r->amplitude = p.attention_factor != 0.0f ? p.attention_factor
                       : p.scaling == BEACON_CUDA_ROPE_SCALING_YARN ? (float)(0.1 * std::log(s) + 1.0) : 1.0f;
        r->turns = std::make_unique<DeviceBuffer>((size_t)half * sizeof(double));
        BC_CUDA(cudaMemcpy(r->turns->ptr, turns.data(), (size_t)half * sizeof(double), cudaMemcpyHostToDevice));
        *out_rope = r.release();
        return BEACON_CUDA_OK;
    });
}

void beacon_cuda_rope_destroy(BeaconCudaRope* rope) { delete rope; }

int32_t beacon_cuda_op_rope_scaled(BeaconCudaContext* ctx, BeaconCudaStream* stream, const BeaconCudaTensor* x,
                                   const BeaconCudaTensor* positions, const BeaconCudaRope* rope,
                                   BeaconCudaTensor** inout_out) {
    return guard([&]() -> int32_t {
        require(ctx && stream && x && positions && rope && inout_out, "rope_scaled: null argument");
        check_stream(ctx, stream, "rope_scaled");
        check_rows(ctx, x, "rope_scaled");
        check_ids(ctx, positions, x->shape[0], "rope_scaled: positions");
        check_rope(ctx, rope, x->shape[2], "rope_scaled");
        DeviceScope dev(ctx);
        OutTensor out(ctx, inout_out, x->shape, x->dtype, "rope_scaled");
        out.check_overlap(x, true, "rope_scaled");
        out.check_overlap(positions, false, "rope_scaled");
        RowArgs a;
        a.seg[0].src = x->data();
        a.seg[0].dst = out.data();
        a.seg[0].heads = (int)x->shape[1];
        a.seg[0].turn = true;
        a.tokens = x->shape[0];
        a.dim = (int)x->shape[2];
        a.positions = static_cast<const int32_t*>(positions->data());
        launch_rows(ctx, a, x->dtype, x->dtype, rope, stream->s);
        out.release();
        return BEACON_CUDA_OK;
    });
}

int32_t beacon_cuda_op_qk_norm_rope(BeaconCudaContext* ctx, BeaconCudaStream* stream, const BeaconCudaTensor* q,
                                    const BeaconCudaTensor* k, const BeaconCudaTensor* q_weight,
                                    const BeaconCudaTensor* k_weight, float eps, const BeaconCudaTensor* positions,
                                    const BeaconCudaRope* rope, BeaconCudaTensor** inout_q, BeaconCudaTensor** inout_k) {
    return guard([&]() -> int32_t {
        require(ctx && stream && q && k && q_weight && k_weight && inout_q && inout_k, "qk_norm_rope: null argument");
        require(positions || !rope, "qk_norm_rope: a rotation needs positions");
        check_stream(ctx, stream, "qk_norm_rope");
        check_rows(ctx, q, "qk_norm_rope");
        check_rows(ctx, k, "qk_norm_rope");
        if (q->dtype != k->dtype) fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, "qk_norm_rope: q and k must have one dtype");
        if (q->shape[0] != k->shape[0] || q->shape[2] != k->shape[2])
            shape_err("qk_norm_rope: q and k must have the same rows and head size");
        for (const BeaconCudaTensor* w : {q_weight, k_weight}) {
            check_tensor(ctx, w, "qk_norm_rope");
            if (w->dtype != BEACON_CUDA_DTYPE_F32 && w->dtype != BEACON_CUDA_DTYPE_F16)
                fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, "qk_norm_rope: weights must be F32 or F16");
            if (w->numel() != q->shape[2]) shape_err("qk_norm_rope: a weight needs one value per head value");
        }
        if (!(eps >= 0.0f)) invalid("qk_norm_rope: eps must not be negative");
        if (positions) check_ids(ctx, positions, q->shape[0], "qk_norm_rope: positions");
        check_rope(ctx, rope, q->shape[2], "qk_norm_rope");
        DeviceScope dev(ctx);
        OutTensor oq(ctx, inout_q, q->shape, q->dtype, "qk_norm_rope"), ok(ctx, inout_k, k->shape, k->dtype, "qk_norm_rope");
        for (const BeaconCudaTensor* other : {q_weight, k_weight, positions}) {
            oq.check_overlap(other, false, "qk_norm_rope");
            ok.check_overlap(other, false, "qk_norm_rope");
        }
        oq.check_overlap(q, true, "qk_norm_rope");
        oq.check_overlap(k, false, "qk_norm_rope");
        ok.check_overlap(k, true, "qk_norm_rope");
        ok.check_overlap(q, false, "qk_norm_rope");
        ok.check_overlap(oq.get(), false, "qk_norm_rope");
        RowArgs a;
        const BeaconCudaTensor* in[2] = {q, k};
        const BeaconCudaTensor* w[2] = {q_weight, k_weight};
        void* dst[2] = {oq.data(), ok.data()};
        for (int i = 0; i < 2; ++i) {
            a.seg[i].src = in[i]->data();
            a.seg[i].dst = dst[i];
            a.seg[i].heads = (int)in[i]->shape[1];
            a.seg[i].weight = w[i]->data();
            a.seg[i].weight_dtype = w[i]->dtype;
            a.seg[i].turn = rope != nullptr;
        }
        a.tokens = q->shape[0];
        a.dim = (int)q->shape[2];
        a.eps = eps;
        a.positions = positions ? static_cast<const int32_t*>(positions->data()) : nullptr;
        launch_rows(ctx, a, q->dtype, q->dtype, rope, stream->s);
        oq.release();
        ok.release();
        return BEACON_CUDA_OK;
    });
}

int32_t beacon_cuda_op_paged_append(BeaconCudaContext* ctx, BeaconCudaStream* stream, BeaconCudaTensor* cache_k,
                                    BeaconCudaTensor* cache_v, const BeaconCudaTensor* new_k,
                                    const BeaconCudaTensor* new_v, const BeaconCudaTensor* page_table,
                                    const BeaconCudaTensor* seq_ids, const BeaconCudaTensor* positions,
                                    const BeaconCudaRope* rope) {
    return guard([&]() -> int32_t {
        require(ctx && stream && cache_k && cache_v && new_k && new_v && page_table && positions,
                "paged_append: null argument");
        check_stream(ctx, stream, "paged_append");
        check_rows(ctx, new_k, "paged_append");
        check_rows(ctx, new_v, "paged_append");
        if (new_k->shape != new_v->shape) shape_err("paged_append: new_k and new_v must have one shape");
        if (new_k->dtype != new_v->dtype) fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, "paged_append: new_k and new_v must have one dtype");
        for (const BeaconCudaTensor* c : {static_cast<const BeaconCudaTensor*>(cache_k), static_cast<const BeaconCudaTensor*>(cache_v)}) {
            check_tensor(ctx, c, "paged_append");
            if (c->dtype != BEACON_CUDA_DTYPE_F32 && c->dtype != BEACON_CUDA_DTYPE_F16 && c->dtype != BEACON_CUDA_DTYPE_BF16)
                fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, "paged_append: caches must be F32, F16 or BF16");
            if (c->shape.size() != 4 || c->shape[2] != new_k->shape[1] || c->shape[3] != new_k->shape[2] || c->shape[1] < 1)
                shape_err("paged_append: caches must be [pages, page_size, heads, dim]");
        }
        if (cache_k->shape != cache_v->shape || cache_k->dtype != cache_v->dtype)
            shape_err("paged_append: both caches must be alike");
        check_tensor(ctx, page_table, "paged_append");
        if (page_table->dtype != BEACON_CUDA_DTYPE_I32) fail(BEACON_CUDA_ERR_UNSUPPORTED_DTYPE, "paged_append: page_table must be I32");
        if (page_table->shape.size() != 2) shape_err("paged_append: page_table must be [B, max_pages]");
        const int64_t T = new_k->shape[0];
        check_ids(ctx, positions, T, "paged_append: positions");
        if (seq_ids) check_ids(ctx, seq_ids, T, "paged_append: seq_ids");
        else if (page_table->shape[0] != T) shape_err("paged_append: without seq_ids every row is a sequence of page_table");
        check_rope(ctx, rope, new_k->shape[2], "paged_append");
        DeviceScope dev(ctx);
        BeaconCudaTensor *pk = cache_k, *pv = cache_v;
        OutTensor ok(ctx, &pk, cache_k->shape, cache_k->dtype, "paged_append"), ov(ctx, &pv, cache_v->shape, cache_v->dtype, "paged_append");
        ok.check_overlap(cache_v, false, "paged_append");
        for (const BeaconCudaTensor* t : {new_k, new_v, page_table, seq_ids, positions}) {
            ok.check_overlap(t, false, "paged_append");
            ov.check_overlap(t, false, "paged_append");
        }
        RowArgs a;
        a.seg[0].src = new_k->data();
        a.seg[1].src = new_v->data();
        a.seg[0].dst = cache_k->data();
        a.seg[1].dst = cache_v->data();
        a.seg[0].heads = a.seg[1].heads = (int)new_k->shape[1];
        a.seg[0].turn = rope != nullptr;
        a.tokens = T;
        a.dim = (int)new_k->shape[2];
        a.positions = static_cast<const int32_t*>(positions->data());
        a.table = static_cast<const int32_t*>(page_table->data());
        a.seq_ids = seq_ids ? static_cast<const int32_t*>(seq_ids->data()) : nullptr;
        a.seqs = page_table->shape[0];
        a.max_pages = page_table->shape[1];
        a.pages = cache_k->shape[0];
        a.page_size = cache_k->shape[1];
        a.err = stream_error_word(stream);
        launch_rows(ctx, a, new_k->dtype, cache_k->dtype, rope, stream->s);
        return BEACON_CUDA_OK;
    });
}

}  // extern "C"
