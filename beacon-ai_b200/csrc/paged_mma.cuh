// paged_mma.cuh -- 16-bit types, warp-level matrix instructions and copies of
// the paged attention kernels.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace bc {

template <typename T>
struct Half2Of;
template <>
struct Half2Of<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};
template <>
struct Half2Of<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
};

// Softmax weights for the value product are rounded to the cache's type. f16
// ends at 2^-24 (normal values at 2^-14), so weights of at most 1 would lose
// their bits from 2^-14 down and vanish below 2^-25, while their sum kept them:
// thousands of small ones beside one large one would be lost from the result.
// They are taken times a power of two that brings the largest near the top of
// the range, and their sums alike, so that nothing else changes.
template <typename T>
constexpr bool kNarrowExponent = false;
template <>
constexpr bool kNarrowExponent<__half> = true;

// 2^x (relative error 2^-22; -inf gives 0).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes to shared memory, or 16 zero bytes when !live (src is not read).
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// d[16 x 8] += a[16 x 16] b[16 x 8], f32 sums.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ unsigned long long as_u64(float2 v) { return *reinterpret_cast<unsigned long long*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)), "l"(as_u64(c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)));
    return *reinterpret_cast<float2*>(&d);
}

// Bounded wait (mbar_wait_bounded) whose limit is already in a register and
// that reads the clock only when the barrier is not there yet.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, long long limit) {
    if (mbar_test_wait(bar, parity)) return true;
    const long long t0 = clock64();
    if (limit >= kBoundedWaitLimit) {
        while (!mbar_try_wait(bar, parity))
            if (clock64() - t0 > limit) return false;
        return true;
    }
    while (!mbar_test_wait(bar, parity))
        if (clock64() - t0 > limit) return false;
    return true;
}

// Rows [row, row + box) of one head, 64 values from x on, to shared memory.
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar))
        : "memory");
}

// The power of two that brings the largest magnitude mx of a 32-bit query row
// to [2^14, 2^15), so that its f16 parts neither overflow nor lose bits, and its
// reciprocal (exponent arithmetic; exponents below 2^-112 stay smaller). Rows
// that are not finite come out as such.
__device__ __forceinline__ float query_scale(float mx, float& inverse) {
    const int e = min(254, max(15, (int)(__float_as_uint(mx) >> 23)));  // mx >= 0
    inverse = __uint_as_float((uint32_t)(e - 14) << 23);
    return __uint_as_float((uint32_t)(268 - e) << 23);
}

// x as a sum of two f16 values (hi: rounded, lo: what that left, rounded).
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

}  // namespace bc
