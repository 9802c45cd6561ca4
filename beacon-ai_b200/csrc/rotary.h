// rotary.h -- rotation tables and the row kernel shared by the rotary, norm
// and cache-append operations (rotary.cu).
#pragma once

#include <atomic>
#include <memory>

#include "internal.h"
#include "kernels.h"

struct BeaconCudaRope {
    BeaconCudaContext* ctx = nullptr;
    int rotary_dim = 0;
    int layout = BEACON_CUDA_ROPE_INTERLEAVED;
    float amplitude = 1.0f;                   // factor on sine and cosine
    std::unique_ptr<bc::DeviceBuffer> turns;  // f64 [rotary_dim / 2]: f_i / 2 pi
};

namespace bc {

// Makes the context's device current for a call and puts back the caller's.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(const BeaconCudaContext* ctx) {
        BC_CUDA(cudaGetDevice(&before));
        if (before == ctx->device)
            before = -1;
        else
            BC_CUDA(cudaSetDevice(ctx->device));
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// The output of an operation: the caller's tensor, checked against the
// result's shape, dtype and inputs, or a new one that is handed over last.
class OutTensor {
   public:
    OutTensor(BeaconCudaContext* ctx, BeaconCudaTensor** inout, const std::vector<int64_t>& shape, int32_t dtype,
              const char* what);
    void* data() const { return t_->data(); }
    BeaconCudaTensor* get() const { return t_; }
    // The output may be `x` itself (same bytes) when in_place, else must not touch it.
    void check_overlap(const BeaconCudaTensor* x, bool in_place, const char* what) const;
    void release() {
        made_.release();
        *inout_ = t_;
    }

   private:
    BeaconCudaTensor** inout_;
    BeaconCudaTensor* t_;
    std::unique_ptr<BeaconCudaTensor> made_;  // freed if the call throws
};

// Tensors of an operation must live on its context.
void check_tensor(const BeaconCudaContext* ctx, const BeaconCudaTensor* t, const char* what);
void check_stream(const BeaconCudaContext* ctx, const BeaconCudaStream* stream, const char* what);
// allow_max_dynamic_smem once per device for a kernel (`done`: one flag word of
// its own, a bit per device): the two driver calls cost more than a launch.
template <typename K>
void allow_smem_once(K kern, const BeaconCudaContext* ctx, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (ctx->device < 64 && (done.load(std::memory_order_acquire) & bit)) return;
    allow_max_dynamic_smem(kern);
    done.fetch_or(bit, std::memory_order_release);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
}  // namespace bc
