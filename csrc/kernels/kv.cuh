// Device helpers of the paged KV cache operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels/common.cuh"
#include "kernels/kv.h"

namespace mpcomm {
namespace kern {

// Makes `device` current for a scope.
class DeviceScope {
 public:
    explicit DeviceScope(int device) {
        int now = -1;
        error_ = static_cast<int>(cudaGetDevice(&now));
        if (error_ || now == device) return;
        error_ = static_cast<int>(cudaSetDevice(device));
        if (!error_) back_ = now;
    }
    ~DeviceScope() {
        if (back_ >= 0) cudaSetDevice(back_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    int error() const { return error_; }

 private:
    int error_ = 0;
    int back_ = -1;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (std::is_same_v<T, __half>) return __half2float(v);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
    else return v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
    else return v;
}

}  // namespace kern
}  // namespace mpcomm
