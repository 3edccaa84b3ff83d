// Element types of the group norm, rotary and attention kernels: single
// element loads and stores, converting from and to fp32 (one rounding).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/ie_cuda_conv.h"

namespace ie_cuda {

// Bytes of one stored element (BF16X2: of one element of one plane).
__host__ __device__ constexpr int element_bytes(int type) { return type == IE_DT_F32 ? 4 : 2; }

template <int T>
__device__ __forceinline__ float load_element(const void* p, int64_t i) {
  if constexpr (T == IE_DT_F32) {
    return static_cast<const float*>(p)[i];
  } else if constexpr (T == IE_DT_F16) {
    return __half2float(static_cast<const __half*>(p)[i]);
  } else {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
}

template <int T>
__device__ __forceinline__ void store_element(void* p, int64_t i, float v) {
  if constexpr (T == IE_DT_F32) {
    static_cast<float*>(p)[i] = v;
  } else if constexpr (T == IE_DT_F16) {
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  } else {
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  }
}

}  // namespace ie_cuda
