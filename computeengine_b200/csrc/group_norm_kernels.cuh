// Group normalization with an activation over channels-last tensors.
#pragma once

#include "element_types.cuh"

namespace ie_cuda {

struct GroupNormArgs {
  const void* x;
  const float* gamma;
  const float* beta;
  void* y;
  int64_t pixels;  // h * w
  int c, c_store, groups, act;
  float eps;
};

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case IE_ACT_RELU:
      return v < 0.0f ? 0.0f : v;  // NaN stays
    case IE_ACT_RELU6:
      return v < 0.0f ? 0.0f : v > 6.0f ? 6.0f : v;
    case IE_ACT_SILU:
      return v / (1.0f + expf(-v));
    case IE_ACT_GELU:
      return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    default:
      return v;
  }
}

// Element e of pixel p of image n; BF16X2 holds two planes of c_store.
template <int T>
__device__ __forceinline__ float gn_load(const void* x, int64_t pixel, int c_store, int c) {
  if constexpr (T == IE_DT_BF16X2) {
    return load_element<IE_DT_BF16>(x, pixel * 2 * c_store + c) +
           load_element<IE_DT_BF16>(x, pixel * 2 * c_store + c_store + c);
  } else {
    return load_element<T>(x, pixel * c_store + c);
  }
}

template <int T>
__device__ __forceinline__ void gn_store(void* y, int64_t pixel, int c_store, int c, float v) {
  if constexpr (T == IE_DT_BF16X2) {
    const float hi = __bfloat162float(__float2bfloat16_rn(v));
    store_element<IE_DT_BF16>(y, pixel * 2 * c_store + c, hi);
    store_element<IE_DT_BF16>(y, pixel * 2 * c_store + c_store + c, v - hi);
  } else {
    store_element<T>(y, pixel * c_store + c, v);
  }
}

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (unsigned i = 0; i < (blockDim.x + 31) / 32; ++i) s += scratch[i];
  __syncthreads();
  return s;
}

// One block per (group, image): mean, variance, then the normalized values,
// three reads of x.
template <int XT, int YT>
__global__ void __launch_bounds__(256) group_norm_simple_kernel(const GroupNormArgs a) {
  __shared__ float scratch[8];
  const int cg = a.c / a.groups;
  const int c0 = blockIdx.x * cg;
  const int64_t p0 = static_cast<int64_t>(blockIdx.y) * a.pixels;
  const int64_t count = a.pixels * cg;
  float sum = 0.0f;
  for (int64_t i = threadIdx.x; i < count; i += blockDim.x) {
    sum += gn_load<XT>(a.x, p0 + i / cg, a.c_store, c0 + static_cast<int>(i % cg));
  }
  const float mean = block_sum(sum, scratch) / static_cast<float>(count);
  sum = 0.0f;
  for (int64_t i = threadIdx.x; i < count; i += blockDim.x) {
    const float d =
        gn_load<XT>(a.x, p0 + i / cg, a.c_store, c0 + static_cast<int>(i % cg)) - mean;
    sum += d * d;
  }
  const float rstd = rsqrtf(block_sum(sum, scratch) / static_cast<float>(count) + a.eps);
  for (int64_t i = threadIdx.x; i < count; i += blockDim.x) {
    const int c = c0 + static_cast<int>(i % cg);
    const float v = (gn_load<XT>(a.x, p0 + i / cg, a.c_store, c) - mean) * rstd;
    const float g = a.gamma == nullptr ? 1.0f : a.gamma[c];
    const float b = a.beta == nullptr ? 0.0f : a.beta[c];
    gn_store<YT>(a.y, p0 + i / cg, a.c_store, c, activate(v * g + b, a.act));
  }
  const int pad = a.c_store - a.c;
  if (blockIdx.x == 0 && pad > 0) {
    for (int64_t i = threadIdx.x; i < a.pixels * pad; i += blockDim.x) {
      gn_store<YT>(a.y, p0 + i / pad, a.c_store, a.c + static_cast<int>(i % pad), 0.0f);
    }
  }
}

}  // namespace ie_cuda
