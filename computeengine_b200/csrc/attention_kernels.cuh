// Attention with a tanh cap, a distance bias and causal, prefix, length and
// document masks.
#pragma once

#include "attention_common.cuh"

namespace ie_cuda {

// One warp per (query row, head), one key at a time, running maximum and sum.
template <int T, int OT>
__global__ void __launch_bounds__(128) attention_simple_kernel(const AttentionArgs a) {
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int h = blockIdx.y;
  if (i >= a.q_len) return;
  int r = blockIdx.z;
  if (a.documents > 0) {  // the document that holds row i
    int lo = 0, hi = a.documents;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.q_offsets[mid + 1] > i) hi = mid;
      else lo = mid + 1;
    }
    if (lo >= a.documents || a.q_offsets[lo] > i) return;
    r = lo;
  }
  const Sequence s = sequence(a, r);
  const int hk = static_cast<int>(static_cast<int64_t>(h) * a.kv_heads / a.q_heads);
  const int64_t qo = s.batch * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2];
  const int64_t ko = s.batch * a.k_stride[0] + s.k0 * a.k_stride[1] + hk * a.k_stride[2];
  const int64_t vo = s.batch * a.v_stride[0] + s.k0 * a.v_stride[1] + hk * a.v_stride[2];
  float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 32 * e;
    q[e] = d < a.head_dim ? load_element<T>(a.q, qo + d) : 0.0f;
  }
  const float slope = a.slopes == nullptr ? 0.0f : a.slopes[h];
  const int place = s.place(i), seen = s.seen(i, a.causal);
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < seen; ++j) {
    float x = 0.0f;
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      if (d < a.head_dim) x += q[e] * load_element<T>(a.k, ko + j * a.k_stride[1] + d);
    }
    for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, w);
    x *= a.scale;
    if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
    x -= slope * fabsf(static_cast<float>(place - j));
    const float top = fmaxf(m, x);
    const float base = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - base), p = expf(x - base);
    m = top;
    l = l * keep + p;
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      if (d < a.head_dim) {
        o[e] = o[e] * keep + p * load_element<T>(a.v, vo + j * a.v_stride[1] + d);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t oo = s.batch * a.o_stride[0] + i * a.o_stride[1] + h * a.o_stride[2];
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 32 * e;
    if (d >= a.head_dim) continue;
    const float y = l == 0.0f ? 0.0f : o[e] * inv;
    if constexpr (OT == IE_DT_BF16X2) {
      const float hi = __bfloat162float(__float2bfloat16_rn(y));
      store_element<IE_DT_BF16>(a.o, oo + d, hi);
      store_element<IE_DT_BF16>(a.o, oo + a.o_lo + d, y - hi);
    } else {
      store_element<OT>(a.o, oo + d, y);
    }
  }
  if (a.lse != nullptr && lane == 0) {
    a.lse[(static_cast<int64_t>(s.batch) * a.q_heads + h) * a.q_len + i] =
        l == 0.0f ? -INFINITY : m + logf(l);
  }
}

}  // namespace ie_cuda
