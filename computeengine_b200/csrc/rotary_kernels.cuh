// Rotary positions over several axes.
#pragma once

#include "element_types.cuh"

namespace ie_cuda {

struct RotaryArgs {
  const void* x;
  const void* positions;
  void* y;
  int64_t tokens, x_token_stride, x_head_stride, y_token_stride, y_head_stride, pos_axis_stride;
  int heads, rot_heads, head_dim, pairs, layout, inverse, pos64, in_place;
  int first[4], section[4];  // first pair and number of pairs of each axis
  uint64_t turns[128];
  uint8_t axis[128];
};

// The two elements of pair i.
__device__ __forceinline__ void rotary_pair(const RotaryArgs& a, int i, int* u, int* v) {
  if (a.layout == IE_ROTARY_PAIRS) {
    *u = 2 * i;
    *v = 2 * i + 1;
  } else if (a.layout == IE_ROTARY_HALVES) {
    *u = i;
    *v = i + a.pairs;
  } else {
    const int ax = a.axis[i];
    *u = a.first[ax] + i;  // 2 * first + (i - first)
    *v = *u + a.section[ax];
  }
}

// cos and sin of pair i at token t.  The product of the position and the
// frequency in 2^-64 turns is the angle modulo one turn, exactly, whatever
// the position; as a signed number it is within half a turn.
__device__ __forceinline__ float2 rotary_angle(const RotaryArgs& a, int64_t t, int i) {
  const int64_t at = a.axis[i] * a.pos_axis_stride + t;
  const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                              : static_cast<const int32_t*>(a.positions)[at];
  const int64_t turn = static_cast<int64_t>(static_cast<uint64_t>(pos) * a.turns[i]);
  float s, c;
  sincospif(static_cast<float>(turn) * 0x1p-63f, &s, &c);
  return make_float2(c, a.inverse ? -s : s);
}

// One block per token, one thread per pair or pass-through element.
template <int XT, int YT>
__global__ void __launch_bounds__(128) rotary_simple_kernel(const __grid_constant__ RotaryArgs a) {
  __shared__ float2 cs[128];
  const int64_t t = blockIdx.x;
  for (int i = threadIdx.x; i < a.pairs; i += blockDim.x) cs[i] = rotary_angle(a, t, i);
  __syncthreads();
  const int rest = a.head_dim - 2 * a.pairs;
  for (int h = 0; h < a.heads; ++h) {
    const int64_t xo = t * a.x_token_stride + h * a.x_head_stride;
    const int64_t yo = t * a.y_token_stride + h * a.y_head_stride;
    if (h < a.rot_heads) {
      for (int i = threadIdx.x; i < a.pairs; i += blockDim.x) {
        int u, v;
        rotary_pair(a, i, &u, &v);
        const float xu = load_element<XT>(a.x, xo + u), xv = load_element<XT>(a.x, xo + v);
        store_element<YT>(a.y, yo + u, xu * cs[i].x - xv * cs[i].y);
        store_element<YT>(a.y, yo + v, xu * cs[i].y + xv * cs[i].x);
      }
    }
    if (!a.in_place) {
      const int from = h < a.rot_heads ? a.head_dim - rest : 0;
      for (int e = from + threadIdx.x; e < a.head_dim; e += blockDim.x) {
        store_element<YT>(a.y, yo + e, load_element<XT>(a.x, xo + e));
      }
    }
  }
}

}  // namespace ie_cuda
