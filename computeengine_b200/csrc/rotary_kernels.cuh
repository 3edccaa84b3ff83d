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
  int block_tokens, block_heads;    // per block
  SmallDivisor units;               // units of a rotated head
  SmallDivisor head_count;          // block_heads
  SmallDivisor copies;              // units of a converted head
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

// Place of one of a unit's 2 W table values (cosines, then sines).
template <int W>
__device__ __forceinline__ int table_at(int units, int unit, int value) {  // of 2 W values
  return W == 1 ? 2 * unit + value : ((value >> 2) * units + unit) * 4 + (value & 3);
}

// One block takes a few tokens (and, when there are few of them, a share of
// their heads): the cosines and sines of a token are taken once for all its
// heads and kept in shared memory, then every thread rotates W pairs at a
// time, loaded and stored as vectors of W elements.  Memory bound; the first
// loads are issued before the angles are known.  Tables lie so that threads of
// neighbouring units read neighbouring 16 bytes (a unit's values in a row
// would be a 4-way bank conflict), and the kernel's parameters are read by
// index only once per block (threads of different indices are served in turn).
// 32760 tokens x 48 heads x 128 bf16: 130 us, 95% of a copy's bandwidth; 4096 x
// 48 heads x 72, fp32 to bf16: 23 us, 57%.
//
// W: pairs per unit; divides the layout's runs of pairs, the elements that are
// not rotated and all strides, and the tensors are aligned to it.
// CW: elements per unit of the heads that are only converted.
template <int XT, int YT, int W, int CW>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float table[];  // [tokens of the block][2 pairs], unit offsets
  constexpr int XB = W * element_bytes(XT), YB = W * element_bytes(YT);
  constexpr int K = XB >= 16 ? 2 : 4;  // units in flight per thread
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.block_tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(a.block_tokens), a.tokens - t0));
  const uint8_t* x = static_cast<const uint8_t*>(a.x);
  uint8_t* y = static_cast<uint8_t*>(a.y);
  const int units = static_cast<int>(a.units.d);
  uint32_t* offsets = reinterpret_cast<uint32_t*>(table + a.block_tokens * 2 * a.pairs);
  for (int i = threadIdx.x; i < units; i += 256) {
    int u, v;
    rotary_pair(a, i * W, &u, &v);
    // PAIRS: 2 W neighbours, as two vectors
    offsets[i] = a.layout == IE_ROTARY_PAIRS ? u | (u + W) << 16 : u | v << 16;
  }
  __syncthreads();

  // units of the rotated heads: [token][head of this block][unit of the head]
  const int h0 = static_cast<int>(blockIdx.y) * a.block_heads;
  const int heads = max(0, min(a.block_heads, a.rot_heads - h0));
  const int items = tokens * heads * units;
  Bytes<XB> xu[K], xv[K];
  uint8_t* yu[K];
  uint8_t* yv[K];
  int at[K];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = base + k * 256;
      if (i >= items) break;
      const uint32_t q = a.units.quotient(i);
      const int unit = static_cast<int>(i - q * a.units.d);
      // one token: q counts whatever heads the block has
      const uint32_t tok = tokens == 1 ? 0 : a.head_count.quotient(q);
      const int64_t h = h0 + static_cast<int>(q - tok * a.head_count.d);
      const uint32_t uv = offsets[unit];
      const uint8_t* px = x + ((t0 + tok) * a.x_token_stride + h * a.x_head_stride) *
                                  element_bytes(XT);
      uint8_t* py = y + ((t0 + tok) * a.y_token_stride + h * a.y_head_stride) * element_bytes(YT);
      const uint32_t u = uv & 0xFFFFu, v = uv >> 16;
      xu[k] = load_bytes<XB>(px + u * element_bytes(XT));
      xv[k] = load_bytes<XB>(px + v * element_bytes(XT));
      yu[k] = py + u * element_bytes(YT);
      yv[k] = py + v * element_bytes(YT);
      at[k] = static_cast<int>(tok) * 2 * a.pairs + (W == 1 ? 2 : 4) * unit;
    }
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < tokens * a.pairs; i += 256) {
    const int tok = i / a.pairs, pair = i - tok * a.pairs;
    const float2 cs = rotary_angle(a, t0 + tok, pair);
    float* c = table + tok * 2 * a.pairs;
    c[table_at<W>(units, pair / W, pair % W)] = cs.x;
    c[table_at<W>(units, pair / W, W + pair % W)] = cs.y;
  }
  __syncthreads();
  for (int base = threadIdx.x; base < items; base += K * 256) {
    if (base >= K * 256) load(base);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (base + k * 256 >= items) break;
      float cs[2 * W];
      if constexpr (W == 1) {
        const float2 c = *reinterpret_cast<const float2*>(table + at[k]);
        cs[0] = c.x;
        cs[1] = c.y;
      } else {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) {
          const float4 c = *reinterpret_cast<const float4*>(table + at[k] + 4 * j * units);
          cs[4 * j] = c.x;
          cs[4 * j + 1] = c.y;
          cs[4 * j + 2] = c.z;
          cs[4 * j + 3] = c.w;
        }
      }
      float f[2 * W];
      {
        float fu[W], fv[W];
        to_floats<XT, W>(xu[k], fu);
        to_floats<XT, W>(xv[k], fv);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          f[e] = fu[e];
          f[W + e] = fv[e];
        }
      }
      float gu[W], gv[W];
      if (a.layout == IE_ROTARY_PAIRS) {
        float g[2 * W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          g[2 * e] = f[2 * e] * cs[e] - f[2 * e + 1] * cs[W + e];
          g[2 * e + 1] = f[2 * e] * cs[W + e] + f[2 * e + 1] * cs[e];
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          gu[e] = g[e];
          gv[e] = g[W + e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          gu[e] = f[e] * cs[e] - f[W + e] * cs[W + e];
          gv[e] = f[e] * cs[W + e] + f[W + e] * cs[e];
        }
      }
      store_bytes<YB>(yu[k], from_floats<YT, W>(gu));
      store_bytes<YB>(yv[k], from_floats<YT, W>(gv));
    }
  }
  if (a.in_place) return;
  // what is only converted: the ends of the rotated heads, and the other heads
  const int rest = (a.head_dim - 2 * a.pairs) / W;
  for (int i = threadIdx.x; i < tokens * heads * rest; i += 256) {
    const int tok = i / (heads * rest), r = i - tok * heads * rest;
    const int64_t h = h0 + r / rest;
    const int e = 2 * a.pairs + r % rest * W;
    float f[W];
    to_floats<XT, W>(load_bytes<XB>(x + ((t0 + tok) * a.x_token_stride + h * a.x_head_stride + e) *
                                            element_bytes(XT)),
                     f);
    store_bytes<YB>(
        y + ((t0 + tok) * a.y_token_stride + h * a.y_head_stride + e) * element_bytes(YT),
        from_floats<YT, W>(f));
  }
  constexpr int CXB = CW * element_bytes(XT), CYB = CW * element_bytes(YT), CK = CXB > 16 ? 2 : 4;
  const uint32_t others = (a.heads - a.rot_heads) * a.copies.d;
  for (int tok = 0; tok < tokens; ++tok) {
    const uint8_t* xt = x + (t0 + tok) * a.x_token_stride * element_bytes(XT);
    uint8_t* yt = y + (t0 + tok) * a.y_token_stride * element_bytes(YT);
    const uint32_t step = gridDim.y * 256;
    for (uint32_t base = blockIdx.y * 256 + threadIdx.x; base < others; base += CK * step) {
      Bytes<CXB> v[CK];
      uint8_t* to[CK];
#pragma unroll
      for (int k = 0; k < CK; ++k) {
        const uint32_t i = base + k * step;
        if (i >= others) break;
        const uint32_t q = a.copies.quotient(i);
        const int64_t h = a.rot_heads + q;
        const uint32_t e = (i - q * a.copies.d) * CW;
        v[k] = load_bytes<CXB>(xt + (h * a.x_head_stride + e) * element_bytes(XT));
        to[k] = yt + (h * a.y_head_stride + e) * element_bytes(YT);
      }
#pragma unroll
      for (int k = 0; k < CK; ++k) {
        if (base + k * step >= others) break;
        float f[CW];
        to_floats<XT, CW>(v[k], f);
        store_bytes<CYB>(to[k], from_floats<YT, CW>(f));
      }
    }
  }
}

}  // namespace ie_cuda
