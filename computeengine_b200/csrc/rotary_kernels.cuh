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

// One block takes a few tokens (and, when there are few of them, a share of
// their heads): the cosines and sines of a token are taken once for all its
// heads and kept in shared memory, then every thread rotates W pairs at a
// time, loaded and stored as vectors of W elements.  Memory bound; the first
// loads are issued before the angles are known.
//
// W: pairs per unit; divides the layout's runs of pairs, the elements that are
// not rotated and all strides, and the tensors are aligned to it.
// CW: elements per unit of the heads that are only converted.
template <int XT, int YT, int W, int CW>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float2 cs[];  // [tokens of the block][pairs]
  constexpr int XB = W * element_bytes(XT), YB = W * element_bytes(YT);
  constexpr int K = XB > 16 ? 2 : 4;  // units in flight per thread
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.block_tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(a.block_tokens), a.tokens - t0));
  const uint8_t* x = static_cast<const uint8_t*>(a.x);
  uint8_t* y = static_cast<uint8_t*>(a.y);

  // units of the rotated heads: [token][head of this block][unit of the head]
  const int h0 = static_cast<int>(blockIdx.y) * a.block_heads;
  const int heads = max(0, min(a.block_heads, a.rot_heads - h0));
  const int per_token = heads * static_cast<int>(a.units.d);
  const int items = tokens * per_token;
  auto place = [&](int i, int* tok, int* pair, int64_t* xo, int64_t* yo) {
    const uint32_t q = a.units.quotient(i);
    *pair = static_cast<int>(i - q * a.units.d) * W;
    // heads of this block: all of them, or (one token) whatever is left
    const uint32_t tk = tokens == 1 ? 0 : a.head_count.quotient(q);
    const int h = static_cast<int>(q - tk * a.head_count.d);
    *tok = static_cast<int>(tk);
    *xo = (t0 + tk) * a.x_token_stride + (h0 + h) * a.x_head_stride;
    *yo = (t0 + tk) * a.y_token_stride + (h0 + h) * a.y_head_stride;
  };
  // memory offsets of the first and second W elements of the unit at `pair`
  auto halves = [&](int pair, int* u, int* v) {
    if (a.layout == IE_ROTARY_PAIRS) {
      *u = 2 * pair;
      *v = 2 * pair + W;
    } else {
      rotary_pair(a, pair, u, v);
    }
  };
  Bytes<XB> xu[K], xv[K];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = base + k * 256;
      if (i >= items) break;
      int tok, pair, u, v;
      int64_t xo, yo;
      place(i, &tok, &pair, &xo, &yo);
      halves(pair, &u, &v);
      xu[k] = load_bytes<XB>(x + (xo + u) * element_bytes(XT));
      xv[k] = load_bytes<XB>(x + (xo + v) * element_bytes(XT));
    }
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < tokens * a.pairs; i += 256) {
    const int tok = i / a.pairs;
    cs[i] = rotary_angle(a, t0 + tok, i - tok * a.pairs);
  }
  __syncthreads();
  for (int base = threadIdx.x; base < items; base += K * 256) {
    if (base >= K * 256) load(base);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = base + k * 256;
      if (i >= items) break;
      int tok, pair, u, v;
      int64_t xo, yo;
      place(i, &tok, &pair, &xo, &yo);
      halves(pair, &u, &v);
      const float2* c = cs + tok * a.pairs + pair;
      float fu[W], fv[W];
      to_floats<XT, W>(xu[k], fu);
      to_floats<XT, W>(xv[k], fv);
      if (a.layout == IE_ROTARY_PAIRS) {
        // fu, fv are 2 W consecutive elements: pairs of neighbours
        float f[2 * W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          f[e] = fu[e];
          f[W + e] = fv[e];
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float p = f[2 * e], q = f[2 * e + 1];
          f[2 * e] = p * c[e].x - q * c[e].y;
          f[2 * e + 1] = p * c[e].y + q * c[e].x;
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          fu[e] = f[e];
          fv[e] = f[W + e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float p = fu[e], q = fv[e];
          fu[e] = p * c[e].x - q * c[e].y;
          fv[e] = p * c[e].y + q * c[e].x;
        }
      }
      store_bytes<YB>(y + (yo + u) * element_bytes(YT), from_floats<YT, W>(fu));
      store_bytes<YB>(y + (yo + v) * element_bytes(YT), from_floats<YT, W>(fv));
    }
  }
  if (a.in_place) return;
  // what is only converted: the ends of the rotated heads, and the other heads
  const int rest = a.head_dim - 2 * a.pairs;
  for (int tok = 0; tok < tokens; ++tok) {
    const int64_t xt = (t0 + tok) * a.x_token_stride, yt = (t0 + tok) * a.y_token_stride;
    for (int i = threadIdx.x; i < heads * (rest / W); i += 256) {
      const int h = h0 + i / (rest / W);
      const int e = 2 * a.pairs + i % (rest / W) * W;
      float f[W];
      to_floats<XT, W>(load_bytes<XB>(x + (xt + h * a.x_head_stride + e) * element_bytes(XT)), f);
      store_bytes<YB>(y + (yt + h * a.y_head_stride + e) * element_bytes(YT),
                      from_floats<YT, W>(f));
    }
    const uint32_t step = gridDim.y * 256;
    const uint32_t others = (a.heads - a.rot_heads) * a.copies.d;
    for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < others; i += step) {
      const uint32_t q = a.copies.quotient(i);
      const int64_t h = a.rot_heads + q;
      const int e = static_cast<int>(i - q * a.copies.d) * CW;
      constexpr int CXB = CW * element_bytes(XT), CYB = CW * element_bytes(YT);
      float f[CW];
      to_floats<XT, CW>(load_bytes<CXB>(x + (xt + h * a.x_head_stride + e) * element_bytes(XT)),
                        f);
      store_bytes<CYB>(y + (yt + h * a.y_head_stride + e) * element_bytes(YT),
                       from_floats<YT, CW>(f));
    }
  }
}

}  // namespace ie_cuda
