// What the attention kernels share: launch arguments, which keys a sequence's
// queries see, the score's cap and bias.
#pragma once

#include "element_types.cuh"

namespace ie_cuda {

constexpr int kMaxSplits = 1024;  // shares of one sequence's keys

struct AttentionArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;
  int64_t q_stride[3], k_stride[3], v_stride[3], o_stride[3];  // batch, token, head
  int64_t o_lo;        // elements from the hi to the lo plane, BF16X2 output
  int batch, q_len, kv_len, q_heads, kv_heads, head_dim;
  int causal, documents;
  const int32_t* kv_lens;
  const int32_t* prefix_lens;
  const int32_t* q_offsets;
  const int32_t* kv_offsets;
  const float* slopes;
  float scale, softcap;
};

// One sequence: its query and key rows within the batch row, and its prefix.
struct Sequence {
  int batch, q0, q1, k0, k1, prefix;

  // Place of query row i among the sequence's keys, counted from k0.
  __device__ __forceinline__ int place(int i) const { return i - q0 + (k1 - k0) - (q1 - q0); }
  // Keys k0 .. k0 + seen - 1 are what query row i sees.
  __device__ __forceinline__ int seen(int i, int causal) const {
    const int length = k1 - k0;
    if (!causal) return length;
    return min(length, max(prefix, max(0, place(i) + 1)));
  }
};

// Sequence r: a batch row, or a document of the one batch row.  Lengths and
// offsets come from device memory and are clamped to the tensors.
__device__ __forceinline__ Sequence sequence(const AttentionArgs& a, int r) {
  Sequence s;
  if (a.documents > 0) {
    s.batch = 0;
    s.q0 = min(max(a.q_offsets[r], 0), a.q_len);
    s.q1 = min(max(a.q_offsets[r + 1], s.q0), a.q_len);
    s.k0 = min(max(a.kv_offsets[r], 0), a.kv_len);
    s.k1 = min(max(a.kv_offsets[r + 1], s.k0), a.kv_len);
  } else {
    s.batch = r;
    s.q0 = 0;
    s.q1 = a.q_len;
    s.k0 = 0;
    s.k1 = a.kv_lens == nullptr ? a.kv_len : min(max(a.kv_lens[r], 0), a.kv_len);
  }
  s.prefix = a.prefix_lens == nullptr ? 0 : max(a.prefix_lens[r], 0);
  return s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- cap * tanh(s / cap), in units of log2 e.  With u = s / cap:
//   |u| <= kTanhLimit   s * (tanh(u) / u), the ratio a polynomial in u^2 (minimax
//                       of tanh u with slope 1 at 0, absolute error below 2.7e-7)
//   beyond              cap * (1 - 2 / (1 + exp(2 u)))
// Either is off by a few 2^-22 of the result, whatever the cap: the second form
// alone is off by that of the cap, 0.1 for scores of 1 under a cap of 10^6.
// Up to kSmallCap the second form's error, 2^-17 then, is far below that of the
// 16-bit weights, and the prompt kernel takes it for all scores of a warp when one is
// beyond kTanhLimit: 284 us against 303 us with both forms (4096 tokens, 16 heads
// of 128, a cap of 2 and nearly all scores beyond it).
constexpr float kTanhLimit = 0.75f;
constexpr float kSmallCap = 64.0f;
constexpr float kTanh1 = -0.33328044414520264f, kTanh2 = 0.13253363966941833f,
                kTanh3 = -0.04986608773469925f, kTanh4 = 0.012750583700835705f;

// u per unit of q.k.  Held below overflow: a cap that small leaves no score.
__device__ __forceinline__ float cap_argument(const AttentionArgs& a) {
  return fminf(fmaxf(a.scale / a.softcap, -1e30f), 1e30f);
}

__device__ __forceinline__ float tanh_ratio(float uu) {
  float p = fmaf(uu, kTanh4, kTanh3);
  p = fmaf(p, uu, kTanh2);
  p = fmaf(p, uu, kTanh1);
  return fmaf(p, uu, 1.0f);
}

// Weights are 2^(score - maximum in use + this), at most 2^15: fp16 would otherwise
// hold those below 2^-14 of the largest with fewer bits and none below 2^-25, which
// many keys behind a heavy one add up to.  The factor cancels in o.
template <int T>
constexpr float kWeightShift = T == IE_DT_F16 ? 7.0f : 0.0f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// The sequence and first query row of a tile of `rows` query rows; false when
// it has none.  Documents: the tiles are counted through all documents.
__device__ __forceinline__ bool tile_sequence(const AttentionArgs& a, int tile, int batch_row,
                                              int rows, Sequence* s, int* row0) {
  if (a.documents == 0) {
    *s = sequence(a, batch_row);
    *row0 = tile * rows;
    return *row0 < s->q1;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int r0 = 0; r0 < a.documents; r0 += 32) {
    const int r = r0 + lane;
    int count = 0;
    if (r < a.documents) {
      const Sequence d = sequence(a, r);
      count = (d.q1 - d.q0 + rows - 1) / rows;
    }
    int sum = count;
    for (int w = 1; w < 32; w <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, sum, w);
      if (lane >= w) sum += up;
    }
    const unsigned hit = __ballot_sync(0xFFFFFFFFu, before + sum > tile);
    if (hit != 0) {
      const int at = __ffs(hit) - 1;
      const int skipped = before + __shfl_sync(0xFFFFFFFFu, sum - count, at);
      *s = sequence(a, r0 + at);
      *row0 = s->q0 + (tile - skipped) * rows;
      return true;
    }
    before += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  return false;
}

// Joins the shares of split sequences: one block per row and head.  The
// shares' weights are taken by all threads at once, then each warp sums every
// fourth share.
template <int OT>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttentionArgs a, int splits,
                                                             const float* part_o,
                                                             const float* part_lse) {
  __shared__ float weight[kMaxSplits], warp_top[4], warp_total[4], warp_y[4][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = int64_t{a.batch} * a.q_heads * a.q_len;
  const int64_t at = blockIdx.x;
  const int i = static_cast<int>(at % a.q_len);
  const int h = static_cast<int>(at / a.q_len % a.q_heads);
  const int64_t b = at / a.q_len / a.q_heads;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // until the shares are written
  float top = -INFINITY;
  for (int s = threadIdx.x; s < splits; s += 128) {
    weight[s] = part_lse[s * rows + at];
    top = max_nan(top, weight[s]);
  }
  for (int w = 16; w > 0; w >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
  for (int w = 0; w < 4; ++w) top = max_nan(top, warp_top[w]);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* o = part_o + at * a.head_dim;
#pragma unroll 4
  for (int s = warp; s < splits; s += 4) {
    const float w = expf(weight[s] - base);
    total += w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      const float v = d < a.head_dim ? o[s * rows * a.head_dim + d] : 0.0f;
      y[e] = fmaf(w, v, y[e]);
    }
  }
  if (lane == 0) warp_total[warp] = total;
#pragma unroll
  for (int e = 0; e < 4; ++e) warp_y[warp][lane + 32 * e] = y[e];
  __syncthreads();
  total = (warp_total[0] + warp_total[1]) + (warp_total[2] + warp_total[3]);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int d = threadIdx.x;
  if (d < a.head_dim) {
    const float v = ((warp_y[0][d] + warp_y[1][d]) + (warp_y[2][d] + warp_y[3][d])) * inv;
    const int64_t oo = b * a.o_stride[0] + i * a.o_stride[1] + h * a.o_stride[2];
    if constexpr (OT == IE_DT_BF16X2) {
      const float hi = __bfloat162float(__float2bfloat16_rn(v));
      store_element<IE_DT_BF16>(a.o, oo + d, hi);
      store_element<IE_DT_BF16>(a.o, oo + a.o_lo + d, v - hi);
    } else {
      store_element<OT>(a.o, oo + d, v);
    }
  }
  if (a.lse != nullptr && d == 0) a.lse[at] = total == 0.0f ? -INFINITY : base + logf(total);
}

}  // namespace ie_cuda
