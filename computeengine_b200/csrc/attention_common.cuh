// What the attention kernels share: launch arguments, which keys a sequence's
// queries see, the score's cap and bias.
#pragma once

#include "element_types.cuh"

namespace ie_cuda {

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

// Joins the shares of split sequences: one warp per row and head.
template <int OT>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttentionArgs a, int splits,
                                                             const float* part_o,
                                                             const float* part_lse) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.q_heads * a.q_len;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (at >= rows) return;
  const int i = static_cast<int>(at % a.q_len);
  const int h = static_cast<int>(at / a.q_len % a.q_heads);
  const int b = static_cast<int>(at / a.q_len / a.q_heads);
  if (a.documents > 0) {  // rows of no document stay as they are
    int lo = 0, hi = a.documents;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.q_offsets[mid + 1] > i) hi = mid;
      else lo = mid + 1;
    }
    if (lo >= a.documents || a.q_offsets[lo] > i) return;
  }
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, part_lse[s * rows + at]);
  const float base = top == -INFINITY ? 0.0f : top;
  float y[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const float w = expf(part_lse[s * rows + at] - base);
    if (w == 0.0f) continue;  // an empty share wrote no o
    sum += w;
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      if (d < a.head_dim) y[e] += w * part_o[(s * rows + at) * a.head_dim + d];
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t oo = b * a.o_stride[0] + i * a.o_stride[1] + h * a.o_stride[2];
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 32 * e;
    if (d >= a.head_dim) continue;
    const float v = y[e] * inv;
    if constexpr (OT == IE_DT_BF16X2) {
      const float hi = __bfloat162float(__float2bfloat16_rn(v));
      store_element<IE_DT_BF16>(a.o, oo + d, hi);
      store_element<IE_DT_BF16>(a.o, oo + a.o_lo + d, v - hi);
    } else {
      store_element<OT>(a.o, oo + d, v);
    }
  }
  if (a.lse != nullptr && lane == 0) a.lse[at] = sum == 0.0f ? -INFINITY : base + logf(sum);
}

}  // namespace ie_cuda
