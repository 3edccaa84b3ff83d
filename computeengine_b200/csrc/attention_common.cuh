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

}  // namespace ie_cuda
