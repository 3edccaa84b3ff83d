// C ABI of the masked attention (declared in include/ie_cuda_conv.h): argument
// checks, choice of the kernel, launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "attention_kernels.cuh"
#include "host_util.h"

using namespace ie_cuda;

namespace {

int check_attention(const ie_attention_desc* d, const ie_attention_mask* m) {
  if (d == nullptr) return fail(IE_INVALID_ARGUMENT, "null descriptor");
  if (d->batch <= 0 || d->q_len <= 0 || d->kv_len <= 0 || d->q_heads <= 0 || d->kv_heads <= 0 ||
      d->head_dim <= 0) {
    return fail(IE_INVALID_ARGUMENT, "Attention expects positive dimensions");
  }
  if (d->q_heads % d->kv_heads != 0) {
    return fail(IE_INVALID_ARGUMENT, "Attention kv_heads must divide q_heads");
  }
  if (d->type != IE_DT_BF16 && d->type != IE_DT_F16) {
    return fail(d->type == IE_DT_F32 || d->type == IE_DT_BF16X2 ? IE_UNSUPPORTED
                                                                : IE_INVALID_ARGUMENT,
                "Attention reads bf16 or f16");
  }
  if (d->o_type != d->type && !(d->o_type == IE_DT_BF16X2 && d->type == IE_DT_BF16)) {
    return fail(IE_INVALID_ARGUMENT, "Attention writes its input type, or split bf16 for bf16");
  }
  if (d->head_dim > 128) return fail(IE_UNSUPPORTED, "Attention head_dim is at most 128");
  if (d->batch > 65535 || d->q_heads > 65535 || d->q_len > (1 << 30) || d->kv_len > (1 << 30)) {
    return fail(IE_UNSUPPORTED, "Attention size out of range (batch and heads < 2^16, lengths "
                                "<= 2^30)");
  }
  if (!std::isfinite(d->scale) || !(d->softcap >= 0.0f) || std::isinf(d->softcap)) {
    return fail(IE_INVALID_ARGUMENT, "Attention scale and softcap must be finite, softcap not "
                                     "negative");
  }
  const int64_t extent[3] = {d->batch, d->q_len, d->q_heads};
  for (int i = 0; i < 3; ++i) {
    if (d->q_stride[i] < 0 || d->k_stride[i] < 0 || d->v_stride[i] < 0 || d->o_stride[i] < 0) {
      return fail(IE_INVALID_ARGUMENT, "strides must not be negative");
    }
    if (extent[i] > 1 && d->o_stride[i] < d->head_dim) {
      return fail(IE_INVALID_ARGUMENT, "the rows of o overlap");
    }
  }
  if (d->o_type == IE_DT_BF16X2 && (d->o_stride[1] % 2 != 0 || d->o_stride[1] < 2 * d->head_dim)) {
    return fail(IE_INVALID_ARGUMENT, "split output: the token stride holds both planes");
  }
  if (m != nullptr) {
    if (m->documents < 0) return fail(IE_INVALID_ARGUMENT, "documents must not be negative");
    if (m->documents > 0) {
      if (d->batch != 1) {
        return fail(IE_INVALID_ARGUMENT, "documents are packed into one batch row");
      }
      if (m->q_offsets == nullptr || m->kv_offsets == nullptr) {
        return fail(IE_INVALID_ARGUMENT, "documents need q_offsets and kv_offsets");
      }
      if (m->kv_lens != nullptr) {
        return fail(IE_INVALID_ARGUMENT, "documents have their lengths in kv_offsets");
      }
    }
    if (m->prefix_lens != nullptr && !m->causal) {
      return fail(IE_INVALID_ARGUMENT, "prefix_lens needs causal");
    }
  }
  return IE_OK;
}

template <int T, int OT>
void launch_simple(const AttentionArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.q_len + 3) / 4), static_cast<unsigned>(a.q_heads),
                  static_cast<unsigned>(a.batch));
  attention_simple_kernel<T, OT><<<grid, 128, 0, s>>>(a);
}

}  // namespace

extern "C" {

size_t ie_cuda_attention_workspace_bytes(const ie_attention_desc*, const ie_attention_mask*) {
  return 0;
}

int ie_cuda_attention(const ie_attention_desc* desc, const ie_attention_mask* mask, const void* q,
                      const void* k, const void* v, void* o, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const int rc = check_attention(desc, mask);
  if (rc != IE_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || o == nullptr) {
    return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  }
  (void)workspace;
  (void)workspace_bytes;
  AttentionArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = o;
  a.lse = lse;
  std::copy_n(desc->q_stride, 3, a.q_stride);
  std::copy_n(desc->k_stride, 3, a.k_stride);
  std::copy_n(desc->v_stride, 3, a.v_stride);
  std::copy_n(desc->o_stride, 3, a.o_stride);
  a.o_lo = desc->o_type == IE_DT_BF16X2 ? desc->o_stride[1] / 2 : 0;
  a.batch = static_cast<int>(desc->batch);
  a.q_len = static_cast<int>(desc->q_len);
  a.kv_len = static_cast<int>(desc->kv_len);
  a.q_heads = desc->q_heads;
  a.kv_heads = desc->kv_heads;
  a.head_dim = desc->head_dim;
  a.scale = desc->scale;
  a.softcap = desc->softcap;
  if (mask != nullptr) {
    a.causal = mask->causal != 0;
    a.documents = mask->documents;
    a.kv_lens = mask->kv_lens;
    a.prefix_lens = mask->prefix_lens;
    a.q_offsets = mask->documents > 0 ? mask->q_offsets : nullptr;
    a.kv_offsets = mask->documents > 0 ? mask->kv_offsets : nullptr;
    a.slopes = mask->slopes;
  }
  const cudaStream_t s = as_stream(stream);
  if (desc->o_type == IE_DT_BF16X2) {
    launch_simple<IE_DT_BF16, IE_DT_BF16X2>(a, s);
  } else if (desc->type == IE_DT_BF16) {
    launch_simple<IE_DT_BF16, IE_DT_BF16>(a, s);
  } else {
    launch_simple<IE_DT_F16, IE_DT_F16>(a, s);
  }
  return check_launch("attention");
}

}  // extern "C"
