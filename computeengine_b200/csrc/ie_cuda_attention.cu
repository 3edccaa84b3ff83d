// C ABI of the masked attention (declared in include/ie_cuda_conv.h): argument
// checks, choice of the kernel, launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "attention_kernels.cuh"
#include "attention_prompt.cuh"
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

constexpr int64_t ceil_div(int64_t v, int64_t m) { return (v + m - 1) / m; }
constexpr int64_t round_up(int64_t v, int64_t m) { return ceil_div(v, m) * m; }

// [batch, len, heads, head_dim] of 16-bit elements, loaded in boxes of 128 rows
// x 64 elements; rows and elements outside read as zeros.
int encode_rows(CUtensorMap* map, const void* p, bool bf16, int64_t head_dim, int64_t len,
                int64_t heads, int64_t batch, const int64_t* stride) {
  const DriverFns& f = driver_fns();
  if (!f.ok) return fail(IE_RUNTIME, "cuTensorMapEncodeTiled entry point unavailable");
  const int64_t extent[4] = {head_dim, len, heads, batch};
  cuuint64_t dims[4], strides[3];
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(extent[i]);
  const int64_t elements[3] = {stride[1], stride[2], stride[0]};
  for (int i = 0; i < 3; ++i) {
    // the stride of an extent of 1 is never used, but has to be a legal one
    strides[i] = static_cast<cuuint64_t>(extent[i + 1] > 1 ? 2 * elements[i]
                                                           : round_up(2 * head_dim, 16));
  }
  const cuuint32_t box[4] = {64, 128, 1, 1}, estrides[4] = {1, 1, 1, 1};
  const CUresult r = f.tiled(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
      const_cast<void*>(p), dims, strides, box, estrides, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    return fail(IE_RUNTIME, "cuTensorMapEncodeTiled failed (%d): attention rows",
                static_cast<int>(r));
  }
  return IE_OK;
}

// Whether TMA can read the tensor: 16-byte aligned rows at positive strides.
bool tma_readable(const void* p, int64_t head_dim, int64_t len, int64_t heads, int64_t batch,
                  const int64_t* stride) {
  const int64_t extent[3] = {batch, len, heads};
  if (head_dim % 8 != 0 || reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i) {
    if (extent[i] > 1 &&
        (stride[i] <= 0 || stride[i] % 8 != 0 || stride[i] >= (int64_t{1} << 38))) {
      return false;
    }
  }
  return true;
}

struct Plan {
  int64_t tiles = 0;  // blocks of 256 query rows per head and batch row
  int splits = 1;
  size_t workspace = 0;
};

// Blocks of the prompt kernel, and into how many shares each block's keys are
// cut when the blocks alone leave more than half of the GPU idle.
Plan plan_for(const ie_attention_desc* d, const ie_attention_mask* m) {
  Plan p;
  const int64_t documents = m == nullptr ? 0 : m->documents;
  p.tiles = documents > 0 ? d->q_len / 256 + documents : ceil_div(d->q_len, 256);
  const int64_t blocks = p.tiles * d->q_heads * d->batch;
  const int64_t key_tiles = ceil_div(d->kv_len, 128);
  constexpr int64_t kSms = 148;
  if (documents == 0 && blocks * 2 <= kSms && key_tiles >= 8) {
    p.splits = static_cast<int>(std::min(kSms / blocks, key_tiles / 4));
  }
  if (p.splits > 1) {
    const int64_t rows = d->batch * d->q_heads * d->q_len;
    p.workspace = static_cast<size_t>(round_up(rows * p.splits * d->head_dim * 4, 256) +
                                      rows * p.splits * 4);
  }
  return p;
}

template <int DP, int T, bool CAP, bool BIAS>
int launch_prompt(const PromptArgs& a, const CUtensorMap* maps, dim3 grid, cudaStream_t s) {
  auto kernel = attention_prompt_kernel<DP, T, CAP, BIAS>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             PromptPlan<DP>::kSmem);
  if (e != cudaSuccess) return fail(IE_RUNTIME, "attention: %s", cudaGetErrorString(e));
  kernel<<<grid, kPromptThreads, PromptPlan<DP>::kSmem, s>>>(a, maps[0], maps[1], maps[2]);
  return check_launch("attention");
}

template <int DP, int T>
int launch_prompt(const PromptArgs& a, const CUtensorMap* maps, dim3 grid, cudaStream_t s) {
  // the variant without cap and bias takes the maximum before the scale
  const bool bias = a.slopes != nullptr || (!(a.scale > 0.0f) && a.softcap == 0.0f);
  if (a.softcap > 0.0f) {
    return bias ? launch_prompt<DP, T, true, true>(a, maps, grid, s)
                : launch_prompt<DP, T, true, false>(a, maps, grid, s);
  }
  return bias ? launch_prompt<DP, T, false, true>(a, maps, grid, s)
              : launch_prompt<DP, T, false, false>(a, maps, grid, s);
}

template <int OT>
int launch_join(const PromptArgs& a, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.q_heads * a.q_len;
  attention_join_kernel<OT><<<static_cast<unsigned>(ceil_div(rows, 4)), 128, 0, s>>>(
      a, a.splits, a.part_o, a.part_lse);
  return check_launch("attention join");
}

template <int T, int OT>
void launch_simple(const AttentionArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.q_len + 3) / 4), static_cast<unsigned>(a.q_heads),
                  static_cast<unsigned>(a.batch));
  attention_simple_kernel<T, OT><<<grid, 128, 0, s>>>(a);
}

}  // namespace

namespace ie_cuda {

// This unit's device error word (each unit's kernels have their own).
int take_attention_error(unsigned int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code));
  const unsigned int zero = 0;
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
  if (e != cudaSuccess) return fail(IE_RUNTIME, "attention error word: %s", cudaGetErrorString(e));
  return IE_OK;
}

}  // namespace ie_cuda

extern "C" {

size_t ie_cuda_attention_workspace_bytes(const ie_attention_desc* desc,
                                         const ie_attention_mask* mask) {
  if (check_attention(desc, mask) != IE_OK) return 0;
  return plan_for(desc, mask).workspace;
}

int ie_cuda_attention(const ie_attention_desc* desc, const ie_attention_mask* mask, const void* q,
                      const void* k, const void* v, void* o, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const int rc = check_attention(desc, mask);
  if (rc != IE_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || o == nullptr) {
    return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  }
  const Plan plan = plan_for(desc, mask);
  if (plan.workspace > 0 &&
      (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 ||
       workspace_bytes < plan.workspace)) {
    return fail(IE_INVALID_ARGUMENT, "Attention needs %zu bytes of 256-byte aligned workspace",
                plan.workspace);
  }
  PromptArgs a{};
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
  const int64_t blocks = plan.tiles * a.q_heads * a.batch;
  if (blocks <= INT_MAX &&
      tma_readable(q, a.head_dim, a.q_len, a.q_heads, a.batch, a.q_stride) &&
      tma_readable(k, a.head_dim, a.kv_len, a.kv_heads, a.batch, a.k_stride) &&
      tma_readable(v, a.head_dim, a.kv_len, a.kv_heads, a.batch, a.v_stride)) {
    const bool bf16 = desc->type == IE_DT_BF16;
    CUtensorMap maps[3];
    int rc2 = encode_rows(&maps[0], q, bf16, a.head_dim, a.q_len, a.q_heads, a.batch, a.q_stride);
    if (rc2 == IE_OK) {
      rc2 = encode_rows(&maps[1], k, bf16, a.head_dim, a.kv_len, a.kv_heads, a.batch, a.k_stride);
    }
    if (rc2 == IE_OK) {
      rc2 = encode_rows(&maps[2], v, bf16, a.head_dim, a.kv_len, a.kv_heads, a.batch, a.v_stride);
    }
    if (rc2 != IE_OK) return rc2;
    a.tiles = static_cast<int>(plan.tiles);
    a.splits = plan.splits;
    a.part_o = static_cast<float*>(workspace);
    a.part_lse = a.splits > 1 ? a.part_o + round_up(int64_t{1} * a.batch * a.q_heads * a.q_len *
                                                        a.splits * a.head_dim, 64)
                              : nullptr;
    a.o_vec = reinterpret_cast<uintptr_t>(o) % 16 == 0 && a.o_lo % 8 == 0;
    for (int i = 0; i < 3; ++i) a.o_vec = a.o_vec && a.o_stride[i] % 8 == 0;
    a.wait_limit_ns = kWaitLimitNs;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.splits));
    if (a.head_dim <= 64) {
      rc2 = bf16 ? launch_prompt<64, IE_DT_BF16>(a, maps, grid, s)
                 : launch_prompt<64, IE_DT_F16>(a, maps, grid, s);
    } else {
      rc2 = bf16 ? launch_prompt<128, IE_DT_BF16>(a, maps, grid, s)
                 : launch_prompt<128, IE_DT_F16>(a, maps, grid, s);
    }
    if (rc2 != IE_OK || a.splits == 1) return rc2;
    return desc->o_type == IE_DT_BF16X2 ? launch_join<IE_DT_BF16X2>(a, s)
           : bf16                       ? launch_join<IE_DT_BF16>(a, s)
                                        : launch_join<IE_DT_F16>(a, s);
  }
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
