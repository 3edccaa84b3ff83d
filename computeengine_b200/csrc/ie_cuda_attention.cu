// C ABI of the masked attention (declared in include/ie_cuda_conv.h): argument
// checks, choice of the kernel, launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "attention_prompt.cuh"
#include "attention_step.cuh"
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
  for (int i = 0; i < 3; ++i) {
    if (d->q_stride[i] < 0 || d->k_stride[i] < 0 || d->v_stride[i] < 0 || d->o_stride[i] < 0) {
      return fail(IE_INVALID_ARGUMENT, "strides must not be negative");
    }
  }
  const bool split = d->o_type == IE_DT_BF16X2;
  if (rows_overlap({d->batch, d->q_len, d->q_heads, split ? 2 : 1},
                   {d->o_stride[0], d->o_stride[1], d->o_stride[2], d->o_stride[1] / 2},
                   d->head_dim)) {
    return fail(IE_INVALID_ARGUMENT, "the rows of o overlap");
  }
  if (split && d->o_stride[1] % 2 != 0) {
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

// [batch, len, heads, head_dim] of 16-bit elements, loaded in boxes of 64
// elements, box_len rows and box_heads heads; what lies outside reads as zeros.
int encode_rows(CUtensorMap* map, const void* p, bool bf16, int64_t head_dim, int64_t len,
                int64_t heads, int64_t batch, const int64_t* stride, int box_len, int box_heads) {
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
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_len),
                             static_cast<cuuint32_t>(box_heads), 1};
  const cuuint32_t estrides[4] = {1, 1, 1, 1};
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

// Shares of each sequence's keys, their partial results in the workspace.
size_t share_bytes(const ie_attention_desc* d, int splits) {
  if (splits <= 1) return 0;
  const int64_t rows = d->batch * d->q_heads * d->q_len * splits;
  return static_cast<size_t>(round_up(rows * d->head_dim * 4, 256) + rows * 4);
}

// The step kernel's tiles: all heads of a kv head and all positions when that
// is at most 16 rows, else 32 positions of one head (documents; unaligned
// tensors of many rows).  Above 16 rows the prompt kernel is faster: 4 x 8
// positions x 4 heads per kv head over 8192 keys took 49 us here and 29 us there (26 us there now).
struct StepTiles {
  int rows, heads;
  int64_t tiles;
  int splits;
};

bool few_rows(const ie_attention_desc* d, const ie_attention_mask* m) {
  return (m == nullptr || m->documents == 0) && d->q_len * (d->q_heads / d->kv_heads) <= 16;
}

StepTiles step_tiles(const ie_attention_desc* d, const ie_attention_mask* m) {
  StepTiles t{};
  if (few_rows(d, m)) {
    t.rows = static_cast<int>(d->q_len);
    t.heads = d->q_heads / d->kv_heads;
    t.tiles = 1;
    // Two blocks for each SM; with ragged lengths three times as many, which
    // evens them out (4 or 10 times the SMs: within 5%, 16 times: 25% slower).
    // Shares of at least 256 keys and, for the precision of their sums, 2^20 at most.
    const int64_t units = d->batch * d->kv_heads;
    const int64_t blocks = (m != nullptr && m->kv_lens != nullptr ? 6 : 2) * kSms;
    const int64_t share =
        std::min<int64_t>(std::max<int64_t>(256, ceil_div(units * d->kv_len, blocks)), 1 << 20);
    t.splits = static_cast<int>(std::min<int64_t>(ceil_div(d->kv_len, share), kMaxSplits));
  } else {
    const int64_t documents = m == nullptr ? 0 : m->documents;
    t.rows = 32;
    t.heads = 1;
    t.tiles = documents > 0 ? d->q_len / 32 + documents : ceil_div(d->q_len, 32);
    t.splits = 1;
  }
  return t;
}

// The prompt kernel's blocks of two row tiles, and into how many shares each
// block's keys are cut when the blocks alone leave half of the GPU idle.  Up to
// 64 positions and several heads per kv head: a tile holds all positions of as
// many of those heads as fit 128 rows, so that their K and V are loaded once.
struct PromptTiles {
  int64_t tiles;
  int64_t head_units;
  int rows, heads;
  bool packed;
  int splits;
};

PromptTiles prompt_tiles(const ie_attention_desc* d, const ie_attention_mask* m) {
  const int64_t documents = m == nullptr ? 0 : m->documents;
  PromptTiles p{documents > 0 ? d->q_len / 256 + documents : ceil_div(d->q_len, 256), d->q_heads,
                128, 1, false, 1};
  const int heads_per_kv = d->q_heads / d->kv_heads;
  if (documents == 0 && d->q_len <= 64 && heads_per_kv > 1) {
    p.packed = true;
    p.rows = static_cast<int>(d->q_len);
    for (int h = 1; h <= heads_per_kv && h * p.rows <= 128; ++h) {
      if (heads_per_kv % h == 0) p.heads = h;
    }
    p.head_units = d->kv_heads * ceil_div(heads_per_kv / p.heads, 2);
  }
  const int64_t blocks = p.tiles * p.head_units * d->batch;
  const int64_t key_tiles = ceil_div(d->kv_len, 128);
  if (documents == 0 && blocks * 2 <= kSms && key_tiles >= 8) {
    p.splits = static_cast<int>(std::min(kSms / blocks, key_tiles / 4));
  }
  return p;
}

// The prompt kernel's workspace: the shares' partial results, or, where a block may
// take more than kFold steps, room for each row's O.
size_t prompt_bytes(const ie_attention_desc* d, const PromptTiles& t) {
  if (t.splits > 1) return share_bytes(d, t.splits);
  if (d->kv_len <= kFold * kStep) return 0;
  return static_cast<size_t>(d->batch * d->q_heads * d->q_len * d->head_dim * 4);
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
int launch_join(const AttentionArgs& a, int splits, const float* part_o, const float* part_lse,
                cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.q_heads * a.q_len;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr{};  // its launch overlaps the end of the kernel before it
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, attention_join_kernel<OT>, a, splits, part_o, part_lse);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(IE_RUNTIME, "attention join: %s", cudaGetErrorString(e));
  }
  return check_launch("attention join");
}

int join(const ie_attention_desc* d, const AttentionArgs& a, int splits, const float* part_o,
         const float* part_lse, cudaStream_t s) {
  return d->o_type == IE_DT_BF16X2 ? launch_join<IE_DT_BF16X2>(a, splits, part_o, part_lse, s)
         : d->o_type == IE_DT_BF16 ? launch_join<IE_DT_BF16>(a, splits, part_o, part_lse, s)
                                   : launch_join<IE_DT_F16>(a, splits, part_o, part_lse, s);
}

template <int DP, int T, int NT, bool VEC>
int launch_step(const StepArgs& a, dim3 grid, cudaStream_t s) {
  auto kernel = attention_step_kernel<DP, T, NT, VEC>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             StepPlan<DP>::kSmem);
  if (e != cudaSuccess) return fail(IE_RUNTIME, "attention: %s", cudaGetErrorString(e));
  kernel<<<grid, kStepThreads, StepPlan<DP>::kSmem, s>>>(a);
  return check_launch("attention");
}

template <int DP, int T, int NT>
int launch_step(const StepArgs& a, dim3 grid, bool vec, cudaStream_t s) {
  return vec ? launch_step<DP, T, NT, true>(a, grid, s) : launch_step<DP, T, NT, false>(a, grid, s);
}

template <int DP, int T>
int launch_step(const StepArgs& a, dim3 grid, bool vec, cudaStream_t s) {
  const int rows = a.tile_rows * a.tile_heads;
  return rows <= 8    ? launch_step<DP, T, 1>(a, grid, vec, s)
         : rows <= 16 ? launch_step<DP, T, 2>(a, grid, vec, s)
                      : launch_step<DP, T, 4>(a, grid, vec, s);
}

int run_step(const ie_attention_desc* d, const ie_attention_mask* m, const AttentionArgs& base,
             bool vec, float* workspace, cudaStream_t s) {
  StepArgs a{};
  static_cast<AttentionArgs&>(a) = base;
  const StepTiles t = step_tiles(d, m);
  a.tile_rows = t.rows;
  a.tile_heads = t.heads;
  a.tiles = static_cast<int>(t.tiles);
  a.splits = t.splits;
  const int64_t rows = d->batch * d->q_heads * d->q_len * a.splits;
  a.part_o = a.splits > 1 ? workspace : nullptr;
  a.part_lse = a.splits > 1 ? workspace + round_up(rows * d->head_dim, 64) : nullptr;
  const int64_t blocks = t.tiles * (d->q_heads / t.heads) * d->batch;
  if (blocks > INT_MAX) return fail(IE_UNSUPPORTED, "Attention has too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.splits));
  const bool bf16 = d->type == IE_DT_BF16;
  int rc;
  if (d->head_dim <= 64) {
    rc = bf16 ? launch_step<64, IE_DT_BF16>(a, grid, vec, s)
              : launch_step<64, IE_DT_F16>(a, grid, vec, s);
  } else {
    rc = bf16 ? launch_step<128, IE_DT_BF16>(a, grid, vec, s)
              : launch_step<128, IE_DT_F16>(a, grid, vec, s);
  }
  if (rc != IE_OK || a.splits == 1) return rc;
  return join(d, a, a.splits, a.part_o, a.part_lse, s);
}

int run_prompt(const ie_attention_desc* d, const ie_attention_mask* m, const AttentionArgs& base,
               float* workspace, cudaStream_t s) {
  PromptArgs a{};
  static_cast<AttentionArgs&>(a) = base;
  const PromptTiles t = prompt_tiles(d, m);
  const int64_t blocks = t.tiles * t.head_units * d->batch;
  if (blocks > INT_MAX) return fail(IE_UNSUPPORTED, "Attention has too many rows");
  const bool bf16 = d->type == IE_DT_BF16;
  CUtensorMap maps[3];
  int rc = encode_rows(&maps[0], a.q, bf16, d->head_dim, d->q_len, d->q_heads, d->batch,
                       d->q_stride, t.rows, t.heads);
  if (rc == IE_OK) {
    rc = encode_rows(&maps[1], a.k, bf16, d->head_dim, d->kv_len, d->kv_heads, d->batch,
                     d->k_stride, kStep, 1);
  }
  if (rc == IE_OK) {
    rc = encode_rows(&maps[2], a.v, bf16, d->head_dim, d->kv_len, d->kv_heads, d->batch,
                     d->v_stride, kStep, 1);
  }
  if (rc != IE_OK) return rc;
  a.head_units = static_cast<int>(t.head_units);
  a.packed = t.packed;
  a.tile_rows = t.rows;
  a.tile_heads = t.heads;
  a.tiles = static_cast<int>(t.tiles);
  a.splits = t.splits;
  const int64_t rows = d->batch * d->q_heads * d->q_len * a.splits;
  a.part_o = workspace;
  a.part_lse = a.splits > 1 ? workspace + round_up(rows * d->head_dim, 64) : nullptr;
  a.o_vec = reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && a.o_lo % 8 == 0;
  for (int i = 0; i < 3; ++i) a.o_vec = a.o_vec && a.o_stride[i] % 8 == 0;
  a.wait_limit_ns = kWaitLimitNs;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.splits));
  if (d->head_dim <= 64) {
    rc = bf16 ? launch_prompt<64, IE_DT_BF16>(a, maps, grid, s)
              : launch_prompt<64, IE_DT_F16>(a, maps, grid, s);
  } else {
    rc = bf16 ? launch_prompt<128, IE_DT_BF16>(a, maps, grid, s)
              : launch_prompt<128, IE_DT_F16>(a, maps, grid, s);
  }
  if (rc != IE_OK || a.splits == 1) return rc;
  return join(d, a, a.splits, a.part_o, a.part_lse, s);
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
  // few rows always run on the step kernel; many rows that TMA cannot read are not split
  return few_rows(desc, mask) ? share_bytes(desc, step_tiles(desc, mask).splits)
                              : prompt_bytes(desc, prompt_tiles(desc, mask));
}

int ie_cuda_attention(const ie_attention_desc* desc, const ie_attention_mask* mask, const void* q,
                      const void* k, const void* v, void* o, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream) {
  int rc = check_attention(desc, mask);
  if (rc != IE_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || o == nullptr) {
    return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  }
  for (const void* p : {q, k, v, static_cast<const void*>(o)}) {
    if (rc == IE_OK) rc = check_aligned(p, 2, "Attention q, k, v and o");
  }
  if (rc == IE_OK) rc = check_aligned(lse, 4, "Attention lse");
  if (mask != nullptr) {
    const void* given[] = {mask->kv_lens, mask->prefix_lens, mask->q_offsets, mask->kv_offsets,
                           mask->slopes};
    for (const void* p : given) {
      if (rc == IE_OK) rc = check_aligned(p, 4, "Attention lengths, offsets and slopes");
    }
  }
  if (rc != IE_OK) return rc;
  const bool few = few_rows(desc, mask);
  const bool kv_tma =
      tma_readable(k, desc->head_dim, desc->kv_len, desc->kv_heads, desc->batch, desc->k_stride) &&
      tma_readable(v, desc->head_dim, desc->kv_len, desc->kv_heads, desc->batch, desc->v_stride);
  const bool tma = kv_tma && tma_readable(q, desc->head_dim, desc->q_len, desc->q_heads,
                                          desc->batch, desc->q_stride);
  const size_t need =
      few ? share_bytes(desc, step_tiles(desc, mask).splits)
          : tma ? prompt_bytes(desc, prompt_tiles(desc, mask)) : size_t{0};
  if (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 ||
                   workspace_bytes < need)) {
    return fail(IE_INVALID_ARGUMENT, "Attention needs %zu bytes of 256-byte aligned workspace",
                need);
  }
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
  if (few || !tma) return run_step(desc, mask, a, kv_tma, static_cast<float*>(workspace), s);
  return run_prompt(desc, mask, a, static_cast<float*>(workspace), s);
}

}  // extern "C"
