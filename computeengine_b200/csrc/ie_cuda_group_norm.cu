// C ABI of the channels-last group normalization (declared in
// include/ie_cuda_conv.h): argument checks, choice of the kernel, launch.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>

#include "group_norm_kernels.cuh"
#include "host_util.h"

using namespace ie_cuda;

namespace {

int check_group_norm(const ie_group_norm_desc* d) {
  if (d == nullptr) return fail(IE_INVALID_ARGUMENT, "null descriptor");
  if (d->n <= 0 || d->c <= 0 || d->h <= 0 || d->w <= 0) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm expects positive dimensions");
  }
  if (d->groups <= 0 || d->c % d->groups != 0) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm groups must divide the channels");
  }
  if (d->c_store < d->c) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm c_store must be at least c");
  }
  if (!(d->eps >= 0.0f) || std::isinf(d->eps)) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm eps must be finite and not negative");
  }
  if (d->act < IE_ACT_NONE || d->act > IE_ACT_GELU) {
    return fail(IE_INVALID_ARGUMENT, "bad activation");
  }
  for (int t : {d->x_type, d->y_type}) {
    if (t < IE_DT_F32 || t > IE_DT_BF16X2) return fail(IE_INVALID_ARGUMENT, "bad element type");
    if (t == IE_DT_BF16X2 && d->c_store % 16 != 0) {
      return fail(IE_INVALID_ARGUMENT, "split tensors hold a multiple of 16 channels per plane");
    }
  }
  if (d->c_store > (1 << 20) || d->h > INT_MAX || d->w > INT_MAX || d->h * d->w > INT_MAX ||
      d->n > 65535) {
    return fail(IE_UNSUPPORTED, "GroupNorm size out of range (c_store <= 2^20, h * w < 2^31, "
                                "n < 2^16)");
  }
  return IE_OK;
}

using Launch = void (*)(const GroupNormArgs&, dim3, cudaStream_t);

template <int XT, int YT>
void launch_simple(const GroupNormArgs& a, dim3 grid, cudaStream_t s) {
  group_norm_simple_kernel<XT, YT><<<grid, 256, 0, s>>>(a);
}

template <int XT>
Launch simple_for(int y_type) {
  switch (y_type) {
    case IE_DT_F32: return launch_simple<XT, IE_DT_F32>;
    case IE_DT_BF16: return launch_simple<XT, IE_DT_BF16>;
    case IE_DT_F16: return launch_simple<XT, IE_DT_F16>;
    default: return launch_simple<XT, IE_DT_BF16X2>;
  }
}

Launch simple_for(int x_type, int y_type) {
  switch (x_type) {
    case IE_DT_F32: return simple_for<IE_DT_F32>(y_type);
    case IE_DT_BF16: return simple_for<IE_DT_BF16>(y_type);
    case IE_DT_F16: return simple_for<IE_DT_F16>(y_type);
    default: return simple_for<IE_DT_BF16X2>(y_type);
  }
}

}  // namespace

extern "C" {

size_t ie_cuda_group_norm_workspace_bytes(const ie_group_norm_desc*) { return 0; }

int ie_cuda_group_norm_nhwc(const ie_group_norm_desc* desc, const void* x, const float* gamma,
                            const float* beta, void* y, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const int rc = check_group_norm(desc);
  if (rc != IE_OK) return rc;
  if (x == nullptr || y == nullptr) return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  if (x == y && desc->x_type != desc->y_type) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm in place needs equal element types");
  }
  (void)workspace;
  (void)workspace_bytes;
  GroupNormArgs a{x, gamma, beta, y, desc->h * desc->w, static_cast<int>(desc->c),
                  static_cast<int>(desc->c_store), static_cast<int>(desc->groups), desc->act,
                  desc->eps};
  simple_for(desc->x_type, desc->y_type)(
      a, dim3(static_cast<unsigned>(desc->groups), static_cast<unsigned>(desc->n)),
      as_stream(stream));
  return check_launch("group_norm");
}

}  // extern "C"
