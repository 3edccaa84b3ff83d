// C ABI of the rotary positions (declared in include/ie_cuda_conv.h).
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "host_util.h"
#include "rotary_kernels.cuh"

using namespace ie_cuda;

namespace {

int check_head_layout(const ie_rotary_desc* d, int* pairs) {
  if (d == nullptr) return fail(IE_INVALID_ARGUMENT, "null descriptor");
  if (d->head_dim <= 0) return fail(IE_INVALID_ARGUMENT, "Rotary expects positive dimensions");
  if (d->head_dim > 256) return fail(IE_UNSUPPORTED, "Rotary head_dim is at most 256");
  if (d->axes < 1 || d->axes > 4) return fail(IE_INVALID_ARGUMENT, "Rotary has 1 to 4 axes");
  int64_t sum = 0;
  for (int a = 0; a < d->axes; ++a) {
    if (d->section[a] < 0) return fail(IE_INVALID_ARGUMENT, "Rotary sections are not negative");
    sum += d->section[a];
  }
  if (sum < 1 || 2 * sum > d->head_dim) {
    return fail(IE_INVALID_ARGUMENT, "Rotary sections must fill 1 to head_dim / 2 pairs");
  }
  if (d->layout < IE_ROTARY_PAIRS || d->layout > IE_ROTARY_AXIS_HALVES) {
    return fail(IE_INVALID_ARGUMENT, "bad rotary layout");
  }
  if (d->freq != IE_ROTARY_FREQ_SHARED && d->freq != IE_ROTARY_FREQ_PER_AXIS) {
    return fail(IE_INVALID_ARGUMENT, "bad rotary frequencies");
  }

  if (!(d->theta > 0.0) || std::isinf(d->theta)) {
    return fail(IE_INVALID_ARGUMENT, "Rotary theta must be positive and finite");
  }
  *pairs = static_cast<int>(sum);
  return IE_OK;
}

using Launch = void (*)(const RotaryArgs&, cudaStream_t);

template <int XT, int YT>
void launch_simple(const RotaryArgs& a, cudaStream_t s) {
  rotary_simple_kernel<XT, YT><<<static_cast<unsigned>(a.tokens), 128, 0, s>>>(a);
}

template <int XT>
Launch simple_for(int y_type) {
  switch (y_type) {
    case IE_DT_F32: return launch_simple<XT, IE_DT_F32>;
    case IE_DT_BF16: return launch_simple<XT, IE_DT_BF16>;
    default: return launch_simple<XT, IE_DT_F16>;
  }
}

Launch simple_for(int x_type, int y_type) {
  switch (x_type) {
    case IE_DT_F32: return simple_for<IE_DT_F32>(y_type);
    case IE_DT_BF16: return simple_for<IE_DT_BF16>(y_type);
    default: return simple_for<IE_DT_F16>(y_type);
  }
}

}  // namespace

extern "C" {

int ie_rotary_plan_init(const ie_rotary_desc* desc, ie_rotary_plan* plan) {
  int pairs = 0;
  const int rc = check_head_layout(desc, &pairs);
  if (rc != IE_OK) return rc;
  if (plan == nullptr) return fail(IE_INVALID_ARGUMENT, "null plan");
  std::memset(plan, 0, sizeof(*plan));
  constexpr long double kTwoPi = 6.283185307179586476925286766559L;
  int i = 0;
  for (int a = 0; a < desc->axes; ++a) {
    for (int j = 0; j < desc->section[a]; ++j, ++i) {
      const long double e = desc->freq == IE_ROTARY_FREQ_SHARED
                                ? static_cast<long double>(i) / pairs
                                : static_cast<long double>(j) / desc->section[a];
      long double t = std::pow(static_cast<long double>(desc->theta), -e) / kTwoPi;
      t -= std::floor(t);  // whole turns per position change nothing
      long double fixed = std::round(t * 0x1p64L);
      if (fixed >= 0x1p64L) fixed = 0.0L;
      plan->turns[i] = static_cast<uint64_t>(fixed);
      plan->axis[i] = static_cast<uint8_t>(a);
    }
    plan->section[a] = desc->section[a];
  }
  plan->head_dim = desc->head_dim;
  plan->axes = desc->axes;
  plan->layout = desc->layout;
  plan->freq = desc->freq;
  plan->pairs = pairs;
  plan->theta = desc->theta;
  return IE_OK;
}

int ie_cuda_rotary(const ie_rotary_desc* desc, const ie_rotary_plan* plan, const void* x,
                   const void* positions, void* y, void* stream) {
  int pairs = 0;
  const int rc = check_head_layout(desc, &pairs);
  if (rc != IE_OK) return rc;
  if (plan == nullptr || x == nullptr || y == nullptr || positions == nullptr) {
    return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  }
  bool same = plan->head_dim == desc->head_dim && plan->axes == desc->axes &&
              plan->layout == desc->layout && plan->freq == desc->freq && plan->pairs == pairs &&
              plan->theta == desc->theta;
  for (int a = 0; a < desc->axes; ++a) same = same && plan->section[a] == desc->section[a];
  if (!same) return fail(IE_INVALID_ARGUMENT, "the rotary plan is of another head layout");
  if (desc->tokens <= 0 || desc->heads <= 0) {
    return fail(IE_INVALID_ARGUMENT, "Rotary expects positive dimensions");
  }
  if (desc->tokens > INT_MAX) return fail(IE_UNSUPPORTED, "Rotary takes at most 2^31 - 1 tokens");
  if (desc->rot_heads < 0 || desc->rot_heads > desc->heads) {
    return fail(IE_INVALID_ARGUMENT, "rot_heads must be between 0 and heads");
  }
  for (int t : {desc->x_type, desc->y_type}) {
    if (t < IE_DT_F32 || t > IE_DT_F16) return fail(IE_INVALID_ARGUMENT, "bad element type");
  }
  if (desc->pos_bits != 32 && desc->pos_bits != 64) {
    return fail(IE_INVALID_ARGUMENT, "positions have 32 or 64 bits");
  }
  if (desc->x_token_stride < 0 || desc->x_head_stride < 0 || desc->y_token_stride < 0 ||
      desc->y_head_stride < 0 || desc->pos_axis_stride < 0) {
    return fail(IE_INVALID_ARGUMENT, "strides must not be negative");
  }
  if ((desc->tokens > 1 && desc->y_token_stride < desc->head_dim) ||
      (desc->heads > 1 && desc->y_head_stride < desc->head_dim)) {
    return fail(IE_INVALID_ARGUMENT, "the tokens or heads of y overlap");
  }
  const bool in_place = x == y;
  if (in_place &&
      (desc->x_type != desc->y_type || desc->x_token_stride != desc->y_token_stride ||
       desc->x_head_stride != desc->y_head_stride)) {
    return fail(IE_INVALID_ARGUMENT, "Rotary in place needs equal types and strides");
  }
  RotaryArgs a{};
  a.x = x;
  a.positions = positions;
  a.y = y;
  a.tokens = desc->tokens;
  a.x_token_stride = desc->x_token_stride;
  a.x_head_stride = desc->x_head_stride;
  a.y_token_stride = desc->y_token_stride;
  a.y_head_stride = desc->y_head_stride;
  a.pos_axis_stride = desc->pos_axis_stride;
  a.heads = desc->heads;
  a.rot_heads = desc->rot_heads;
  a.head_dim = desc->head_dim;
  a.pairs = pairs;
  a.layout = desc->layout;
  a.inverse = desc->inverse != 0;
  a.pos64 = desc->pos_bits == 64;
  a.in_place = in_place;
  for (int s = 0, first = 0; s < desc->axes; ++s) {
    a.first[s] = first;
    a.section[s] = desc->section[s];
    first += desc->section[s];
  }
  std::memcpy(a.turns, plan->turns, sizeof(a.turns));
  std::memcpy(a.axis, plan->axis, sizeof(a.axis));
  simple_for(desc->x_type, desc->y_type)(a, as_stream(stream));
  return check_launch("rotary");
}

}  // extern "C"
