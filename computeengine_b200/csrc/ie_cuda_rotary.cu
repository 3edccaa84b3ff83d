// C ABI of the rotary positions (declared in include/ie_cuda_conv.h).
#include <cuda_runtime.h>

#include <algorithm>
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

using Launch = void (*)(const RotaryArgs&, dim3, cudaStream_t);

template <int XT, int YT, int W, int CW>
void launch(const RotaryArgs& a, dim3 grid, cudaStream_t s) {
  const size_t smem = sizeof(float2) * a.block_tokens * a.pairs + sizeof(uint32_t) * a.units.d;
  rotary_kernel<XT, YT, W, CW><<<grid, 256, smem, s>>>(a);
}

template <int XT, int YT>
Launch launch_for(int w, bool copy8) {
  switch (w) {
    case 8: return copy8 ? launch<XT, YT, 8, 8> : launch<XT, YT, 8, 1>;
    case 4: return copy8 ? launch<XT, YT, 4, 8> : launch<XT, YT, 4, 1>;
    case 2: return copy8 ? launch<XT, YT, 2, 8> : launch<XT, YT, 2, 1>;
    default: return copy8 ? launch<XT, YT, 1, 8> : launch<XT, YT, 1, 1>;
  }
}

template <int XT>
Launch launch_for(int y_type, int w, bool copy8) {
  switch (y_type) {
    case IE_DT_F32: return launch_for<XT, IE_DT_F32>(w, copy8);
    case IE_DT_BF16: return launch_for<XT, IE_DT_BF16>(w, copy8);
    default: return launch_for<XT, IE_DT_F16>(w, copy8);
  }
}

Launch launch_for(int x_type, int y_type, int w, bool copy8) {
  switch (x_type) {
    case IE_DT_F32: return launch_for<IE_DT_F32>(y_type, w, copy8);
    case IE_DT_BF16: return launch_for<IE_DT_BF16>(y_type, w, copy8);
    default: return launch_for<IE_DT_F16>(y_type, w, copy8);
  }
}

// Whether both tensors can be read and written in vectors of w elements.
bool vectors_of(const ie_rotary_desc* d, const void* x, const void* y, int w) {
  const uintptr_t bytes_x = std::min(16, w * element_bytes(d->x_type));
  const uintptr_t bytes_y = std::min(16, w * element_bytes(d->y_type));
  return reinterpret_cast<uintptr_t>(x) % bytes_x == 0 &&
         reinterpret_cast<uintptr_t>(y) % bytes_y == 0 && d->x_token_stride % w == 0 &&
         d->x_head_stride % w == 0 && d->y_token_stride % w == 0 && d->y_head_stride % w == 0;
}

// The widest unit that every run of pairs, the elements behind them and the
// strides are a multiple of.
int unit_width(const ie_rotary_desc* d, const void* x, const void* y, int pairs) {
  for (int w : {8, 4, 2}) {
    bool fits = vectors_of(d, x, y, w) && pairs % w == 0 && (d->head_dim - 2 * pairs) % w == 0;
    if (d->layout == IE_ROTARY_AXIS_HALVES) {
      for (int s = 0; s < d->axes; ++s) fits = fits && d->section[s] % w == 0;
    }
    if (fits) return w;
  }
  return 1;
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
      const long double t = std::pow(static_cast<long double>(desc->theta), -e) / kTwoPi;
      if (!(t < 1.0L)) {  // above, long double has no 2^-64 turns left
        return fail(IE_UNSUPPORTED, "Rotary frequencies are below one turn per position");
      }
      const long double fixed = std::round(t * 0x1p64L);
      plan->turns[i] = fixed < 0x1p64L ? static_cast<uint64_t>(fixed) : 0;  // a whole turn
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
  int rc = check_head_layout(desc, &pairs);
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
  if (desc->tokens > INT_MAX || desc->heads > 65535) {
    return fail(IE_UNSUPPORTED, "Rotary takes at most 2^31 - 1 tokens of 2^16 - 1 heads");
  }
  if (desc->rot_heads < 0 || desc->rot_heads > desc->heads) {
    return fail(IE_INVALID_ARGUMENT, "rot_heads must be between 0 and heads");
  }
  for (int t : {desc->x_type, desc->y_type}) {
    if (t < IE_DT_F32 || t > IE_DT_F16) return fail(IE_INVALID_ARGUMENT, "bad element type");
  }
  if (desc->pos_bits != 32 && desc->pos_bits != 64) {
    return fail(IE_INVALID_ARGUMENT, "positions have 32 or 64 bits");
  }
  rc = check_aligned(x, element_bytes(desc->x_type), "Rotary x");
  if (rc == IE_OK) rc = check_aligned(y, element_bytes(desc->y_type), "Rotary y");
  if (rc == IE_OK) rc = check_aligned(positions, desc->pos_bits / 8, "Rotary positions");
  if (rc != IE_OK) return rc;
  if (desc->x_token_stride < 0 || desc->x_head_stride < 0 || desc->y_token_stride < 0 ||
      desc->y_head_stride < 0 || desc->pos_axis_stride < 0) {
    return fail(IE_INVALID_ARGUMENT, "strides must not be negative");
  }
  if (rows_overlap({desc->tokens, int64_t{desc->heads}},
                   {desc->y_token_stride, desc->y_head_stride}, desc->head_dim)) {
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
  const int w = unit_width(desc, x, y, pairs);
  const bool copy8 = desc->head_dim % 8 == 0 && vectors_of(desc, x, y, 8);
  a.units = SmallDivisor::of(static_cast<uint32_t>(pairs / w));
  a.copies = SmallDivisor::of(static_cast<uint32_t>(copy8 ? desc->head_dim / 8 : desc->head_dim));
  // Tokens per block: about eight units a thread, as long as that leaves four
  // blocks per SM; heads are shared out among blocks when there are fewer
  // tokens than SMs (one token per block then).
  constexpr int64_t kMaxItems = 1 << 15;
  const int64_t units = std::max<int64_t>(1, int64_t{desc->rot_heads} * (pairs / w));
  int64_t block_tokens = std::min<int64_t>(8, std::max<int64_t>(1, 2048 / units));
  block_tokens = std::max<int64_t>(1, std::min(block_tokens, desc->tokens / (4 * kSms)));
  // a block's units stay below 2^16 (SmallDivisor)
  int64_t shares = 1;
  if (block_tokens == 1) {
    shares = std::max((units + kMaxItems - 1) / kMaxItems,
                      std::min((units + 255) / 256, (kSms + desc->tokens - 1) / desc->tokens));
  }
  a.block_tokens = static_cast<int>(block_tokens);
  a.block_heads = static_cast<int>((desc->rot_heads + shares - 1) / shares);
  if (a.block_heads == 0) a.block_heads = 1;
  a.head_count = SmallDivisor::of(static_cast<uint32_t>(a.block_heads));
  const dim3 grid(static_cast<unsigned>((desc->tokens + block_tokens - 1) / block_tokens),
                  static_cast<unsigned>(shares));
  launch_for(desc->x_type, desc->y_type, w, copy8)(a, grid, as_stream(stream));
  return check_launch("rotary");
}

}  // extern "C"
