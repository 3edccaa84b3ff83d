// C ABI of the channels-last group normalization (declared in
// include/ie_cuda_conv.h): argument checks, choice of the kernel, launch.
#include <cuda_runtime.h>

#include <algorithm>
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
  constexpr int64_t kMaxPixels = 1 << 30;
  if (d->c_store > (1 << 20) || d->h > kMaxPixels || d->w > kMaxPixels ||
      d->h * d->w > kMaxPixels || d->n > 65535) {
    return fail(IE_UNSUPPORTED, "GroupNorm size out of range (c_store <= 2^20, h * w <= 2^30, "
                                "n < 2^16)");
  }
  return IE_OK;
}

constexpr int64_t ceil_div(int64_t v, int64_t m) { return (v + m - 1) / m; }

constexpr int64_t kSms = 148;
constexpr int64_t kSmemPerSm = 227 * 1024;
// Bytes of x that the two-kernel path normalizes per pair of launches: with
// the y they become they stay in the 126 MB L2 between the two reads.
constexpr int64_t kWaveBytes = 72 << 20;

int64_t item_bytes(int x_type, int v) {
  return int64_t{v} * element_bytes(x_type) * (x_type == IE_DT_BF16X2 ? 2 : 1);
}

struct Plan {
  int v = 1;
  bool cluster = false;
  int range_groups = 1, ranges = 1;  // channel ranges of whole groups
  int blocks = 1;                    // per image and range: cluster size, or statistics blocks
  int64_t smem = 0;
  // two-kernel path: (image, range) units of one pair of launches
  int64_t wave_images = 1;
  int wave_ranges = 1;
  int apply_blocks = 1;
  int64_t workspace = 0;
};

// Whether ranges of g groups begin and end on vectors of v channels.
bool range_fits(const ie_group_norm_desc* d, int64_t g, int v) {
  return d->groups % g == 0 && (g == d->groups || g * (d->c / d->groups) % v == 0);
}

// The choice between one kernel that holds x in shared memory and two that
// read it twice, and the split of the work, by an estimate of the time: blocks
// run in waves over the SMs; a wave costs about 4 us of latencies (load, join,
// store), more with the cluster's barriers, and all of them together no less
// than the bytes at the measured 6.5 TB/s.  Pieces of a pixel narrower than
// 128 bytes waste part of each DRAM access.
Plan plan_for(const ie_group_norm_desc* d, int v) {
  Plan best;
  const int64_t cg = d->c / d->groups, pixels = d->h * d->w;
  const int64_t xb = item_bytes(d->x_type, 1), yb = item_bytes(d->y_type, 1);
  best.v = v;
  double best_ns = 1e30;
  for (int64_t g = 1; v > 1 && g <= d->groups; ++g) {
    if (!range_fits(d, g, v)) continue;
    const int64_t ranges = d->groups / g;
    const int64_t stored = d->c_store - (ranges - 1) * g * cg;  // of the last range
    const int64_t cols = ceil_div(std::max(stored, g * cg), v);
    if (cols > kGnThreads) break;
    const int64_t rows = kGnThreads / cols;
    const double segment = static_cast<double>(g * cg * xb);
    const double waste = segment < 32 ? 2.0 : segment < 64 ? 1.5 : segment < 128 ? 1.15 : 1.0;
    for (int blocks = 1; blocks <= 16; blocks *= 2) {
      const int64_t share = ceil_div(pixels, blocks);
      const int64_t held = ceil_div(share, rows) * kGnThreads * item_bytes(d->x_type, v);
      const int64_t smem = held + (v + 1) * kGnThreads * 4 + (20 + 8 * blocks) * g + 32;
      if (smem > kSmemPerSm || (blocks > 1 && share * (blocks - 1) >= pixels)) continue;
      const int64_t per_sm = std::min<int64_t>(4, (kSmemPerSm + 1024) / (smem + 1024));
      const int64_t total = d->n * ranges * blocks;
      const int64_t waves = ceil_div(total, kSms * per_sm);
      const double latency = blocks > 8 ? 5500.0 : blocks > 1 ? 4500.0 : 4000.0;
      // one wave: no SM can do better than its own share of the bandwidth
      const double busy = static_cast<double>(std::min<int64_t>(total, kSms)) / kSms;
      const double bytes = static_cast<double>(d->n * pixels * d->c) * static_cast<double>(xb + yb);
      // with few blocks on an SM, one's loads, arithmetic and stores leave the
      // memory idle in turn (measured: one block per SM reaches half of it)
      const double overlap = per_sm == 1 ? 2.0 : per_sm == 2 ? 1.4 : per_sm == 3 ? 1.15 : 1.0;
      const double ns = latency + std::max(latency * static_cast<double>(waves - 1),
                                           waste * overlap * bytes / (6500.0 * busy));
      if (ns < best_ns) {
        best_ns = ns;
        best.cluster = true;
        best.range_groups = static_cast<int>(g);
        best.ranges = static_cast<int>(ranges);
        best.blocks = blocks;
        best.smem = smem;
      }
    }
  }
  // two kernels: a second launch, x read again from L2 (about twice as fast)
  const double two_ns = 9000.0 + static_cast<double>(d->n * pixels * d->c_store) *
                                     (1.5 * static_cast<double>(xb) + static_cast<double>(yb)) /
                                     6500.0;
  if (best.cluster && best_ns <= two_ns) return best;
  best.cluster = false;
  // ranges: whole pixels if the threads cover them and the image fits a wave,
  // else the narrowest range of at least 256 bytes
  const int64_t image = pixels * d->c_store * xb;
  best.range_groups = static_cast<int>(d->groups);
  const bool whole = ceil_div(d->c, v) <= kGnThreads && image <= kWaveBytes;
  if (!whole) {
    best.range_groups = 0;
    for (int64_t g = 1; g <= d->groups; ++g) {
      if (!range_fits(d, g, v)) continue;
      // several groups only within the threads' columns
      if (best.range_groups > 0 && ceil_div(g * cg, v) > kGnThreads) break;
      best.range_groups = static_cast<int>(g);
      if (g * cg * xb >= 256) break;
    }
  }
  const int64_t channels = best.range_groups * cg;
  best.ranges = static_cast<int>(d->groups / best.range_groups);
  const int64_t rows = std::max<int64_t>(1, kGnThreads / ceil_div(channels, v));
  if (image <= kWaveBytes) {
    best.wave_images = std::min(d->n, std::max<int64_t>(1, kWaveBytes / image));
    best.wave_ranges = best.ranges;
  } else {
    best.wave_images = 1;
    best.wave_ranges = static_cast<int>(
        std::min<int64_t>(best.ranges, std::max<int64_t>(1, kWaveBytes * best.ranges / image)));
  }
  const int64_t units = best.wave_images * best.wave_ranges;
  best.blocks = static_cast<int>(
      std::max<int64_t>(1, std::min(2 * kSms / units, ceil_div(pixels, kGnBatch * rows))));
  best.apply_blocks = static_cast<int>(
      std::max<int64_t>(1, std::min(2 * kSms / units, ceil_div(pixels, 4 * rows))));
  best.smem = (v + 1) * kGnThreads * 4 + 4 * best.range_groups;
  best.workspace = units * best.blocks * best.range_groups * static_cast<int64_t>(sizeof(float2));
  return best;
}

// Vectors of 16 bytes of x where pixels, pointers and ranges allow it.
int vector_width(const ie_group_norm_desc* d) {
  const int v = d->x_type == IE_DT_F32 ? 4 : 8;
  if (d->c_store % v != 0) return 1;
  // a group wider than the threads' columns must be a range of its own
  const int64_t cg = d->c / d->groups;
  for (int64_t g = 1; g <= d->groups; ++g) {
    if (!range_fits(d, g, v)) continue;
    if (ceil_div(g * cg, v) <= kGnThreads || (g == 1 && cg % v == 0)) return v;
    break;
  }
  return 1;
}

template <class Kernel>
int allow_smem(Kernel kernel, int64_t smem, bool wide_cluster) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e == cudaSuccess && wide_cluster) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }
  return e == cudaSuccess ? IE_OK : fail(IE_RUNTIME, "group_norm: %s", cudaGetErrorString(e));
}

template <int XT, int YT, int V, int ACT>
int launch_cluster(const GroupNormArgs& a, const Plan& p, int64_t images, cudaStream_t s) {
  auto kernel = group_norm_cluster_kernel<XT, YT, V, ACT>;
  const int rc = allow_smem(kernel, p.smem, p.blocks > 8);
  if (rc != IE_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(images * p.ranges * p.blocks));
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.smem);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(p.blocks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(IE_RUNTIME, "group_norm: %s", cudaGetErrorString(e));
  }
  return check_launch("group_norm");
}

template <int XT, int YT, int V, int ACT>
int launch_two(GroupNormArgs a, const Plan& p, int64_t images, cudaStream_t s) {
  auto stats = group_norm_stats_kernel<XT, V>;
  auto apply = group_norm_apply_kernel<XT, YT, V, ACT>;
  const int64_t apply_smem = 8 * p.range_groups;
  int rc = allow_smem(stats, p.smem, false);
  if (rc == IE_OK) rc = allow_smem(apply, apply_smem, false);
  for (int64_t i = 0; rc == IE_OK && i < images; i += p.wave_images) {
    a.first_image = i;
    const int64_t wave = std::min(p.wave_images, images - i);
    for (int r = 0; rc == IE_OK && r < p.ranges; r += p.wave_ranges) {
      a.first_range = r;
      a.launch_ranges = std::min(p.wave_ranges, p.ranges - r);
      const int64_t units = wave * a.launch_ranges;
      stats<<<static_cast<unsigned>(units * p.blocks), kGnThreads, p.smem, s>>>(a);
      rc = check_launch("group_norm statistics");
      if (rc != IE_OK) break;
      apply<<<static_cast<unsigned>(units * p.apply_blocks), kGnThreads, apply_smem, s>>>(
          a, p.apply_blocks);
      rc = check_launch("group_norm");
    }
  }
  return rc;
}

template <int XT, int YT, int ACT>
int launch(const GroupNormArgs& a, const Plan& p, int64_t images, cudaStream_t s) {
  constexpr int V = XT == IE_DT_F32 ? 4 : 8;
  if (p.v == 1) return launch_two<XT, YT, 1, ACT>(a, p, images, s);
  return p.cluster ? launch_cluster<XT, YT, V, ACT>(a, p, images, s)
                   : launch_two<XT, YT, V, ACT>(a, p, images, s);
}

template <int XT, int YT>
int launch(int act, GroupNormArgs a, const Plan& p, int64_t images, cudaStream_t s) {
  if (act == IE_ACT_SILU) return launch<XT, YT, kActSilu>(a, p, images, s);
  if (act == IE_ACT_GELU) return launch<XT, YT, kActGelu>(a, p, images, s);
  a.low = act == IE_ACT_NONE ? -INFINITY : 0.0f;
  a.high = act == IE_ACT_RELU6 ? 6.0f : INFINITY;
  return launch<XT, YT, kActClamp>(a, p, images, s);
}

template <int XT>
int launch(int y_type, int act, const GroupNormArgs& a, const Plan& p, int64_t images, cudaStream_t s) {
  switch (y_type) {
    case IE_DT_F32: return launch<XT, IE_DT_F32>(act, a, p, images, s);
    case IE_DT_BF16: return launch<XT, IE_DT_BF16>(act, a, p, images, s);
    case IE_DT_F16: return launch<XT, IE_DT_F16>(act, a, p, images, s);
    default: return launch<XT, IE_DT_BF16X2>(act, a, p, images, s);
  }
}

int launch(int x_type, int y_type, int act, const GroupNormArgs& a, const Plan& p,
           int64_t images, cudaStream_t s) {
  switch (x_type) {
    case IE_DT_F32: return launch<IE_DT_F32>(y_type, act, a, p, images, s);
    case IE_DT_BF16: return launch<IE_DT_BF16>(y_type, act, a, p, images, s);
    case IE_DT_F16: return launch<IE_DT_F16>(y_type, act, a, p, images, s);
    default: return launch<IE_DT_BF16X2>(y_type, act, a, p, images, s);
  }
}

}  // namespace

extern "C" {

size_t ie_cuda_group_norm_workspace_bytes(const ie_group_norm_desc* desc) {
  if (check_group_norm(desc) != IE_OK) return 0;
  // what unaligned tensors need, too
  return static_cast<size_t>(
      std::max(plan_for(desc, vector_width(desc)).workspace, plan_for(desc, 1).workspace));
}

int ie_cuda_group_norm_nhwc(const ie_group_norm_desc* desc, const void* x, const float* gamma,
                            const float* beta, void* y, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const int rc = check_group_norm(desc);
  if (rc != IE_OK) return rc;
  if (x == nullptr || y == nullptr) return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  if (x == y && desc->x_type != desc->y_type) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm in place needs equal element types");
  }
  int v = vector_width(desc);
  const uintptr_t y_bytes =
      std::min<uintptr_t>(16, static_cast<uintptr_t>(v) * element_bytes(desc->y_type));
  if (reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(y) % y_bytes != 0) {
    v = 1;
  }
  const Plan p = plan_for(desc, v);
  if (p.workspace > 0 &&
      (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
       workspace_bytes < static_cast<size_t>(p.workspace))) {
    return fail(IE_INVALID_ARGUMENT, "GroupNorm needs %lld bytes of 16-byte aligned workspace",
                static_cast<long long>(p.workspace));
  }
  GroupNormArgs a{};
  a.x = x;
  a.gamma = gamma;
  a.beta = beta;
  a.y = y;
  a.pixels = static_cast<int>(desc->h * desc->w);
  a.c = static_cast<int>(desc->c);
  a.c_store = static_cast<int>(desc->c_store);
  a.group_channels = static_cast<int>(desc->c / desc->groups);
  a.eps = desc->eps;
  a.range_groups = p.range_groups;
  a.ranges = p.ranges;
  a.blocks = p.blocks;
  a.share = static_cast<int>(ceil_div(a.pixels, p.blocks));
  for (int last = 0; last < 2; ++last) {
    const int64_t channels = int64_t{p.range_groups} * a.group_channels;
    const int64_t stored = last ? desc->c_store - (p.ranges - 1) * channels : channels;
    a.cols[last] = static_cast<int>(ceil_div(stored, p.v));
    a.rows[last] = std::max(1, kGnThreads / a.cols[last]);
  }
  a.partial = static_cast<float2*>(workspace);
  return launch(desc->x_type, desc->y_type, desc->act, a, p, desc->n, as_stream(stream));
}

}  // extern "C"
