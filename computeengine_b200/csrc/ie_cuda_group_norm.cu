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

constexpr int64_t kSmemPerSm = 227 * 1024;
int64_t item_bytes(int x_type, int v) {
  return int64_t{v} * element_bytes(x_type) * (x_type == IE_DT_BF16X2 ? 2 : 1);
}

int64_t scratch_bytes(int v) { return int64_t{v + 2} * kGnThreads * 4; }

struct Plan {
  int v = 1;
  bool cluster = false;
  int range_groups = 1, ranges = 1;  // channel ranges of whole groups
  int blocks = 1;                    // per image and range: cluster size, or statistics blocks
  int64_t smem = 0;
  // two-kernel path
  int joined = 1;  // statistics blocks of a cluster
  int apply_blocks = 1;
  int64_t workspace = 0;
};

// Whether ranges of g groups begin and end on vectors of v channels.
bool range_fits(const ie_group_norm_desc* d, int64_t g, int v) {
  return d->groups % g == 0 && (g == d->groups || g * (d->c / d->groups) % v == 0);
}

// The choice between one kernel that holds x in shared memory and two that
// read it twice, and the split of an image's work.  It does not depend on the
// number of images, so an image's result is the same in every batch.
//
// One kernel: channel ranges of whole groups, at least 64 bytes of a pixel (32
// where that saves a larger cluster; narrower pieces waste part of each DRAM
// access), cut into blocks of pixels of at most 32768 elements and half an SM's
// shared memory, so that one block's loads cover another's arithmetic: 32
// images of 56 x 56 x 256 fp32 take 56 us in clusters of 2 (59 when clusters of
// 8 and a quarter of the size, not timed since, took 70).  Up to 8 blocks are a cluster; ranges too
// large for that take two kernels, 256 blocks an image at most.
Plan plan_for(const ie_group_norm_desc* d, int v) {
  Plan p;
  const int64_t cg = d->c / d->groups, pixels = d->h * d->w;
  const int64_t xb = item_bytes(d->x_type, 1), yb = item_bytes(d->y_type, 1);
  p.v = v;
  auto smem_for = [&](int64_t g, int blocks) {
    const int64_t stored = d->c_store - (d->groups / g - 1) * g * cg;  // of the last range
    const int64_t cols = ceil_div(std::max(stored, g * cg), v);
    if (cols > kGnThreads) return int64_t{1} << 40;
    const int64_t rows = kGnThreads / cols;
    return ceil_div(ceil_div(pixels, blocks), rows) * kGnThreads * item_bytes(d->x_type, v) +
           scratch_bytes(v) + static_cast<int64_t>(sizeof(Stat)) * (2 + blocks) * g + 16;
  };
  auto fits = [&](int64_t g, int blocks) {
    const int64_t share = ceil_div(pixels, blocks);
    return smem_for(g, blocks) <= kSmemPerSm / 2 - 1024 && share * g * cg <= 32768 &&
           (blocks == 1 || share * (blocks - 1) < pixels);
  };
  auto accept = [&](int64_t g, int blocks) {
    p.cluster = true;
    p.range_groups = static_cast<int>(g);
    p.ranges = static_cast<int>(d->groups / g);
    p.blocks = blocks;
    p.smem = smem_for(g, blocks);
  };
  for (int64_t segment = 64; v > 1 && segment >= 32 && !p.cluster; segment /= 2) {
    int64_t g = 1;
    while (g < d->groups && !(range_fits(d, g, v) && g * cg * xb >= segment)) ++g;
    if (!range_fits(d, g, v)) break;
    for (int blocks = 1; blocks <= 8 && !p.cluster; blocks *= 2) {
      if (fits(g, blocks)) accept(g, blocks);
    }
  }
  // small images: at least 16 KB a block
  for (int64_t g = p.range_groups + 1;
       p.cluster && p.blocks == 1 && g <= d->groups && p.range_groups * cg * pixels * xb < 16384 &&
       g * cg <= kGnThreads * v;
       ++g) {
    if (range_fits(d, g, v) && fits(g, 1)) accept(g, 1);
  }
  if (p.cluster) return p;
  // ranges: whole pixels if the threads cover them, else the narrowest range of
  // at least 256 bytes
  p.range_groups = static_cast<int>(d->groups);
  if (ceil_div(d->c, v) > kGnThreads) {
    p.range_groups = 0;
    for (int64_t g = 1; g <= d->groups; ++g) {
      if (!range_fits(d, g, v)) continue;
      // several groups only within the threads' columns
      if (p.range_groups > 0 && ceil_div(g * cg, v) > kGnThreads) break;
      p.range_groups = static_cast<int>(g);
      if (g * cg * xb >= 256) break;
    }
  }
  const int64_t channels = p.range_groups * cg;
  p.ranges = static_cast<int>(d->groups / p.range_groups);
  const int64_t rows = std::max<int64_t>(1, kGnThreads / ceil_div(channels, v));
  const int64_t units = d->n * p.ranges;
  int64_t blocks = std::min(ceil_div(pixels * channels * xb, 32768), int64_t{256});
  blocks = std::max<int64_t>(1, std::min(blocks, ceil_div(pixels, kGnBatch * rows)));
  if (blocks > kGnCluster) {  // whole clusters, and every block has pixels
    blocks -= blocks % kGnCluster;
    while (blocks > kGnCluster && ceil_div(pixels, blocks) * (blocks - 1) >= pixels) {
      blocks -= kGnCluster;
    }
    p.joined = kGnCluster;
  }
  p.blocks = static_cast<int>(blocks);
  p.apply_blocks = static_cast<int>(std::max<int64_t>(
      1, std::min(std::max(4 * kSms / units, ceil_div(pixels * channels * (xb + yb), 262144)),
                  ceil_div(pixels, 4 * rows))));
  p.smem = scratch_bytes(v) + static_cast<int64_t>(sizeof(Stat)) * p.range_groups;
  p.workspace =
      units * (p.blocks / p.joined) * p.range_groups * static_cast<int64_t>(sizeof(float4));
  return p;
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
int allow_smem(Kernel kernel, int64_t smem) {
  const cudaError_t e = cudaFuncSetAttribute(
      kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  return e == cudaSuccess ? IE_OK : fail(IE_RUNTIME, "group_norm: %s", cudaGetErrorString(e));
}

template <class Kernel>
int launch_clusters(Kernel kernel, int64_t blocks, int cluster, int64_t smem, cudaStream_t s,
                    const GroupNormArgs& a) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
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
int launch_cluster(const GroupNormArgs& a, const Plan& p, int64_t images, cudaStream_t s) {
  auto kernel = group_norm_cluster_kernel<XT, YT, V, ACT>;
  const int rc = allow_smem(kernel, p.smem);
  if (rc != IE_OK) return rc;
  return launch_clusters(kernel, images * p.ranges * p.blocks, p.blocks, p.smem, s, a);
}

template <int XT, int YT, int V, int ACT>
int launch_two(const GroupNormArgs& a, const Plan& p, int64_t images, cudaStream_t s) {
  auto stats = group_norm_stats_kernel<XT, V>;
  auto apply = group_norm_apply_kernel<XT, YT, V, ACT>;
  const int64_t apply_smem = static_cast<int64_t>(sizeof(Stat)) * p.range_groups;
  int rc = allow_smem(stats, p.smem);
  if (rc == IE_OK) rc = allow_smem(apply, apply_smem);
  const int64_t units = images * p.ranges;
  if (rc == IE_OK) rc = launch_clusters(stats, units * p.blocks, p.joined, p.smem, s, a);
  if (rc != IE_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units * p.apply_blocks));
  cfg.blockDim = dim3(kGnThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(apply_smem);
  cfg.stream = s;
  cudaLaunchAttribute attr{};  // its launch overlaps the end of the statistics kernel
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, apply, a, p.apply_blocks);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(IE_RUNTIME, "group_norm: %s", cudaGetErrorString(e));
  }
  return check_launch("group_norm");
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
  int rc = check_group_norm(desc);
  if (rc != IE_OK) return rc;
  if (x == nullptr || y == nullptr) return fail(IE_INVALID_ARGUMENT, "null tensor or buffer");
  rc = check_aligned(x, element_bytes(desc->x_type), "GroupNorm x");
  if (rc == IE_OK) rc = check_aligned(y, element_bytes(desc->y_type), "GroupNorm y");
  if (rc == IE_OK) rc = check_aligned(gamma, 4, "GroupNorm gamma");
  if (rc == IE_OK) rc = check_aligned(beta, 4, "GroupNorm beta");
  if (rc != IE_OK) return rc;
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
  a.parts = p.blocks / p.joined;
  a.part_share = a.share * p.joined;
  for (int last = 0; last < 2; ++last) {
    const int64_t channels = int64_t{p.range_groups} * a.group_channels;
    const int64_t stored = last ? desc->c_store - (p.ranges - 1) * channels : channels;
    a.cols[last] = static_cast<int>(ceil_div(stored, p.v));
    a.rows[last] = std::max(1, kGnThreads / a.cols[last]);
  }
  a.partial = static_cast<float4*>(workspace);
  return launch(desc->x_type, desc->y_type, desc->act, a, p, desc->n, as_stream(stream));
}

}  // extern "C"
