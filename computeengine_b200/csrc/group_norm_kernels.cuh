// Group normalization with an activation over channels-last tensors.
//
// A thread owns V neighbouring channels (one 16-byte load of x) and strides
// over the pixels, so everything it does is per channel and a group may begin
// and end anywhere in a vector.  Statistics: each batch of pixels gives its
// exact mean and sum of squared differences per channel, joined with what the
// thread has by the pairwise update of Chan, Golub and LeVeque (1979); threads,
// then blocks are joined the same way in a fixed order.  A mean far from zero
// therefore costs no precision and results do not depend on timing.
//
// group_norm_cluster_kernel: a channel range of an image is held in the shared
// memory of one block or a cluster of up to 16, so x is read once.
// group_norm_stats_kernel, group_norm_apply_kernel: for images that do not fit;
// the second read of x comes out of L2.
#pragma once

#include <cooperative_groups.h>


#include "element_types.cuh"

namespace ie_cuda {

struct GroupNormArgs {
  const void* x;
  const float* gamma;
  const float* beta;
  void* y;
  int pixels;  // h * w
  int c, c_store, group_channels;
  float low, high;  // of the clamp
  float eps;
  int range_groups;     // groups per channel range
  int ranges;           // channel ranges of an image
  int first_range;      // of this launch (two-kernel path)
  int64_t first_image;  // of this launch
  int blocks;           // pixel blocks per image and range
  int share;            // pixels of a block
  int cols[2], rows[2]; // threads over a range's vectors and pixels: inner, last range
  float2* partial;      // two-kernel path: mean and sum of squared differences,
                        // [image of this launch][range of this launch][block][range_groups]
  int launch_ranges;    // ranges of this launch
};

constexpr int kGnThreads = 256;
constexpr int kGnBatch = 4;  // pixels per exact mean

// Kinds of activation: a clamp to [low, high] (none, ReLU, ReLU6), SiLU, GELU.
enum { kActClamp = 0, kActSilu = 1, kActGelu = 2 };

template <int ACT>
__device__ __forceinline__ float activate(float v, float low, float high) {
  if constexpr (ACT == kActClamp) {
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(low));  // NaN stays
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(high));
    return v;
  } else if constexpr (ACT == kActSilu) {
    // v / (1 + 2^(-v log2 e)) on the special function unit: each of its two
    // results is within two steps of fp32
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return v * r;
  } else {
    return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
  }
}

// V channels of one pixel as they lie in memory (BF16X2: of both planes).
template <int T, int V>
struct Item {
  static constexpr int kBytes = V * element_bytes(T);
  Bytes<kBytes> v;
  Bytes<T == IE_DT_BF16X2 ? kBytes : 2> lo;
};

// Element offset of channel c of a pixel, and of the lo plane behind it.
template <int T>
__device__ __forceinline__ int64_t channel_at(int64_t pixel, int c_store, int c) {
  return pixel * (T == IE_DT_BF16X2 ? 2 * c_store : c_store) + c;
}

template <int T, int V>
__device__ __forceinline__ Item<T, V> load_item(const void* x, int64_t at, int c_store) {
  Item<T, V> i;
  const uint8_t* p = static_cast<const uint8_t*>(x) + at * element_bytes(T);
  i.v = load_bytes<Item<T, V>::kBytes>(p);
  if constexpr (T == IE_DT_BF16X2) i.lo = load_bytes<Item<T, V>::kBytes>(p + 2 * c_store);
  return i;
}

template <int T, int V>
__device__ __forceinline__ void item_floats(const Item<T, V>& i, float (&f)[V]) {
  if constexpr (T == IE_DT_BF16X2) {
    float l[V];
    to_floats<IE_DT_BF16, V>(i.v, f);
    to_floats<IE_DT_BF16, V>(i.lo, l);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] += l[e];
  } else {
    to_floats<T, V>(i.v, f);
  }
}

template <int T, int V>
__device__ __forceinline__ void store_item(void* y, int64_t at, int c_store, const float (&f)[V]) {
  uint8_t* p = static_cast<uint8_t*>(y) + at * element_bytes(T);
  if constexpr (T == IE_DT_BF16X2) {
    float h[V], l[V];
    const auto hi = from_floats<IE_DT_BF16, V>(f);
    to_floats<IE_DT_BF16, V>(hi, h);
#pragma unroll
    for (int e = 0; e < V; ++e) l[e] = f[e] - h[e];
    store_bytes<V * 2>(p, hi);
    store_bytes<V * 2>(p + 2 * c_store, from_floats<IE_DT_BF16, V>(l));
  } else {
    store_bytes<V * element_bytes(T)>(p, from_floats<T, V>(f));
  }
}

// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ void add_pair(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma_pair(float& d0, float& d1, float a0, float a1, float b0,
                                         float b1) {  // d += a * b
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 d, {%0, %1};\n\tfma.rn.f32x2 d, a, b, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "+f"(d0), "+f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
template <int V>
__device__ __forceinline__ void add_to(float (&a)[V], const float (&b)[V]) {  // a += b
  if constexpr (V == 1) {
    a[0] += b[0];
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) add_pair(a[e], a[e + 1], b[e], b[e + 1]);
  }
}
template <int V>
__device__ __forceinline__ void add_squares(float (&a)[V], const float (&b)[V],
                                            const float (&minus)[V]) {  // a += (b + minus)^2
  if constexpr (V == 1) {
    const float d = b[0] + minus[0];
    a[0] += d * d;
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      float d0 = b[e], d1 = b[e + 1];
      add_pair(d0, d1, minus[e], minus[e + 1]);
      fma_pair(a[e], a[e + 1], d0, d1, d0, d1);
    }
  }
}

// Running statistics of V channels over the pixels a thread has seen.
template <int V>
struct Running {
  float mean[V], m2[V];
  int n = 0;

  __device__ __forceinline__ Running() {
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.0f;
  }
  // Joins k > 0 pixels with sum s and squares q about their mean.
  __device__ __forceinline__ void join(int k, const float (&batch_mean)[V], const float (&q)[V]) {
    const float share = static_cast<float>(k) / static_cast<float>(n + k);
    const float weight = static_cast<float>(n) * share;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = n == 0 ? 0.0f : batch_mean[e] - mean[e];
      mean[e] = n == 0 ? batch_mean[e] : fmaf(d, share, mean[e]);
      m2[e] += fmaf(d * d, weight, q[e]);
    }
    n += k;
  }
  // A whole batch in registers.
  __device__ __forceinline__ void add(const float (&f)[kGnBatch][V]) {
    float s[V], q[V], minus[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s[e] = f[0][e];
      q[e] = 0.0f;
    }
#pragma unroll
    for (int i = 1; i < kGnBatch; ++i) add_to<V>(s, f[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s[e] *= 1.0f / kGnBatch;
      minus[e] = -s[e];
    }
#pragma unroll
    for (int i = 0; i < kGnBatch; ++i) add_squares<V>(q, f[i], minus);
    join(kGnBatch, s, q);
  }
  // One pixel.
  __device__ __forceinline__ void add(const float (&f)[V]) {
    float q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = 0.0f;
    join(1, f, q);
  }
};

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sums each thread's V channels into the groups of the block's channel range:
// out[g], in an order that is always the same.  Thread t holds the channels
// (t % cols) * V .. of the range, rows = threads per column.  First slices of
// the rows of each channel are summed by all threads, then a warp sums a
// group.  scratch holds (V + 1) * threads floats.  (A single group wider than
// the threads' columns: group_channels is what the columns hold.)
template <int V>
__device__ __forceinline__ void group_sums(const float (&v)[V], int cols, int rows,
                                           int group_channels, int groups, float* scratch,
                                           float* out) {
  const int width = cols * V, t = threadIdx.x, lane = t & 31;
  if (t < cols * rows) {  // [rows][width]
#pragma unroll
    for (int e = 0; e < V; ++e) scratch[t * V + e] = v[e];
  }
  __syncthreads();
  float* partial = scratch;  // [slices][width]
  int slices = 1;
  if (width >= kGnThreads) {  // a channel's sum replaces its first row
    for (int ch = t; ch < width; ch += kGnThreads) {
      float s = scratch[ch];
      for (int k = 1; k < rows; ++k) s += scratch[k * width + ch];
      scratch[ch] = s;
    }
  } else {
    partial = scratch + V * kGnThreads;
    slices = kGnThreads / width;
    const int slice = t / width, ch = t - slice * width;
    if (slice < slices) {
      float s = 0.0f;
#pragma unroll 4
      for (int k = slice; k < rows; k += slices) s += scratch[k * width + ch];
      partial[t] = s;
    }
  }
  __syncthreads();
  // lanes over the group's channels, and over slices when they are few
  int lanes = 1, shift = 0;
  while (lanes < group_channels && lanes < 32) {
    lanes <<= 1;
    ++shift;
  }
  for (int g = t >> 5; g < groups; g += kGnThreads / 32) {
    float s = 0.0f;
    for (int k = lane >> shift; k < slices; k += 32 >> shift) {
      const float* row = partial + k * width + g * group_channels;
      for (int ch = lane & (lanes - 1); ch < group_channels; ch += lanes) s += row[ch];
    }
    s = warp_sum(s);
    if (lane == 0) out[g] = s;
  }
  __syncthreads();
}

// Joins the statistics of `blocks` pixel blocks, block k's at at(k), into the
// mean and 1 / sigma of a group.
template <class At>
__device__ __forceinline__ float2 join_blocks(const GroupNormArgs& a, int group_channels,
                                              const At& at) {
  float s = 0.0f, q = 0.0f;
  for (int k = 0; k < a.blocks; ++k) {
    const int w = min(a.pixels, (k + 1) * a.share) - k * a.share;
    if (w > 0) s += static_cast<float>(w) * at(k).x;
  }
  const float mu = a.blocks == 1 ? at(0).x : s / static_cast<float>(a.pixels);
  for (int k = 0; k < a.blocks; ++k) {
    const int w = min(a.pixels, (k + 1) * a.share) - k * a.share;
    if (w <= 0) continue;
    const float2 o = at(k);
    const float d = o.x - mu;
    q += o.y + static_cast<float>(w) * static_cast<float>(group_channels) * d * d;
  }
  const float size = static_cast<float>(a.pixels) * static_cast<float>(group_channels);
  return make_float2(mu, 1.0f / sqrtf(q / size + a.eps));
}

// Geometry shared by the kernels: the block's channel range.
struct Range {
  int c0, channels, cols, rows, group_channels;
  __device__ __forceinline__ Range(const GroupNormArgs& a, int range) {
    const int last = range == a.ranges - 1;  // carries the padding channels
    group_channels = a.group_channels;
    channels = a.range_groups * group_channels;
    c0 = range * channels;
    cols = a.cols[last];
    rows = a.rows[last];
  }
};

// mul and add of the V channels from c: gamma / sigma, and beta less the mean's
// share of it.  stat: mean and 1 / sigma of the range's groups; the thread's
// first channel is `inner` channels into group `first`.
template <int V>
__device__ __forceinline__ void channel_affine(const GroupNormArgs& a, int c, int first, int inner,
                                               const float2* stat, float (&mul)[V],
                                               float (&add)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool in = c + e < a.c;
    const float2 st = in ? stat[first] : make_float2(0.0f, 0.0f);
    mul[e] = in && a.gamma != nullptr ? st.y * a.gamma[c + e] : st.y;
    add[e] = fmaf(-st.x, mul[e], in && a.beta != nullptr ? a.beta[c + e] : 0.0f);
    if (++inner == a.group_channels) {
      inner = 0;
      ++first;
    }
  }
}

// Normalizes, activates and stores one item; channels past c become zero
// (mul and add are zero there, but x may hold anything).
template <int YT, int V, int ACT>
__device__ __forceinline__ void finish_item(const GroupNormArgs& a, float (&f)[V],
                                            const float (&mul)[V], const float (&add)[V],
                                            uint8_t* y, int valid) {
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = activate<ACT>(fmaf(f[e], mul[e], add[e]), a.low, a.high);
  if (valid < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < valid ? f[e] : 0.0f;
  }
  store_item<YT, V>(y, 0, a.c_store, f);
}

// One cluster per (image, channel range); each block holds its pixels' items
// in shared memory.  The copies are issued at once, so the whole range is in
// flight; a thread reads back only what it copied itself.
template <int XT, int YT, int V, int ACT>
__global__ void __launch_bounds__(kGnThreads, 4) group_norm_cluster_kernel(const GroupNormArgs a) {
  namespace cg = cooperative_groups;
  constexpr int kItem = Item<XT, V>::kBytes * (XT == IE_DT_BF16X2 ? 2 : 1);
  static_assert(Item<XT, V>::kBytes == 16, "16-byte copies");
  extern __shared__ __align__(16) uint8_t smem[];
  float2* own = reinterpret_cast<float2*>(smem);    // [range_groups] of this block
  float2* stat = own + a.range_groups;              // [range_groups] mean, 1 / sigma
  float2* others = stat + a.range_groups;           // [blocks][range_groups]
  float* sums = reinterpret_cast<float*>(others + a.blocks * a.range_groups);  // [range_groups]
  float* scratch = sums + a.range_groups;
  uint8_t* items = reinterpret_cast<uint8_t*>(scratch + (V + 1) * kGnThreads);
  items += (16 - reinterpret_cast<uintptr_t>(items) % 16) % 16;

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = a.blocks > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(a.blocks);
  const int64_t image = unit / static_cast<uint32_t>(a.ranges);
  const int range = static_cast<int>(unit - image * a.ranges);
  const Range r(a, range);
  const int row = threadIdx.x / r.cols, col = threadIdx.x - row * r.cols;
  const int from = rank * a.share;
  const int count = max(0, min(a.pixels, from + a.share) - from);
  const int64_t p0 = image * a.pixels + from;
  const int c = r.c0 + col * V;

  uint8_t* mine = items + threadIdx.x * 16;
  constexpr int kStep = kGnThreads * kItem;
  const int n = row < r.rows && row < count ? (count - row + r.rows - 1) / r.rows : 0;
  {
    const int64_t x_step = static_cast<int64_t>(r.rows) * channel_at<XT>(1, a.c_store, 0) *
                           element_bytes(XT);
    const uint8_t* from_x = static_cast<const uint8_t*>(a.x) +
                            channel_at<XT>(p0 + row, a.c_store, c) * element_bytes(XT);
    uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
    for (int i = 0; i < n; ++i, from_x += x_step, to += kStep) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from_x) : "memory");
      if constexpr (XT == IE_DT_BF16X2) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kGnThreads * 16),
                     "l"(from_x + 2 * a.c_store)
                     : "memory");
      }
    }
  }
  // the thread's place among the groups, while the copies are under way
  const int first = col * V / r.group_channels, inner = col * V - first * r.group_channels;
  asm volatile("cp.async.wait_all;" ::: "memory");

  auto item = [&](int i, float(&f)[V]) {
    Item<XT, V> it;
    it.v = load_bytes<16>(mine + i * kStep);
    if constexpr (XT == IE_DT_BF16X2) it.lo = load_bytes<16>(mine + i * kStep + kGnThreads * 16);
    item_floats<XT, V>(it, f);
  };
  // the block's mean of each group, then the squares about it
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = 0.0f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    float f[V];
    item(i, f);
    add_to<V>(v, f);
  }
  group_sums<V>(v, r.cols, r.rows, r.group_channels, a.range_groups, scratch, sums);
  const float inv = 1.0f / (static_cast<float>(count) * static_cast<float>(r.group_channels));
  {
    float minus[V];
    int g = first, in_group = inner;
#pragma unroll
    for (int e = 0; e < V; ++e) {  // padding channels: the group's that would follow
      minus[e] = -sums[min(g, a.range_groups - 1)] * inv;
      v[e] = 0.0f;
      if (++in_group == r.group_channels) {
        in_group = 0;
        ++g;
      }
    }
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      float f[V];
      item(i, f);
      add_squares<V>(v, f, minus);
    }
  }
  for (int g = threadIdx.x; g < a.range_groups; g += kGnThreads) own[g].x = sums[g] * inv;
  __syncthreads();
  group_sums<V>(v, r.cols, r.rows, r.group_channels, a.range_groups, scratch, sums);
  for (int g = threadIdx.x; g < a.range_groups; g += kGnThreads) own[g].y = sums[g];

  // the blocks' statistics, in rank order
  if (a.blocks > 1) {
    cluster.sync();
    const int all = a.blocks * a.range_groups;
    for (int i = threadIdx.x; i < all; i += kGnThreads) {
      const int k = i / a.range_groups;
      others[i] = *cluster.map_shared_rank(own + (i - k * a.range_groups), k);
    }
    cluster.barrier_arrive();  // waited for at the end: no block leaves while others read
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.range_groups; g += kGnThreads) {
    stat[g] = join_blocks(a, r.group_channels, [&](int k) {
      return a.blocks > 1 ? others[k * a.range_groups + g] : own[g];
    });
  }
  __syncthreads();
  float g[V], b[V];
  if (n > 0) channel_affine<V>(a, c, first, inner, stat, g, b);
  uint8_t* y = static_cast<uint8_t*>(a.y) +
               channel_at<YT>(p0 + row, a.c_store, c) * element_bytes(YT);
  const int64_t y_step = static_cast<int64_t>(r.rows) * channel_at<YT>(1, a.c_store, 0) *
                         element_bytes(YT);
#pragma unroll(ACT == kActGelu ? 1 : 2)
  for (int i = 0; i < n; ++i, y += y_step) {
    float f[V];
    item(i, f);
    finish_item<YT, V, ACT>(a, f, g, b, y, a.c - c);
  }
  if (a.blocks > 1) cluster.barrier_wait();
}

// Statistics of one block of pixels of an image and channel range.
template <int XT, int V>
__global__ void __launch_bounds__(kGnThreads, 2) group_norm_stats_kernel(const GroupNormArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  float* sums = reinterpret_cast<float*>(smem);  // [range_groups]
  float* scratch = sums + a.range_groups;
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(a.blocks);
  const int block = static_cast<int>(blockIdx.x - unit * a.blocks);
  const uint32_t of_launch = unit / static_cast<uint32_t>(a.launch_ranges);
  const int range = a.first_range + static_cast<int>(unit - of_launch * a.launch_ranges);
  const int64_t image = a.first_image + of_launch;
  const Range r(a, range);
  const int all = (r.channels + V - 1) / V;  // padding channels have no statistics
  const int cols = min(all, kGnThreads), rows = kGnThreads / cols;
  const int row = threadIdx.x / cols, col = threadIdx.x - row * cols;
  const int from = block * a.share;
  const int count = max(0, min(a.pixels, from + a.share) - from);
  const int64_t p0 = image * a.pixels + from;
  Running<V> run;
  // more columns than threads: the range is one group
  for (int at = col; row < rows && row < count && at < all; at += cols) {
    const int c = r.c0 + at * V;
    constexpr int K = XT == IE_DT_BF16X2 ? 1 : 2;  // batches in flight
    const int64_t step = static_cast<int64_t>(rows) * channel_at<XT>(1, a.c_store, 0);
    int64_t from_x = channel_at<XT>(p0 + row, a.c_store, c);
    int left = (count - row + rows - 1) / rows;  // pixels of this thread
    for (; left >= K * kGnBatch; left -= K * kGnBatch) {
      Item<XT, V> it[K * kGnBatch];
#pragma unroll
      for (int e = 0; e < K * kGnBatch; ++e, from_x += step) {
        it[e] = load_item<XT, V>(a.x, from_x, a.c_store);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float f[kGnBatch][V];
#pragma unroll
        for (int e = 0; e < kGnBatch; ++e) item_floats<XT, V>(it[k * kGnBatch + e], f[e]);
        run.add(f);
      }
    }
    for (; left > 0; --left, from_x += step) {
      float f[V];
      item_floats<XT, V>(load_item<XT, V>(a.x, from_x, a.c_store), f);
      run.add(f);
    }
  }
  // the block's mean of each group, then each channel's squares about it
  const int group_channels = all > cols ? cols * V : r.group_channels;
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = run.n > 0 ? run.mean[e] * static_cast<float>(run.n) : 0.0f;
  group_sums<V>(v, cols, rows, group_channels, a.range_groups, scratch, sums);
  const float inv = 1.0f / (static_cast<float>(count) * static_cast<float>(r.group_channels));
  int g = col * V / group_channels, inner = col * V - g * group_channels;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float d = run.mean[e] - sums[min(g, a.range_groups - 1)] * inv;
    v[e] = run.n > 0 ? fmaf(d * d, static_cast<float>(run.n), run.m2[e]) : 0.0f;
    if (++inner == group_channels) {
      inner = 0;
      ++g;
    }
  }
  // [unit][group][block], so that a warp reads a group's blocks side by side
  float2* to = a.partial + static_cast<int64_t>(unit) * a.range_groups * a.blocks + block;
  for (int i = threadIdx.x; i < a.range_groups; i += kGnThreads) {
    to[static_cast<int64_t>(i) * a.blocks].x = sums[i] * inv;
  }
  __syncthreads();
  group_sums<V>(v, cols, rows, group_channels, a.range_groups, scratch, sums);
  for (int i = threadIdx.x; i < a.range_groups; i += kGnThreads) {
    to[static_cast<int64_t>(i) * a.blocks].y = sums[i];
  }
}

// Joins the blocks' statistics (every block of the launch for itself) and
// normalizes.  Blocks run over the pixels from the end, which L2 still holds.
template <int XT, int YT, int V, int ACT>
__global__ void __launch_bounds__(kGnThreads, V == 8 && XT == IE_DT_BF16X2 ? 2 : 4)
    group_norm_apply_kernel(const GroupNormArgs a,
                                                                      int apply_blocks) {
  extern __shared__ __align__(16) uint8_t smem[];
  float2* stat = reinterpret_cast<float2*>(smem);
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(apply_blocks);
  const int block = apply_blocks - 1 - static_cast<int>(blockIdx.x - unit * apply_blocks);
  const uint32_t of_launch = unit / static_cast<uint32_t>(a.launch_ranges);
  const int range = a.first_range + static_cast<int>(unit - of_launch * a.launch_ranges);
  const int64_t image = a.first_image + of_launch;
  const Range r(a, range);
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < a.range_groups; g += kGnThreads / 32) {
    const float2* p = a.partial + (static_cast<int64_t>(unit) * a.range_groups + g) * a.blocks;
    float s = 0.0f, q = 0.0f;
    for (int k = lane; k < a.blocks; k += 32) {
      const int w = min(a.pixels, (k + 1) * a.share) - k * a.share;
      if (w > 0) s += static_cast<float>(w) * p[k].x;
    }
    const float mu = warp_sum(s) / static_cast<float>(a.pixels);
    for (int k = lane; k < a.blocks; k += 32) {
      const int w = min(a.pixels, (k + 1) * a.share) - k * a.share;
      if (w <= 0) continue;
      const float2 o = p[k];
      const float d = o.x - mu;
      q += o.y + static_cast<float>(w) * static_cast<float>(r.group_channels) * d * d;
    }
    q = warp_sum(q);
    const float size = static_cast<float>(a.pixels) * static_cast<float>(r.group_channels);
    if (lane == 0) stat[g] = make_float2(mu, 1.0f / sqrtf(q / size + a.eps));
  }
  __syncthreads();
  const int share = (a.pixels + apply_blocks - 1) / apply_blocks;
  const int from = block * share;
  const int count = max(0, min(a.pixels, from + share) - from);
  const int64_t p0 = image * a.pixels + from;
  // padding channels may make the last range wider than the block
  for (int col0 = 0; col0 < r.cols; col0 += kGnThreads) {
    const int cols = min(r.cols - col0, kGnThreads), rows = kGnThreads / cols;
    const int row = threadIdx.x / cols, col = col0 + threadIdx.x - row * cols;
    if (row >= rows || row >= count) continue;
    const int c = r.c0 + col * V;
    const int first = col * V / r.group_channels;
    float mul[V], add[V];
    channel_affine<V>(a, c, first, col * V - first * r.group_channels, stat, mul, add);
    constexpr int K = ACT == kActGelu || XT == IE_DT_BF16X2 ? 2 : 4;
    const int64_t x_step = static_cast<int64_t>(rows) * channel_at<XT>(1, a.c_store, 0);
    const int64_t y_step = static_cast<int64_t>(rows) * channel_at<YT>(1, a.c_store, 0) *
                           element_bytes(YT);
    int64_t from_x = channel_at<XT>(p0 + row, a.c_store, c);
    uint8_t* y = static_cast<uint8_t*>(a.y) +
                 channel_at<YT>(p0 + row, a.c_store, c) * element_bytes(YT);
    int left = (count - row + rows - 1) / rows;
    for (; left >= K; left -= K) {
      Item<XT, V> it[K];
#pragma unroll
      for (int e = 0; e < K; ++e, from_x += x_step) {
        it[e] = load_item<XT, V>(a.x, from_x, a.c_store);
      }
#pragma unroll
      for (int e = 0; e < K; ++e, y += y_step) {
        float f[V];
        item_floats<XT, V>(it[e], f);
        finish_item<YT, V, ACT>(a, f, mul, add, y, a.c - c);
      }
    }
    for (; left > 0; --left, from_x += x_step, y += y_step) {
      float f[V];
      item_floats<XT, V>(load_item<XT, V>(a.x, from_x, a.c_store), f);
      finish_item<YT, V, ACT>(a, f, mul, add, y, a.c - c);
    }
  }
}

}  // namespace ie_cuda
