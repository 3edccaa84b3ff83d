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

#include <type_traits>

#include "element_types.cuh"

namespace ie_cuda {

struct GroupNormArgs {
  const void* x;
  const float* gamma;
  const float* beta;
  void* y;
  int64_t pixels;  // h * w
  int c, c_store, groups, act;
  float eps;
  int range_groups;     // groups per channel range
  int ranges;           // channel ranges of an image
  int first_range;      // of this launch (two-kernel path)
  int64_t first_image;  // of this launch
  int blocks;           // pixel blocks per image and range
  float2* partial;      // two-kernel path: mean and sum of squared differences,
                        // [image of this launch][range of this launch][block][range_groups]
  int launch_ranges;    // ranges of this launch
};

constexpr int kGnThreads = 256;
constexpr int kGnBatch = 8;  // pixels per exact mean

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case IE_ACT_RELU:
      return v < 0.0f ? 0.0f : v;  // NaN stays
    case IE_ACT_RELU6:
      return v < 0.0f ? 0.0f : v > 6.0f ? 6.0f : v;
    case IE_ACT_SILU:
      return __fdividef(v, 1.0f + __expf(-v));
    case IE_ACT_GELU:
      return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    default:
      return v;
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

// Running statistics of V channels over the pixels a thread has seen.
template <int V>
struct Running {
  float mean[V], m2[V];
  int n = 0;

  __device__ __forceinline__ Running() {
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.0f;
  }
  // A batch of k > 0 pixels, MAX at most (0: any number); get(i, f) reads
  // pixel i, twice.
  template <int MAX, class Get>
  __device__ __forceinline__ void add(int k, const Get& get) {
    float s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.0f;
    auto sum = [&](int i) {
      float f[V];
      get(i, f);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += f[e];
    };
    auto squares = [&](int i) {
      float f[V];
      get(i, f);
#pragma unroll
      for (int e = 0; e < V; ++e) q[e] += (f[e] - s[e]) * (f[e] - s[e]);
    };
    const float inv = 1.0f / static_cast<float>(k);
    if constexpr (MAX > 0) {
#pragma unroll
      for (int i = 0; i < MAX; ++i) {
        if (i < k) sum(i);
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < k; ++i) sum(i);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] *= inv;
    if constexpr (MAX > 0) {
#pragma unroll
      for (int i = 0; i < MAX; ++i) {
        if (i < k) squares(i);
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < k; ++i) squares(i);
    }
    const float share = static_cast<float>(k) / static_cast<float>(n + k);
    const float weight = static_cast<float>(n) * share;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = n == 0 ? 0.0f : s[e] - mean[e];
      mean[e] = n == 0 ? s[e] : mean[e] + d * share;
      m2[e] += q[e] + d * d * weight;
    }
    n += k;
  }
};

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Joins the threads' channels into the groups of the block's channel range:
// out[g] = (mean, sum of squared differences).  Thread t holds the channels
// (t % cols) * V .. of the range, rows = threads per column; scratch holds
// (2 * V + 2) * threads floats.  First every channel's rows are joined in
// slices, so that all threads take part; then a warp joins a group's channels.
// (A single group wider than the threads' columns: every thread's channels are
// that group's.)
template <int V>
__device__ __forceinline__ void join_threads(const Running<V>& r, int cols, int rows,
                                             int group_channels, int groups, float* scratch,
                                             float2* out) {
  const int width = cols * V;
  float* mean = scratch;                   // [rows][width]
  float* m2 = mean + V * kGnThreads;       // [rows][width]
  float* count = m2 + V * kGnThreads;      // [rows][cols]
  float* joined = count + kGnThreads;      // [slices][cols]
  const int t = threadIdx.x;
  if (t < cols * rows) {
    const int at = t / cols * width + t % cols * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      mean[at + e] = r.mean[e];
      m2[at + e] = r.m2[e];
    }
    count[t] = static_cast<float>(r.n);
  }
  __syncthreads();
  // slices of whole rows; a slice's result replaces its first row
  const int slices = max(1, min(rows, kGnThreads / width));
  const int deep = (rows + slices - 1) / slices;
  for (int i = t; i < slices * width; i += kGnThreads) {
    const int slice = i / width, ch = i - slice * width, col = ch / V;
    const int from = slice * deep, to = min(rows, from + deep);
    float n = 0.0f, s = 0.0f, q = 0.0f;
    for (int k = from; k < to; ++k) {
      n += count[k * cols + col];
      s += count[k * cols + col] * mean[k * width + ch];
    }
    const float mu = n > 0.0f ? s / n : 0.0f;
    for (int k = from; k < to; ++k) {
      const float w = count[k * cols + col], d = mean[k * width + ch] - mu;
      if (w > 0.0f) q += m2[k * width + ch] + w * d * d;
    }
    if (from < rows) {
      mean[from * width + ch] = mu;
      m2[from * width + ch] = q;
    }
    joined[slice * cols + col] = n;  // the same from each of the column's channels
  }
  __syncthreads();
  const int lane = t & 31;
  for (int g = t >> 5; g < groups; g += kGnThreads / 32) {
    const int entries = slices * group_channels;
    float n = 0.0f, s = 0.0f, q = 0.0f;
    for (int i = lane; i < entries; i += 32) {
      const int slice = i / group_channels, ch = g * group_channels + i - slice * group_channels;
      const float w = joined[slice * cols + ch / V];
      if (w > 0.0f) {
        n += w;
        s += w * mean[slice * deep * width + ch];
      }
    }
    n = warp_sum(n);
    const float mu = warp_sum(s) / n;
    for (int i = lane; i < entries; i += 32) {
      const int slice = i / group_channels, ch = g * group_channels + i - slice * group_channels;
      const float w = joined[slice * cols + ch / V];
      const float d = w > 0.0f ? mean[slice * deep * width + ch] - mu : 0.0f;
      if (w > 0.0f) q += m2[slice * deep * width + ch] + w * d * d;
    }
    q = warp_sum(q);
    if (lane == 0) out[g] = make_float2(mu, q);
  }
  __syncthreads();
}

// Geometry shared by the kernels: the block's channel range.
struct Range {
  int c0, channels, cols, rows, group_channels;
  __device__ __forceinline__ Range(const GroupNormArgs& a, int range, int v) {
    group_channels = a.c / a.groups;
    c0 = range * a.range_groups * group_channels;
    channels = a.range_groups * group_channels;
    // the last range carries the padding channels
    const int stored = range == a.ranges - 1 ? a.c_store - c0 : channels;
    cols = (stored + v - 1) / v;
    rows = max(1, kGnThreads / cols);
  }
};

// Normalizes, activates and stores one item; channels past c become zero
// (mul and add are zero there, but x may hold anything).
template <int YT, int V, int ACT>
__device__ __forceinline__ void finish_item(const GroupNormArgs& a, float (&f)[V],
                                            const float (&mul)[V], const float (&add)[V],
                                            int64_t pixel, int c) {
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = activate(fmaf(f[e], mul[e], add[e]), ACT);
  if (c + V > a.c) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = c + e < a.c ? f[e] : 0.0f;
  }
  store_item<YT, V>(a.y, channel_at<YT>(pixel, a.c_store, c), a.c_store, f);
}

// Runs body(std::integral_constant<int, act>) for the activation, so that the
// choice is made once and not per element.
template <class Body>
__device__ __forceinline__ void with_activation(int act, const Body& body) {
  switch (act) {
    case IE_ACT_RELU: body(std::integral_constant<int, IE_ACT_RELU>()); break;
    case IE_ACT_RELU6: body(std::integral_constant<int, IE_ACT_RELU6>()); break;
    case IE_ACT_SILU: body(std::integral_constant<int, IE_ACT_SILU>()); break;
    case IE_ACT_GELU: body(std::integral_constant<int, IE_ACT_GELU>()); break;
    default: body(std::integral_constant<int, IE_ACT_NONE>()); break;
  }
}

// One cluster per (image, channel range); each block holds its pixels' items
// in shared memory.  The copies are issued at once, so the whole range is in
// flight; a thread reads back only what it copied itself.
template <int XT, int YT, int V>
__global__ void __launch_bounds__(kGnThreads, 4) group_norm_cluster_kernel(const GroupNormArgs a) {
  namespace cg = cooperative_groups;
  constexpr int kItem = Item<XT, V>::kBytes * (XT == IE_DT_BF16X2 ? 2 : 1);
  static_assert(Item<XT, V>::kBytes == 16, "16-byte copies");
  extern __shared__ __align__(16) uint8_t smem[];
  float2* own = reinterpret_cast<float2*>(smem);  // [range_groups] of this block
  float2* stat = own + a.range_groups;            // [range_groups] mean, 1 / sigma
  float* scratch = reinterpret_cast<float*>(stat + a.range_groups);
  uint8_t* items = reinterpret_cast<uint8_t*>(scratch + (2 * V + 2) * kGnThreads);
  items += (16 - reinterpret_cast<uintptr_t>(items) % 16) % 16;

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = a.blocks > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  const int unit = static_cast<int>(blockIdx.x) / a.blocks;
  const int range = unit % a.ranges;
  const int64_t image = unit / a.ranges;
  const Range r(a, range, V);
  const int col = threadIdx.x % r.cols, row = threadIdx.x / r.cols;
  const bool works = row < r.rows;
  const int64_t share = (a.pixels + a.blocks - 1) / a.blocks;
  const int64_t from = rank * share;
  const int count = static_cast<int>(max(int64_t{0}, min(a.pixels, from + share) - from));
  const int64_t p0 = image * a.pixels + from;
  const int c = r.c0 + col * V;

  uint8_t* mine = items + threadIdx.x * 16;
  constexpr int kStep = kGnThreads * kItem;
  if (works) {
    const uint8_t* x = static_cast<const uint8_t*>(a.x);
    int i = 0;
    for (int p = row; p < count; p += r.rows, ++i) {
      const uint8_t* from_x = x + channel_at<XT>(p0 + p, a.c_store, c) * element_bytes(XT);
      const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(mine + i * kStep));
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from_x) : "memory");
      if constexpr (XT == IE_DT_BF16X2) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kGnThreads * 16),
                     "l"(from_x + 2 * a.c_store)
                     : "memory");
      }
    }
  }
  float g[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    g[e] = works && a.gamma != nullptr && c + e < a.c ? a.gamma[c + e] : 1.0f;
    b[e] = works && a.beta != nullptr && c + e < a.c ? a.beta[c + e] : 0.0f;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  auto item = [&](int i, float(&f)[V]) {
    Item<XT, V> it;
    it.v = load_bytes<16>(mine + i * kStep);
    if constexpr (XT == IE_DT_BF16X2) it.lo = load_bytes<16>(mine + i * kStep + kGnThreads * 16);
    item_floats<XT, V>(it, f);
  };
  const int n = works && row < count ? (count - row + r.rows - 1) / r.rows : 0;
  Running<V> run;
  if (n > 0) run.template add<0>(n, item);
  join_threads<V>(run, r.cols, r.rows, r.group_channels, a.range_groups, scratch, own);

  // the blocks' statistics, in rank order
  if (a.blocks > 1) cluster.sync();
  for (int gi = threadIdx.x; gi < a.range_groups; gi += kGnThreads) {
    float total = 0.0f, s = 0.0f, q = 0.0f, mu = own[gi].x;
    if (a.blocks > 1) {
      for (int k = 0; k < a.blocks; ++k) {
        const float w = static_cast<float>(
            max(int64_t{0}, min(a.pixels, (k + 1) * share) - k * share));
        const float2 o = *cluster.map_shared_rank(own + gi, k);
        total += w;
        if (w > 0.0f) s += w * o.x;
      }
      mu = s / total;
    }
    for (int k = 0; k < a.blocks; ++k) {
      const float w = static_cast<float>(
          max(int64_t{0}, min(a.pixels, (k + 1) * share) - k * share));
      if (w == 0.0f) continue;
      const float2 o = a.blocks > 1 ? *cluster.map_shared_rank(own + gi, k) : own[gi];
      const float d = o.x - mu;
      q += o.y + w * static_cast<float>(r.group_channels) * d * d;
    }
    const float size = static_cast<float>(a.pixels) * static_cast<float>(r.group_channels);
    stat[gi] = make_float2(mu, 1.0f / sqrtf(q / size + a.eps));
  }
  if (a.blocks > 1) {
    cluster.sync();  // no block leaves while another reads its statistics
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int gi = (c + e - r.c0) / r.group_channels;
    const float2 st = works && c + e < a.c ? stat[gi] : make_float2(0.0f, 0.0f);
    g[e] *= st.y;
    b[e] = fmaf(-st.x, g[e], b[e]);  // the mean goes into the addend
  }
  with_activation(a.act, [&](auto act) {
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      float f[V];
      item(i, f);
      finish_item<YT, V, decltype(act)::value>(a, f, g, b,
                                               p0 + row + static_cast<int64_t>(i) * r.rows, c);
    }
  });
}

// Statistics of one block of pixels of an image and channel range.
template <int XT, int V>
__global__ void __launch_bounds__(kGnThreads, 2) group_norm_stats_kernel(const GroupNormArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  float* scratch = reinterpret_cast<float*>(smem);
  float2* own = reinterpret_cast<float2*>(scratch + (2 * V + 2) * kGnThreads);
  const int block = blockIdx.x % a.blocks;
  const int64_t unit = blockIdx.x / a.blocks;
  const int range = a.first_range + static_cast<int>(unit % a.launch_ranges);
  const int64_t image = a.first_image + unit / a.launch_ranges;
  const Range r(a, range, V);
  const int all = (r.channels + V - 1) / V;  // padding channels have no statistics
  const int cols = min(all, kGnThreads), rows = kGnThreads / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const int64_t share = (a.pixels + a.blocks - 1) / a.blocks;
  const int64_t from = block * share;
  const int64_t count = max(int64_t{0}, min(a.pixels, from + share) - from);
  const int64_t p0 = image * a.pixels + from;
  Running<V> run;
  // more columns than threads: the range is one group
  for (int at = col; row < rows && at < all; at += cols) {
    const int c = r.c0 + at * V;
    for (int64_t p = row; p < count; p += kGnBatch * rows) {
      const int64_t left = (count - p + rows - 1) / rows;
      const int k = left < kGnBatch ? static_cast<int>(left) : kGnBatch;
      Item<XT, V> it[kGnBatch];
#pragma unroll
      for (int e = 0; e < kGnBatch; ++e) {
        if (e < k) {
          it[e] = load_item<XT, V>(a.x, channel_at<XT>(p0 + p + int64_t{e} * rows, a.c_store, c),
                                   a.c_store);
        }
      }
      run.template add<kGnBatch>(k, [&](int e, float(&f)[V]) { item_floats<XT, V>(it[e], f); });
    }
  }
  join_threads<V>(run, cols, rows, all > cols ? cols * V : r.group_channels, a.range_groups,
                  scratch, own);
  for (int g = threadIdx.x; g < a.range_groups; g += kGnThreads) {
    a.partial[(unit * a.blocks + block) * a.range_groups + g] = own[g];
  }
}

// Joins the blocks' statistics (every block of the launch for itself) and
// normalizes.  Blocks run over the pixels from the end, which L2 still holds.
template <int XT, int YT, int V>
__global__ void __launch_bounds__(kGnThreads, 2) group_norm_apply_kernel(const GroupNormArgs a,
                                                                      int apply_blocks) {
  extern __shared__ __align__(16) uint8_t smem[];
  float2* stat = reinterpret_cast<float2*>(smem);
  const int block = apply_blocks - 1 - static_cast<int>(blockIdx.x % apply_blocks);
  const int64_t unit = blockIdx.x / apply_blocks;
  const int range = a.first_range + static_cast<int>(unit % a.launch_ranges);
  const int64_t image = a.first_image + unit / a.launch_ranges;
  const Range r(a, range, V);
  const int64_t part = (a.pixels + a.blocks - 1) / a.blocks;
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < a.range_groups; g += kGnThreads / 32) {
    const float2* p = a.partial + unit * a.blocks * a.range_groups + g;
    float s = 0.0f, q = 0.0f;
    for (int k = lane; k < a.blocks; k += 32) {
      const float w =
          static_cast<float>(max(int64_t{0}, min(a.pixels, (k + 1) * part) - k * part));
      if (w > 0.0f) s += w * p[k * a.range_groups].x;
    }
    const float mu = warp_sum(s) / static_cast<float>(a.pixels);
    for (int k = lane; k < a.blocks; k += 32) {
      const float w =
          static_cast<float>(max(int64_t{0}, min(a.pixels, (k + 1) * part) - k * part));
      if (w == 0.0f) continue;
      const float2 o = p[k * a.range_groups];
      const float d = o.x - mu;
      q += o.y + w * static_cast<float>(r.group_channels) * d * d;
    }
    q = warp_sum(q);
    const float size = static_cast<float>(a.pixels) * static_cast<float>(r.group_channels);
    if (lane == 0) stat[g] = make_float2(mu, 1.0f / sqrtf(q / size + a.eps));
  }
  __syncthreads();
  const int64_t share = (a.pixels + apply_blocks - 1) / apply_blocks;
  const int64_t from = block * share;
  const int64_t count = max(int64_t{0}, min(a.pixels, from + share) - from);
  const int64_t p0 = image * a.pixels + from;
  // padding channels may make the last range wider than the block
  for (int col0 = 0; col0 < r.cols; col0 += kGnThreads) {
    const int cols = min(r.cols - col0, kGnThreads), rows = kGnThreads / cols;
    const int col = col0 + threadIdx.x % cols, row = threadIdx.x / cols;
    if (row >= rows) continue;
    const int c = r.c0 + col * V;
    float mul[V], add[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      mul[e] = add[e] = 0.0f;
      if (c + e < a.c) {
        const float2 st = stat[(c + e - r.c0) / r.group_channels];
        mul[e] = a.gamma == nullptr ? st.y : st.y * a.gamma[c + e];
        // the mean goes into the addend
        add[e] = fmaf(-st.x, mul[e], a.beta == nullptr ? 0.0f : a.beta[c + e]);
      }
    }
    constexpr int K = XT == IE_DT_BF16X2 ? 2 : 4;
    with_activation(a.act, [&](auto act) {
      for (int64_t p = row; p < count; p += K * rows) {
        Item<XT, V> it[K];
#pragma unroll
        for (int e = 0; e < K; ++e) {
          if (p + int64_t{e} * rows < count) {
            it[e] = load_item<XT, V>(a.x, channel_at<XT>(p0 + p + int64_t{e} * rows, a.c_store, c),
                                     a.c_store);
          }
        }
#pragma unroll
        for (int e = 0; e < K; ++e) {
          if (p + int64_t{e} * rows >= count) break;
          float f[V];
          item_floats<XT, V>(it[e], f);
          finish_item<YT, V, decltype(act)::value>(a, f, mul, add, p0 + p + int64_t{e} * rows, c);
        }
      }
    });
  }
}

}  // namespace ie_cuda
