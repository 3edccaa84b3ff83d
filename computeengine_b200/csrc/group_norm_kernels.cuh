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
// memory of one block or a cluster of up to 8, so x is read once.
// group_norm_stats_kernel, group_norm_apply_kernel: for images that do not fit.
// 32 x 56 x 56 x 256 fp32 (held): 59 us, 3.5 TB/s of x and y; 512 x 512 x 128
// bf16 (read twice): 50 us, 2.7 TB/s of x and y, 4.0 TB/s with the second read.
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
  int blocks;           // pixel blocks per image and range
  int share;            // pixels of a block
  int parts, part_share;  // two-kernel path: clusters of blocks, and their pixels
  int cols[2], rows[2]; // threads over a range's vectors and pixels: inner, last range
  float2* partial;      // two-kernel path: mean and sum of squared differences,
                        // [image][range][range_groups][part]
};

constexpr int kGnThreads = 256;
constexpr int kGnBatch = 4;  // pixels per exact mean
constexpr int kGnCluster = 4;  // blocks of the statistics kernel joined before memory

// Kinds of activation: a clamp to [low, high] (none, ReLU, ReLU6), SiLU, GELU.
enum { kActClamp = 0, kActSilu = 1, kActGelu = 2 };

// 1 / x for 1 <= x, 0 from 2^126 on.
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int ACT, int V>
__device__ __forceinline__ void activate(float (&v)[V], float low, float high) {
  if constexpr (ACT == kActClamp) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(v[e]) : "f"(v[e]), "f"(low));  // NaN stays
      asm("min.NaN.f32 %0, %1, %2;" : "=f"(v[e]) : "f"(v[e]), "f"(high));
    }
  } else if constexpr (ACT == kActSilu) {
    // v / (1 + 2^(-v log2 e)) on the special function unit, within a few steps
    // of fp32.  It takes 16 results a cycle and SM, which exponential and
    // reciprocal for each value would make the bound; so two values share the
    // reciprocal of their denominators' product, where that has a normal one.
    // Where it has not, each takes its own: a NaN stays in its channel, and far
    // below zero v / infinity is 0.
    constexpr float kNormal = 0x1p126f;
    float d[V];
    bool shared = true;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float x;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x) : "f"(v[e] * -1.4426950408889634f));
      d[e] = 1.0f + x;
      if (e % 2 == 1) shared = shared && d[e - 1] * d[e] <= kNormal;
    }
    if (V % 2 == 1) shared = shared && d[V - 1] <= kNormal;
    if (shared) {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float other = e + 1 < V ? d[e + 1] : 1.0f;
        const float r = reciprocal(d[e] * other);
        v[e] *= r * other;
        if (e + 1 < V) v[e + 1] *= r * d[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= reciprocal(d[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.5f * v[e] * (1.0f + erff(v[e] * 0.70710678118654752f));
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

// Two fp32 values in one register pair, two operations per instruction (sm_100).
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 floats_of(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// V channels as pairs; V == 1: the second of the one pair is zero.
template <int V>
struct Pairs {
  static constexpr int kCount = (V + 1) / 2;
  uint64_t p[kCount];

  __device__ __forceinline__ float operator[](int e) const {
    const float2 f = floats_of(p[e / 2]);
    return e % 2 == 0 ? f.x : f.y;
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) p[i] = pair_of(f[2 * i], 2 * i + 1 < V ? f[2 * i + 1] : 0.0f);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kCount; ++i) p[i] = 0;
  }
  __device__ __forceinline__ void add(const Pairs& o) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) p[i] = add2(p[i], o.p[i]);
  }
  __device__ __forceinline__ void add_squares(const Pairs& o, const Pairs& minus) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const uint64_t d = add2(o.p[i], minus.p[i]);
      p[i] = fma2(d, d, p[i]);
    }
  }
};

template <int T, int V>
__device__ __forceinline__ Pairs<V> item_pairs(const Item<T, V>& i) {
  Pairs<V> r;
  if constexpr (V == 1) {
    float f[1];
    to_floats<T == IE_DT_BF16X2 ? static_cast<int>(IE_DT_BF16) : T, 1>(i.v, f);
    if constexpr (T == IE_DT_BF16X2) {
      float l[1];
      to_floats<IE_DT_BF16, 1>(i.lo, l);
      f[0] += l[0];
    }
    r.set(f);
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      if constexpr (T == IE_DT_F32) {
        r.p[k] = pair_of(__uint_as_float(i.v.r[2 * k]), __uint_as_float(i.v.r[2 * k + 1]));
      } else {
        const float2 f = unpack_pair<T>(i.v.r[k]);
        r.p[k] = pair_of(f.x, f.y);
        if constexpr (T == IE_DT_BF16X2) {
          const float2 l = unpack_pair<T>(i.lo.r[k]);
          r.p[k] = add2(r.p[k], pair_of(l.x, l.y));
        }
      }
    }
  }
  return r;
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
  Pairs<V> mean, m2;
  int n = 0;

  __device__ __forceinline__ Running() {
    mean.zero();
    m2.zero();
  }
  // Joins k > 0 pixels of the given mean and squares about it.
  __device__ __forceinline__ void join(int k, const Pairs<V>& batch, const Pairs<V>& squares) {
    if (n == 0) {
      mean = batch;
      m2 = squares;
    } else {
      const float share = static_cast<float>(k) / static_cast<float>(n + k);
      const float weight = static_cast<float>(n) * share;
      const uint64_t share2 = pair_of(share, share), weight2 = pair_of(weight, weight);
      const uint64_t minus1 = pair_of(-1.0f, -1.0f);
#pragma unroll
      for (int i = 0; i < Pairs<V>::kCount; ++i) {
        const uint64_t d = fma2(mean.p[i], minus1, batch.p[i]);
        mean.p[i] = fma2(d, share2, mean.p[i]);
        m2.p[i] = add2(m2.p[i], fma2(mul2(d, d), weight2, squares.p[i]));
      }
    }
    n += k;
  }
  // A whole batch in registers.
  __device__ __forceinline__ void add(const Pairs<V> (&f)[kGnBatch]) {
    Pairs<V> s = f[0], q, minus;
#pragma unroll
    for (int i = 1; i < kGnBatch; ++i) s.add(f[i]);
    const uint64_t inv = pair_of(1.0f / kGnBatch, 1.0f / kGnBatch);
    const uint64_t minus_inv = pair_of(-1.0f / kGnBatch, -1.0f / kGnBatch);
#pragma unroll
    for (int i = 0; i < Pairs<V>::kCount; ++i) {
      minus.p[i] = mul2(s.p[i], minus_inv);
      s.p[i] = mul2(s.p[i], inv);
    }
    q.zero();
#pragma unroll
    for (int i = 0; i < kGnBatch; ++i) q.add_squares(f[i], minus);
    join(kGnBatch, s, q);
  }
  // One pixel.
  __device__ __forceinline__ void add(const Pairs<V>& f) {
    Pairs<V> q;
    q.zero();
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
__device__ __forceinline__ void group_sums(const Pairs<V>& v, int cols, int rows,
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
                                               const float2* stat, Pairs<V>* mul_pairs,
                                               Pairs<V>* add_pairs) {
  float mul[V], add[V];
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
  mul_pairs->set(mul);
  add_pairs->set(add);
}

// Normalizes, activates and stores one item; channels past c are zero before
// the activation already (mul and add are zero there, but x may hold anything).
template <int YT, int V, int ACT>
__device__ __forceinline__ void finish_item(const GroupNormArgs& a, const Pairs<V>& x,
                                            const Pairs<V>& mul, const Pairs<V>& add, uint8_t* y,
                                            int valid) {
  float f[V];
#pragma unroll
  for (int i = 0; i < Pairs<V>::kCount; ++i) {
    const float2 r = floats_of(fma2(x.p[i], mul.p[i], add.p[i]));
    f[2 * i] = r.x;
    if (2 * i + 1 < V) f[2 * i + 1] = r.y;
  }
  if (valid < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < valid ? f[e] : 0.0f;
  }
  activate<ACT, V>(f, a.low, a.high);
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

  auto item = [&](int i) {
    Item<XT, V> it;
    it.v = load_bytes<16>(mine + i * kStep);
    if constexpr (XT == IE_DT_BF16X2) it.lo = load_bytes<16>(mine + i * kStep + kGnThreads * 16);
    return item_pairs<XT, V>(it);
  };
  // the block's mean of each group, then the squares about it
  Pairs<V> v;
  v.zero();
#pragma unroll 4
  for (int i = 0; i < n; ++i) v.add(item(i));
  group_sums<V>(v, r.cols, r.rows, r.group_channels, a.range_groups, scratch, sums);
  const float inv = 1.0f / (static_cast<float>(count) * static_cast<float>(r.group_channels));
  {
    float minus[V];
    int g = first, in_group = inner;
#pragma unroll
    for (int e = 0; e < V; ++e) {  // padding channels: the group's that would follow
      minus[e] = -sums[min(g, a.range_groups - 1)] * inv;
      if (++in_group == r.group_channels) {
        in_group = 0;
        ++g;
      }
    }
    Pairs<V> minus_pairs;
    minus_pairs.set(minus);
    v.zero();
#pragma unroll 4
    for (int i = 0; i < n; ++i) v.add_squares(item(i), minus_pairs);
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
  Pairs<V> g, b;
  if (n > 0) channel_affine<V>(a, c, first, inner, stat, &g, &b);
  uint8_t* y = static_cast<uint8_t*>(a.y) +
               channel_at<YT>(p0 + row, a.c_store, c) * element_bytes(YT);
  const int64_t y_step = static_cast<int64_t>(r.rows) * channel_at<YT>(1, a.c_store, 0) *
                         element_bytes(YT);
#pragma unroll(ACT == kActGelu ? 1 : 2)
  for (int i = 0; i < n; ++i, y += y_step) {
    finish_item<YT, V, ACT>(a, item(i), g, b, y, a.c - c);
  }
  if (a.blocks > 1) cluster.barrier_wait();
}

// Statistics of one block of pixels of an image and channel range.
template <int XT, int V>
__global__ void __launch_bounds__(kGnThreads, 2) group_norm_stats_kernel(const GroupNormArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem[];
  float2* own = reinterpret_cast<float2*>(smem);  // [range_groups] of this block
  float* sums = reinterpret_cast<float*>(own + a.range_groups);  // [range_groups]
  float* scratch = sums + a.range_groups;
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(a.blocks);
  const int block = static_cast<int>(blockIdx.x - unit * a.blocks);
  const int64_t image = unit / static_cast<uint32_t>(a.ranges);
  const int range = static_cast<int>(unit - image * a.ranges);
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
    constexpr int K = XT == IE_DT_BF16X2 ? 2 : 4;  // batches in flight
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
        Pairs<V> f[kGnBatch];
#pragma unroll
        for (int e = 0; e < kGnBatch; ++e) f[e] = item_pairs<XT, V>(it[k * kGnBatch + e]);
        run.add(f);
      }
    }
    for (; left > 0; --left, from_x += step) {
      run.add(item_pairs<XT, V>(load_item<XT, V>(a.x, from_x, a.c_store)));
    }
  }
  // the second kernel may be launched; it waits for this one's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the block's mean of each group, then each channel's squares about it
  const int group_channels = all > cols ? cols * V : r.group_channels;
  Pairs<V> sum = run.mean;
  const uint64_t seen = pair_of(static_cast<float>(run.n), static_cast<float>(run.n));
#pragma unroll
  for (int i = 0; i < Pairs<V>::kCount; ++i) sum.p[i] = mul2(sum.p[i], seen);
  group_sums<V>(sum, cols, rows, group_channels, a.range_groups, scratch, sums);
  const float inv = 1.0f / (static_cast<float>(count) * static_cast<float>(r.group_channels));
  int g = col * V / group_channels, inner = col * V - g * group_channels;
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float d = run.mean[e] - sums[min(g, a.range_groups - 1)] * inv;
    v[e] = run.n > 0 ? fmaf(d * d, static_cast<float>(run.n), run.m2[e]) : 0.0f;
    if (++inner == group_channels) {
      inner = 0;
      ++g;
    }
  }
  for (int i = threadIdx.x; i < a.range_groups; i += kGnThreads) own[i].x = sums[i] * inv;
  __syncthreads();
  sum.set(v);
  group_sums<V>(sum, cols, rows, group_channels, a.range_groups, scratch, sums);
  for (int i = threadIdx.x; i < a.range_groups; i += kGnThreads) own[i].y = sums[i];
  // A cluster's blocks are joined here, so that the second kernel's blocks,
  // which each join them all, find few parts: [unit][group][part].
  cg::cluster_group cluster = cg::this_cluster();
  const int size = static_cast<int>(cluster.num_blocks());
  cluster.sync();
  const int part = block / size, first_pixel = part * a.part_share;
  const int pixels = min(a.pixels, first_pixel + a.part_share) - first_pixel;
  for (int i = static_cast<int>(cluster.block_rank()) * kGnThreads + threadIdx.x;
       i < a.range_groups; i += kGnThreads * size) {
    float s = 0.0f, q = 0.0f;
    float2 o[kGnCluster];
#pragma unroll
    for (int k = 0; k < kGnCluster; ++k) {
      o[k] = k < size ? *cluster.map_shared_rank(own + i, k) : make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 0; k < kGnCluster; ++k) {
      const int w = min(pixels, (k + 1) * a.share) - k * a.share;
      if (k < size && w > 0) s += static_cast<float>(w) * o[k].x;
    }
    const float mu = s / static_cast<float>(pixels);
#pragma unroll
    for (int k = 0; k < kGnCluster; ++k) {
      const int w = min(pixels, (k + 1) * a.share) - k * a.share;
      const float d = o[k].x - mu;
      if (k < size && w > 0) {
        q += o[k].y + static_cast<float>(w) * static_cast<float>(r.group_channels) * d * d;
      }
    }
    a.partial[(static_cast<int64_t>(unit) * a.range_groups + i) * a.parts + part] =
        make_float2(mu, q);
  }
  cluster.sync();  // no block leaves while another reads its statistics
}

// Joins the blocks' statistics (every block of the launch for itself) and
// normalizes.  Every block runs over its pixels from their end: the statistics
// kernel's blocks, all on the GPU at once, read the ends last, so L2 holds them.
template <int XT, int YT, int V, int ACT>
__global__ void __launch_bounds__(kGnThreads, V == 8 && XT == IE_DT_BF16X2 ? 2 : 4)
    group_norm_apply_kernel(const GroupNormArgs a,
                                                                      int apply_blocks) {
  extern __shared__ __align__(16) uint8_t smem[];
  float2* stat = reinterpret_cast<float2*>(smem);
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(apply_blocks);
  const int block = static_cast<int>(blockIdx.x - unit * apply_blocks);
  const int64_t image = unit / static_cast<uint32_t>(a.ranges);
  const int range = static_cast<int>(unit - image * a.ranges);
  const Range r(a, range);
  const int lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // until the statistics are written
  for (int g = threadIdx.x >> 5; g < a.range_groups; g += kGnThreads / 32) {
    const float2* p = a.partial + (static_cast<int64_t>(unit) * a.range_groups + g) * a.parts;
    // up to 64 parts stay in registers between the mean and the squares
    const float2 mine[2] = {lane < a.parts ? p[lane] : make_float2(0.0f, 0.0f),
                            lane + 32 < a.parts ? p[lane + 32] : make_float2(0.0f, 0.0f)};
    auto pixels_of = [&](int k) {
      return static_cast<float>(max(0, min(a.pixels, (k + 1) * a.part_share) - k * a.part_share));
    };
    float s = 0.0f, q = 0.0f;
    for (int k = lane, i = 0; k < a.parts; k += 32, ++i) {
      if (pixels_of(k) > 0.0f) s += pixels_of(k) * (i == 0 ? mine[0] : i == 1 ? mine[1] : p[k]).x;
    }
    const float mu = warp_sum(s) / static_cast<float>(a.pixels);
    for (int k = lane, i = 0; k < a.parts; k += 32, ++i) {
      const float2 o = i == 0 ? mine[0] : i == 1 ? mine[1] : p[k];
      const float d = o.x - mu;
      if (pixels_of(k) > 0.0f) {
        q += o.y + pixels_of(k) * static_cast<float>(r.group_channels) * d * d;
      }
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
    Pairs<V> mul, add;
    channel_affine<V>(a, c, first, col * V - first * r.group_channels, stat, &mul, &add);
    constexpr int K = ACT == kActGelu || XT == IE_DT_BF16X2 ? 2 : 4;
    const int64_t x_step = -static_cast<int64_t>(rows) * channel_at<XT>(1, a.c_store, 0);
    const int64_t y_step = -static_cast<int64_t>(rows) * channel_at<YT>(1, a.c_store, 0) *
                           element_bytes(YT);
    const int64_t last = p0 + count - 1 - row;
    int64_t from_x = channel_at<XT>(last, a.c_store, c);
    uint8_t* y = static_cast<uint8_t*>(a.y) + channel_at<YT>(last, a.c_store, c) * element_bytes(YT);
    int left = (count - row + rows - 1) / rows;
    for (; left >= K; left -= K) {
      Item<XT, V> it[K];
#pragma unroll
      for (int e = 0; e < K; ++e, from_x += x_step) {
        it[e] = load_item<XT, V>(a.x, from_x, a.c_store);
      }
#pragma unroll
      for (int e = 0; e < K; ++e, y += y_step) {
        finish_item<YT, V, ACT>(a, item_pairs<XT, V>(it[e]), mul, add, y, a.c - c);
      }
    }
    for (; left > 0; --left, from_x += x_step, y += y_step) {
      finish_item<YT, V, ACT>(a, item_pairs<XT, V>(load_item<XT, V>(a.x, from_x, a.c_store)), mul,
                              add, y, a.c - c);
    }
  }
}

}  // namespace ie_cuda
