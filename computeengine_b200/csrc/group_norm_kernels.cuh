// Group normalization with an activation over channels-last tensors.
//
// A thread owns V neighbouring channels (one 16-byte load of x) and strides
// over the pixels, so everything it does is per channel and a group may begin
// and end anywhere in a vector.  Statistics: a thread takes each channel's mean, and
// the squares about it, from differences to a pixel or to the mean so far; threads,
// then blocks are joined by the differences of their means to one value of the group
// (its first channel at the image's first pixel) and the squares about their mean
// (Chan, Golub and LeVeque 1979), all in fp32 and in a fixed order.  The mean, kept as
// two numbers, is subtracted before the scale.  So errors follow the spread, however
// far the mean is from zero, and results do not depend on timing.
//
// group_norm_cluster_kernel: a channel range of an image is held in the shared
// memory of one block or a cluster of up to 8, so x is read once.
// group_norm_stats_kernel, group_norm_apply_kernel: for images that do not fit.
// 32 x 56 x 56 x 256 fp32 (held): 56 us, 3.7 TB/s of x and y; 512 x 512 x 128
// bf16 (read twice): 53 us, 2.5 TB/s of x and y, 3.8 TB/s with the second read.
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
  float4* partial;      // two-kernel path: [image][range][range_groups][part]
};

constexpr int kGnThreads = 256;
constexpr int kGnBatch = 4;    // a thread's pixels, at least, in a statistics block
constexpr int kGnCluster = 4;  // blocks of the statistics kernel joined before memory

// Kinds of activation: a clamp to [low, high] (none, ReLU, ReLU6), SiLU, GELU.
enum { kActClamp = 0, kActSilu = 1, kActGelu = 2 };

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
  __device__ __forceinline__ Pairs plus(const Pairs& o) const {
    Pairs r;
#pragma unroll
    for (int i = 0; i < kCount; ++i) r.p[i] = add2(p[i], o.p[i]);
    return r;
  }
  __device__ __forceinline__ Pairs times(float f) const {
    Pairs r;
    const uint64_t f2 = pair_of(f, f);
#pragma unroll
    for (int i = 0; i < kCount; ++i) r.p[i] = mul2(p[i], f2);
    return r;
  }
  __device__ __forceinline__ void add_product(const Pairs& a, const Pairs& b) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) p[i] = fma2(a.p[i], b.p[i], p[i]);
  }
  __device__ __forceinline__ void add_squares(const Pairs& d) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) p[i] = fma2(d.p[i], d.p[i], p[i]);
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

// Running statistics of V channels over the pixels a thread has seen: the mean is
// pivot + rest, and pivot moves with it, so that sums of a batch's differences to it
// and of their squares lose no more than the squares of the means' differences.
template <int V>
struct Running {
  Pairs<V> pivot, rest, m2, m2_rest;
  int n = 0;

  __device__ __forceinline__ Running() {
    pivot.zero();
    rest.zero();
    m2.zero();
    m2_rest.zero();
  }
  // The next K pixels, the k-th of them at(k).
  template <int K, class At>
  __device__ __forceinline__ void add(const At& at) {
    if (n == 0) pivot = at(0);
    const Pairs<V> minus = pivot.times(-1.0f);
    Pairs<V> sum, squares;
    sum.zero();
    squares.zero();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Pairs<V> d = at(k).plus(minus);
      sum.add(d);
      squares.add_squares(d);
    }
    const float share = static_cast<float>(K) / static_cast<float>(n + K);
    const float weight = static_cast<float>(n) * share;
    const uint64_t share2 = pair_of(share, share), weight2 = pair_of(weight, weight);
    const uint64_t inv = pair_of(1.0f / K, 1.0f / K), minus1 = pair_of(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < Pairs<V>::kCount; ++i) {
      const uint64_t mean = mul2(sum.p[i], inv);  // of the batch, as difference to pivot
      const uint64_t d = fma2(rest.p[i], minus1, mean);
      const uint64_t about_mean = fma2(mul2(sum.p[i], minus1), mean, squares.p[i]);
      // what the running sum of squares cuts off each time goes into the next term
      const uint64_t term = add2(fma2(mul2(d, d), weight2, about_mean), m2_rest.p[i]);
      const uint64_t total = add2(m2.p[i], term);
      m2_rest.p[i] = add2(fma2(total, minus1, m2.p[i]), term);
      m2.p[i] = total;
      const uint64_t moved = fma2(d, share2, rest.p[i]);
      const uint64_t to = add2(pivot.p[i], moved);
      rest.p[i] = add2(fma2(to, minus1, pivot.p[i]), moved);
      pivot.p[i] = to;
    }
    n += K;
  }
  // The mean as difference to `base`.
  __device__ __forceinline__ Pairs<V> mean(const Pairs<V>& base) const {
    return pivot.plus(base.times(-1.0f)).plus(rest);
  }
};

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// A group's statistics: mean + rest is its mean (below the last join, `mean` is the
// value that differences are taken to), squares the sum of squares about it.
struct Stat {
  float mean, rest, squares;
};

// The same with `mean` the mean rounded, and 1 / sigma in the place of the squares.
__device__ __forceinline__ Stat finished(const Stat& s, float size, float eps) {
  const float mean = s.mean + s.rest;
  const float back = mean - s.mean;  // what of rest went into mean; the rest is exact
  const float squares = s.squares < 0.0f ? 0.0f : s.squares;  // a rounding below; NaN stays
  return {mean, (s.mean - (mean - back)) + (s.rest - back), 1.0f / sqrtf(squares / size + eps)};
}

// Block-wide joins of what each thread holds of V channels: thread t has the
// channels (t % cols) * V .. of the range, rows = threads per column, whose `count`
// pixels are dealt to the rows in turn.  First slices of the rows of each channel are
// joined by all threads, then a warp joins a group.  scratch holds (V + 2) * threads
// floats, 16-byte aligned.  Everything that needs a division is made before the data.
template <int V>
struct Columns {
  int cols, rows, width, count;
  int all;             // columns of the range; more than cols: it is a single group
  int group_channels;  // of the columns held (all > cols: all of them)
  int groups;
  bool wide;           // threads own channels, not slices of them
  int slices, slice, channel;  // of rows; this thread's
  int shift;           // lanes over a group's channels; the others over slices
  int each, extra;     // pixels of row k: each + (k < extra)
  float inv_size, inv_slices, inv_pixels;  // of a group, and of this thread's slice

  __device__ __forceinline__ Columns(int cols, int rows, int all, int count, int group_channels,
                                     int groups, float size)
      : cols(cols), rows(rows), width(cols * V), count(count), all(all),
        group_channels(group_channels), groups(groups), inv_size(1.0f / size) {
    const int t = threadIdx.x;
    wide = width >= kGnThreads;
    slices = wide ? 1 : kGnThreads / width;
    slice = wide ? 0 : t / width;
    channel = t - slice * width;
    shift = 0;
    while ((1 << shift) < group_channels && shift < 5) ++shift;
    each = count / rows;
    extra = count - each * rows;
    inv_slices = 1.0f / static_cast<float>(slices);
    const float p = pixels(slice);
    inv_pixels = p > 0.0f ? 1.0f / p : 0.0f;
  }
  // ceil(v / slices) of -slices < v <= 256
  __device__ __forceinline__ float per_slice(int v) const {
    return ceilf((static_cast<float>(v) - 0.5f) * inv_slices);
  }
  __device__ __forceinline__ float pixels(int k) const {  // of slice k
    return static_cast<float>(each) * per_slice(rows - k) + fmaxf(per_slice(extra - k), 0.0f);
  }
};

template <int V>
__device__ __forceinline__ void put_channels(const Pairs<V>& v, const Columns<V>& c,
                                             float* scratch) {
  const int t = threadIdx.x;
  if (t >= c.cols * c.rows) return;  // [rows][width]
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const float2 lo = floats_of(v.p[e / 2]), hi = floats_of(v.p[e / 2 + 1]);
      *reinterpret_cast<float4*>(scratch + t * V + e) = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) scratch[t * V + e] = v[e];
  }
}

// Joins each thread's means (0 where it has no pixel) and squares into stat[g].rest and
// stat[g].squares.
template <int V>
__device__ __forceinline__ void join_threads(const Pairs<V>& mean, const Pairs<V>& squares,
                                             const Columns<V>& c, float* scratch, Stat* stat) {
  const int t = threadIdx.x, lane = t & 31;
  put_channels<V>(mean, c, scratch);
  __syncthreads();
  // The slice's rows of a channel, about the first of them: the squares about it are
  // at most as many times those about their mean as there are rows, below 2 V.
  auto join_rows = [&](int ch) {
    const float first = scratch[c.slice * c.width + ch];
    float s = 0.0f, q = 0.0f;
#pragma unroll 4
    for (int k = c.slice; k < c.rows; k += c.slices) {
      const float w = static_cast<float>(c.each + (k < c.extra ? 1 : 0));
      const float d = scratch[k * c.width + ch] - first, wd = w * d;
      s += wd;
      q = fmaf(wd, d, q);
    }
    const float m = s * c.inv_pixels;
    return make_float2(first + m, q - s * m);
  };
  auto sum_rows = [&](int ch) {
    float s = 0.0f;
#pragma unroll 4
    for (int k = c.slice; k < c.rows; k += c.slices) s += scratch[k * c.width + ch];
    return s;
  };
  float* part_mean = scratch;  // [slices][width], and the squares
  float* part_squares = scratch + c.width;
  if (c.wide) {  // over a channel's first two rows
    for (int ch = t; ch < c.width; ch += kGnThreads) {
      const float2 r = join_rows(ch);
      part_mean[ch] = r.x;
      if (c.rows > 1) part_squares[ch] = r.y;
    }
  } else {
    part_mean = scratch + V * kGnThreads;
    part_squares = part_mean + kGnThreads;
    float2 r = make_float2(0.0f, 0.0f);
    if (c.slice < c.slices) r = join_rows(c.channel);
    __syncthreads();
    put_channels<V>(squares, c, scratch);
    __syncthreads();
    if (c.slice < c.slices) {
      part_mean[t] = r.x;
      part_squares[t] = r.y + sum_rows(c.channel);
    }
  }
  __syncthreads();
  const int shift = c.shift, lanes = 1 << shift, ch0 = lane & (lanes - 1);
  // pixels of a slice (all > cols: of a thread's columns)
  auto weight = [&](int k, int ch) {
    if (c.all <= c.cols) return c.pixels(k);
    return static_cast<float>(c.count * ((c.all - ch / V + c.cols - 1) / c.cols));
  };
  for (int g = t >> 5; g < c.groups; g += kGnThreads / 32) {
    const float first = part_mean[g * c.group_channels];
    float s = 0.0f, q = 0.0f;
    for (int k = lane >> shift; k < c.slices; k += 32 >> shift) {
      const int row = k * c.width + g * c.group_channels;
      float w = weight(k, 0);
      for (int ch = ch0; ch < c.group_channels; ch += lanes) {
        if (c.all > c.cols) w = weight(k, ch);
        s = fmaf(w, part_mean[row + ch] - first, s);
        if (!c.wide || c.rows > 1) q += part_squares[row + ch];
      }
    }
    const float m = warp_sum(s) * c.inv_size;
    for (int k = lane >> shift; k < c.slices; k += 32 >> shift) {
      const int row = k * c.width + g * c.group_channels;
      float w = weight(k, 0);
      for (int ch = ch0; ch < c.group_channels; ch += lanes) {
        if (c.all > c.cols) w = weight(k, ch);
        const float d = (part_mean[row + ch] - first) - m;
        q = fmaf(w * d, d, q);
      }
    }
    q = warp_sum(q);
    if (lane == 0) {
      stat[g].rest = first + m;
      stat[g].squares = q;
    }
  }
  __syncthreads();
  if (!c.wide) return;
  put_channels<V>(squares, c, scratch);
  __syncthreads();
  for (int ch = t; ch < c.width; ch += kGnThreads) scratch[ch] = sum_rows(ch);
  __syncthreads();
  for (int g = t >> 5; g < c.groups; g += kGnThreads / 32) {
    float s = 0.0f;
    for (int ch = lane; ch < c.group_channels; ch += 32) s += scratch[g * c.group_channels + ch];
    s = warp_sum(s);
    if (lane == 0) stat[g].squares += s;
  }
  __syncthreads();
}

// Joins the statistics of `blocks` blocks of `share` pixels, all about one value:
// first the means, then the squares about their mean.
template <class At>
__device__ __forceinline__ Stat join_blocks(int blocks, int share, int pixels, int group_channels,
                                            const At& at) {
  auto pixels_of = [&](int k) {
    return static_cast<float>(min(pixels, (k + 1) * share) - k * share);
  };
  float s = 0.0f, q = 0.0f;
  for (int k = 0; k < blocks; ++k) {
    if (pixels_of(k) > 0.0f) s = fmaf(pixels_of(k), at(k).rest, s);
  }
  const float mean = s / static_cast<float>(pixels);
  for (int k = 0; k < blocks; ++k) {
    if (pixels_of(k) > 0.0f) {
      const float d = at(k).rest - mean;
      q += at(k).squares + pixels_of(k) * static_cast<float>(group_channels) * d * d;
    }
  }
  return {at(0).mean, mean, q};
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

// The value of a group that its statistics are about.
template <int XT>
__device__ __forceinline__ float group_base(const GroupNormArgs& a, const Range& r, int64_t image,
                                            int g) {
  const int64_t at = channel_at<XT>(image * a.pixels, a.c_store, r.c0 + g * r.group_channels);
  float v = load_element<XT>(a.x, at);
  if constexpr (XT == IE_DT_BF16X2) v += load_element<XT>(a.x, at + a.c_store);
  return v;
}

// Of the groups of V channels, the first `inner` channels into group g; 0 for padding.
template <int V>
__device__ __forceinline__ Pairs<V> group_bases(const Stat* stat, int groups, int group_channels,
                                                int g, int inner) {
  float base[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    base[e] = g < groups ? stat[g].mean : 0.0f;
    if (++inner == group_channels) {
      inner = 0;
      ++g;
    }
  }
  Pairs<V> p;
  p.set(base);
  return p;
}

// Of the V channels from c: the mean to subtract, gamma / sigma, and beta less the
// share of what the mean lacks.  stat: the range's groups; the thread's first channel
// is `inner` channels into group `first`.
template <int V>
struct Affine {
  Pairs<V> minus, mul, add;
};

template <int V>
__device__ __forceinline__ void channel_affine(const GroupNormArgs& a, int c, int first, int inner,
                                               const Stat* stat, Affine<V>* affine) {
  float minus[V], mul[V], add[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool in = c + e < a.c;
    const Stat st = in ? stat[first] : Stat{0.0f, 0.0f, 0.0f};
    minus[e] = -st.mean;
    mul[e] = in && a.gamma != nullptr ? st.squares * a.gamma[c + e] : st.squares;
    add[e] = fmaf(-st.rest, mul[e], in && a.beta != nullptr ? a.beta[c + e] : 0.0f);
    if (++inner == a.group_channels) {
      inner = 0;
      ++first;
    }
  }
  affine->minus.set(minus);
  affine->mul.set(mul);
  affine->add.set(add);
}

// Normalizes, activates and stores one item; channels past c are zero before
// the activation already (mul and add are zero there, but x may hold anything).
template <int YT, int V, int ACT>
__device__ __forceinline__ void finish_item(const GroupNormArgs& a, const Pairs<V>& x,
                                            const Affine<V>& affine, uint8_t* y, int valid) {
  float f[V];
#pragma unroll
  for (int i = 0; i < Pairs<V>::kCount; ++i) {
    const float2 r = floats_of(
        fma2(add2(x.p[i], affine.minus.p[i]), affine.mul.p[i], affine.add.p[i]));
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
  float* scratch = reinterpret_cast<float*>(smem);
  Stat* own = reinterpret_cast<Stat*>(scratch + (V + 2) * kGnThreads);  // of this block
  Stat* stat = own + a.range_groups;                                    // of the image
  Stat* others = stat + a.range_groups;                                 // [blocks][range_groups]
  uint8_t* items = reinterpret_cast<uint8_t*>(others + a.blocks * a.range_groups);
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
  for (int g = threadIdx.x; g < a.range_groups; g += kGnThreads) {
    own[g].mean = group_base<XT>(a, r, image, g);
  }
  const Columns<V> columns(r.cols, r.rows, r.cols, count, r.group_channels, a.range_groups,
                           static_cast<float>(count) * static_cast<float>(r.group_channels));
  const float inv_n = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
  asm volatile("cp.async.wait_all;" ::: "memory");

  auto item = [&](int i) {
    Item<XT, V> it;
    it.v = load_bytes<16>(mine + i * kStep);
    if constexpr (XT == IE_DT_BF16X2) it.lo = load_bytes<16>(mine + i * kStep + kGnThreads * 16);
    return item_pairs<XT, V>(it);
  };
  // the thread's differences to its first pixel, and their squares (of at most 28
  // pixels, by the shared memory: at most 28 times the squares about their mean)
  __syncthreads();  // the groups' values
  Pairs<V> mean, squares;
  mean.zero();
  squares.zero();
  if (n > 0) {
    const Pairs<V> first_pixel = item(0), minus = first_pixel.times(-1.0f);
#pragma unroll 4
    for (int i = 1; i < n; ++i) {
      const Pairs<V> d = item(i).plus(minus);
      mean.add(d);
      squares.add_squares(d);
    }
    const Pairs<V> sum = mean;
    mean = sum.times(inv_n);
    squares.add_product(sum, mean.times(-1.0f));
    const Pairs<V> base = group_bases<V>(own, a.range_groups, r.group_channels, first, inner);
    mean.add(first_pixel.plus(base.times(-1.0f)));
  }
  join_threads<V>(mean, squares, columns, scratch, own);

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
    Stat all = own[g];
    if (a.blocks > 1) {
      all = join_blocks(a.blocks, a.share, a.pixels, r.group_channels,
                        [&](int k) { return others[k * a.range_groups + g]; });
    }
    stat[g] = finished(all, static_cast<float>(a.pixels) * static_cast<float>(r.group_channels),
                       a.eps);
  }
  __syncthreads();
  Affine<V> affine;
  if (n > 0) channel_affine<V>(a, c, first, inner, stat, &affine);
  uint8_t* y = static_cast<uint8_t*>(a.y) +
               channel_at<YT>(p0 + row, a.c_store, c) * element_bytes(YT);
  const int64_t y_step = static_cast<int64_t>(r.rows) * channel_at<YT>(1, a.c_store, 0) *
                         element_bytes(YT);
#pragma unroll(ACT == kActGelu ? 1 : 2)
  for (int i = 0; i < n; ++i, y += y_step) {
    finish_item<YT, V, ACT>(a, item(i), affine, y, a.c - c);
  }
  if (a.blocks > 1) cluster.barrier_wait();
}

// Statistics of one block of pixels of an image and channel range.
template <int XT, int V>
__global__ void __launch_bounds__(kGnThreads, 2) group_norm_stats_kernel(const GroupNormArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem[];
  float* scratch = reinterpret_cast<float*>(smem);
  Stat* own = reinterpret_cast<Stat*>(scratch + (V + 2) * kGnThreads);  // of this block
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
  // the groups' values are on their way while the pixels are read
  const float own_base =
      threadIdx.x < a.range_groups ? group_base<XT>(a, r, image, threadIdx.x) : 0.0f;
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
      run.template add<K * kGnBatch>([&](int e) { return item_pairs<XT, V>(it[e]); });
    }
    for (; left > 0; --left, from_x += step) {
      const Pairs<V> f = item_pairs<XT, V>(load_item<XT, V>(a.x, from_x, a.c_store));
      run.template add<1>([&](int) { return f; });
    }
  }
  // the second kernel may be launched; it waits for this one's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Columns<V> columns(cols, rows, all, count, all > cols ? cols * V : r.group_channels,
                           a.range_groups,
                           static_cast<float>(count) * static_cast<float>(r.group_channels));
  for (int g = threadIdx.x; g < a.range_groups; g += kGnThreads) {
    own[g].mean = g < kGnThreads ? own_base : group_base<XT>(a, r, image, g);
  }
  __syncthreads();
  Pairs<V> base;
  {
    const int first = all > cols ? 0 : col * V / r.group_channels;
    base = group_bases<V>(own, a.range_groups, r.group_channels, first,
                          col * V - first * r.group_channels);
  }
  Pairs<V> mean = run.mean(base);
  if (run.n == 0) mean.zero();
  join_threads<V>(mean, run.m2, columns, scratch, own);
  // A cluster's blocks are joined here, so that the second kernel's blocks,
  // which each join them all, find few parts: [unit][group][part].
  cg::cluster_group cluster = cg::this_cluster();
  const int size_of_cluster = static_cast<int>(cluster.num_blocks());
  cluster.sync();
  const int part = block / size_of_cluster;
  const int pixels = min(a.pixels, (part + 1) * a.part_share) - part * a.part_share;
  for (int i = static_cast<int>(cluster.block_rank()) * kGnThreads + threadIdx.x;
       i < a.range_groups; i += kGnThreads * size_of_cluster) {
    Stat o[kGnCluster];
#pragma unroll
    for (int k = 0; k < kGnCluster; ++k) {
      o[k] = *cluster.map_shared_rank(own + i, min(k, size_of_cluster - 1));
    }
    Stat part_stat = o[0];
    if (size_of_cluster > 1) {  // kGnCluster
      part_stat = join_blocks(kGnCluster, a.share, pixels, r.group_channels,
                              [&](int k) { return o[k]; });
    }
    a.partial[(static_cast<int64_t>(unit) * a.range_groups + i) * a.parts + part] =
        make_float4(part_stat.mean, part_stat.rest, part_stat.squares, 0.0f);
  }
  cluster.sync();  // no block leaves while another reads its statistics
}

// Joins the blocks' statistics (every block of the launch for itself) and
// normalizes.  Every block runs over its pixels from their end: the statistics
// kernel's blocks, all on the GPU at once, read the ends last, so L2 holds them.
template <int XT, int YT, int V, int ACT>
__global__ void __launch_bounds__(kGnThreads, V == 8 && XT == IE_DT_BF16X2 ? 2 : 4)
    group_norm_apply_kernel(const GroupNormArgs a, int apply_blocks) {
  extern __shared__ __align__(16) uint8_t smem[];
  Stat* stat = reinterpret_cast<Stat*>(smem);
  const uint32_t unit = blockIdx.x / static_cast<uint32_t>(apply_blocks);
  const int block = static_cast<int>(blockIdx.x - unit * apply_blocks);
  const int64_t image = unit / static_cast<uint32_t>(a.ranges);
  const int range = static_cast<int>(unit - image * a.ranges);
  const Range r(a, range);
  const int lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // until the statistics are written
  for (int g = threadIdx.x >> 5; g < a.range_groups; g += kGnThreads / 32) {
    const float4* p = a.partial + (static_cast<int64_t>(unit) * a.range_groups + g) * a.parts;
    // up to 64 parts stay in registers between the means and the squares
    const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4 mine[2] = {lane < a.parts ? p[lane] : none,
                            lane + 32 < a.parts ? p[lane + 32] : none};
    auto part = [&](int k, int i) {
      const float4 v = i == 0 ? mine[0] : i == 1 ? mine[1] : p[k];
      return Stat{v.x, v.y, v.z};
    };
    auto pixels_of = [&](int k) {
      return static_cast<float>(max(0, min(a.pixels, (k + 1) * a.part_share) - k * a.part_share));
    };
    float s = 0.0f, q = 0.0f;
    for (int k = lane, i = 0; k < a.parts; k += 32, ++i) {
      if (pixels_of(k) > 0.0f) s = fmaf(pixels_of(k), part(k, i).rest, s);
    }
    const float mean = warp_sum(s) / static_cast<float>(a.pixels);
    for (int k = lane, i = 0; k < a.parts; k += 32, ++i) {
      const Stat o = part(k, i);
      const float d = o.rest - mean;
      if (pixels_of(k) > 0.0f) {
        q += o.squares + pixels_of(k) * static_cast<float>(r.group_channels) * d * d;
      }
    }
    q = warp_sum(q);
    if (lane == 0) {  // lane 0 holds a part
      const float size = static_cast<float>(a.pixels) * static_cast<float>(r.group_channels);
      stat[g] = finished({mine[0].x, mean, q}, size, a.eps);
    }
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
    Affine<V> affine;
    channel_affine<V>(a, c, first, col * V - first * r.group_channels, stat, &affine);
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
        finish_item<YT, V, ACT>(a, item_pairs<XT, V>(it[e]), affine, y, a.c - c);
      }
    }
    for (; left > 0; --left, from_x += x_step, y += y_step) {
      finish_item<YT, V, ACT>(a, item_pairs<XT, V>(load_item<XT, V>(a.x, from_x, a.c_store)),
                              affine, y, a.c - c);
    }
  }
}

}  // namespace ie_cuda
