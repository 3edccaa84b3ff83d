// Attention for few query rows (single tokens), and for tensors that TMA
// cannot read.
//
// All query heads that read one kv head are columns of one tile, so K and V
// are read once: S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16, keys (and
// then elements of the head) as its 16 rows and eight query rows as its
// columns.  The other way round half of the operand would be empty for up to
// eight rows, and the softmax would run over the empty half too (735 warp
// instructions per 16 keys instead of about 250).  Bound by the memory: a
// block's four warps take keys 16 at a time, each into its own ring of
// asynchronous copies (no barrier between warps), with a running maximum and
// sum per row; long sequences are cut into shares for many blocks.  The warps'
// results are joined in shared memory, the shares' by a second kernel.
// 64 tokens over 1024 keys, 32 heads of 128: 160 us, 6.7 TB/s; one token over
// 65536 keys: 49 us, 5.4 TB/s.
#pragma once

#include "attention_common.cuh"

namespace ie_cuda {

constexpr int kStepThreads = 128;
constexpr int kStepStages = 2;  // three blocks per SM; 3 stages and two blocks: 2% slower
constexpr int kStepKeys = 16;

struct StepArgs : AttentionArgs {
  int tile_rows;    // query positions of a tile
  int tile_heads;   // query heads of a tile; tile_rows * tile_heads <= 8 NT
  int tiles;        // tiles of positions per sequence (documents: upper bound in all)
  int splits;       // shares of each sequence's keys
  float* part_o;    // splits > 1: fp32 [splits][batch][q_heads][q_len][head_dim]
  float* part_lse;  //             fp32 [splits][batch][q_heads][q_len]
};

template <int DP>
struct StepPlan {
  static constexpr int kRow = DP * 2;                              // bytes of a key's row
  static constexpr int kStage = 2 * kStepKeys * kRow;              // K and V of 16 keys
  static constexpr int kSmem = 4 * kStepStages * kStage;
};

template <int T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (T == IE_DT_BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
  } else {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
  }
}

// The transpose of an 8 x 8 matrix of 16-bit elements held across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(v));
  return y;
}

// Byte of 16-byte chunk c of key row r in a tile of rows of DP elements: the
// chunk's place is turned by the row, so eight rows' chunks share no bank.
template <int DP>
__device__ __forceinline__ uint32_t step_at(int r, int c) {
  return static_cast<uint32_t>(r * StepPlan<DP>::kRow + ((c ^ (r & 7)) << 4));
}

// NT: columns / 8.  VEC: K and V in 16-byte aligned rows of a multiple of 8
// elements.
template <int DP, int T, int NT, bool VEC>
__global__ void __launch_bounds__(kStepThreads) attention_step_kernel(const StepArgs a) {
  using P = StepPlan<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float row_m[4][8 * NT], row_l[4][8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads_per_kv = a.q_heads / a.kv_heads;
  const int head_tiles = a.q_heads / a.tile_heads;

  // ---- which rows and keys
  const int h0 = static_cast<int>(blockIdx.x % head_tiles) * a.tile_heads;
  const int64_t rest = blockIdx.x / head_tiles;
  const int tile = a.tiles - 1 - static_cast<int>(rest / a.batch);
  Sequence seq;
  int row0 = 0;
  if (!tile_sequence(a, tile, static_cast<int>(rest % a.batch), a.tile_rows, &seq, &row0)) return;
  const int hk = h0 / heads_per_kv;
  const int positions = min(a.tile_rows, seq.q1 - row0);
  const int rows = a.tile_heads * a.tile_rows;
  const int all = seq.seen(row0 + positions - 1, a.causal);
  const int share = (((all + a.splits - 1) / a.splits) + 63) / 64 * 64;
  const int from = min(all, share * static_cast<int>(blockIdx.y));
  const int to = min(all, from + share);

  const uint16_t* k = static_cast<const uint16_t*>(a.k) + seq.batch * a.k_stride[0] +
                      int64_t{seq.k0} * a.k_stride[1] + hk * a.k_stride[2];
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + seq.batch * a.v_stride[0] +
                      int64_t{seq.k0} * a.v_stride[1] + hk * a.v_stride[2];
  uint8_t* ring = smem + warp * kStepStages * P::kStage;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

  // Copies K and V of the next 16 keys of this warp into a stage; rows past
  // `to` and elements past head_dim are zeros.  A lane copies chunk lane %
  // kChunks of the rows lane / kChunks + i * kRows.
  constexpr int kStride = 4 * kStepKeys;
  constexpr int kChunks = DP / 8, kRows = 32 / kChunks, kCopies = kStepKeys / kRows;
  const int first = from + warp * kStepKeys;
  const int my_row = lane / kChunks, my_chunk = lane % kChunks;
  const bool my_data = my_chunk * 8 < a.head_dim;
  const uint16_t* k_next = k + (my_data ? my_chunk * 8 : 0) + (first + my_row) * a.k_stride[1];
  const uint16_t* v_next = v + (my_data ? my_chunk * 8 : 0) + (first + my_row) * a.v_stride[1];
  const int64_t k_rows = kRows * a.k_stride[1], v_rows = kRows * a.v_stride[1];
  const bool whole = a.head_dim == DP;  // every chunk of a row holds data
  int key_next = first;
  auto fetch = [&](int stage) {
    const uint32_t at = ring_at + stage * P::kStage;
    if (VEC && whole && key_next + kStepKeys <= to) {
      const uint16_t* kp = k_next;
      const uint16_t* vp = v_next;
#pragma unroll
      for (int i = 0; i < kCopies; ++i, kp += k_rows, vp += v_rows) {
        const uint32_t s = at + step_at<DP>(my_row + i * kRows, my_chunk);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(kp) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s + kStepKeys * P::kRow),
                     "l"(vp)
                     : "memory");
      }
    } else if constexpr (VEC) {
#pragma unroll 1
      for (int i = 0; i < kCopies; ++i) {
        const int r = my_row + i * kRows;
        const bool in = key_next + r < to && my_data;
        const int bytes = in ? 16 : 0;
        const uint16_t* kp = in ? k_next + i * kRows * a.k_stride[1] : k;
        const uint16_t* vp = in ? v_next + i * kRows * a.v_stride[1] : v;
        const uint32_t s = at + step_at<DP>(r, my_chunk);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(kp), "r"(bytes)
                     : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s + kStepKeys * P::kRow),
                     "l"(vp), "r"(bytes)
                     : "memory");
      }
    } else {
      uint8_t* p = ring + stage * P::kStage;
      for (int e = lane; e < kStepKeys * DP; e += 32) {
        const int r = e / DP, d = e % DP;
        const bool in = key_next + r < to && d < a.head_dim;
        const int64_t j = in ? key_next + r : 0;
        uint16_t* at_k = reinterpret_cast<uint16_t*>(p + step_at<DP>(r, d / 8)) + d % 8;
        at_k[0] = in ? k[j * a.k_stride[1] + d] : uint16_t{0};
        at_k[kStepKeys * DP] = in ? v[j * a.v_stride[1] + d] : uint16_t{0};
      }
      __syncwarp();
    }
    key_next += kStride;
    k_next += kStride * a.k_stride[1];
    v_next += kStride * a.v_stride[1];
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStepStages - 1; ++s) fetch(s);

  // ---- Q^T as mma operand: column lane / 4 of each tile of eight is query row
  // n, head h0 + n / tile_rows and position row0 + n % tile_rows
  uint32_t q[NT][DP / 16][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + lane / 4;
    const int pos = row0 + r % a.tile_rows;
    const bool valid = r < rows && pos < seq.q1;
    const uint16_t* qr = static_cast<const uint16_t*>(a.q) + seq.batch * a.q_stride[0] +
                         int64_t{valid ? pos : row0} * a.q_stride[1] +
                         (valid ? h0 + r / a.tile_rows : h0) * a.q_stride[2];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int d = 16 * s + 8 * half + 2 * (lane & 3);
        const uint32_t lo = valid && d < a.head_dim ? qr[d] : 0u;
        const uint32_t hi = valid && d + 1 < a.head_dim ? qr[d + 1] : 0u;
        q[n][s][half] = lo | hi << 16;
      }
    }
  }
  // ---- this thread's softmax rows: columns 2 (lane % 4) and the next
  constexpr float kLog2e = 1.4426950408889634f;
  const float scale = a.scale * kLog2e;
  const bool cap = a.softcap > 0.0f;
  const float cap_arg = cap ? cap_argument(a) : 0.0f;
  const float cap_out = a.softcap * kLog2e;
  const bool bias = a.slopes != nullptr;
  float slope[NT][2];
  int place[NT][2], seen[NT][2];
  float o[NT][DP / 16][4], top[NT][2], sum[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * n + 2 * (lane & 3) + i;
      const int pos = row0 + r % a.tile_rows;
      const bool valid = r < rows && pos < seq.q1;
      seen[n][i] = valid ? min(to, seq.seen(pos, a.causal)) : 0;
      place[n][i] = valid ? seq.place(pos) : 0;
      slope[n][i] = valid && bias ? a.slopes[h0 + r / a.tile_rows] * kLog2e : 0.0f;
      top[n][i] = -INFINITY;
      sum[n][i] = 0.0f;
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][d][e] = 0.0f;
    }
  }

  // ldmatrix rows of this lane: K as it lies (keys 0-7, 8-15, then the next
  // eight elements), V transposed (elements 0-7, 8-15, then the next keys)
  const int k_row = lane & 15, k_half = lane >> 4;
  const int v_row = (lane & 7) + (lane >> 4) * 8, v_half = lane >> 3 & 1;
  int stage = 0;
  for (int key = first; key < to; key += kStride) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStepStages - 2) : "memory");
    __syncwarp();
    fetch(stage == 0 ? kStepStages - 1 : stage - 1);
    const uint32_t k_at = ring_at + stage * P::kStage, v_at = k_at + kStepKeys * P::kRow;
    stage = stage == kStepStages - 1 ? 0 : stage + 1;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t m[4];
      ldmatrix4<false>(m, k_at + step_at<DP>(k_row, 2 * d + k_half));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_16816<T>(s[n], m, q[n][d][0], q[n][d][1]);
    }
    // s[n][2 half + i]: key lane / 4 + 8 half, row column i
    uint32_t p[NT][2];
    const int j0 = key + lane / 4;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (cap) {
        float u[4];
        bool small = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u[e] = s[n][e] * cap_arg;
          small = small && fabsf(u[e]) <= kTanhLimit;
          s[n][e] *= scale * tanh_ratio(u[e] * u[e]);
        }
        if (__any_sync(0xFFFFFFFFu, !small)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float far = fmaf(-2.0f * cap_out, reciprocal(1.0f + ex2(u[e] * (2.0f * kLog2e))),
                                   cap_out);
            s[n][e] = fabsf(u[e]) <= kTanhLimit ? s[n][e] : far;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= scale;
      }
      float t[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = s[n][2 * half + i];
          const int j = j0 + 8 * half;
          // subtracted as integers: fp32 does not hold every place behind 2^24
          if (bias) x -= slope[n][i] * fabsf(static_cast<float>(place[n][i] - j));
          s[n][2 * half + i] = j < seen[n][i] ? x : -INFINITY;
        }
        t[i] = max_nan(top[n][i], max_nan(s[n][i], s[n][2 + i]));
      }
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) {
        t[0] = max_nan(t[0], __shfl_xor_sync(0xFFFFFFFFu, t[0], w));
        t[1] = max_nan(t[1], __shfl_xor_sync(0xFFFFFFFFu, t[1], w));
      }
      // as in the prompt kernel: the maximum in use moves when it grew by 2^8
      bool moved[2];
      float factor[2], base[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        moved[i] = !(t[i] - top[n][i] <= 8.0f) && t[i] != -INFINITY;
        factor[i] = moved[i] && top[n][i] != -INFINITY ? ex2(top[n][i] - t[i]) : 1.0f;
        if (moved[i]) top[n][i] = t[i];
        base[i] = top[n][i] == -INFINITY ? 0.0f : top[n][i] - kWeightShift<T>;
      }
      if (__any_sync(0xFFFFFFFFu, moved[0] || moved[1])) {
        sum[n][0] *= factor[0];
        sum[n][1] *= factor[1];
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][d][e] *= factor[e & 1];
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float p0 = ex2(s[n][2 * half] - base[0]), p1 = ex2(s[n][2 * half + 1] - base[1]);
        sum[n][0] += p0;
        sum[n][1] += p1;
        p[n][half] = transpose8(pack_pair<T>(p0, p1));
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t m[4];
      ldmatrix4<true>(m, v_at + step_at<DP>(v_row, 2 * d + v_half));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // added here: the tensor core would cut off what lies below o's last place
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_16816<T>(y, m, p[n][0], p[n][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][d][e] += y[e];
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  // ---- join the warps: [warp][row][DP] fp32 over the rings
  float* all_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float l = sum[n][i];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, w);
      const int r = 8 * n + 2 * (lane & 3) + i;
      if (lane < 4) {
        row_m[warp][r] = top[n][i];
        row_l[warp][r] = l;
      }
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        float* to_o = all_o + (warp * 8 * NT + r) * DP + 16 * d + lane / 4;
        to_o[0] = o[n][d][i];
        to_o[8] = o[n][d][2 + i];
      }
    }
  }
  __syncthreads();
  const int64_t part_rows = int64_t{a.batch} * a.q_heads * a.q_len;
  for (int r = warp; r < rows; r += 4) {
    const int pos = row0 + r % a.tile_rows, h = h0 + r / a.tile_rows;
    if (pos >= seq.q1) continue;
    float t = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) t = max_nan(t, row_m[w][r]);
    const float base = t == -INFINITY ? 0.0f : t;
    float f[4], l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = row_m[w][r] == -INFINITY ? 0.0f : ex2(row_m[w][r] - base);
      if (f[w] != 0.0f) l += f[w] * row_l[w][r];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t at = (int64_t{seq.batch} * a.q_heads + h) * a.q_len + pos;
    const float lse =
        l == 0.0f ? -INFINITY : (base + (log2f(l) - kWeightShift<T>)) * 0.6931471805599453f;
    const int64_t oo = seq.batch * a.o_stride[0] + pos * a.o_stride[1] + h * a.o_stride[2];
    if (lane == 0) {
      if (a.splits > 1) {
        a.part_lse[blockIdx.y * part_rows + at] = lse;
      } else if (a.lse != nullptr) {
        a.lse[at] = lse;
      }
    }
    for (int d = lane; d < a.head_dim; d += 32) {
      float y = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (f[w] != 0.0f) y += f[w] * all_o[(w * 8 * NT + r) * DP + d];
      }
      y *= inv;
      if (a.splits > 1) {
        a.part_o[(blockIdx.y * part_rows + at) * a.head_dim + d] = y;
      } else if (a.o_lo != 0) {
        const float hi = __bfloat162float(__float2bfloat16_rn(y));
        store_element<IE_DT_BF16>(a.o, oo + d, hi);
        store_element<IE_DT_BF16>(a.o, oo + a.o_lo + d, y - hi);
      } else {
        store_element<T>(a.o, oo + d, y);
      }
    }
  }
}

}  // namespace ie_cuda
