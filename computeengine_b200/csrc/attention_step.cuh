// Attention for few query rows (single tokens), and for tensors that TMA
// cannot read.
//
// All query heads that read one kv head are rows of one tile, so K and V are
// read once: 16 rows are one mma.sync m16n8k16 operand, two at most.  Bound by
// the memory: a block's four warps take keys 16 at a time, each into its own
// ring of asynchronous copies (no barrier between warps), with a running
// maximum and sum per row; long sequences are cut into shares for many blocks.
// The warps' results are joined in shared memory, the shares' by a second
// kernel.
#pragma once

#include "attention_common.cuh"

namespace ie_cuda {

constexpr int kStepThreads = 128;
constexpr int kStepStages = 3;
constexpr int kStepKeys = 16;

struct StepArgs : AttentionArgs {
  int tile_rows;    // query positions of a tile
  int tile_heads;   // query heads of a tile; tile_rows * tile_heads <= 16 MT
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

// Byte of 16-byte chunk c of key row r in a tile of rows of DP elements: the
// chunk's place is turned by the row, so eight rows' chunks share no bank.
template <int DP>
__device__ __forceinline__ uint32_t step_at(int r, int c) {
  return static_cast<uint32_t>(r * StepPlan<DP>::kRow + ((c ^ (r & 7)) << 4));
}

// VEC: K and V in 16-byte aligned rows of a multiple of 8 elements.
template <int DP, int T, int MT, bool VEC>
__global__ void __launch_bounds__(kStepThreads) attention_step_kernel(const StepArgs a) {
  using P = StepPlan<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float row_m[4][16 * MT], row_l[4][16 * MT];
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
  const int chunks = (a.head_dim + 7) / 8;  // of a row that hold data

  // copies K and V of keys key .. key + 15 into a stage; rows past `to` and
  // elements past head_dim are zeros
  auto fetch = [&](int stage, int key) {
    const uint32_t at = ring_at + stage * P::kStage;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kStepKeys * DP / 8 / 32; ++i) {
        const int e = i * 32 + lane, r = e / (DP / 8), c = e % (DP / 8);
        const bool in = key + r < to && c < chunks;
        const int64_t j = in ? key + r : 0;
        const int bytes = in ? 16 : 0, cc = in ? c : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + step_at<DP>(r, c)),
                     "l"(k + j * a.k_stride[1] + cc * 8), "r"(bytes)
                     : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         at + kStepKeys * P::kRow + step_at<DP>(r, c)),
                     "l"(v + j * a.v_stride[1] + cc * 8), "r"(bytes)
                     : "memory");
      }
    } else {
      uint8_t* p = ring + stage * P::kStage;
      for (int e = lane; e < kStepKeys * DP; e += 32) {
        const int r = e / DP, d = e % DP;
        const bool in = key + r < to && d < a.head_dim;
        const int64_t j = in ? key + r : 0;
        uint16_t* at_k = reinterpret_cast<uint16_t*>(p + step_at<DP>(r, d / 8)) + d % 8;
        at_k[0] = in ? k[j * a.k_stride[1] + d] : uint16_t{0};
        at_k[kStepKeys * DP] = in ? v[j * a.v_stride[1] + d] : uint16_t{0};
      }
      __syncwarp();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int first = from + warp * kStepKeys;
  constexpr int kStride = 4 * kStepKeys;
#pragma unroll
  for (int s = 0; s < kStepStages - 1; ++s) fetch(s, first + s * kStride);

  // ---- Q as mma operands: this thread's rows are lane / 4 and lane / 4 + 8 of
  // each 16-row tile, row r being head h0 + r / tile_rows, position row0 + r % tile_rows
  uint32_t q[MT][DP / 16][4];
  int seen[MT][2], head[MT][2], place[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * m + lane / 4 + 8 * i;
      const int pos = row0 + r % a.tile_rows;
      const bool valid = r < rows && pos < seq.q1;
      head[m][i] = valid ? h0 + r / a.tile_rows : h0;
      seen[m][i] = valid ? min(to, seq.seen(pos, a.causal)) : 0;
      place[m][i] = valid ? seq.place(pos) : 0;
      const uint16_t* qr = static_cast<const uint16_t*>(a.q) + seq.batch * a.q_stride[0] +
                           int64_t{valid ? pos : row0} * a.q_stride[1] +
                           head[m][i] * a.q_stride[2];
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int d = 16 * s + 8 * half + 2 * (lane & 3);
          const uint32_t lo = valid && d < a.head_dim ? qr[d] : 0u;
          const uint32_t hi = valid && d + 1 < a.head_dim ? qr[d + 1] : 0u;
          q[m][s][2 * half + i] = lo | hi << 16;
        }
      }
    }
  }
  constexpr float kLog2e = 1.4426950408889634f;
  const float scale = a.scale * kLog2e;
  const bool cap = a.softcap > 0.0f;
  const float cap_in = cap ? 2.0f * kLog2e * a.scale / a.softcap : 0.0f;
  const float cap_out = a.softcap * kLog2e;
  float slope[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      slope[m][i] = a.slopes == nullptr ? 0.0f : a.slopes[head[m][i]] * kLog2e;
    }
  }

  float o[MT][DP / 8][4], top[MT][2], sum[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[m][i] = -INFINITY;
      sum[m][i] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][n][e] = 0.0f;
    }
  }

  int stage = 0;
  for (int key = first; key < to; key += kStride) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStepStages - 2) : "memory");
    __syncwarp();
    fetch((stage + kStepStages - 1) % kStepStages, key + (kStepStages - 1) * kStride);
    const uint32_t k_at = ring_at + stage * P::kStage, v_at = k_at + kStepKeys * P::kRow;
    stage = (stage + 1) % kStepStages;
    float s[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][n][e] = 0.0f;
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      // matrices: keys 0-7 and 8-15, each with the two halves of 16 elements
      uint32_t b[4];
      ldmatrix4<false>(b, k_at + step_at<DP>((lane & 7) + (lane >> 4) * 8, 2 * d + (lane >> 3 & 1)));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma_16816<T>(s[m][0], q[m][d], b[0], b[1]);
        mma_16816<T>(s[m][1], q[m][d], b[2], b[3]);
      }
    }
    uint32_t p[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float t = top[m][i];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = key + 8 * n + 2 * (lane & 3) + e;
            float x = s[m][n][2 * i + e];
            if (cap) {
              x = cap_out - __fdividef(2.0f * cap_out, 1.0f + ex2(x * cap_in));
            } else {
              x *= scale;
            }
            x -= slope[m][i] * fabsf(static_cast<float>(place[m][i] - j));
            x = j < seen[m][i] ? x : -INFINITY;
            s[m][n][2 * i + e] = x;
            t = max_nan(t, x);
          }
        }
        t = max_nan(t, __shfl_xor_sync(0xFFFFFFFFu, t, 1));
        t = max_nan(t, __shfl_xor_sync(0xFFFFFFFFu, t, 2));
        // as in the prompt kernel: the maximum in use moves when it grew by 2^8
        const bool moved = !(t - top[m][i] <= 8.0f) && t != -INFINITY;
        const float factor = moved && top[m][i] != -INFINITY ? ex2(top[m][i] - t) : 1.0f;
        if (moved) top[m][i] = t;
        if (__any_sync(0xFFFFFFFFu, moved)) {
          sum[m][i] *= factor;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            o[m][n][2 * i] *= factor;
            o[m][n][2 * i + 1] *= factor;
          }
        }
        const float base = top[m][i] == -INFINITY ? 0.0f : top[m][i];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2(s[m][n][2 * i] - base), p1 = ex2(s[m][n][2 * i + 1] - base);
          sum[m][i] += p0 + p1;
          p[m][2 * n + i] = pack_pair<T>(p0, p1);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      // matrices: keys 0-7 and 8-15 of 8 elements, then of the next 8
      uint32_t b[4];
      ldmatrix4<true>(b, v_at + step_at<DP>((lane & 7) + (lane >> 3 & 1) * 8, 2 * d + (lane >> 4)));
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma_16816<T>(o[m][2 * d], p[m], b[0], b[1]);
        mma_16816<T>(o[m][2 * d + 1], p[m], b[2], b[3]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();

  // ---- join the warps: [warp][row][DP] fp32 over the rings
  float* all_o = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float l = sum[m][i];
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
      l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
      const int r = 16 * m + lane / 4 + 8 * i;
      if ((lane & 3) == 0) {
        row_m[warp][r] = top[m][i];
        row_l[warp][r] = l;
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        *reinterpret_cast<float2*>(all_o + (warp * 16 * MT + r) * DP + 8 * n + 2 * (lane & 3)) =
            make_float2(o[m][n][2 * i], o[m][n][2 * i + 1]);
      }
    }
  }
  __syncthreads();
  const int64_t part_rows = int64_t{a.batch} * a.q_heads * a.q_len;
  for (int r = warp; r < rows; r += 4) {
    const int pos = row0 + r % a.tile_rows, h = h0 + r / a.tile_rows;
    if (pos >= seq.q1) continue;
    float t = -INFINITY;
    for (int w = 0; w < 4; ++w) t = max_nan(t, row_m[w][r]);
    const float base = t == -INFINITY ? 0.0f : t;
    float f[4], l = 0.0f;
    for (int w = 0; w < 4; ++w) {
      f[w] = row_m[w][r] == -INFINITY ? 0.0f : ex2(row_m[w][r] - base);
      if (f[w] != 0.0f) l += f[w] * row_l[w][r];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t at = (int64_t{seq.batch} * a.q_heads + h) * a.q_len + pos;
    const float lse = l == 0.0f ? -INFINITY : (base + log2f(l)) * 0.6931471805599453f;
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
      for (int w = 0; w < 4; ++w) {
        if (f[w] != 0.0f) y += f[w] * all_o[(w * 16 * MT + r) * DP + d];
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
