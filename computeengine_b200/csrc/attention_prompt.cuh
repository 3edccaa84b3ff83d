// Attention for many query rows on the tensor cores.
//
// One block works on 256 query rows of one head and sequence as two tiles of
// 128, over the keys in tiles of 128:
//   S = Q K^T            tcgen05.mma, both operands in shared memory, S in TMEM
//   P = exp2(S - max)    one thread per row: the row's maximum and sum need no
//                        exchange; P goes back over S in TMEM as 16-bit values
//   O += P V             tcgen05.mma with P as the TMEM operand, O in TMEM
// While the threads of one tile take their exponentials, the tensor core works
// for the other one.  Warps 0-3 and 4-7 hold the rows of the tiles, warp 8
// issues the MMAs, warp 9 the TMA loads of Q, K and V, warp 10 clears the rows
// of V behind the sequence's end (0 * NaN would reach O).
#pragma once

#include "attention_common.cuh"
#include "ptx.cuh"

namespace ie_cuda {

constexpr unsigned kErrAttnQ = 0x201, kErrAttnKv = 0x202, kErrAttnEmpty = 0x203,
                   kErrAttnS = 0x204, kErrAttnP = 0x205, kErrAttnO = 0x206, kErrAttnFix = 0x207;

constexpr int kPromptThreads = 384;

struct PromptArgs : AttentionArgs {
  int tiles;           // blocks of 256 rows per (head, batch row), documents: upper bound
  int splits;          // shares of each sequence's keys
  float* part_o;       // splits > 1: fp32 [splits][batch][q_heads][q_len][head_dim]
  float* part_lse;     //             fp32 [splits][batch][q_heads][q_len]
  int o_vec;           // rows of o can be written in 16-byte pieces
  uint64_t wait_limit_ns;
};

template <int DP>
struct PromptPlan {
  static constexpr int kCols = DP / 64;               // 128-byte wide column blocks of a tile
  static constexpr int kTile = kCols * 128 * 128;     // bytes of a 128-row tile
  static constexpr int kStages = DP == 128 ? 5 : 8;   // K and V tiles in flight
  static constexpr int kSmem = 2 * kTile + kStages * kTile + 1024 + 256;
};

template <int DP, int T, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kPromptThreads, 1)
    attention_prompt_kernel(const PromptArgs a, const __grid_constant__ CUtensorMap map_q,
                            const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v) {
  using P = PromptPlan<DP>;
  constexpr int kStages = P::kStages;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which rows and keys
  const int h = blockIdx.x % a.q_heads;
  const int batch_row = blockIdx.x / a.q_heads % a.batch;
  const int tile = a.tiles - 1 - static_cast<int>(blockIdx.x / a.q_heads / a.batch);  // causal: longest first
  Sequence seq;
  int row0 = 0;
  if (!tile_sequence(a, tile, batch_row, 256, &seq, &row0)) return;
  const int length = seq.k1 - seq.k0;
  // key tiles of each row tile: up to what its last row sees
  int tiles_t[2];
  for (int t = 0; t < 2; ++t) {
    const int last = min(row0 + 128 * (t + 1), seq.q1) - 1;
    tiles_t[t] = row0 + 128 * t < seq.q1 ? (seq.seen(last, a.causal) + 127) / 128 : 0;
  }
  int begin = 0;
  {
    const int all = max(tiles_t[0], tiles_t[1]);
    const int share = (all + a.splits - 1) / a.splits;
    begin = share * static_cast<int>(blockIdx.y);
    for (int t = 0; t < 2; ++t) tiles_t[t] = max(0, min(tiles_t[t], begin + share) - begin);
  }
  const int tiles = max(tiles_t[0], tiles_t[1]);

  // ---- shared memory
  uint8_t* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* q_tile = base;
  uint8_t* ring = base + 2 * P::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kStages * P::kTile);
  uint64_t* q_full = bars;                 // [2]
  uint64_t* s_full = bars + 2;             // [2]
  uint64_t* p_full = bars + 4;             // [2]
  uint64_t* o_full = bars + 6;             // [2]
  uint64_t* short_full = bars + 8;         // the last V tile, when it is cut short
  uint64_t* fixed = bars + 9;              // and its rows behind the end are cleared
  uint64_t* drain = bars + 10;
  uint64_t* kv_full = bars + 11;           // [kStages]
  uint64_t* kv_empty = bars + 11 + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11 + 2 * kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* loads_issued = const_cast<int*>(abort_flag) + 1;

  if (warp == 8) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 128);
        mbar_init(&o_full[i], 1);
      }
      mbar_init(short_full, 1);
      mbar_init(fixed, 32);
      mbar_init(drain, 1);
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&kv_full[i], 1);
        mbar_init(&kv_empty[i], 1);
      }
      *abort_flag = 0;
      *loads_issued = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // TMEM columns: S (and P over it) of tile t at 128 t, O at 256 + DP t
  const bool last_short = length % 128 != 0 && begin + tiles == (length + 127) / 128;

  if (warp >= 8) {
    setmaxnreg_dec<56>();
    if (warp == 9 && lane == 0) {
      // ------------------------------------------------ TMA loads
      const int hk = static_cast<int>(static_cast<int64_t>(h) * a.kv_heads / a.q_heads);
      bool ok = tiles > 0;
      for (int t = 0; t < 2 && ok; ++t) {
        if (tiles_t[t] == 0) continue;
        mbar_arrive_expect_tx(&q_full[t], P::kTile);
        for (int c = 0; c < P::kCols; ++c) {
          tma_load_4d(q_tile + t * P::kTile + c * 16384, &map_q, &q_full[t], 64 * c,
                      row0 + 128 * t, h, seq.batch);
        }
      }
      // ring order: K0, K1, V0, K2, V1, ... : V of a tile is needed after K of the next
      int issued = 0;
      const int total = 2 * tiles;
      for (int i = 0; ok && i < total; ++i) {
        // i = 0: K0; then pairs (K_{j+1}, V_j); the last V has no K before it
        const bool is_k = i == 0 || (i % 2 == 1 && i < total - 1);
        const int j = i == 0 ? 0 : is_k ? (i + 1) / 2 : i == total - 1 ? tiles - 1 : i / 2 - 1;
        const int s = i % kStages;
        if (!mbar_wait(&kv_empty[s], ((i / kStages) & 1) ^ 1u, abort_flag, kErrAttnEmpty,
                       a.wait_limit_ns)) {
          break;
        }
        // a barrier of its own lets warp 10 wait for this load from the start
        uint64_t* full = last_short && i == total - 1 ? short_full : &kv_full[s];
        mbar_arrive_expect_tx(full, P::kTile);
        const int row = seq.k0 + (begin + j) * 128;
        for (int c = 0; c < P::kCols; ++c) {
          tma_load_4d(ring + s * P::kTile + c * 16384, is_k ? &map_k : &map_v, full, 64 * c,
                      row, hk, seq.batch);
        }
        issued = i + 1;
      }
      *loads_issued = issued;
    } else if (warp == 8 && lane == 0) {
      // ------------------------------------------------ MMA issuer
      const int ksteps = (a.head_dim + 15) / 16;
      const uint32_t idesc_s = make_idesc_f16(128, 128, T == IE_DT_BF16, false);
      const uint32_t idesc_o = make_idesc_f16(128, ksteps * 16, T == IE_DT_BF16, true);
      const uint64_t q_desc = make_smem_desc(smem_u32(q_tile), 16, 1024, 2);
      const uint64_t k_desc = make_smem_desc(smem_u32(ring), 16, 1024, 2);
      const uint64_t v_desc = make_smem_desc(smem_u32(ring), 16384, 1024, 2);
      bool ok = tiles > 0;
      auto wait_kv = [&](int i) {
        return mbar_wait(&kv_full[i % kStages], (i / kStages) & 1, abort_flag, kErrAttnKv,
                         a.wait_limit_ns);
      };
      auto scores = [&](int t, int i) {  // S_t = Q_t K^T, K in ring slot of load i
        const uint64_t qd = q_desc + ((t * P::kTile) >> 4);
        const uint64_t kd = k_desc + (((i % kStages) * P::kTile) >> 4);
        for (int s = 0; s < ksteps; ++s) {
          const uint64_t at = ((s / 4) * 16384 + (s % 4) * 32) >> 4;
          mma_f16(tmem + 128 * t, qd + at, kd + at, idesc_s, s > 0);
        }
        tc_commit(&s_full[t]);
      };
      auto outputs = [&](int t, int i, bool add) {  // O_t += P_t V, V in ring slot of load i
        const uint64_t vd = v_desc + (((i % kStages) * P::kTile) >> 4);
        for (int s = 0; s < 8; ++s) {
          mma_f16_ta(tmem + 256 + DP * t, tmem + 128 * t + 8 * s, vd + ((s * 2048) >> 4), idesc_o,
                     add || s > 0);
        }
      };
      // load index of K_j and V_j in the ring's order
      auto k_at = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
      auto v_at = [&](int j) { return j == tiles - 1 ? 2 * tiles - 1 : 2 * j + 2; };
      for (int t = 0; t < 2 && ok; ++t) {
        if (tiles_t[t] == 0) continue;
        ok = mbar_wait(&q_full[t], 0, abort_flag, kErrAttnQ, a.wait_limit_ns) && wait_kv(0);
        if (ok) scores(t, 0);
      }
      if (ok) tc_commit(&kv_empty[0]);
      for (int j = 0; ok && j < tiles; ++j) {
        if (j + 1 < tiles) ok = wait_kv(k_at(j + 1));
        if (last_short && j == tiles - 1) {
          ok = ok && mbar_wait(fixed, 0, abort_flag, kErrAttnFix, a.wait_limit_ns);
        } else {
          ok = ok && wait_kv(v_at(j));
        }
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= tiles_t[t]) continue;
          ok = mbar_wait(&p_full[t], j & 1, abort_flag, kErrAttnP, a.wait_limit_ns);
          if (!ok) break;
          tc_fence_after();
          outputs(t, v_at(j), j > 0);
          if (j + 1 < tiles_t[t]) {
            scores(t, k_at(j + 1));
          } else {
            tc_commit(&o_full[t]);
          }
        }
        if (!ok) break;
        if (j + 1 < tiles) tc_commit(&kv_empty[k_at(j + 1) % kStages]);
        tc_commit(&kv_empty[v_at(j) % kStages]);
      }
      // every MMA done before tensor memory is released, on the abort path too
      tc_commit(drain);
      int dummy_abort = 0;
      mbar_wait(drain, 0, &dummy_abort, kErrAttnO, a.wait_limit_ns);
    } else if (warp == 10 && last_short && tiles > 0) {
      // ------------------------------------------------ rows of V behind the end
      const int i = 2 * tiles - 1, s = i % kStages;  // the last load is the last tile's V
      if (mbar_wait_warp(short_full, 0, abort_flag, kErrAttnKv, a.wait_limit_ns)) {
        uint8_t* v = ring + s * P::kTile;
        const int from = length % 128;
        for (int e = lane; e < (128 - from) * 8 * P::kCols; e += 32) {
          const int c = e / ((128 - from) * 8), r = e % ((128 - from) * 8);
          *reinterpret_cast<uint4*>(v + c * 16384 + from * 128 + r * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        mbar_arrive(fixed);
      }
    }
  } else {
    // ------------------------------------------------ rows
    setmaxnreg_inc<224>();
    const int t = warp >> 2;
    const int row = row0 + 128 * t + (threadIdx.x & 127);
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + 128 * t + lanes, o_at = tmem + 256 + DP * t + lanes;
    const bool valid = row < seq.q1;
    const int seen = valid ? seq.seen(row, a.causal) : 0;
    // what every row of this tile sees, and what the sequence's rows are biased by
    const int all_see =
        row0 + 128 * t < seq.q1 ? seq.seen(row0 + 128 * t, a.causal) : 0;
    constexpr float kLog2e = 1.4426950408889634f;
    const float scale = a.scale * kLog2e;
    const float cap_in = CAP ? 2.0f * kLog2e * a.scale / a.softcap : 0.0f;
    const float cap_out = CAP ? a.softcap * kLog2e : 0.0f;
    const float slope = BIAS && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.0f;
    const float place = static_cast<float>(valid ? seq.place(row) : 0);
    // x is the score in units of log2 e (plain: before the scale)
    constexpr bool kScaled = CAP || BIAS;
    const float to_log2 = kScaled ? 1.0f : scale;

    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    const int n = tiles_t[t];
    for (int j = 0; j < n; ++j) {
      if (!mbar_wait_warp(&s_full[t], j & 1, abort_flag, kErrAttnS, a.wait_limit_ns)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sr[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_at + 32 * c, sr[c]);
      const int key0 = (begin + j) * 128;
      float x[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld_wait(sr[c]);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[32 * c + e] = __uint_as_float(sr[c][e]);
      }
      if constexpr (CAP) {
#pragma unroll
        for (int e = 0; e < 128; ++e) {
          // cap * tanh(s / cap) = cap * (1 - 2 / (1 + exp(2 s / cap)))
          const float u = ex2(x[e] * cap_in);
          x[e] = cap_out - __fdividef(2.0f * cap_out, 1.0f + u);
        }
      } else if constexpr (BIAS) {
#pragma unroll
        for (int e = 0; e < 128; ++e) x[e] *= scale;
      }
      if constexpr (BIAS) {
        const float from = place - static_cast<float>(key0);
#pragma unroll
        for (int e = 0; e < 128; ++e) x[e] -= slope * fabsf(from - static_cast<float>(e));
      }
      if (key0 + 128 > all_see) {
        const int vis = seen - key0;
#pragma unroll
        for (int e = 0; e < 128; ++e) x[e] = e < vis ? x[e] : -INFINITY;
      }
      float top = m;
#pragma unroll
      for (int e = 0; e < 128; ++e) top = max_nan(top, x[e]);
      // The maximum in use moves only when it grew by more than 2^8: until then
      // the weights stay below 256, which both 16-bit types hold as well as 1.
      float factor = 1.0f;
      const bool moved = !((top - m) * to_log2 <= 8.0f) && top != -INFINITY;
      if (moved) {
        factor = m == -INFINITY ? 1.0f : ex2((m - top) * to_log2);
        m = top;
      }
      if (j > 0 && __any_sync(0xFFFFFFFFu, moved)) {
        // the tile's earlier O (S of this tile follows it in the tensor core's order)
        l *= factor;
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(o_at + 32 * c, r);
          tmem_ld_wait(r);
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * factor);
          tmem_st_32x32b_x32(o_at + 32 * c, r);
        }
      }
      const float base = m == -INFINITY ? 0.0f : m * to_log2;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float p0 = ex2(fmaf(x[64 * c + 2 * e], to_log2, -base));
          const float p1 = ex2(fmaf(x[64 * c + 2 * e + 1], to_log2, -base));
          sum[e & 1] += p0;
          sum[2 + (e & 1)] += p1;
          p[e] = pack_pair<T>(p0, p1);
        }
        tmem_st_32x32b_x32(s_at + 32 * c, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
    }
    if (n > 0 && ok) ok = mbar_wait_warp(&o_full[t], 0, abort_flag, kErrAttnO, a.wait_limit_ns);
    tc_fence_after();
    if (ok) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const bool none = l == 0.0f;
      const int64_t at = (static_cast<int64_t>(seq.batch) * a.q_heads + h) * a.q_len + row;
      const float lse = none ? -INFINITY : (m * to_log2 + log2f(l)) * 0.6931471805599453f;
      const int64_t part_rows = static_cast<int64_t>(a.batch) * a.q_heads * a.q_len;
      if (valid) {
        if (a.splits > 1) {
          a.part_lse[blockIdx.y * part_rows + at] = lse;
        } else if (a.lse != nullptr) {
          a.lse[at] = lse;
        }
      }
      const int64_t oo = static_cast<int64_t>(seq.batch) * a.o_stride[0] +
                         static_cast<int64_t>(row) * a.o_stride[1] +
                         static_cast<int64_t>(h) * a.o_stride[2];
      float* part = a.splits > 1 ? a.part_o + (blockIdx.y * part_rows + at) * a.head_dim : nullptr;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        if (32 * c >= a.head_dim) break;
        uint32_t r[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(o_at + 32 * c, r);
          tmem_ld_wait(r);
        }
        if (valid) {
          float y[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = none ? 0.0f : __uint_as_float(r[e]) * inv;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            const int d = 32 * c + e;
            if (d >= a.head_dim) break;  // head_dim is a multiple of 8 here
            if (a.splits > 1) {
              for (int f = 0; f < 8; ++f) part[d + f] = y[e + f];
              continue;
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) hi[f] = pack_pair<T>(y[e + 2 * f], y[e + 2 * f + 1]);
            if (a.o_lo != 0) {
#pragma unroll
              for (int f = 0; f < 4; ++f) {
                lo[f] = pack_pair<T>(y[e + 2 * f] - __uint_as_float(hi[f] << 16),
                                 y[e + 2 * f + 1] - __uint_as_float(hi[f] & 0xFFFF0000u));
              }
            }
            uint16_t* o = static_cast<uint16_t*>(a.o) + oo + d;
            if (a.o_vec) {
              *reinterpret_cast<uint4*>(o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              if (a.o_lo != 0) {
                *reinterpret_cast<uint4*>(o + a.o_lo) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            } else {
              for (int f = 0; f < 8; ++f) {
                o[f] = static_cast<uint16_t>(hi[f / 2] >> (16 * (f & 1)));
                if (a.o_lo != 0) o[a.o_lo + f] = static_cast<uint16_t>(lo[f / 2] >> (16 * (f & 1)));
              }
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
    }
  }

  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    // no TMA load may still be writing this block's shared memory when it ends
    int dummy_abort = 0;
    for (int t = 0; t < 2; ++t) {
      if (tiles_t[t] > 0) mbar_wait(&q_full[t], 0, &dummy_abort, kErrAttnQ, a.wait_limit_ns);
    }
    const int issued = *loads_issued;
    for (int i = max(0, issued - kStages); i < issued; ++i) {
      const bool cut = last_short && i == 2 * tiles - 1;
      mbar_wait(cut ? short_full : &kv_full[i % kStages], cut ? 0 : (i / kStages) & 1,
                &dummy_abort, kErrAttnKv, a.wait_limit_ns);
    }
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ie_cuda
