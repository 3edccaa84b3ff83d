// Attention for many query rows on the tensor cores.
//
// One block works on two tiles of 128 query rows of one sequence, over the keys
// in steps of 64:
//   S = Q K^T            tcgen05.mma, both operands in shared memory, S in TMEM
//   P = exp2(S - max)    one thread per row: the row's maximum and sum need no
//                        exchange; P goes back over S in TMEM as 16-bit values
//   O += P V             tcgen05.mma with P as the TMEM operand, O in TMEM
// The rows of a tile are 128 positions of one head, or, for few positions, all
// positions of several heads that read the same kv head.
//
// From P in TMEM to the next S there pass the MMAs and 400 cycles of latency.
// Tiles with heads of 128 have two S buffers, so the threads of a row always
// find the next S; with one S of 128 keys they waited a third of the time.  The
// price is that S of 64 keys costs 49 cycles per 16 elements of the head where
// half of one of 128 keys costs 32 (Q is read from shared memory for each), so a
// head of 128 runs at most at 79% of the tensor core's rate.  With heads of 64
// there is room for two blocks per SM instead.  Then the exponentials are the
// longest single part (16 a cycle and SM: 60 us of 113 to 126 us for 4096 tokens, 16
// heads of 64); a polynomial on the FMA pipes for a quarter of them changed nothing.
// Warps 0-3 and 4-7 hold the rows of the tiles, warps 8 and 9 issue their MMAs
// (one thread for both tiles took about 2200 cycles a step, 1200 of them between
// its waits and the MMAs), warp 10 the TMA loads of Q, K and V; it also
// clears the rows of V behind the sequence's end (0 * NaN would reach O).  Warp 11
// is idle: it completes the warpgroup that gives its registers away.
// The weights are rounded to the 16-bit type, half a step of each, as the tensor
// core takes them; their sum is that of the unrounded ones.
// 4096 tokens, 16 heads of 128, no mask: 126 to 137 us, 1000 to 1090 TFLOP/s; of 64:
// 113 to 126 us, 543 to 608 TFLOP/s.
#pragma once

#include "attention_common.cuh"
#include "ptx.cuh"

namespace ie_cuda {

constexpr unsigned kErrAttnQ = 0x201, kErrAttnKv = 0x202, kErrAttnEmpty = 0x203,
                   kErrAttnS = 0x204, kErrAttnP = 0x205, kErrAttnO = 0x206, kErrAttnFix = 0x207;

constexpr int kPromptThreads = 384;
constexpr int kStep = 64;      // keys per step
// The tensor core cuts off what lies below its fp32 sum's last place.  For keys
// of equal weight that was 0.6% of o after 2^20 of them: so after this many steps
// (2^15 keys, 0.02%) O is put away, added to what was put away before (in fp32,
// rounded to nearest), and begins anew.  So does the weights' sum: additions of equal
// weights to a long sum all round the same way.
constexpr int kFold = 512;

struct PromptArgs : AttentionArgs {
  int tiles;           // blocks per (head unit, batch row), documents: upper bound in all
  int head_units;      // blocks side by side: heads, or (packed) pairs of head tiles
  int packed;          // a tile holds several heads of a kv head
  int tile_rows;       // positions of a tile: 128, packed: q_len
  int tile_heads;      // heads of a tile: 1, packed: tile_rows * tile_heads <= 128
  int splits;          // shares of each sequence's keys
  // splits > 1, or more than kFold steps: fp32 [splits][batch][q_heads][q_len][head_dim]
  float* part_o;
  float* part_lse;     // splits > 1: fp32 [splits][batch][q_heads][q_len]
  int o_vec;           // rows of o can be written in 16-byte pieces
  uint64_t wait_limit_ns;
};

template <int DP>
struct PromptPlan {
  static constexpr int kCols = DP / 64;               // 128-byte wide column blocks of a tile
  static constexpr int kQ = kCols * 128 * 128;        // bytes of 128 rows of Q
  static constexpr int kKv = kCols * kStep * 128;     // bytes of a step's K or V
  // Heads of 128: two S buffers per tile, one block per SM.  Heads of 64: one S
  // buffer, so that two blocks share the SM's tensor memory (and its registers):
  // four tiles hide each other's latencies.
  static constexpr int kBuffers = DP == 128 ? 2 : 1;
  static constexpr int kBlocks = DP == 128 ? 1 : 2;   // per SM
  static constexpr int kColumns = DP == 128 ? 512 : 256;  // of tensor memory
  static constexpr int kSlot = 2 * kKv;               // V of a step, K of one ahead
  static constexpr int kStages = DP == 128 ? 5 : 4;
  // barriers, and for heads of 64, whose threads have no register to spare, what a row
  // keeps between the points where O is put away
  static constexpr bool kKeptInSmem = DP == 64;
  static constexpr int kSmem =
      2 * kQ + kStages * kSlot + 1024 + 512 + (kKeptInSmem ? 256 * 8 : 0);
};

// True in one thread of the (converged) warp.  The compiler then knows that
// one thread runs what follows: with `lane == 0` it walks the warp's active
// threads around every MMA, which took 81 to 87 cycles an MMA instead of the 65 that
// it takes then (128 x 128 x 16).
__device__ __forceinline__ bool elect_one() {
  uint32_t yes = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "@p mov.b32 %0, 1;\n\t}"
      : "+r"(yes));
  return yes != 0;
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// The warp's bounded wait, with every lane looking first: a phase that is
// already complete costs one look and a vote instead of a branch to one lane.
__device__ __forceinline__ bool wait_ready(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                           unsigned site, uint64_t limit_ns) {
  if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
  return mbar_wait_warp(bar, parity, abort_flag, site, limit_ns);
}

__device__ __forceinline__ void unpair(uint64_t v, float* a, float* b) {
  const float2 f = floats_of(v);
  *a = f.x;
  *b = f.y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float y;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

__device__ __forceinline__ uint64_t tanh_ratio2(uint64_t uu) {
  uint64_t p = fma2(uu, pair_of(kTanh4, kTanh4), pair_of(kTanh3, kTanh3));
  p = fma2(p, uu, pair_of(kTanh2, kTanh2));
  p = fma2(p, uu, pair_of(kTanh1, kTanh1));
  return fma2(p, uu, pair_of(1.0f, 1.0f));
}

template <int DP, int T, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kPromptThreads, PromptPlan<DP>::kBlocks)
    attention_prompt_kernel(const PromptArgs a, const __grid_constant__ CUtensorMap map_q,
                            const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v) {
  using P = PromptPlan<DP>;
  constexpr int kStages = P::kStages, kBuffers = P::kBuffers;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which rows and keys
  const int unit = blockIdx.x % a.head_units;
  const int batch_row = blockIdx.x / a.head_units % a.batch;
  // causal: longest first
  const int tile = a.tiles - 1 - static_cast<int>(blockIdx.x / a.head_units / a.batch);
  Sequence seq;
  int row0 = 0;
  if (!tile_sequence(a, tile, batch_row, a.packed ? a.tile_rows : 256, &seq, &row0)) return;
  const int length = seq.k1 - seq.k0;
  const int heads_per_kv = a.q_heads / a.kv_heads;
  // first head and position of each row tile; the kv head is the same
  int head_t[2] = {unit, unit}, row_t[2] = {row0, row0 + 128}, hk = unit / heads_per_kv;
  bool some_t[2] = {true, row0 + 128 < seq.q1};
  if (a.packed) {
    const int groups = heads_per_kv / a.tile_heads, pairs = (groups + 1) / 2;
    hk = unit / pairs;
    for (int t = 0; t < 2; ++t) {
      const int group = unit % pairs * 2 + t;
      head_t[t] = hk * heads_per_kv + group * a.tile_heads;
      row_t[t] = row0;
      some_t[t] = group < groups;
    }
  }
  // steps of each row tile: up to what its last position sees
  int steps_t[2];
  for (int t = 0; t < 2; ++t) {
    const int last = min(row_t[t] + a.tile_rows, seq.q1) - 1;
    steps_t[t] = some_t[t] ? (seq.seen(last, a.causal) + kStep - 1) / kStep : 0;
  }
  int begin = 0;
  if (a.splits > 1) {
    const int all = max(steps_t[0], steps_t[1]);
    const int share = (all + a.splits - 1) / a.splits;
    begin = share * static_cast<int>(blockIdx.y);
    for (int t = 0; t < 2; ++t) steps_t[t] = max(0, min(steps_t[t], begin + share) - begin);
  }
  const int steps = max(steps_t[0], steps_t[1]);

  // ---- shared memory
  uint8_t* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* q_tile = base;
  uint8_t* ring = base + 2 * P::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kStages * P::kSlot);
  uint64_t* q_full = bars;                 // [2]
  uint64_t* s_full = bars + 2;             // [2][buffers]
  uint64_t* p_full = bars + 6;             // [2][buffers]
  uint64_t* fixed = bars + 10;             // the last V's rows behind the end are cleared
  uint64_t* drain = bars + 11;             // [2]
  uint64_t* kv_full = bars + 13;           // [kStages]
  uint64_t* kv_empty = bars + 13 + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13 + 2 * kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* loads_issued = const_cast<int*>(abort_flag) + 1;

  const bool last_short =
      length % kStep != 0 && begin + steps == (length + kStep - 1) / kStep;
  // A slot of the ring holds what a tile's MMAs wait for together: K of the
  // first kBuffers steps, then V of a step and K of the step kBuffers ahead.
  const int slots = steps > 0 ? steps + 1 : 0;
  auto load_slot = [&](int i, int slot) {
    uint64_t* full = &kv_full[slot];
    const int first = i == 0 ? 0 : i - 1;  // steps of the two halves
    const int second = i == 0 && kBuffers == 1 ? steps : i + kBuffers - 1;
    mbar_arrive_expect_tx(full, second < steps ? 2 * P::kKv : P::kKv);
    uint8_t* to = ring + slot * P::kSlot;
    for (int c = 0; c < P::kCols; ++c) {
      tma_load_4d(to + c * (kStep * 128), i == 0 ? &map_k : &map_v, full, 64 * c,
                  seq.k0 + (begin + first) * kStep, hk, seq.batch);
    }
    for (int c = 0; c < P::kCols && second < steps; ++c) {
      tma_load_4d(to + P::kKv + c * (kStep * 128), &map_k, full, 64 * c,
                  seq.k0 + (begin + second) * kStep, hk, seq.batch);
    }
  };
  if (warp == 8) {
    tmem_alloc(tmem_slot, P::kColumns);
    tmem_relinquish();
  } else if (warp == 10) {
    // barriers 0 .. 12 + 2 kStages in their order above, one per lane
    for (int i = lane; i < 13 + 2 * kStages; i += 32) {
      mbar_init(&bars[i], i >= 6 && i < 10 ? 4           // p_full: a lane of each warp
                          : i == 10        ? 32          // fixed
                          : i >= 13 + kStages ? 2        // kv_empty: both MMA warps
                                              : 1);
    }
    if (lane == 0) {
      *abort_flag = 0;
      *loads_issued = 0;
    }
    fence_mbar_init();
    __syncwarp();
    if (elect_one()) {  // the first loads need no other warp
      for (int i = 0; i < min(slots, kStages); ++i) {
        if (i < 2 && steps_t[i] > 0) {
          mbar_arrive_expect_tx(&q_full[i], P::kCols * a.tile_rows * a.tile_heads * 128);
          for (int c = 0; c < P::kCols; ++c) {
            tma_load_4d(q_tile + i * P::kQ + c * 16384, &map_q, &q_full[i], 64 * c, row_t[i],
                        head_t[i], seq.batch);
          }
        }
        load_slot(i, i);
      }
    }
  }
  if (a.packed && warp < 8) {
    // rows of Q that no head fills: zeros, or what another block left there could
    // be NaN, for which a row would look for a new maximum at every step
    const int rows = a.tile_rows * a.tile_heads;
    for (int i = rows * 8 + static_cast<int>(threadIdx.x); i < 128 * 8; i += 256) {
      for (int c = 0; c < 2 * P::kCols; ++c) {
        *reinterpret_cast<uint4*>(q_tile + c * 16384 + i * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // TMEM columns: S buffer b of tile t (and P over it) at 64 (kBuffers t + b),
  // O of tile t behind them
  constexpr int kO = 2 * kBuffers * kStep;

  if (warp >= 8) {
    setmaxnreg_dec<P::kBlocks == 1 ? 120 : 48>();
    if (warp == 10) {
      // ------------------------------------------------ TMA loads
      if (elect_one()) {
        int issued = min(slots, kStages), slot = 0;
        uint32_t phase = 0;
        for (int i = kStages; i < slots; ++i) {
          if (!mbar_wait(&kv_empty[slot], phase, abort_flag, kErrAttnEmpty, a.wait_limit_ns)) break;
          load_slot(i, slot);
          issued = i + 1;
          if (++slot == kStages) {
            slot = 0;
            phase ^= 1u;
          }
        }
        *loads_issued = issued;
      }
      __syncwarp();
      // Rows of the last V behind the end, when all loads are issued: a wait from
      // the start would have the whole block's time for its limit.
      if (last_short && steps > 0) {
        const int last = (slots - 1) % kStages;
        if (mbar_wait_warp(&kv_full[last], ((slots - 1) / kStages) & 1, abort_flag, kErrAttnKv,
                           a.wait_limit_ns)) {
          uint8_t* v = ring + last * P::kSlot;
          const int from = length % kStep, pieces = (kStep - from) * 8;
          for (int e = lane; e < pieces * P::kCols; e += 32) {
            *reinterpret_cast<uint4*>(v + e / pieces * (kStep * 128) + from * 128 +
                                      e % pieces * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          mbar_arrive(fixed);
        }
      }
    } else if (warp < 10 && elect_one()) {
      // ------------------------------------------------ MMAs of tile t
      const int t = warp - 8, n = steps_t[t];
      const int ksteps = (a.head_dim + 15) / 16;
      const uint32_t idesc_s = make_idesc_f16(128, kStep, T == IE_DT_BF16, false);
      const uint32_t idesc_o = make_idesc_f16(128, ksteps * 16, T == IE_DT_BF16, true);
      const uint64_t q_desc = make_smem_desc(smem_u32(q_tile + t * P::kQ), 16, 1024, 2);
      const uint64_t k_desc = make_smem_desc(smem_u32(ring), 16, 1024, 2);
      const uint64_t v_desc = make_smem_desc(smem_u32(ring), kStep * 128, 1024, 2);
      const uint32_t s_tmem = tmem + kBuffers * kStep * t, o_tmem = tmem + kO + DP * t;
      int slot = 0;
      uint32_t phase = 0;
      auto advance = [&] {
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1u;
        }
      };
      // the slot is free once this tile's MMAs so far are done, or at once
      auto release = [&](int i, bool used) {
        if (used) tc_commit(&kv_empty[i]);
        else mbar_arrive(&kv_empty[i]);
      };
      // Unrolled: an MMA takes 33 to 65 cycles, a loop around it up to 86.
      auto scores = [&](int s, uint32_t k_offset) {  // S of step s = Q K^T
        const uint64_t kd = k_desc + (k_offset >> 4);
        const uint32_t d = s_tmem + kStep * (s % kBuffers);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          if (k < ksteps) {
            mma_f16(d, q_desc + (((k / 4) * 16384 + (k % 4) * 32) >> 4),
                    kd + (((k / 4) * (kStep * 128) + (k % 4) * 32) >> 4), idesc_s, k > 0);
          }
        }
      };
      bool ok = n == 0 || mbar_wait(&q_full[t], 0, abort_flag, kErrAttnQ, a.wait_limit_ns);
      if (ok && steps > 0) {
        ok = mbar_wait(&kv_full[0], 0, abort_flag, kErrAttnKv, a.wait_limit_ns);
        if (ok) {
          for (int s = 0; s < kBuffers; ++s) {
            if (s < n) scores(s, s * P::kKv);
            if (n > 0) tc_commit(&s_full[2 * t + s]);
          }
          release(0, n > 0);
          advance();
        }
      }
      for (int s = 0; ok && s < steps; ++s) {
        ok = last_short && s == steps - 1
                 ? mbar_wait(fixed, 0, abort_flag, kErrAttnFix, a.wait_limit_ns)
                 : mbar_wait(&kv_full[slot], phase, abort_flag, kErrAttnKv, a.wait_limit_ns);
        if (ok && s < n) {
          ok = mbar_wait(&p_full[2 * t + s % kBuffers], (s / kBuffers) & 1, abort_flag, kErrAttnP,
                         a.wait_limit_ns);
        }
        if (!ok) break;
        if (s < n) {
          tc_fence_after();
          const uint64_t vd = v_desc + ((slot * P::kSlot) >> 4);
          const uint32_t p = s_tmem + kStep * (s % kBuffers);
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k) {
            mma_f16_ta(o_tmem, p + 8 * k, vd + ((k * 2048) >> 4), idesc_o,
                       s % kFold > 0 || k > 0);
          }
          if (s + kBuffers < n) scores(s + kBuffers, slot * P::kSlot + P::kKv);
          // S of that step is there, or (behind the last) just O += P V of step s
          tc_commit(&s_full[2 * t + s % kBuffers]);
        }
        release(slot, s < n);
        advance();
      }
      // every MMA done before tensor memory is released, on the abort path too
      tc_commit(&drain[t]);
      int dummy_abort = 0;
      mbar_wait(&drain[t], 0, &dummy_abort, kErrAttnO, a.wait_limit_ns);
    }
  } else {
    // ------------------------------------------------ rows
    setmaxnreg_inc<P::kBlocks == 1 ? 192 : 96>();
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;
    const int row = row_t[t] + r % a.tile_rows, h = head_t[t] + r / a.tile_rows;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + kBuffers * kStep * t + lanes, o_at = tmem + kO + DP * t + lanes;
    const bool valid = some_t[t] && r < a.tile_rows * a.tile_heads && row < seq.q1;
    const int seen = valid ? seq.seen(row, a.causal) : 0;
    // what every row of this tile sees, and the first row's place
    const int all_see = some_t[t] ? seq.seen(row_t[t], a.causal) : 0;
    const int all_past = some_t[t] ? seq.place(row_t[t]) : 0;
    constexpr float kLog2e = 1.4426950408889634f;
    const float scale = a.scale * kLog2e;
    const float cap_arg = CAP ? cap_argument(a) : 0.0f;
    const float cap_out = CAP ? a.softcap * kLog2e : 0.0f;
    // scores up to here go through the polynomial
    const float cap_limit = CAP ? kTanhLimit / fabsf(cap_arg) : 0.0f;
    const float slope = BIAS && valid && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.0f;
    const int place = valid ? seq.place(row) : 0;
    // x is the score in units of log2 e (plain: before the scale)
    constexpr bool kScaled = CAP || BIAS;
    const float to_log2 = kScaled ? 1.0f : scale;
    auto capped = [&](float s) {
      const float u = ex2(s * (2.0f * kLog2e * cap_arg));
      return cap_out - __fdividef(2.0f * cap_out, 1.0f + u);
    };
    auto capped_pair = [&](uint64_t s) {
      const uint64_t u = mul2(s, pair_of(cap_arg, cap_arg));
      return mul2(mul2(s, pair_of(scale, scale)), tanh_ratio2(mul2(u, u)));
    };

    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    const int n = steps_t[t];
    // the row among all rows, and among the shares' rows
    auto lse_at = [&] {
      return (static_cast<int64_t>(seq.batch) * a.q_heads + h) * a.q_len + row;
    };
    auto part_at = [&] {
      return blockIdx.y * (static_cast<int64_t>(a.batch) * a.q_heads * a.q_len) + lse_at();
    };
    // the maximum in use when O was put away, and the weights' sum then
    float2 kept = make_float2(-INFINITY, 0.0f);
    float2* const kept_at =
        P::kKeptInSmem ? reinterpret_cast<float2*>(ring + kStages * P::kSlot + 512) + threadIdx.x
                       : &kept;
    auto kept_factor = [&](float m_kept) {
      return m_kept == m ? 1.0f : ex2((m_kept - m) * to_log2);
    };
#pragma unroll 1
    for (int s = 0; ok && s < n;) {
      if (s > 0) {
        // O += P V of the step before comes before S of this step (one buffer) or of the next
        const int then = s + kBuffers - 1;
        if (!wait_ready(&s_full[2 * t + then % kBuffers], (then / kBuffers) & 1, abort_flag,
                        kErrAttnO, a.wait_limit_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float2 before = s == kFold ? make_float2(m, 0.0f) : *kept_at;
        const float factor = kept_factor(before.x);
        float4* to = reinterpret_cast<float4*>(a.part_o + part_at() * a.head_dim);
#pragma unroll 1
        for (int c = 0; c < a.head_dim; c += 32, to += 8) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld_32x32b_x32(o_at + c, o);
          tmem_ld_wait(o);
          if (valid) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (c + 4 * i >= a.head_dim) break;
              const float4 old = s == kFold ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : to[i];
              to[i] = make_float4(fmaf(old.x, factor, __uint_as_float(o[4 * i])),
                                  fmaf(old.y, factor, __uint_as_float(o[4 * i + 1])),
                                  fmaf(old.z, factor, __uint_as_float(o[4 * i + 2])),
                                  fmaf(old.w, factor, __uint_as_float(o[4 * i + 3])));
            }
          }
        }
        __syncwarp();
        *kept_at = make_float2(m, fmaf(before.y, factor, l));
        l = 0.0f;
      }
      const int stop = min(n, s + kFold);
#pragma unroll 1
      for (; s < stop; ++s) {
        if (!wait_ready(&s_full[2 * t + s % kBuffers], (s / kBuffers) & 1, abort_flag, kErrAttnS,
                        a.wait_limit_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t s_now = s_at + kStep * (s % kBuffers);
        const int key0 = (begin + s) * kStep;
        float x[kStep];
        {
          uint32_t sr[2][32];
          tmem_ld_32x32b_x32(s_now, sr[0]);
          tmem_ld_32x32b_x32(s_now + 32, sr[1]);
          tmem_ld_wait(sr[0]);
          tmem_ld_wait(sr[1]);
#pragma unroll
          for (int e = 0; e < kStep; ++e) x[e] = __uint_as_float(sr[e / 32][e % 32]);
        }
        if constexpr (CAP) {
          float hi[2] = {x[0], x[0]}, lo[2] = {x[0], x[0]};
#pragma unroll
          for (int e = 0; e < kStep; e += 4) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              hi[c] = max3(hi[c], x[e + 2 * c], x[e + 2 * c + 1]);
              lo[c] = min3(lo[c], x[e + 2 * c], x[e + 2 * c + 1]);
            }
          }
          const bool small = max_nan(hi[0], hi[1]) <= cap_limit &&
                             min3(lo[0], lo[1], lo[1]) >= -cap_limit;
          if (__all_sync(0xFFFFFFFFu, small)) {
#pragma unroll
            for (int e = 0; e < kStep; e += 2) {
              unpair(capped_pair(pair_of(x[e], x[e + 1])), &x[e], &x[e + 1]);
            }
          } else if (a.softcap <= kSmallCap) {
#pragma unroll
            for (int e = 0; e < kStep; ++e) x[e] = capped(x[e]);
          } else {
#pragma unroll
            for (int e = 0; e < kStep; e += 2) {
              float t[2];
              unpair(capped_pair(pair_of(x[e], x[e + 1])), &t[0], &t[1]);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                x[e + k] = fabsf(x[e + k]) <= cap_limit ? t[k] : capped(x[e + k]);
              }
            }
          }
        }
        if constexpr (BIAS) {
          // subtracted as integers: fp32 does not hold every place behind 2^24
          const float from = static_cast<float>(place - key0);
          const float factor = CAP ? 1.0f : scale;
          if (all_past >= key0 + kStep - 1) {  // no key lies ahead of its row
            const uint64_t f2 = pair_of(factor, factor), s2 = pair_of(slope, slope);
            const uint64_t c2 = pair_of(-slope * from, -slope * from);
#pragma unroll
            for (int e = 0; e < kStep; e += 2) {
              const uint64_t c =
                  fma2(s2, pair_of(static_cast<float>(e), static_cast<float>(e + 1)), c2);
              const uint64_t y = CAP ? add2(pair_of(x[e], x[e + 1]), c)
                                     : fma2(pair_of(x[e], x[e + 1]), f2, c);
              unpair(y, &x[e], &x[e + 1]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < kStep; ++e) {
              x[e] = x[e] * factor - slope * fabsf(from - static_cast<float>(e));
            }
          }
        }
        if (key0 + kStep > all_see) {
          const int vis = seen - key0;
#pragma unroll
          for (int e = 0; e < kStep; ++e) x[e] = e < vis ? x[e] : -INFINITY;
        }
        float hi[4] = {m, m, m, m};
#pragma unroll
        for (int e = 0; e < kStep; e += 8) {
#pragma unroll
          for (int c = 0; c < 4; ++c) hi[c] = max3(hi[c], x[e + 2 * c], x[e + 2 * c + 1]);
        }
        const float top = max_nan(max3(hi[0], hi[1], hi[2]), hi[3]);
        // The maximum in use moves only when it grew by more than 2^8: until then
        // the weights stay below 2^8 (fp16: 2^15), which the types hold as well as 1.
        float factor = 1.0f;
        const bool moved = !((top - m) * to_log2 <= 8.0f) && top != -INFINITY;
        if (moved) {
          factor = m == -INFINITY ? 1.0f : ex2((m - top) * to_log2);
          m = top;
        }
        if (s > 0 && __any_sync(0xFFFFFFFFu, moved)) {
          l *= factor;
          // O += P V of the step before this one comes before S of this step (one
          // buffer) or of the next
          if (kBuffers == 2 && !wait_ready(&s_full[2 * t + ((s + 1) & 1)], ((s + 1) >> 1) & 1,
                                           abort_flag, kErrAttnO, a.wait_limit_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(o_at + 16 * c, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st_32x32b_x16(o_at + 16 * c, o);
          }
        }
        const float base = m == -INFINITY ? 0.0f : m * to_log2 - kWeightShift<T>;
        const uint64_t to2 = pair_of(to_log2, to_log2), base2 = pair_of(-base, -base);
        uint64_t sum[2] = {0, 0};
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          uint64_t y = pair_of(x[2 * e], x[2 * e + 1]);
          y = kScaled ? add2(y, base2) : fma2(y, to2, base2);
          float p0, p1;
          unpair(y, &p0, &p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          sum[e & 1] = add2(sum[e & 1], pair_of(p0, p1));
          p[e] = pack_pair<T>(p0, p1);
        }
        tmem_st_32x32b_x32(s_now, p);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + s % kBuffers]);
        float s0, s1;
        unpair(add2(sum[0], sum[1]), &s0, &s1);
        l += s0 + s1;
      }
    }
    if (n > 0 && ok) {
      // what follows the last step's O += P V
      const int behind = n + kBuffers - 1;
      ok = wait_ready(&s_full[2 * t + behind % kBuffers], (behind / kBuffers) & 1, abort_flag,
                      kErrAttnO, a.wait_limit_ns);
    }
    tc_fence_after();
    if (ok) {
      float share_kept = 0.0f;  // what was put away counts by
      if (n > kFold) {
        share_kept = kept_factor(kept_at->x);
        l = fmaf(kept_at->y, share_kept, l);
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const bool none = l == 0.0f;
      const float lse =
          none ? -INFINITY : (m * to_log2 + (log2f(l) - kWeightShift<T>)) * 0.6931471805599453f;
      if (valid) {
        if (a.splits > 1) {
          a.part_lse[part_at()] = lse;
        } else if (a.lse != nullptr) {
          a.lse[lse_at()] = lse;
        }
      }
      const int64_t oo = static_cast<int64_t>(seq.batch) * a.o_stride[0] +
                         static_cast<int64_t>(row) * a.o_stride[1] +
                         static_cast<int64_t>(h) * a.o_stride[2];
      float* part = a.part_o + part_at() * a.head_dim;  // splits > 1, or n > kFold
      // 32 columns at a time through the warp's share of the tile's Q (its MMAs
      // are done): a row's pieces are written side by side by neighbouring
      // threads, not by the one thread that holds the row.
      uint8_t* stage = q_tile + t * P::kQ + (warp & 3) * 4096;
      // 32 rows of `pieces` 16-byte pieces each; row r of `to` is lane r's
      auto write_rows = [&](int pieces, uint64_t to, int limit) {
        __syncwarp();
        const int c = lane % pieces;
#pragma unroll 1
        for (int r0 = lane / pieces; r0 < 32; r0 += 32 / pieces) {
          const uint64_t to_r = __shfl_sync(0xFFFFFFFFu, to, r0);
          const bool write = __shfl_sync(0xFFFFFFFFu, static_cast<int>(valid), r0) != 0;
          if (write && c < limit) {
            *reinterpret_cast<uint4*>(to_r + 16 * c) =
                *reinterpret_cast<const uint4*>(stage + (r0 * pieces + (c ^ (r0 & (pieces - 1)))) * 16);
          }
        }
        __syncwarp();
      };
      auto put = [&](int pieces, int c, uint4 v) {
        *reinterpret_cast<uint4*>(stage + (lane * pieces + (c ^ (lane & (pieces - 1)))) * 16) = v;
      };
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        if (32 * c >= a.head_dim) break;
        uint32_t acc[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(o_at + 32 * c, acc);
          tmem_ld_wait(acc);
        }
        const int left = a.head_dim - 32 * c;  // a multiple of 8
        if (n > kFold && valid) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            if (e < left) {
              const float4 old = *reinterpret_cast<const float4*>(part + 32 * c + e);
              const float o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                acc[e + i] =
                    __float_as_uint(fmaf(o[i], share_kept, __uint_as_float(acc[e + i])));
              }
            }
          }
        }
        __syncwarp();
        float y[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) y[e] = none ? 0.0f : __uint_as_float(acc[e]) * inv;
        if (a.splits > 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            put(8, e, make_uint4(__float_as_uint(y[4 * e]), __float_as_uint(y[4 * e + 1]),
                                 __float_as_uint(y[4 * e + 2]), __float_as_uint(y[4 * e + 3])));
          }
          write_rows(8, reinterpret_cast<uint64_t>(part + 32 * c), left / 4);
          continue;
        }
        uint16_t* o = static_cast<uint16_t*>(a.o) + oo + 32 * c;
        uint32_t hi[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) hi[e] = pack_pair<T>(y[2 * e], y[2 * e + 1]);
        if (a.o_vec) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            put(4, e, make_uint4(hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3]));
          }
          write_rows(4, reinterpret_cast<uint64_t>(o), left / 8);
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (e < left) o[e] = static_cast<uint16_t>(hi[e / 2] >> (16 * (e & 1)));
          }
        }
        if (a.o_lo != 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            hi[e] = pack_pair<T>(y[2 * e] - __uint_as_float(hi[e] << 16),
                                 y[2 * e + 1] - __uint_as_float(hi[e] & 0xFFFF0000u));
          }
          if (a.o_vec) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              put(4, e, make_uint4(hi[4 * e], hi[4 * e + 1], hi[4 * e + 2], hi[4 * e + 3]));
            }
            write_rows(4, reinterpret_cast<uint64_t>(o + a.o_lo), left / 8);
          } else if (valid) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (e < left) o[a.o_lo + e] = static_cast<uint16_t>(hi[e / 2] >> (16 * (e & 1)));
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
      if (steps_t[t] > 0) mbar_wait(&q_full[t], 0, &dummy_abort, kErrAttnQ, a.wait_limit_ns);
    }
    const int issued = *loads_issued;
    for (int i = max(0, issued - kStages); i < issued; ++i) {
      mbar_wait(&kv_full[i % kStages], (i / kStages) & 1, &dummy_abort, kErrAttnKv,
                a.wait_limit_ns);
    }
  }
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, P::kColumns);
  }
}

}  // namespace ie_cuda
