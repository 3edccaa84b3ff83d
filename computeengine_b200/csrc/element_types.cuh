// Element types of the group norm, rotary and attention kernels: single
// element loads and stores, converting from and to fp32 (one rounding).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/ie_cuda_conv.h"

namespace ie_cuda {

// Bytes of one stored element (BF16X2: of one element of one plane).
__host__ __device__ constexpr int element_bytes(int type) { return type == IE_DT_F32 ? 4 : 2; }

template <int T>
__device__ __forceinline__ float load_element(const void* p, int64_t i) {
  if constexpr (T == IE_DT_F32) {
    return static_cast<const float*>(p)[i];
  } else if constexpr (T == IE_DT_F16) {
    return __half2float(static_cast<const __half*>(p)[i]);
  } else {
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
}

template <int T>
__device__ __forceinline__ void store_element(void* p, int64_t i, float v) {
  if constexpr (T == IE_DT_F32) {
    static_cast<float*>(p)[i] = v;
  } else if constexpr (T == IE_DT_F16) {
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  } else {
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  }
}

// B bytes at p, which is aligned to min(B, 16).
template <int B>
struct Bytes {
  uint32_t r[(B + 3) / 4];
};

template <int B>
__device__ __forceinline__ Bytes<B> load_bytes(const void* p) {
  Bytes<B> v;
  if constexpr (B % 16 == 0) {
#pragma unroll
    for (int i = 0; i < B / 16; ++i) {
      const uint4 q = static_cast<const uint4*>(p)[i];
      v.r[4 * i] = q.x;
      v.r[4 * i + 1] = q.y;
      v.r[4 * i + 2] = q.z;
      v.r[4 * i + 3] = q.w;
    }
  } else if constexpr (B == 8) {
    const uint2 q = *static_cast<const uint2*>(p);
    v.r[0] = q.x;
    v.r[1] = q.y;
  } else if constexpr (B == 4) {
    v.r[0] = *static_cast<const uint32_t*>(p);
  } else {
    static_assert(B == 2, "2, 4, 8 or a multiple of 16 bytes");
    v.r[0] = *static_cast<const uint16_t*>(p);
  }
  return v;
}

template <int B>
__device__ __forceinline__ void store_bytes(void* p, const Bytes<B>& v) {
  if constexpr (B % 16 == 0) {
#pragma unroll
    for (int i = 0; i < B / 16; ++i) {
      static_cast<uint4*>(p)[i] =
          make_uint4(v.r[4 * i], v.r[4 * i + 1], v.r[4 * i + 2], v.r[4 * i + 3]);
    }
  } else if constexpr (B == 8) {
    *static_cast<uint2*>(p) = make_uint2(v.r[0], v.r[1]);
  } else if constexpr (B == 4) {
    *static_cast<uint32_t*>(p) = v.r[0];
  } else {
    static_assert(B == 2, "2, 4, 8 or a multiple of 16 bytes");
    *static_cast<uint16_t*>(p) = static_cast<uint16_t>(v.r[0]);
  }
}

// Two 16-bit elements as fp32, and back with one rounding each.
template <int T>
__device__ __forceinline__ float2 unpack_pair(uint32_t r) {
  if constexpr (T == IE_DT_F16) {
    return __half22float2(*reinterpret_cast<const __half2*>(&r));
  } else {
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
  }
}

template <int T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t y;
  if constexpr (T == IE_DT_F16) {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  }
  return y;
}

// W elements of type T as they lie in memory, to and from fp32.
template <int T, int W>
__device__ __forceinline__ void to_floats(const Bytes<W * element_bytes(T)>& v, float (&f)[W]) {
  if constexpr (T == IE_DT_F32) {
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = __uint_as_float(v.r[i]);
  } else if constexpr (W == 1) {
    f[0] = unpack_pair<T>(v.r[0]).x;
  } else {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float2 q = unpack_pair<T>(v.r[i]);
      f[2 * i] = q.x;
      f[2 * i + 1] = q.y;
    }
  }
}

template <int T, int W>
__device__ __forceinline__ Bytes<W * element_bytes(T)> from_floats(const float (&f)[W]) {
  Bytes<W * element_bytes(T)> v;
  if constexpr (T == IE_DT_F32) {
#pragma unroll
    for (int i = 0; i < W; ++i) v.r[i] = __float_as_uint(f[i]);
  } else if constexpr (W == 1) {
    v.r[0] = pack_pair<T>(f[0], 0.0f) & 0xFFFFu;
  } else {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) v.r[i] = pack_pair<T>(f[2 * i], f[2 * i + 1]);
  }
  return v;
}

// 1 / x for 1 <= x on the special function unit, 0 from 2^126 on.
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// x / d for x * d < 2^32, with m = 2^32 / d rounded up: x * m / 2^32 is too
// large by less than x / 2^32 < 1 / d.
struct SmallDivisor {
  uint32_t d, m;
  __host__ __device__ static SmallDivisor of(uint32_t d) {
    return {d, d == 1 ? 0u : static_cast<uint32_t>(((uint64_t{1} << 32) + d - 1) / d)};
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    return d == 1 ? x : __umulhi(x, m);
  }
};

}  // namespace ie_cuda
