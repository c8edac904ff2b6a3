// Device helpers of the 8-bit pool: e4m3 conversions, a page's power-of-two
// scale, and the search for the sequence that owns a row of a ragged batch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "yl_kvpath.h"

namespace ylk {

// Two e4m3 codes (low byte first) -> two halves.  Exact: every e4m3 value is a
// normal half.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return h;
}

// Two floats -> two e4m3 codes (`lo` in the low byte), to nearest even,
// magnitudes above 448 to 448, NaN to e4m3's NaN.
__device__ __forceinline__ uint16_t float2_to_e4m3x2(float lo, float hi) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
  return c;
}

__device__ __forceinline__ float2 half2_bits_to_float2(uint32_t h) {
  __half2 v;
  memcpy(&v, &h, 4);
  return __half22float2(v);
}

// The 16-bit types of the entry points: conversions of packed pairs, the bit
// pattern of infinity (every larger magnitude pattern is a NaN) and the
// largest finite value.
struct Bf16 {
  static constexpr uint32_t kInf = 0x7f80u;
  static constexpr float kMax = 3.38953139e38f;
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
  }
};
struct Fp16 {
  static constexpr uint32_t kInf = 0x7c00u;
  static constexpr float kMax = 65504.f;
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return half2_bits_to_float2(w); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t w;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
  }
};

constexpr int kScaleExpMin = -100;
constexpr int kScaleExpMax = 120;

// 2^ceil(log2(amax / 448)) with its exponent clamped.  With amax = 1.m * 2^e
// and 448 = 1.75 * 2^8 the exponent is e - 8 where 1.m <= 1.75, else e - 7; a
// subnormal or zero amax falls to the clamp.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t b = __float_as_uint(amax);
  int k = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = max(kScaleExpMin, min(kScaleExpMax, k));
  return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

__device__ __forceinline__ bool good_scale(float s) { return s > 0.f && s < __int_as_float(0x7f800000); }

// The largest i in [0, n) with key(i) <= x, for key(0) <= x and key not
// decreasing, found by a whole warp: 32 probes a round, so n <= 1024 takes two
// dependent loads.  Any key values give an i in range.
template <typename Key>
__device__ __forceinline__ int warp_find(int n, int64_t x, int lane, Key key) {
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 31) >> 5;
    const int i = lo + lane * step;
    const bool le = lane == 0 || (lane * step < len && key(i) <= x);
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, le));
    len = min(step, len - last * step);
    lo += last * step;
  }
  return lo;
}

}  // namespace ylk
