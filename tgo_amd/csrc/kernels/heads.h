// heads.h -- rows of heads for the kernels that rotate them (rope.hip, cache_rows.hip):
// loads and stores of runs of elements, and a pair's angle.
#pragma once

#include "operators.h"

namespace tgohip {

// N consecutive elements as f32: 16-byte loads where N allows, else 8.
template <int N, bool F16>
__device__ __forceinline__ void rope_load(const void* p, int64_t off, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = F16 ? (float)((const half_t*)p)[off] : ((const float*)p)[off];
  } else if constexpr (N == 2) {
    v[0] = F16 ? (float)((const half_t*)p)[off] : ((const float*)p)[off];
    v[1] = F16 ? (float)((const half_t*)p)[off + 1] : ((const float*)p)[off + 1];
  } else if constexpr (!F16) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4_t f = *(const float4_t*)((const float*)p + off + j);
#pragma unroll
      for (int e = 0; e < 4; e++) v[j + e] = f[e];
    }
  } else if constexpr (N == 4) {
    const half4_t h = *(const half4_t*)((const half_t*)p + off);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)h[e];
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      const half8_t h = *(const half8_t*)((const half_t*)p + off + j);
#pragma unroll
      for (int e = 0; e < 8; e++) v[j + e] = (float)h[e];
    }
  }
}
template <int N, bool F16>
__device__ __forceinline__ void rope_store(void* p, int64_t off, const float (&v)[N]) {
  if constexpr (N <= 2) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      if (F16) ((half_t*)p)[off + j] = (half_t)v[j];
      else ((float*)p)[off + j] = v[j];
    }
  } else if constexpr (!F16) {
#pragma unroll
    for (int j = 0; j < N; j += 4) *(float4_t*)((float*)p + off + j) = float4_t{v[j], v[j + 1], v[j + 2], v[j + 3]};
  } else if constexpr (N == 4) {
    *(half4_t*)((half_t*)p + off) = half4_t{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      half8_t h;
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = (half_t)v[j + e];
      *(half8_t*)((half_t*)p + off + j) = h;
    }
  }
}

// cos and sin of one pair of one row, times m. The turns are reduced in double
// (positions to 2^31 keep 2^-23 of a turn and better), the rest in f32 with the
// angle's second half as a first-order correction: within 2 ulp of 1.
__device__ __forceinline__ float2 rope_angle(int32_t pos, double turns_per_position, float m) {
#pragma clang fp contract(off)  // every kernel that inlines this computes the same bits
  double x = (double)pos * turns_per_position;
  x = 2.0 * (x - rint(x));
  const float hi = (float)x, lo = (float)(x - (double)hi) * 3.14159265f;
  float s, c;
  sincospif(hi, &s, &c);
  return float2{m * fmaf(-lo, s, c), m * fmaf(lo, c, s)};
}

}  // namespace tgohip
