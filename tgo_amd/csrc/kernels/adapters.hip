// adapters.hip -- low-rank adapters of many requests beside a shared projection:
// y[t] = base[t] + s (x[t] . down^T) . up^T with the adapter of the request that
// row t belongs to, or y[t] = base[t] where it has none.
//
// Rows are sorted by adapter (AdapterTile: up to 16 TB rows of one adapter), so
// each product is a small matrix product and an adapter is read once per tile.
// With ranks up to 128 the work is far below the matrix unit's: x, base and y
// bound it, and for a few rows the two launches' latency.
//   adapter_down_kernel  u = x . down^T over a share of K, f32 planes
//   adapter_up_kernel    sums the planes in order, y = base + s u . up^T
// Both use v_mfma_f32_16x16x32_f16 (16x16x16 for rank 16): lane (l16, q) =
// (lane % 16, lane / 16) holds row or column l16 of an operand at k 8q + [0,8),
// and of the result column l16, rows 4q + [0,4).
#include "operators.h"

#include <algorithm>

namespace tgohip {

// x of rows `off` elements in, at k .. k + 8: the hi part, and lo where there is one.
template <int XK>
__device__ __forceinline__ void adapter_load_x(const AdapterArgs& a, int64_t off, half8_t& hi, half8_t& lo) {
  if constexpr (XK == XK_F32) {
    const float4_t u = *(const float4_t*)((const float*)a.x + off), v = *(const float4_t*)((const float*)a.x + off + 4);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float f = j < 4 ? u[j & 3] : v[j & 3];
      hi[j] = (half_t)f;
      lo[j] = (half_t)(f - (float)hi[j]);
    }
  } else {
    hi = *(const half8_t*)((const half_t*)a.x + off);
    if constexpr (XK == XK_X2) lo = *(const half8_t*)((const half_t*)a.x + (int64_t)a.T * a.K + off);
  }
}

// Waves take 32-k steps of the workgroup's share of K in turn, so that every
// wave streams its own lines of x and down, and their sums meet in LDS.
template <int XK, int TB, int RB>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a) {
  __shared__ float part[4][16][RB * 16];
  const AdapterTile t = a.tiles[blockIdx.x];
  if (t.adapter < 0) return;
  const AdapterEntry e = a.table[t.adapter];
  if (e.rank_pad == 0 || e.rank_pad > RB * 16) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
  const int nrb = e.rank_pad / 16, ntb = (t.n + 15) / 16;
  const int steps = a.K / 32;
  const int s0 = (int)((int64_t)steps * blockIdx.y / gridDim.y), s1 = (int)((int64_t)steps * (blockIdx.y + 1) / gridDim.y);
  int64_t row[TB];
#pragma unroll
  for (int b = 0; b < TB; b++) row[b] = (int64_t)a.perm[t.start + min(b * 16 + l16, t.n - 1)] * a.K + 8 * q;
  const half_t* dn = e.down + (int64_t)l16 * a.K + 8 * q;
  float4_t acc[TB][RB] = {};
#pragma unroll 2
  for (int s = s0 + wave; s < s1; s += 4) {
    half8_t d[RB], hi[TB], lo[TB];
#pragma unroll
    for (int b = 0; b < TB; b++)
      if (b < ntb) adapter_load_x<XK>(a, row[b] + 32 * s, hi[b], lo[b]);
#pragma unroll
    for (int r = 0; r < RB; r++)
      if (r < nrb) d[r] = *(const half8_t*)(dn + (int64_t)r * 16 * a.K + 32 * s);
#pragma unroll
    for (int b = 0; b < TB; b++)
#pragma unroll
      for (int r = 0; r < RB; r++)
        if (b < ntb && r < nrb) {
          acc[b][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[b], d[r], acc[b][r], 0, 0, 0);
          if (XK != XK_F16) acc[b][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[b], d[r], acc[b][r], 0, 0, 0);
        }
  }
  float* u = a.u + ((int64_t)blockIdx.y * a.T + t.start) * kAdapterMaxRank;
#pragma unroll
  for (int b = 0; b < TB; b++) {
    if (b >= ntb) break;
    if (b) __syncthreads();
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) part[wave][4 * q + i][r * 16 + l16] = acc[b][r][i];
    __syncthreads();
    for (int i = tid; i < 16 * e.rank_pad; i += 256) {
      const int m = i / e.rank_pad, r = i - m * e.rank_pad;
      if (b * 16 + m < t.n)
        u[(b * 16 + m) * kAdapterMaxRank + r] = (part[0][m][r] + part[1][m][r]) + (part[2][m][r] + part[3][m][r]);
    }
  }
}

template <bool YF16>
__device__ __forceinline__ float4_t adapter_load_base(const AdapterArgs& a, int64_t off) {
  if (!a.base) return float4_t{0.f, 0.f, 0.f, 0.f};
  if constexpr (YF16) {
    const half4_t h = *(const half4_t*)((const half_t*)a.base + off);
    return float4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
  }
  return *(const float4_t*)((const float*)a.base + off);
}
template <bool YF16>
__device__ __forceinline__ void adapter_store_y(const AdapterArgs& a, int64_t off, float4_t v) {
  if constexpr (YF16) *(half4_t*)((half_t*)a.y + off) = half4_t{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
  else *(float4_t*)((float*)a.y + off) = v;
}

// Columns [a.cols * blockIdx.y, + a.cols) of a tile's rows, 16 columns a wave at a
// time: up's 16 rows are the A operand, so a lane holds four neighbouring columns
// of row l16 of y.
template <int TB, int RB, bool YF16>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a) {
  constexpr int KB = RB == 1 ? 1 : RB / 2;  // products along the rank: 32 wide, or one 16 wide
  __shared__ __attribute__((aligned(16))) float us[TB * 16][RB * 16 + 4];
  const AdapterTile t = a.tiles[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.y * a.cols, n1 = min(n0 + a.cols, a.N);
  AdapterEntry e{};
  if (t.adapter >= 0) e = a.table[t.adapter];
  const int ntb = (t.n + 15) / 16;
  // an adapter of a larger rank than the launch was captured for: its rows are NaN
  if (e.rank_pad > RB * 16) {
    e.rank_pad = RB * 16;
    e.scale = NAN;
  }
  if (e.rank_pad == 0) {
    if (a.base == a.y) return;
    const int w = (n1 - n0) / 4;
    for (int i = tid; i < t.n * w; i += 256) {
      const int m = i / w;
      const int64_t off = (int64_t)a.perm[t.start + m] * a.N + n0 + 4 * (i - m * w);
      adapter_store_y<YF16>(a, off, adapter_load_base<YF16>(a, off));
    }
    return;
  }
  for (int i = tid; i < TB * 16 * RB * 16; i += 256) {
    const int m = i / (RB * 16), r = i - m * (RB * 16);
    float s = 0.f;
    if (m < t.n && r < e.rank_pad)
      for (int p = 0; p < a.splits; p++) s += a.u[((int64_t)p * a.T + t.start + m) * kAdapterMaxRank + r];
    us[m][r] = s;
  }
  __syncthreads();
  // u of row l16 of each block as an f16 pair, scaled by a power of two to a
  // largest value in [1, 2): 22 bits of it, wherever f16's range ends
  half8_t uh[TB][KB], ul[TB][KB];
  float scale[TB];
  int64_t row[TB];
  const int kq = RB == 1 ? 4 * q : 8 * q;
#pragma unroll
  for (int b = 0; b < TB; b++) {
    row[b] = (int64_t)a.perm[t.start + min(b * 16 + l16, t.n - 1)] * a.N + 4 * q;
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < KB; k++)
#pragma unroll
      for (int j = 0; j < (RB == 1 ? 4 : 8); j++) top = fmaxf(top, fabsf(us[b * 16 + l16][32 * k + kq + j]));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int ex = (int)((__float_as_uint(top) >> 23) & 255) - 127;
    ex = top > 0.f && ex < 128 ? max(-100, min(100, ex)) : 0;
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
    scale[b] = e.scale * __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
    for (int k = 0; k < KB; k++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float f = RB == 1 && j >= 4 ? 0.f : us[b * 16 + l16][32 * k + kq + j] * down;
        uh[b][k][j] = (half_t)f;
        ul[b][k][j] = (half_t)(f - (float)uh[b][k][j]);
      }
  }
  const int nkb = RB == 1 ? 1 : (e.rank_pad + 31) / 32;
#pragma unroll 2
  for (int n = n0 + 16 * wave; n < n1; n += 64) {
    const half_t* up = e.up + (int64_t)(n + l16) * e.rank_pad + kq;
    half8_t w[KB];
    float4_t base[TB];
#pragma unroll
    for (int k = 0; k < KB; k++) {
      if constexpr (RB == 1) {
        const half4_t h = *(const half4_t*)up;
        w[0] = half8_t{h[0], h[1], h[2], h[3], 0, 0, 0, 0};
      } else {
        w[k] = half8_t{};
        if (k < nkb && 32 * k + kq < e.rank_pad) w[k] = *(const half8_t*)(up + 32 * k);
      }
    }
#pragma unroll
    for (int b = 0; b < TB; b++)
      if (b < ntb) base[b] = adapter_load_base<YF16>(a, row[b] + n);
#pragma unroll
    for (int b = 0; b < TB; b++) {
      if (b >= ntb) break;
      float4_t acc = {};
      if constexpr (RB == 1) {
        const half4_t w4 = {w[0][0], w[0][1], w[0][2], w[0][3]};
        const half4_t h4 = {uh[b][0][0], uh[b][0][1], uh[b][0][2], uh[b][0][3]};
        const half4_t l4 = {ul[b][0][0], ul[b][0][1], ul[b][0][2], ul[b][0][3]};
        acc = __builtin_amdgcn_mfma_f32_16x16x16f16(w4, l4, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x16f16(w4, h4, acc, 0, 0, 0);
      } else {
#pragma unroll
        for (int k = 0; k < KB; k++)
          if (k < nkb) {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[k], ul[b][k], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[k], uh[b][k], acc, 0, 0, 0);
          }
      }
      float4_t y;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = fmaf(scale[b], acc[i], base[b][i]);
      if (b * 16 + l16 < t.n) adapter_store_y<YF16>(a, row[b] + n, y);
    }
  }
}

template <int XK, int TB, int RB>
static void adapters_launch(const AdapterArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((adapter_down_kernel<XK, TB, RB>), dim3((unsigned)a.ntiles, (unsigned)a.splits), dim3(256), 0, st, a);
  const dim3 grid((unsigned)a.ntiles, (unsigned)((a.N + a.cols - 1) / a.cols));
  if (a.y_f16) hipLaunchKernelGGL((adapter_up_kernel<TB, RB, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_up_kernel<TB, RB, false>), grid, dim3(256), 0, st, a);
}
template <int XK, int TB>
static void adapters_rank(const AdapterArgs& a, int rank_pad, hipStream_t st) {
  if (rank_pad <= 16) adapters_launch<XK, TB, 1>(a, st);
  else if (rank_pad <= 32) adapters_launch<XK, TB, 2>(a, st);
  else if (rank_pad <= 64) adapters_launch<XK, TB, 4>(a, st);
  else adapters_launch<XK, TB, 8>(a, st);
}

void launch_adapters(const AdapterArgs& args, int tile_rows, int rank_pad, int ncu, hipStream_t st) {
  AdapterArgs a = args;
  // about two workgroups per CU along N, each with at least 64 columns a wave
  const int per_tile = std::max(1, 2 * ncu / a.ntiles);
  a.cols = std::max(256, (a.N / per_tile + 63) / 64 * 64);
  const bool few = tile_rows <= 16;
  switch (a.xk) {
    case XK_F32: few ? adapters_rank<XK_F32, 1>(a, rank_pad, st) : adapters_rank<XK_F32, 4>(a, rank_pad, st); break;
    case XK_F16: few ? adapters_rank<XK_F16, 1>(a, rank_pad, st) : adapters_rank<XK_F16, 4>(a, rank_pad, st); break;
    default: few ? adapters_rank<XK_X2, 1>(a, rank_pad, st) : adapters_rank<XK_X2, 4>(a, rank_pad, st); break;
  }
}

}  // namespace tgohip
