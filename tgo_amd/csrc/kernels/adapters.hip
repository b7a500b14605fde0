// adapters.hip -- low-rank adapters of many requests beside a shared projection:
// y[t] = base[t] + s (x[t] . down^T) . up^T with the adapter of the request that
// row t belongs to, or y[t] = base[t] where it has none.
//
// Rows are sorted by adapter (AdapterTile: up to 16 TB rows of one adapter), so
// each product is a small matrix product and an adapter is read once per tile.
// With ranks up to 128 the work is far below the matrix unit's: x, base and y
// bound it, and for a few rows the two launches' latency.
//   adapter_down_kernel  u = x . down^T over a share of K, f32 planes
//   adapter_pair_kernel  (tiles of 64 rows) the planes' sums, as scaled f16 pairs
//   adapter_up_kernel    y = base + s u . up^T; with tiles of 16 rows it sums the
//                        planes itself, a launch less
// Measured, the three together (us; bytes are x, base, y and each adapter once):
//   1 row, rank 16, [4096, 4096]                8.6, 3.7 and 4.1 of them the kernels
//   128 rows of 32 adapters, [4096, 6144]       10.6, 1.8 TB/s
//   1152 rows, rank 64, [4096, 24576]           95, 3.7 TB/s: 15, 5 and 77
//   8000 f16 rows, rank 24, [12288, 4096]       77, 4.0 TB/s: 39, 5 and 33
// The kernels are built for the set's largest rank, RB blocks of 16: a tile of a smaller
// one loads its last rows again and multiplies them for nothing. Two adapters of rank 16
// over [4096, 6144], alone in their set and beside one of rank 128: 128 f32 rows 7.5 and
// 13.1, 1152 f32 rows 24 and 36, 8000 f16 rows 105 and 143.
// Both products in one launch, each workgroup computing its tile's u, was slower for
// all but the smallest K: one row of [4096, 4096] 9.4 us for 8.0, 128 rows of
// [12288, 4096] 27.9 for 12.0, 16 rows of [1024, 4096] 6.1 for 6.9.
// Both use v_mfma_f32_16x16x32_f16 (16x16x16 for rank 16): lane (l16, q) =
// (lane % 16, lane / 16) holds row or column l16 of an operand at eight k of its own,
// the same of both operands, and of the result column l16, rows 4q + [0,4).
#include "operators.h"

#include <algorithm>

namespace tgohip {

// Eight f32 as f16 hi + lo: to 2^-22 of each, or to 2^-25 (half of f16's smallest step)
// where that is more, as the projection that y's base comes from carries them.
__device__ __forceinline__ void adapter_split(float4_t u, float4_t v, half8_t& hi, half8_t& lo) {
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float f = j < 4 ? u[j & 3] : v[j & 3];
    hi[j] = (half_t)f;
    lo[j] = (half_t)(f - (float)hi[j]);
  }
}
// Eight values of x at `off` elements, as the hi part of the product (and lo).
template <int XK>
__device__ __forceinline__ void adapter_load_x(const AdapterArgs& a, int64_t off, half8_t& hi, half8_t& lo) {
  if constexpr (XK == XK_F32) {
    const float4_t u = *(const float4_t*)((const float*)a.x + off), v = *(const float4_t*)((const float*)a.x + off + 4);
    adapter_split(u, v, hi, lo);
  } else {
    hi = *(const half8_t*)((const half_t*)a.x + off);
    if constexpr (XK == XK_X2) lo = *(const half8_t*)((const half_t*)a.x + (int64_t)a.T * a.K + off);
  }
}

// Up to 16 rows of a tile, 64-k units [s0, s1) of its workgroup's share: waves take
// runs of two units in turn. A lane's two loads of a unit lie side by side (its k are
// 16q + 8g + [0,8)), so that a unit is whole lines of x and down.
template <int XK, int RB>
__device__ __forceinline__ void adapter_down_16(const AdapterArgs& a, const AdapterTile& t, const AdapterEntry& e, int s0,
                                                int s1, int wave, float4_t (&acc)[1][RB]) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4, nrb = e.rank_pad / 16;
  // rows past the tile and ranks past the adapter repeat the last ones, whose results are not stored
  const int64_t row = (int64_t)a.perm[t.start + min(l16, t.n - 1)] * a.K + 16 * q;
  const half_t* dn = e.down + (int64_t)l16 * a.K + 16 * q;
  for (int j = 0; s0 + 8 * (j / 2) + 2 * wave + j % 2 < s1; j++) {
    const int k = 64 * (s0 + 8 * (j / 2) + 2 * wave + j % 2);
    half8_t d[RB][2], hi[2], lo[2];
#pragma unroll
    for (int g = 0; g < 2; g++) {
      adapter_load_x<XK>(a, row + k + 8 * g, hi[g], lo[g]);
#pragma unroll
      for (int r = 0; r < RB; r++) d[r][g] = *(const half8_t*)(dn + (int64_t)min(r, nrb - 1) * 16 * a.K + k + 8 * g);
    }
#pragma unroll
    for (int g = 0; g < 2; g++)
#pragma unroll
      for (int r = 0; r < RB; r++) {
        acc[0][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[g], d[r][g], acc[0][r], 0, 0, 0);
        if (XK != XK_F16) acc[0][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[g], d[r][g], acc[0][r], 0, 0, 0);
      }
  }
}

constexpr int kAdapterNt = 2;  // the nt bit: x is read once
typedef __attribute__((address_space(3))) char* adapter_lds;
// s_waitcnt vmcnt(0) lgkmcnt(0), and no memory access moves across it.
__device__ __forceinline__ void adapter_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
}

// Up to 64 rows: x goes through 16 KiB of LDS that are the wave's own by DMA, whole
// lines of a row at a time, 16-byte chunks XOR-swizzled by the row. Eight waves a CU,
// each with its buffer on its way, keep the memory busy; no wave waits for another.
// 7000 f16 rows of K = 12288 and a rank of 24: 37 us, 4.6 TB/s; loaded to registers as
// half lines 56 us, as the unit above 43 (L1 holds half of what is in flight); without
// the nt bit 40. At rank 128 f16 rows and pairs take more than 256 registers with their
// sums, and a CU holds four waves.
template <int XK, int RB>
__device__ __forceinline__ void adapter_down_64(const AdapterArgs& a, const AdapterTile& t, const AdapterEntry& e, int s0,
                                                int s1, int wave, adapter_lds buf, float4_t (&acc)[4][RB]) {
  constexpr int RBY = XK == XK_F32 ? 256 : 128;  // bytes of a row's unit in one plane
  constexpr int CH = RBY / 16, RPI = 64 / CH, NI = 64 / RPI;  // its chunks, rows per instruction, instructions
  constexpr int U = XK == XK_F16 && RB <= 4 ? 2 : 1;  // units in the buffer (rank 128: no registers for two)
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4, nrb = e.rank_pad / 16;
  int64_t at[NI];  // byte offset of the lane's chunk, row by row
#pragma unroll
  for (int n = 0; n < NI; n++) {
    const int m = n * RPI + lane / CH;
    at[n] = (int64_t)a.perm[t.start + min(m, t.n - 1)] * a.K * (RBY / 64) + 16 * ((lane % CH) ^ (m & 7));
  }
  const half_t* dn = e.down + (int64_t)l16 * a.K + 16 * q;
  for (int s = s0 + U * wave; s < s1; s += 4 * U) {
    half8_t d[U][RB][2];
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (s + u >= s1) break;
      const char* x = (const char*)a.x + (int64_t)(s + u) * RBY;
#pragma unroll
      for (int p = 0; p < (XK == XK_X2 ? 2 : 1); p++)
#pragma unroll
        for (int n = 0; n < NI; n++)
          __builtin_amdgcn_global_load_lds(
              (const __attribute__((address_space(1))) void*)(x + p * (int64_t)a.T * a.K * 2 + at[n]),
              (__attribute__((address_space(3))) void*)(buf + 8192 * (u + p) + 1024 * n), 16, 0, kAdapterNt);
#pragma unroll
      for (int r = 0; r < RB; r++)
#pragma unroll
        for (int g = 0; g < 2; g++)
          d[u][r][g] = *(const half8_t*)(dn + (int64_t)min(r, nrb - 1) * 16 * a.K + 64 * (s + u) + 8 * g);
    }
    adapter_wait();
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (s + u >= s1) break;
#pragma unroll
      for (int b = 0; b < 4; b++)
#pragma unroll
        for (int g = 0; g < 2; g++) {
          const adapter_lds row = buf + (16 * b + l16) * RBY;
          half8_t hi, lo;
          if constexpr (XK == XK_F32) {
            typedef __attribute__((address_space(3))) float4_t* f4;
            const int c = 4 * q + 2 * g;
            adapter_split(*(f4)(row + 16 * (c ^ (l16 & 7))), *(f4)(row + 16 * ((c + 1) ^ (l16 & 7))), hi, lo);
          } else {
            typedef __attribute__((address_space(3))) half8_t* h8;
            const int c = 16 * ((2 * q + g) ^ (l16 & 7));
            hi = *(h8)(row + 8192 * u + c);
            if constexpr (XK == XK_X2) lo = *(h8)(row + 8192 + c);
          }
#pragma unroll
          for (int r = 0; r < RB; r++) {
            acc[b][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, d[u][r][g], acc[b][r], 0, 0, 0);
            if (XK != XK_F16) acc[b][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, d[u][r][g], acc[b][r], 0, 0, 0);
          }
        }
    }
    adapter_wait();  // the reads have returned before the next DMA
  }
}

// The waves' sums of TB blocks of rows meet in LDS and go to the share's plane.
template <int TB, int RB>
__device__ __forceinline__ void adapter_down_out(const AdapterArgs& a, const AdapterTile& t, int rank_pad, int wave,
                                                 const float4_t (&acc)[TB][RB], float (*part)[16][RB * 16]) {
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, q = lane >> 4;
  float* u = a.u + ((int64_t)blockIdx.y * a.T + t.start) * kAdapterMaxRank;
#pragma unroll
  for (int b = 0; b < TB; b++) {
    if (b) __syncthreads();
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) part[wave][4 * q + i][r * 16 + l16] = acc[b][r][i];
    __syncthreads();
    for (int i = tid; i < 16 * RB * 16; i += 256) {
      const int m = i / (RB * 16), r = i % (RB * 16);
      if (b * 16 + m < t.n && r < rank_pad)
        u[(b * 16 + m) * kAdapterMaxRank + r] = (part[0][m][r] + part[1][m][r]) + (part[2][m][r] + part[3][m][r]);
    }
  }
}

template <int XK, int TB, int RB>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a) {
  constexpr int kPart = 4 * 16 * RB * 16 * 4, kBuf = TB > 1 ? 4 * 16384 : 0;
  __shared__ __attribute__((aligned(1024))) char mem[kPart > kBuf ? kPart : kBuf];
  const AdapterTile t = a.tiles[blockIdx.x];
  if (t.adapter < 0) return;
  const AdapterEntry e = a.table[t.adapter];
  if (e.rank_pad == 0 || e.rank_pad > RB * 16) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), units = a.K / 64;
  const int s0 = (int)((int64_t)units * blockIdx.y / gridDim.y);
  const int s1 = (int)((int64_t)units * (blockIdx.y + 1) / gridDim.y);
  float (*part)[16][RB * 16] = (float(*)[16][RB * 16])mem;
  if (TB == 1 || t.n <= 16) {
    float4_t acc[1][RB] = {};
    adapter_down_16<XK, RB>(a, t, e, s0, s1, wave, acc);
    adapter_down_out<1, RB>(a, t, e.rank_pad, wave, acc, part);
  } else {
    float4_t acc[4][RB] = {};
    adapter_down_64<XK, RB>(a, t, e, s0, s1, wave, (adapter_lds)mem + 16384 * wave, acc);
    __syncthreads();  // part lies where the DMA went
    adapter_down_out<4, RB>(a, t, e.rank_pad, wave, acc, part);
  }
}

// A piece of a row of base or y: four f32 or eight f16 columns, 16 bytes.
template <bool YF16>
__device__ __forceinline__ void adapter_load_piece(const AdapterArgs& a, int64_t off, float (&v)[YF16 ? 8 : 4]) {
  if (!a.base) {
#pragma unroll
    for (int j = 0; j < (YF16 ? 8 : 4); j++) v[j] = 0.f;
  } else if constexpr (YF16) {
    const half8_t h = *(const half8_t*)((const half_t*)a.base + off);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)h[j];
  } else {
    const float4_t f = *(const float4_t*)((const float*)a.base + off);
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = f[j];
  }
}
template <bool YF16>
__device__ __forceinline__ void adapter_store_piece(const AdapterArgs& a, int64_t off, const float (&v)[YF16 ? 8 : 4]) {
  if constexpr (YF16) {
    half8_t h;
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = (half_t)v[j];
    *(half8_t*)((half_t*)a.y + off) = h;
  } else {
    *(float4_t*)((float*)a.y + off) = float4_t{v[0], v[1], v[2], v[3]};
  }
}
// Orders a wave's own LDS writes before its other lanes' reads (and back).
__device__ __forceinline__ void adapter_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ half4_t adapter_low(half8_t v) { return half4_t{v[0], v[1], v[2], v[3]}; }

// The power of two that brings a row whose largest magnitude is `top` to [1, 2), and
// its inverse: u is carried as an f16 pair of that scale, 22 bits of its largest
// value wherever f16's range ends.
__device__ __forceinline__ void adapter_power(float top, float& down, float& up) {
  int ex = (int)((__float_as_uint(top) >> 23) & 255) - 127;
  ex = top > 0.f && ex < 128 ? max(-100, min(100, ex)) : 0;
  down = __uint_as_float((uint32_t)(127 - ex) << 23);
  up = __uint_as_float((uint32_t)(127 + ex) << 23);
}

// Sums the planes of a tile's rows in their order and leaves them as pairs,
// [hi 128 | lo 128] a row, 0 from the adapter's rank to the launch's, two ranks a lane.
template <int RB>
__global__ __launch_bounds__(256) void adapter_pair_kernel(AdapterArgs a) {
  constexpr int LR = RB * 8;  // lanes per row
  const AdapterTile t = a.tiles[blockIdx.x];
  const int m = blockIdx.y * (256 / LR) + threadIdx.x / LR, r = threadIdx.x % LR * 2;
  if (t.adapter < 0 || m >= t.n) return;
  const bool in = r < a.table[t.adapter].rank_pad;
  const int64_t pos = t.start + m;
  const float* u = a.u + pos * kAdapterMaxRank + (in ? r : 0);
  float s0 = 0.f, s1 = 0.f;
  for (int p0 = 0; p0 < a.splits; p0 += 4) {
    float2 v[4];
#pragma unroll
    for (int p = 0; p < 4; p++) v[p] = *(const float2*)(u + (int64_t)min(p0 + p, a.splits - 1) * a.T * kAdapterMaxRank);
#pragma unroll
    for (int p = 0; p < 4; p++) {
      s0 += p0 + p < a.splits ? v[p].x : 0.f;
      s1 += p0 + p < a.splits ? v[p].y : 0.f;
    }
  }
  s0 = in ? s0 : 0.f;
  s1 = in ? s1 : 0.f;
  float top = fmaxf(fabsf(s0), fabsf(s1)), down, up;
#pragma unroll
  for (int o = LR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  adapter_power(top, down, up);
  s0 *= down;
  s1 *= down;
  const half2_t hi = {(half_t)s0, (half_t)s1};
  half_t* dst = a.pair + pos * 2 * kAdapterMaxRank + r;
  *(half2_t*)dst = hi;
  *(half2_t*)(dst + kAdapterMaxRank) = half2_t{(half_t)(s0 - (float)hi[0]), (half_t)(s1 - (float)hi[1])};
  if (r == 0) a.pair_scale[pos] = up;
}

// u of row l16 (16 rows in LDS) as the lane's operands of the second product.
template <int RB>
__device__ __forceinline__ void adapter_operand(const float (&us)[16][RB * 16 + 4], int l16, int q,
                                                half8_t (&uh)[(RB + 1) / 2], half8_t (&ul)[(RB + 1) / 2], float& scale) {
  constexpr int KB = (RB + 1) / 2, E = RB == 1 ? 4 : 8;
  float top = 0.f, down, up;
#pragma unroll
  for (int k = 0; k < KB; k++)
#pragma unroll
    for (int j = 0; j < E; j++) top = fmaxf(top, fabsf(us[l16][32 * k + E * q + j]));
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  adapter_power(top, down, up);
  scale *= up;
#pragma unroll
  for (int k = 0; k < KB; k++)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float f = j < E ? us[l16][32 * k + E * q + (j < E ? j : 0)] * down : 0.f;
      uh[k][j] = (half_t)f;
      ul[k][j] = (half_t)(f - (float)uh[k][j]);
    }
}

// y of 16 rows (m0 on) of a tile, columns n, n + step, ... below n1, 64 at a time by
// one wave: up's rows are the A operand, so a lane holds four neighbouring columns of
// row l16. The next round's up and base are loaded before this one's products, which
// cross the wave's own LDS (ys) so that base and y move in runs of 64 columns of a row.
template <int RB, bool YF16>
__device__ __forceinline__ void adapter_columns(const AdapterArgs& a, const AdapterTile& t, const AdapterEntry& e,
                                                const half8_t (&uh)[(RB + 1) / 2], const half8_t (&ul)[(RB + 1) / 2],
                                                float scale, int m0, int n, int n1, int step, float (*ys)[68]) {
  constexpr int KB = (RB + 1) / 2;   // products along the rank: 32 wide, or one 16 wide
  constexpr int E = RB == 1 ? 4 : 8; // of which a lane holds E
  constexpr int PE = YF16 ? 8 : 4;   // columns of a 16-byte piece of base or y
  constexpr int PL = 64 / PE;        // lanes per row's run
  constexpr int NP = 16 * PL / 64;   // pieces a lane holds
  const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
  const int prow = lane / PL, pcol = lane % PL * PE;
  int64_t off[NP];  // this lane's pieces of the rows
  bool live[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int m = m0 + i * (64 / PL) + prow;
    live[i] = m < t.n;
    off[i] = (int64_t)a.perm[t.start + min(m, t.n - 1)] * a.N + pcol;
  }
  half8_t w[4][KB];
  float base[NP][PE];
  auto load = [&](int n) {
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const half_t* up = e.up + (int64_t)min(n + 16 * c + l16, a.N - 1) * e.rank_pad + E * q;
#pragma unroll
      for (int k = 0; k < KB; k++) {
        if constexpr (RB == 1) {
          const half4_t h = *(const half4_t*)up;
          w[c][0] = half8_t{h[0], h[1], h[2], h[3], 0, 0, 0, 0};
        } else {
          // past the adapter's rank u is 0, and up reads its first values again
          w[c][k] = *(const half8_t*)(up + (32 * k + 8 * q < e.rank_pad ? 32 * k : 8 * q < e.rank_pad ? 0 : -8 * q));
        }
      }
    }
    const int back = n + pcol < n1 ? 0 : pcol;  // behind the last column: the run's first piece again
#pragma unroll
    for (int i = 0; i < NP; i++) adapter_load_piece<YF16>(a, off[i] + n - back, base[i]);
  };
  if (n < n1) load(n);
  for (; n < n1; n += step) {
    half8_t wc[4][KB];
    float bc[NP][PE];
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int k = 0; k < KB; k++) wc[c][k] = w[c][k];
#pragma unroll
    for (int i = 0; i < NP; i++)
#pragma unroll
      for (int j = 0; j < PE; j++) bc[i][j] = base[i][j];
    if (n + step < n1) load(n + step);
#pragma unroll
    for (int c = 0; c < 4; c++) {
      float4_t acc = {};
#pragma unroll
      for (int k = 0; k < KB; k++) {
        if constexpr (RB == 1) {
          acc = __builtin_amdgcn_mfma_f32_16x16x16f16(adapter_low(wc[c][0]), adapter_low(ul[0]), acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x16f16(adapter_low(wc[c][0]), adapter_low(uh[0]), acc, 0, 0, 0);
        } else {
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(wc[c][k], ul[k], acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(wc[c][k], uh[k], acc, 0, 0, 0);
        }
      }
      *(float4_t*)&ys[l16][16 * c + 4 * q] = acc * scale;
    }
    adapter_wave_sync();
#pragma unroll
    for (int i = 0; i < NP; i++) {
      float y[PE];
#pragma unroll
      for (int j = 0; j < PE; j += 4) {
        const float4_t v = *(const float4_t*)&ys[i * (64 / PL) + prow][pcol + j];
#pragma unroll
        for (int g = 0; g < 4; g++) y[j + g] = bc[i][j + g] + v[g];
      }
      if (live[i] && n + pcol < n1) adapter_store_piece<YF16>(a, off[i] + n, y);
    }
    adapter_wave_sync();
  }
}

// A tile's rows without an adapter: y = base, eight pieces a thread in flight (one at a
// time, 1152 rows of which 528 have none took 103 us instead of 96). False: the rows have
// one, in e.
template <int RB, bool YF16>
__device__ __forceinline__ bool adapter_copies(const AdapterArgs& a, const AdapterTile& t, AdapterEntry& e, int n0,
                                               int n1) {
  e = AdapterEntry{};
  if (t.adapter >= 0) e = a.table[t.adapter];
  // an adapter of a larger rank than the launch was captured for: its rows are NaN
  if (e.rank_pad > RB * 16) {
    e.rank_pad = RB * 16;
    e.scale = NAN;
  }
  if (e.rank_pad) return false;
  if (a.base == a.y) return true;
  constexpr int PE = YF16 ? 8 : 4;
  const int w = (n1 - n0) / PE, all = t.n * w;
  for (int i0 = threadIdx.x; i0 < all; i0 += 8 * 256) {
    int64_t off[8];
    float v[8][PE];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int i = min(i0 + 256 * u, all - 1), m = i / w;
      off[u] = (int64_t)a.perm[t.start + m] * a.N + n0 + PE * (i - m * w);
      adapter_load_piece<YF16>(a, off[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (i0 + 256 * u < all) adapter_store_piece<YF16>(a, off[u], v[u]);
  }
  return true;
}

// Columns [a.cols * blockIdx.y, + a.cols) of a tile's rows. A wave takes 16 of the
// rows; a tile of fewer blocks of rows shares its columns among the waves instead.
// With one block of rows per tile (TB = 1) the planes are summed and scaled here, else
// they come as adapter_pair_kernel's pairs.
template <int TB, int RB, bool YF16>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a) {
  constexpr int KB = (RB + 1) / 2, E = RB == 1 ? 4 : 8;
  __shared__ __attribute__((aligned(16))) float us[TB == 1 ? 16 : 1][RB * 16 + 4];
  __shared__ __attribute__((aligned(16))) float stage[4][16][68];
  const AdapterTile t = a.tiles[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.y * a.cols, n1 = min(n0 + a.cols, a.N);
  AdapterEntry e;
  if (adapter_copies<RB, YF16>(a, t, e, n0, n1)) return;
  const int ntb = (t.n + 15) / 16, share = ntb == 1 ? 4 : ntb == 2 ? 2 : 1;  // waves that share a block's columns
  const int m0 = 16 * (wave / share);
  half8_t uh[KB], ul[KB];
  float scale = e.scale;
  if constexpr (TB == 1) {
    for (int i = tid; i < 16 * RB * 16; i += 256) {
      const int m = i / (RB * 16), r = i - m * (RB * 16);
      // every plane's load in flight, summed in their order: as many loads as there may be
      // planes, the last one again where a batch has fewer
      float s = 0.f, v[kAdapterMaxSplits];
      const bool in = m < t.n && r < e.rank_pad;
      const float* u = a.u + ((int64_t)t.start + (in ? m : 0)) * kAdapterMaxRank + (in ? r : 0);
#pragma unroll
      for (int p = 0; p < kAdapterMaxSplits; p++) v[p] = u[(int64_t)min(p, a.splits - 1) * a.T * kAdapterMaxRank];
#pragma unroll
      for (int p = 0; p < kAdapterMaxSplits; p++) s += p < a.splits ? v[p] : 0.f;
      us[m][r] = in ? s : 0.f;
    }
    __syncthreads();
    adapter_operand<RB>(us, l16, q, uh, ul, scale);
  } else {
    if (m0 >= t.n) return;
    const int64_t pos = t.start + min(m0 + l16, t.n - 1);
    const half_t* p = a.pair + pos * 2 * kAdapterMaxRank + E * q;
    scale *= a.pair_scale[pos];
#pragma unroll
    for (int k = 0; k < KB; k++) {  // RB = 1 uses the first half of what it loads
      uh[k] = *(const half8_t*)(p + 32 * k);
      ul[k] = *(const half8_t*)(p + kAdapterMaxRank + 32 * k);
    }
  }
  adapter_columns<RB, YF16>(a, t, e, uh, ul, scale, m0, n0 + 64 * (wave % share), n1, 64 * share, stage[wave]);
}

template <int XK, int TB, int RB>
static void adapters_launch(const AdapterArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.ntiles, (unsigned)((a.N + a.cols - 1) / a.cols));
  const dim3 shares((unsigned)a.ntiles, (unsigned)a.splits);
  hipLaunchKernelGGL((adapter_down_kernel<XK, TB, RB>), shares, dim3(256), 0, st, a);
  constexpr int kPairRows = 256 / (RB * 8);  // rows of a workgroup
  const dim3 pairs((unsigned)a.ntiles, (16 * TB + kPairRows - 1) / kPairRows);
  if (TB > 1) hipLaunchKernelGGL((adapter_pair_kernel<RB>), pairs, dim3(256), 0, st, a);
  if (a.y_f16) hipLaunchKernelGGL((adapter_up_kernel<TB, RB, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((adapter_up_kernel<TB, RB, false>), grid, dim3(256), 0, st, a);
}
template <int XK, int TB>
static void adapters_rank(const AdapterArgs& a, hipStream_t st) {
  if (a.rank_pad <= 16) adapters_launch<XK, TB, 1>(a, st);
  else if (a.rank_pad <= 32) adapters_launch<XK, TB, 2>(a, st);
  else if (a.rank_pad <= 64) adapters_launch<XK, TB, 4>(a, st);
  else adapters_launch<XK, TB, 8>(a, st);
}

void launch_adapters(const AdapterArgs& args, int tile_rows, int ncu, hipStream_t st) {
  AdapterArgs a = args;
  const bool one = tile_rows <= 16;
  // Columns per workgroup of the second kernel, us for 1152 mixed rows of rank 64 over
  // [4096, 24576] and 8000 f16 rows of rank 24 over [12288, 4096]: 128 columns 98, 84;
  // 256 96, 79; 512 101, 79; 1024 119, 85.
  a.cols = 256;
  switch (a.xk) {
    case XK_F32: one ? adapters_rank<XK_F32, 1>(a, st) : adapters_rank<XK_F32, 4>(a, st); break;
    case XK_F16: one ? adapters_rank<XK_F16, 1>(a, st) : adapters_rank<XK_F16, 4>(a, st); break;
    default: one ? adapters_rank<XK_X2, 1>(a, st) : adapters_rank<XK_X2, 4>(a, st); break;
  }
}

}  // namespace tgohip
