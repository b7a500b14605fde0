// cache_rows.hip -- rows of the 8-bit cache: written from a projection's output (norm,
// rotation, quantisation), read back, moved.
//
// A row y of d values is held as codes c and one scale s = max(max|y| / top, 2^-40) with
// c = y / s to the nearest (ties to even): int8 (top 127) or e4m3 (top 448). It stands for
// c s. A row with a value that is not finite, or past 2^40, has the scale NaN and codes 0:
// all of it stands for NaN, and no code is ever one.
#include "heads.h"

#include <algorithm>

namespace tgohip {

constexpr float kCacheMost = 0x1p40f, kCacheLeast = 0x1p-40f;

template <bool F8>
__device__ __forceinline__ uint32_t cache_codes4(float a, float b, float c, float d) {
  if constexpr (F8) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    const uint32_t w0 = (uint32_t)(int)rintf(a) & 255u, w1 = (uint32_t)(int)rintf(b) & 255u;
    const uint32_t w2 = (uint32_t)(int)rintf(c) & 255u, w3 = (uint32_t)(int)rintf(d);
    return w0 | w1 << 8 | w2 << 16 | w3 << 24;
  }
}
template <bool F8>
__device__ __forceinline__ void cache_values4(uint32_t w, float s, float* v) {
  if constexpr (F8) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[0] = a[0] * s;
    v[1] = a[1] * s;
    v[2] = b[0] * s;
    v[3] = b[1] * s;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (float)(int8_t)(w >> (8 * i)) * s;
  }
}

// One head of one row, by D / 8 neighbouring lanes: lane j holds 4 / V units of 2V
// elements, unit u = j + D / 8 i. A unit of the rotated part is V pairs, in the half layout two runs of V,
// others 2V neighbouring elements from 2V u on.
template <int V, bool HALF, int D, bool F8, bool XF16>
__device__ __forceinline__ void cache_store_head(const CacheStoreArgs& a, int t, int h, int j, const float2* cs) {
  constexpr int LPH = D / 8, NU = 4 / V;
  const int kind = h < a.H ? 0 : h < a.H + a.c.Hkv ? 1 : 2;
  const int hh = kind == 0 ? h : kind == 1 ? h - a.H : h - a.H - a.c.Hkv;
  int32_t slot = 0;
  if (kind) {
    slot = a.slots[t];
    if ((uint32_t)slot >= (uint32_t)a.c.capacity) return;  // all lanes of the head alike
  }
  const void* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  const int64_t off = kind == 0   ? t * a.q_row + hh * a.q_head
                      : kind == 1 ? t * a.k_row + hh * a.k_head
                                  : t * a.v_row + hh * a.v_head;
  const int turned = kind < 2 ? a.rd / (2 * V) : 0, pairs = a.rd / 2;
  float A[NU][V], B[NU][V];
  int ja[NU], jb[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int u = j + LPH * i;
    const bool split = HALF && u < turned;
    ja[i] = split ? V * u : 2 * V * u;
    jb[i] = split ? pairs + V * u : ja[i] + V;
    rope_load<V, XF16>(src, off + ja[i], A[i]);
    rope_load<V, XF16>(src, off + jb[i], B[i]);
  }
  const float* gain = kind == 0 ? a.q_gain : kind == 1 ? a.k_gain : nullptr;
  if (gain) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NU; i++)
#pragma unroll
      for (int e = 0; e < V; e++) ss += A[i][e] * A[i][e] + B[i][e] * B[i][e];
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    const float sc = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
    for (int i = 0; i < NU; i++) {
      float ga[V], gb[V];
      rope_load<V, false>(gain, ja[i], ga);
      rope_load<V, false>(gain, jb[i], gb);
#pragma unroll
      for (int e = 0; e < V; e++) {
        A[i][e] = A[i][e] * sc * ga[e];
        B[i][e] = B[i][e] * sc * gb[e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int u = j + LPH * i;
    if (u >= turned) continue;
    float p[2 * V];
#pragma unroll
    for (int e = 0; e < V; e++) {
      p[e] = A[i][e];
      p[V + e] = B[i][e];
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
      const float2 w = cs[V * u + e];
      const int x = HALF ? e : 2 * e, y = HALF ? V + e : 2 * e + 1;
      const float f = p[x], g = p[y];
      p[x] = fmaf(f, w.x, -(g * w.y));
      p[y] = fmaf(f, w.y, g * w.x);
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
      A[i][e] = p[e];
      B[i][e] = p[V + e];
    }
  }
  if (kind == 0) {
    const int64_t to = t * a.out_row + hh * a.out_head;
#pragma unroll
    for (int i = 0; i < NU; i++) {
      if (a.out_f16) {
        rope_store<V, true>(a.q_out, to + ja[i], A[i]);
        rope_store<V, true>(a.q_out, to + jb[i], B[i]);
      } else {
        rope_store<V, false>(a.q_out, to + ja[i], A[i]);
        rope_store<V, false>(a.q_out, to + jb[i], B[i]);
      }
    }
    return;
  }
  float peak = 0.f;  // infinite where a value is past kCacheMost or NaN
#pragma unroll
  for (int i = 0; i < NU; i++)
#pragma unroll
    for (int e = 0; e < V; e++) {
      const float x = fabsf(A[i][e]), y = fabsf(B[i][e]);
      peak = fmaxf(peak, x <= kCacheMost ? x : INFINITY);
      peak = fmaxf(peak, y <= kCacheMost ? y : INFINITY);
    }
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o, 64));
  const bool bad = peak == INFINITY;
  const float scale = fmaxf(peak / (F8 ? 448.f : 127.f), kCacheLeast), inv = 1.0f / scale;
  const int64_t row = a.c.row(slot, hh);
  uint8_t* to = (kind == 1 ? a.c.k : a.c.v) + row * D;
  if (j == 0) (kind == 1 ? a.c.ks : a.c.vs)[row] = bad ? NAN : scale;
#pragma unroll
  for (int i = 0; i < NU; i++) {
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      x[e] = bad ? 0.f : A[i][e % V] * inv;
      y[e] = bad ? 0.f : B[i][e % V] * inv;
    }
    const uint32_t w0 = cache_codes4<F8>(x[0], x[1], x[2], x[3]), w1 = cache_codes4<F8>(y[0], y[1], y[2], y[3]);
    if constexpr (V == 4) {
      *(uint32_t*)(to + ja[i]) = w0;
      *(uint32_t*)(to + jb[i]) = w1;
    } else {
      to[ja[i]] = (uint8_t)w0;
      to[jb[i]] = (uint8_t)w1;
    }
  }
}

template <int V, bool HALF, int D, bool F8, bool XF16>
__global__ __launch_bounds__(256) void cache_store_kernel(CacheStoreArgs a) {
  extern __shared__ float2 cs[];  // [rows][pairs]
  constexpr int LPH = D / 8;
  const int heads = a.H + 2 * a.c.Hkv, h0 = blockIdx.y * a.slice, n = min(a.slice, heads - h0);
  const int t0 = blockIdx.x * a.rows, rows = min(a.rows, a.T - t0), pairs = a.rd / 2;
  if (pairs && h0 < a.H + a.c.Hkv) {
    for (int i = threadIdx.x; i < rows * pairs; i += 256) {
      const int t = i / pairs;
      cs[i] = rope_angle(a.positions[t0 + t], a.inv_freq[i - t * pairs], a.attention);
    }
    __syncthreads();
  }
  for (int r = threadIdx.x / LPH; r < rows * a.slice; r += 256 / LPH) {
    const int t = (int)(((uint64_t)r * a.magic) >> 32), h = r - t * a.slice;
    if (h < n) cache_store_head<V, HALF, D, F8, XF16>(a, t0 + t, h0 + h, threadIdx.x % LPH, cs + t * pairs);
  }
}

template <int V, bool HALF, int D, bool F8>
static void cache_store_launch(const CacheStoreArgs& a, hipStream_t st) {
  const int heads = a.H + 2 * a.c.Hkv;
  const dim3 grid((unsigned)((a.T + a.rows - 1) / a.rows), (unsigned)((heads + a.slice - 1) / a.slice));
  const size_t lds = (size_t)a.rows * (a.rd / 2) * sizeof(float2);
  if (a.x_f16) hipLaunchKernelGGL((cache_store_kernel<V, HALF, D, F8, true>), grid, dim3(256), lds, st, a);
  else hipLaunchKernelGGL((cache_store_kernel<V, HALF, D, F8, false>), grid, dim3(256), lds, st, a);
}
template <int V, int D>
static void cache_store_form(const CacheStoreArgs& a, hipStream_t st) {
  if (a.half) a.c.f8 ? cache_store_launch<V, true, D, true>(a, st) : cache_store_launch<V, true, D, false>(a, st);
  else a.c.f8 ? cache_store_launch<V, false, D, true>(a, st) : cache_store_launch<V, false, D, false>(a, st);
}

void launch_cache_store(const CacheStoreArgs& args, int ncu, hipStream_t st) {
  CacheStoreArgs a = args;
  const int heads = a.H + 2 * a.c.Hkv, at_once = 256 / (a.c.d / 8);
  // Few rows: their heads spread over workgroups, down to one head for each group of
  // lanes; many: a workgroup takes all heads of up to 16 rows, and their angles once.
  a.slice = heads;
  while (a.slice > at_once && (int64_t)a.T * ((heads + a.slice - 1) / a.slice) < 2 * ncu)
    a.slice = std::max(at_once, (a.slice + 1) / 2);
  a.rows = 1;
  while (a.rows < 16 && (int64_t)a.T * ((heads + a.slice - 1) / a.slice) / (2 * a.rows) >= 4 * ncu) a.rows *= 2;
  a.magic = (((uint64_t)1 << 32) + a.slice - 1) / a.slice;
  const auto fits = [](const void* p, int64_t row, int64_t head, int f16) {
    const int n = f16 ? 8 : 4;
    return (uintptr_t)p % 16 == 0 && row % n == 0 && head % n == 0;
  };
  const bool wide = a.rd % 8 == 0 && fits(a.k, a.k_row, a.k_head, a.x_f16) && fits(a.v, a.v_row, a.v_head, a.x_f16) &&
                    (!a.H || (fits(a.q, a.q_row, a.q_head, a.x_f16) && fits(a.q_out, a.out_row, a.out_head, a.out_f16))) &&
                    (uintptr_t)a.q_gain % 16 == 0 && (uintptr_t)a.k_gain % 16 == 0;
  if (a.c.d == 128) wide ? cache_store_form<4, 128>(a, st) : cache_store_form<1, 128>(a, st);
  else wide ? cache_store_form<4, 64>(a, st) : cache_store_form<1, 64>(a, st);
}

// ---------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------

// D / 8 lanes a row, eight codes each, kReadRows rows a lane with their loads in flight.
constexpr int kReadRows = 4;

template <int D, bool F8, bool F16, bool WIDE>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadArgs a) {
  constexpr int LPH = D / 8, GR = 256 / LPH;
  const int which = a.out[0] ? blockIdx.y : 1, j = threadIdx.x % LPH;
  const uint8_t* codes = which ? a.c.v : a.c.k;
  const float* scales = which ? a.c.vs : a.c.ks;
  const uint32_t total = (uint32_t)a.T * a.c.Hkv, r0 = blockIdx.x * (GR * kReadRows) + threadIdx.x / LPH;
  uint2 w[kReadRows];
  float s[kReadRows];
  int64_t to[kReadRows];
#pragma unroll
  for (int i = 0; i < kReadRows; i++) {
    const uint32_t r = min(r0 + i * GR, total - 1), t = r / a.c.Hkv, h = r - t * a.c.Hkv;
    const int32_t slot = a.slots[t];
    const bool in = (uint32_t)slot < (uint32_t)a.c.capacity;
    const int64_t row = a.c.row(in ? slot : 0, h);
    w[i] = *(const uint2*)(codes + row * D + 8 * j);
    s[i] = scales[row];
    if (!in) {
      w[i] = make_uint2(0, 0);
      s[i] = 0.f;
    }
    to[i] = t * a.row[which] + h * a.head[which] + 8 * j;
  }
#pragma unroll
  for (int i = 0; i < kReadRows; i++) {
    if (r0 + i * GR >= total) continue;
    float v[8];
    cache_values4<F8>(w[i].x, s[i], v);
    cache_values4<F8>(w[i].y, s[i], v + 4);
    if constexpr (WIDE) {
      rope_store<8, F16>(a.out[which], to[i], v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float one[1] = {v[e]};
        rope_store<1, F16>(a.out[which], to[i] + e, one);
      }
    }
  }
}

template <int D, bool F8>
static void cache_read_launch(const CacheReadArgs& a, bool wide, hipStream_t st) {
  const uint64_t total = (uint64_t)a.T * a.c.Hkv, per = 256 / (D / 8) * kReadRows;
  const dim3 grid((unsigned)((total + per - 1) / per), a.out[0] && a.out[1] ? 2 : 1);
  if (a.f16) {
    if (wide) hipLaunchKernelGGL((cache_read_kernel<D, F8, true, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((cache_read_kernel<D, F8, true, false>), grid, dim3(256), 0, st, a);
  } else {
    if (wide) hipLaunchKernelGGL((cache_read_kernel<D, F8, false, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((cache_read_kernel<D, F8, false, false>), grid, dim3(256), 0, st, a);
  }
}

void launch_cache_read(const CacheReadArgs& a, int ncu, hipStream_t st) {
  (void)ncu;
  bool wide = true;
  for (int i = 0; i < 2; i++) {
    const int n = a.f16 ? 8 : 4;
    wide = wide && (!a.out[i] || ((uintptr_t)a.out[i] % 16 == 0 && a.row[i] % n == 0 && a.head[i] % n == 0));
  }
  if (a.c.d == 128) a.c.f8 ? cache_read_launch<128, true>(a, wide, st) : cache_read_launch<128, false>(a, wide, st);
  else a.c.f8 ? cache_read_launch<64, true>(a, wide, st) : cache_read_launch<64, false>(a, wide, st);
}

// ---------------------------------------------------------------------------
// moving
// ---------------------------------------------------------------------------

// D / 16 lanes a row, 16 bytes each.
template <int D>
__global__ __launch_bounds__(256) void cache_move_kernel(CacheMoveArgs a) {
  constexpr int LPR = D / 16, PER = 256 / LPR, N = (kCacheMoveSeg + PER - 1) / PER;
  const CacheMoveBatch b = a.batch[blockIdx.x];
  const int layer = blockIdx.y / a.c.Hkv, h = blockIdx.y % a.c.Hkv;
  const int64_t first = layer * a.layer_rows;
  uint8_t* codes = (blockIdx.z ? a.c.v : a.c.k) + first * D;
  float* scales = (blockIdx.z ? a.c.vs : a.c.ks) + first;
  const int j = threadIdx.x % LPR, g = threadIdx.x / LPR;
  for (int s0 = 0; s0 < b.n; s0 += kCacheMoveSeg) {
    const int n = min(kCacheMoveSeg, b.n - s0);
    uint4 w[N];
    float s[N];
    int64_t to[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int m = b.start + s0 + min(g + i * PER, n - 1);
      const int64_t from = a.c.row(a.src[m], h);
      to[i] = a.c.row(a.dst[m], h);
      w[i] = *(const uint4*)(codes + from * D + 16 * j);
      s[i] = scales[from];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (g + i * PER >= n) continue;
      *(uint4*)(codes + to[i] * D + 16 * j) = w[i];
      if (j == 0) scales[to[i]] = s[i];
    }
    __syncthreads();
  }
}

void launch_cache_move(const CacheMoveArgs& a, hipStream_t st) {
  const dim3 grid(a.batches, a.layers * a.c.Hkv, 2);
  if (a.c.d == 128) hipLaunchKernelGGL((cache_move_kernel<128>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((cache_move_kernel<64>), grid, dim3(256), 0, st, a);
}

}  // namespace tgohip
