// cache_rows.hip -- rows of the 8-bit cache: written from a projection's output (norm,
// rotation, quantisation), read back, moved.
//
// A row y of d values is held as codes c and one scale s = max(max|y| / top, 2^-40) with
// c = y / s, rounded to f32 and then to the nearest (ties to even): int8 (top 127) or e4m3 (top 448). It stands for
// c s. A row with a value that is not finite, or past 2^40, has the scale NaN and codes 0:
// all of it stands for NaN, and no code is ever one.
//
// All three are bound by the rows' bytes. Measured (a large copy here 4.7 TB/s), us of the kernel: store
// of 16384 rows of 80 f16 heads of 128 dims, normed, half of each rotated, 639 MB, 141, 4.5 TB/s;
// of 1152 rows of 48 f32 heads, 50 MB, 12; of one row 3.3, 7 with the call.
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

// Sum and maximum over LPH (8 or 16) neighbouring lanes, in all of them: DPP moves within
// a row of 16 lanes (exchanges of 1 and 2 lanes, then mirrors of 8 and 16).
template <int CTRL>
__device__ __forceinline__ float cache_dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int LPH, typename F>
__device__ __forceinline__ float cache_over_lanes(float v, F f) {
  v = f(v, cache_dpp<0xb1>(v));
  v = f(v, cache_dpp<0x4e>(v));
  v = f(v, cache_dpp<0x141>(v));
  if (LPH == 16) v = f(v, cache_dpp<0x140>(v));
  return v;
}

// Elements of one head of one row in D / 8 neighbouring lanes: lane j holds 4 / V units of
// 2V, unit u = j + D / 8 i. A unit of the rotated part is V pairs, in the half layout two runs
// of V; others are 2V neighbouring elements from 2V u on.
template <int V>
struct HeadRow {
  float A[4 / V][V], B[4 / V][V];
};

// Rows [t0, t0 + rows) of head h, row t0 + phase, then every P-th. What belongs to the head
// (its tensor, gains, places) is taken once, a row is loaded while the one before is worked on.
template <int KIND, int V, bool HALF, int D, bool F8, bool XF16>
__device__ __forceinline__ void cache_store_rows(const CacheStoreArgs& a, int t0, int rows, int h, int phase, int P, int j,
                                                 const float2* cs) {
  constexpr int LPH = D / 8, NU = 4 / V;
  const int turned = KIND < 2 ? a.rd / (2 * V) : 0, pairs = a.rd / 2;
  const void* src = KIND == 0 ? a.q : KIND == 1 ? a.k : a.v;
  const int64_t row = KIND == 0 ? a.q_row : KIND == 1 ? a.k_row : a.v_row;
  const int64_t head = KIND == 0 ? a.q_head : KIND == 1 ? a.k_head : a.v_head;
  int ja[NU], jb[NU];
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int u = j + LPH * i;
    const bool split = HALF && u < turned;
    ja[i] = split ? V * u : 2 * V * u;
    jb[i] = split ? pairs + V * u : ja[i] + V;
  }
  const float* gain = KIND == 0 ? a.q_gain : KIND == 1 ? a.k_gain : nullptr;
  HeadRow<V> g;
  if (gain) {
#pragma unroll
    for (int i = 0; i < NU; i++) {
      rope_load<V, false>(gain, ja[i], g.A[i]);
      rope_load<V, false>(gain, jb[i], g.B[i]);
    }
  }
  const auto load = [&](int t, HeadRow<V>& x, int32_t& slot) {
    const int64_t off = t * row + h * head;
#pragma unroll
    for (int i = 0; i < NU; i++) {
      rope_load<V, XF16>(src, off + ja[i], x.A[i]);
      rope_load<V, XF16>(src, off + jb[i], x.B[i]);
    }
    if (KIND) slot = a.slots[t];
  };
  HeadRow<V> x, next;
  int32_t slot = 0, next_slot = 0;
  if (phase < rows) load(t0 + phase, next, next_slot);
  for (int t = phase; t < rows; t += P) {
    x = next;
    slot = next_slot;
    load(t0 + min(t + P, rows - 1), next, next_slot);
    if (gain) {
      const auto mean = [&](float k2) {  // of the squares, and eps k2
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
          for (int e = 0; e < V; e++) ss += x.A[i][e] * x.A[i][e] + x.B[i][e] * x.B[i][e];
        return cache_over_lanes<LPH>(ss, [](float p, float q) { return p + q; }) * (1.f / D) + k2;
      };
      float ms = mean(a.eps);
      if (!(ms > 0x1p-84f && ms < 0x1p120f)) {
        // squares that leave f32's range, or may: the row by a power of two, eps by its square
        const float k = ms < 1.f ? 0x1p100f : 0x1p-64f;
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
          for (int e = 0; e < V; e++) {
            x.A[i][e] *= k;
            x.B[i][e] *= k;
          }
        ms = mean(a.eps * k * k);
      }
      const float sc = 1.f / sqrtf(ms);
#pragma unroll
      for (int i = 0; i < NU; i++)
#pragma unroll
        for (int e = 0; e < V; e++) {
          x.A[i][e] = x.A[i][e] * sc * g.A[i][e];
          x.B[i][e] = x.B[i][e] * sc * g.B[i][e];
        }
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const int u = j + LPH * i;
      if (u >= turned) continue;
      float p[2 * V];
#pragma unroll
      for (int e = 0; e < V; e++) {
        p[e] = x.A[i][e];
        p[V + e] = x.B[i][e];
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float2 w = cs[t * pairs + V * u + e];
        const int m = HALF ? e : 2 * e, n = HALF ? V + e : 2 * e + 1;
        const float f = p[m], r = p[n];
        p[m] = fmaf(f, w.x, -(r * w.y));
        p[n] = fmaf(f, w.y, r * w.x);
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        x.A[i][e] = p[e];
        x.B[i][e] = p[V + e];
      }
    }
    if constexpr (KIND == 0) {
      const int64_t to = (t0 + t) * a.out_row + h * a.out_head;
#pragma unroll
      for (int i = 0; i < NU; i++) {
        if (a.out_f16) {
          rope_store<V, true>(a.q_out, to + ja[i], x.A[i]);
          rope_store<V, true>(a.q_out, to + jb[i], x.B[i]);
        } else {
          rope_store<V, false>(a.q_out, to + ja[i], x.A[i]);
          rope_store<V, false>(a.q_out, to + jb[i], x.B[i]);
        }
      }
    } else {
      float peak = 0.f;  // infinite where a value is past kCacheMost or NaN
#pragma unroll
      for (int i = 0; i < NU; i++)
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float m = fabsf(x.A[i][e]), n = fabsf(x.B[i][e]);
          peak = fmaxf(peak, m <= kCacheMost ? m : INFINITY);
          peak = fmaxf(peak, n <= kCacheMost ? n : INFINITY);
        }
      peak = cache_over_lanes<LPH>(peak, [](float p, float q) { return fmaxf(p, q); });
      const bool bad = peak == INFINITY;
      const float scale = fmaxf(peak / (F8 ? 448.f : 127.f), kCacheLeast);
      const float inv = 1.f / scale;
      // y / scale as a division rounds it: the product with a rounded reciprocal is off by up to two
      // steps, its remainder (exact by fma) times that reciprocal corrects it. us of 16384 rows of 80
      // f16 heads / 1152 of 48 f32 heads, with reading back: 156 / 14.9; by divisions 161 / 15.2; by v_rcp_f32
      // alone, codes of half steps to either side, 154 / 14.5.
      const auto quotient = [=](float y) {
        const float q = y * inv;
        return fmaf(fmaf(-q, scale, y), inv, q);
      };
      if ((uint32_t)slot >= (uint32_t)a.c.capacity) continue;  // all lanes of the head alike
      const int64_t at = a.c.row(slot, h);
      uint8_t* to = (KIND == 1 ? a.c.k : a.c.v) + at * D;
      if (j == 0) (KIND == 1 ? a.c.ks : a.c.vs)[at] = bad ? NAN : scale;
#pragma unroll
      for (int i = 0; i < NU; i++) {
        float m[4], n[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          m[e] = bad ? 0.f : quotient(x.A[i][e % V]);
          n[e] = bad ? 0.f : quotient(x.B[i][e % V]);
        }
        const uint32_t w0 = cache_codes4<F8>(m[0], m[1], m[2], m[3]), w1 = cache_codes4<F8>(n[0], n[1], n[2], n[3]);
        if constexpr (V == 4) {
          *(uint32_t*)(to + ja[i]) = w0;
          *(uint32_t*)(to + jb[i]) = w1;
        } else {
          to[ja[i]] = (uint8_t)w0;
          to[jb[i]] = (uint8_t)w1;
        }
      }
    }
  }
}

template <int V, bool HALF, int D, bool F8, bool XF16>
__global__ __launch_bounds__(256) void cache_store_kernel(CacheStoreArgs a) {
  extern __shared__ float2 cs[];  // [rows][pairs]
  constexpr int LPH = D / 8, GR = 256 / LPH;
  const int heads = a.H + 2 * a.c.Hkv, h0 = blockIdx.y * a.slice, hn = min(h0 + a.slice, heads);
  const int t0 = blockIdx.x * a.rows, rows = min(a.rows, a.T - t0), pairs = a.rd / 2;
  if (pairs && h0 < a.H + a.c.Hkv) {
    for (int i = threadIdx.x; i < rows * pairs; i += 256) {
      const int t = i / pairs;
      cs[i] = rope_angle(a.positions[t0 + t], a.inv_freq[i - t * pairs], a.attention);
    }
    __syncthreads();
  }
  // GR heads at a time, the last few of the slice with their rows shared by several groups of lanes
  const int g = threadIdx.x / LPH, j = threadIdx.x % LPH;
  for (int h = h0; h < hn; h += GR) {
    const int n = min(GR, hn - h), P = GR / n, phase = g / n, mine = h + g % n;
    if (phase >= P) continue;
    if (mine < a.H) cache_store_rows<0, V, HALF, D, F8, XF16>(a, t0, rows, mine, phase, P, j, cs);
    else if (mine < a.H + a.c.Hkv) cache_store_rows<1, V, HALF, D, F8, XF16>(a, t0, rows, mine - a.H, phase, P, j, cs);
    else cache_store_rows<2, V, HALF, D, F8, XF16>(a, t0, rows, mine - a.H - a.c.Hkv, phase, P, j, cs);
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
  // Few rows: their heads spread over workgroups, down to one head for each group of lanes. Spread /
  // all by one workgroup, us of 48 f32 heads in a graph: one row 3.1 / 4.7, 64 rows 3.6 / 5.2. Many: a
  // workgroup takes all heads of up to 16 rows, and their angles once. Up to 1 / 4 / 16 / 64
  // rows, us with 17 and 4 of reading them back: 16384 of 80 f16 heads 169 / 161 / 157 / 157,
  // 1152 of 48 f32 heads 14.8 each.
  a.slice = heads;
  while (a.slice > at_once && (int64_t)a.T * ((heads + a.slice - 1) / a.slice) < 2 * ncu)
    a.slice = std::max(at_once, (a.slice + 1) / 2);
  a.rows = 1;
  while (a.rows < 16 && (int64_t)a.T * ((heads + a.slice - 1) / a.slice) / (2 * a.rows) >= 4 * ncu) a.rows *= 2;
  const auto fits = [](const void* p, int64_t row, int64_t head, int f16) {
    const int n = f16 ? 8 : 4;
    return (uintptr_t)p % 16 == 0 && row % n == 0 && head % n == 0;
  };
  // Units of eight elements, where every head starts on 16 bytes, / of two, us with the same: 16384
  // rows 157 / 214, 1152 14.8 / 17.8.
  const bool wide = a.rd % 8 == 0 && fits(a.k, a.k_row, a.k_head, a.x_f16) && fits(a.v, a.v_row, a.v_head, a.x_f16) &&
                    (!a.H || (fits(a.q, a.q_row, a.q_head, a.x_f16) && fits(a.q_out, a.out_row, a.out_head, a.out_f16))) &&
                    (uintptr_t)a.q_gain % 16 == 0 && (uintptr_t)a.k_gain % 16 == 0;
  if (a.c.d == 128) wide ? cache_store_form<4, 128>(a, st) : cache_store_form<1, 128>(a, st);
  else wide ? cache_store_form<4, 64>(a, st) : cache_store_form<1, 64>(a, st);
}

// ---------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------

// D / 8 lanes a row, eight codes each, kReadRows rows a lane with their loads in flight: with 1 / 2 /
// 4 / 8, us for 131072 rows of 8 heads of 128 dims to f16, 182 / 167 / 154 / 154. Bound by its
// bytes: 814 MB, 5.3 TB/s.
constexpr int kReadRows = 4;

template <int D, bool F8, bool F16>
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
    // by elements: they may start anywhere, and become wide stores as they are
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float one[1] = {v[e]};
      rope_store<1, F16>(a.out[which], to[i] + e, one);
    }
  }
}

template <int D, bool F8>
static void cache_read_launch(const CacheReadArgs& a, hipStream_t st) {
  const uint64_t total = (uint64_t)a.T * a.c.Hkv, per = 256 / (D / 8) * kReadRows;
  const dim3 grid((unsigned)((total + per - 1) / per), a.out[0] && a.out[1] ? 2 : 1);
  if (a.f16) hipLaunchKernelGGL((cache_read_kernel<D, F8, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((cache_read_kernel<D, F8, false>), grid, dim3(256), 0, st, a);
}

void launch_cache_read(const CacheReadArgs& a, hipStream_t st) {
  if (a.c.d == 128) a.c.f8 ? cache_read_launch<128, true>(a, st) : cache_read_launch<128, false>(a, st);
  else a.c.f8 ? cache_read_launch<64, true>(a, st) : cache_read_launch<64, false>(a, st);
}

// ---------------------------------------------------------------------------
// moving
// ---------------------------------------------------------------------------

// D / 16 lanes a row, 16 bytes each, of K and of V; FEW: the moves are in f. Bound by its bytes,
// read and written (pieces of 128): 448 rows of 36 layers of 8 heads of 128 dims, 68 MB, 18 us,
// and 16 a call where calls follow each other, 4.2 TB/s beside a large copy's 4.7. K and V
// by workgroups of their own and a row's two scales behind its codes took 27.
template <int D, bool FEW>
__global__ __launch_bounds__(256) void cache_move_kernel(CacheMoveArgs a, CacheMoveFew f) {
  constexpr int LPR = D / 16, PER = 256 / LPR, N = kCacheMoveSeg / PER;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const CacheMoveBatch b = FEW ? f.batch[blockIdx.x] : a.batch[blockIdx.x];
  const int layer = blockIdx.y / a.c.Hkv, h = blockIdx.y % a.c.Hkv;
  const int64_t first = layer * a.layer_rows;
  const int j = threadIdx.x % LPR, g = threadIdx.x / LPR;
  for (int s0 = 0; s0 < b.n; s0 += kCacheMoveSeg) {
    const int n = min(kCacheMoveSeg, b.n - s0);
    u4 k[N], v[N];
    float ks[N], vs[N];
    int64_t to[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int m = b.start + s0 + min(g + i * PER, n - 1);
      const int32_t src = FEW ? f.src[m] : a.src[m], dst = FEW ? f.dst[m] : a.dst[m];
      const int64_t from = first + a.c.row(src, h);
      to[i] = first + a.c.row(dst, h);
      k[i] = *(const u4*)(a.c.k + from * D + 16 * j);
      v[i] = *(const u4*)(a.c.v + from * D + 16 * j);
      ks[i] = a.c.ks[from];
      vs[i] = a.c.vs[from];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (g + i * PER >= n) continue;
      *(u4*)(a.c.k + to[i] * D + 16 * j) = k[i];
      *(u4*)(a.c.v + to[i] * D + 16 * j) = v[i];
      if (j == 0) {
        a.c.ks[to[i]] = ks[i];
        a.c.vs[to[i]] = vs[i];
      }
    }
    __syncthreads();
  }
}

template <int D>
static void cache_move_launch(const CacheMoveArgs& a, const CacheMoveFew& f, hipStream_t st) {
  if (f.n) hipLaunchKernelGGL((cache_move_kernel<D, true>), dim3(a.batches, a.layers * a.c.Hkv), dim3(256), 0, st, a, f);
  else hipLaunchKernelGGL((cache_move_kernel<D, false>), dim3(a.batches, a.layers * a.c.Hkv), dim3(256), 0, st, a, f);
}

void launch_cache_move(const CacheMoveArgs& a, const CacheMoveFew& f, hipStream_t st) {
  if (a.c.d == 128) cache_move_launch<128>(a, f, st);
  else cache_move_launch<64>(a, f, st);
}

}  // namespace tgohip
