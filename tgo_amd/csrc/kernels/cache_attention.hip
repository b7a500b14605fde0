// cache_attention.hip -- attention over the 8-bit paged cache: single tokens, chunks of
// new tokens, trees of drafted tokens; grouped heads.
//
// Codes are exact in f16 and stay as they are in both products; the rows' scales go into
// the softmax, in f32. With S_k = q . c_k the score of key k in log2 units is S_k a_k,
// a_k = scale log2(e) k_scale_k, and
//   o = sum_k 2^(S_k a_k + b_k - m) d_k / sum_k 2^(S_k a_k + b_k - m) / v_scale_k,
// b_k = log2(v_scale_k) and d_k the value's codes: the probabilities that the second
// product takes hold their value's scale, so that their largest is near 1 whatever the
// scales are, and the sum takes it out again. m moves along (online softmax), and only
// when a probability would leave its range.
#include "operators.h"
#include "waits.h"

#include <algorithm>

namespace tgohip {

typedef __attribute__((address_space(3))) char* lds_t;
constexpr int kNonTemporal = 2;  // the nt bit: a context's rows are read once
// The reference starts at kCacheNoMax; where a term passes it by more than 2^kCacheTop (f16
// ends at 2^16) it moves to the row's largest, kCacheLift less, so that small terms
// keep an absolute error of 2^(-25 - kCacheLift) of that one's. Past kCacheFar a step of f32
// is more than 1/4: the reference is then the largest itself, and differences stay exact.
constexpr float kCacheNoMax = -1.0e30f, kCacheFar = 4194304.f, kCacheLift = 7.f, kCacheTop = 15.f;
// Scales as the store writes them: kept within these, so that a key's probability is lost
// from the sum only where it is below 2^-46 of the largest (126 bits of f32's exponent
// less the 80 between two scales).
constexpr float kScaleLeast = 0x1p-40f, kScaleMost = 0x1p40f;

constexpr int kFewTile = 32;   // keys of a wave's tile
constexpr int kFewWaves = 4;
constexpr int kFewRows = 32;   // rows of an item

// Eight codes as f16, exact. int8: 1024 + (c + 128) is the f16 whose low byte is c + 128.
template <bool F8>
__device__ __forceinline__ half8_t cache_half8(uint32_t a, uint32_t b) {
  typedef half2_t h2;
  h2 r[4];
  if constexpr (F8) {
    r[0] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
    r[1] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
    r[2] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
    r[3] = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
  } else {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const h2 off = {(half_t)-1152.f, (half_t)-1152.f};
    r[0] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + off;
    r[1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + off;
    r[2] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
    r[3] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
  }
  return half8_t{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

// What a key's scales are in the softmax: a_k, b_k and 1 / v_scale_k. A value row that
// stands for NaN makes its key's score NaN.
struct KeyScales {
  float a, b, inv;
};
__device__ __forceinline__ KeyScales cache_scales(float ks, float vs, float qscale) {
  KeyScales r;
  const float v = fminf(fmaxf(vs, kScaleLeast), kScaleMost);
  r.a = vs == vs ? ks * qscale : NAN;
  r.b = __builtin_amdgcn_logf(v);
  r.inv = 1.0f / v;
  return r;
}

template <bool QF16>
__device__ __forceinline__ void cache_load_q(const void* q, int64_t off, half8_t& hi, half8_t& lo) {
  if constexpr (QF16) {
    hi = *(const half8_t*)((const half_t*)q + off);
  } else {
    const float4_t a = *(const float4_t*)((const float*)q + off), b = *(const float4_t*)((const float*)q + off + 4);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float f = j < 4 ? a[j & 3] : b[j & 3];
      hi[j] = (half_t)f;
      lo[j] = (half_t)(f - (float)hi[j]);
    }
  }
}

__device__ __forceinline__ void cache_out4(const CacheAttnArgs& a, int64_t off, float4_t v) {
  if (a.out_form == OUT_F32) {
    *(float4_t*)((float*)a.out + off) = v;
    return;
  }
  half4_t hv, lv;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    hv[e] = (half_t)v[e];
    lv[e] = (half_t)(v[e] - (float)hv[e]);
  }
  *(half4_t*)((half_t*)a.out + off) = hv;
  if (a.out_form == OUT_X2) *(half4_t*)((half_t*)a.out + a.out_lo + off) = lv;
}

// Which of the 32 keys from position t0 on a token sees, as bits. mask: its tree's.
// 64-bit shifts here go by amounts of the whole wave only: with a lane's amount in the last
// register that the wave has allocated, v_lshlrev_b64 has shifted by the lane's v0 instead
// (one register pair is read where one register is the amount, and the second lies past
// the allocation), on gfx950 and with the compiler none the wiser.
__device__ __forceinline__ uint32_t cache_ones(int n) {  // the lowest n bits, all from 32 on
  return n >= 32 ? ~0u : n > 0 ? (1u << n) - 1 : 0u;
}
__device__ __forceinline__ uint32_t cache_visible(const CacheItem& it, int tok, uint64_t mask, int t0) {
  uint32_t v;
  if (it.tree) {
    const int off = it.shift - t0;  // keys before the tree's
    v = off >= 32  ? ~0u
        : off > 0  ? ((uint32_t)mask << off) | cache_ones(off)
        : off > -64 ? (uint32_t)(mask >> -off)
                    : 0u;
  } else {
    v = cache_ones(tok + it.shift + 1 - t0);
  }
  return v & cache_ones(it.kv_hi - t0);
}

// LDS tiles hold rows of D bytes, their 16-byte chunks XOR-swizzled: K's so that the 16
// rows of one chunk that a quarter wave reads touch distinct banks, V's so that the 16
// rows of a half wave's transposing reads (rows 0..7 and 16..23, or those + 8) do.
template <int D>
__device__ __forceinline__ int cache_k_swz(int r) {
  return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int cache_v_swz(int r) {
  return D == 128 ? ((r >> 1) & 3) | ((r >> 4) & 1) << 2 : ((r >> 2) & 1) | ((r >> 4) & 1) << 1;
}

// Items of up to 16 RB rows. kFewWaves waves take tiles of 32 keys in turn, each through
// two LDS buffers of its own, filled by DMA through the page table; their results meet in
// LDS. S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: lane (l16, g) holds row
// l16 of each block of 16 rows, its scores at keys 16 kb + 4g + i, and of O^T dims
// 16 db + 4g + i.
template <int D>
struct CacheLds {
  char tiles[kFewWaves * 4 * kFewTile * D] __attribute__((aligned(1024)));
  float4_t scales[kFewWaves][3 * kFewTile / 4];
  float2 refs[kFewWaves][kFewRows];
};

template <int D, bool QF16, bool F8, int RB>
__device__ __forceinline__ void cache_rows_body(const CacheAttnArgs& a, CacheLds<D>& lds) {
  constexpr int TB = kFewTile * D, RPI = 1024 / D, NI = kFewTile / RPI, NS = D / 32, ND = D / 16;
  auto& tiles = lds.tiles;
  auto& scales = lds.scales;
  const CacheItem it = a.items[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const lds_t base = (lds_t)tiles + wave * 4 * TB;  // K and V of the even tiles, then of the odd ones
  float* mine = (float*)scales[wave];
  const uint32_t* table = a.pages + (int64_t)it.seq * a.max_pages;
  const int first = it.kv_lo + wave * kFewTile, step = kFewWaves * kFewTile;

  // The row of the lane's key (lane % 32) of the tile at t0; past the item's keys its last one.
  const auto key_page = [&](int t0) { return table[min(t0 + (lane & 31), it.kv_hi - 1) >> a.c.bshift]; };
  const auto key_row = [&](int t0, uint32_t page) {
    const int p = min(t0 + (lane & 31), it.kv_hi - 1);
    return (int)(((page * (uint32_t)a.c.Hkv + (uint32_t)it.kvh) << a.c.bshift) + (uint32_t)(p & ((1 << a.c.bshift) - 1)));
  };
  const auto dma = [&](int row, lds_t K, lds_t V) {
#pragma unroll
    for (int n = 0; n < NI; n++) {
      const int r = n * RPI + lane / (D / 16), c = lane % (D / 16);
      const int64_t at = (int64_t)__shfl(row, r, 64) * D;
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(a.c.k + at + 16 * (c ^ cache_k_swz<D>(r))),
          (__attribute__((address_space(3))) void*)(K + 1024 * n), 16, 0, kNonTemporal);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(a.c.v + at + 16 * (c ^ cache_v_swz<D>(r))),
          (__attribute__((address_space(3))) void*)(V + 1024 * n), 16, 0, kNonTemporal);
    }
  };

  // the first tile's rows and scales, the second's pages
  float ks = 0.f, vs = 1.f;
  uint32_t page = 0;
  if (first < it.kv_hi) {
    const int row = key_row(first, key_page(first));
    dma(row, base, base + TB);
    ks = a.c.ks[row];
    vs = a.c.vs[row];
    if (first + step < it.kv_hi) page = key_page(first + step);
  }

  half8_t qh[RB][NS], ql[RB][QF16 ? 1 : NS];
  float m[RB], l[RB];
  float4_t o[RB][ND];
  int tok[RB];
  uint64_t mask[RB];
#pragma unroll
  for (int b = 0; b < RB; b++) {
    const int r = 16 * b + l16, row = it.r0 + (r < it.nr ? r : 0), head = it.kvh * a.G + row % a.G;
    tok[b] = row / a.G;
    mask[b] = it.tree ? a.masks[it.q0 + tok[b]] : 0;
    const int64_t at = (int64_t)(it.q0 + tok[b]) * a.q_row + head * D;
    // step s of the first product takes dims 64 (s / 2) + 16 g + 8 (s % 2) + [0, 8): one
    // 16-byte read of K serves two steps
#pragma unroll
    for (int s = 0; s < NS; s++)
      cache_load_q<QF16>(a.q, at + 64 * (s / 2) + 16 * g + 8 * (s % 2), qh[b][s], ql[b][QF16 ? 0 : s]);
    m[b] = kCacheNoMax;
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; d++) o[b][d] = float4_t{};
  }
  // from here on a tile is seen in part by some row
  const int partly = it.tree ? it.shift : it.r0 / a.G + it.shift + 1;

  const auto tile = [&](int t0, lds_t K, lds_t V, lds_t Kn, lds_t Vn) {
    pack_wait();  // the tile has landed, and what was read of the other buffer has returned
    const KeyScales sk = cache_scales(ks, vs, a.qscale);
    if (lane < 32) {
      mine[lane] = sk.a;
      mine[kFewTile + lane] = sk.b;
      mine[2 * kFewTile + lane] = sk.inv;
    }
    if (t0 + step < it.kv_hi) {
      const int row = key_row(t0 + step, page);
      dma(row, Kn, Vn);
      ks = a.c.ks[row];
      vs = a.c.vs[row];
      if (t0 + 2 * step < it.kv_hi) page = key_page(t0 + 2 * step);
    }
    pack_wave_sync();
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    float4_t sc[RB][2];
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
#pragma unroll
      for (int b = 0; b < RB; b++) sc[b][kb] = float4_t{};
      const int r = 16 * kb + l16;
#pragma unroll
      for (int h = 0; h < D / 64; h++) {
        const u4 w = *(__attribute__((address_space(3))) u4*)(K + r * D + 16 * ((4 * h + g) ^ cache_k_swz<D>(r)));
        const half8_t k0 = cache_half8<F8>(w[0], w[1]), k1 = cache_half8<F8>(w[2], w[3]);
#pragma unroll
        for (int b = 0; b < RB; b++) {
          sc[b][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[b][2 * h], sc[b][kb], 0, 0, 0);
          sc[b][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[b][2 * h + 1], sc[b][kb], 0, 0, 0);
          if (!QF16) {
            sc[b][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[b][QF16 ? 0 : 2 * h], sc[b][kb], 0, 0, 0);
            sc[b][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[b][QF16 ? 0 : 2 * h + 1], sc[b][kb], 0, 0, 0);
          }
        }
      }
    }
    const bool masked = t0 + kFewTile > partly || t0 + kFewTile > it.kv_hi;
    half8_t ph[RB], pl[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) {
      const uint32_t vis = masked ? cache_visible(it, tok[b], mask[b], t0) >> (4 * g) : ~0u;
      float top = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        const float4_t ka = *(const float4_t*)(mine + 16 * kb + 4 * g);
        const float4_t kv = *(const float4_t*)(mine + kFewTile + 16 * kb + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float t = fmaf(sc[b][kb][i], ka[i], kv[i]);
          if (masked && !(vis >> (16 * kb + i) & 1)) t = -INFINITY;
          sc[b][kb][i] = t;
          top = fmaxf(top, t);
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const bool need = top > m[b] + kCacheTop;
      if (__builtin_amdgcn_ballot_w64(need)) {
        const float mnew = need ? (fabsf(top) > kCacheFar ? top : top - kCacheLift) : m[b];
        const float alpha = __builtin_amdgcn_exp2f(m[b] - mnew);
        l[b] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; d++) o[b][d] *= alpha;
        m[b] = mnew;
      }
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        const float4_t inv = *(const float4_t*)(mine + 2 * kFewTile + 16 * kb + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float p = __builtin_amdgcn_exp2f(sc[b][kb][i] - m[b]);
          const half_t h = (half_t)p;
          ph[b][4 * kb + i] = h;
          if (!QF16) pl[b][4 * kb + i] = (half_t)(p - (float)h);
          l[b] = fmaf(p, inv[i], l[b]);
        }
      }
    }
    // V^T: in each 16-lane group lane j names 8 bytes of the key that is index j / 2 of the
    // group's eight (4g + [0,4) and 16 + 4g + [0,4), as the scores lie) at dims 8 (j % 2) on,
    // and receives dim j of the eight
    typedef int i2 __attribute__((ext_vector_type(2)));
    const int vr = ((l16 >> 1) & 3) + 16 * (l16 >> 3) + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; d++) {
      const i2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (__attribute__((address_space(3))) i2*)(V + vr * D + 16 * (d ^ cache_v_swz<D>(vr)) + 8 * (l16 & 1)));
      const half8_t va = cache_half8<F8>((uint32_t)w[0], (uint32_t)w[1]);
#pragma unroll
      for (int b = 0; b < RB; b++) {
        o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[b], o[b][d], 0, 0, 0);
        if (!QF16) o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[b], o[b][d], 0, 0, 0);
      }
    }
  };
  for (int t0 = first; t0 < it.kv_hi; t0 += 2 * step) {
    tile(t0, base, base + TB, base + 2 * TB, base + 3 * TB);
    if (t0 + step < it.kv_hi) tile(t0 + step, base + 2 * TB, base + 3 * TB, base, base + TB);
  }

  // The waves' rows meet: each brings its own to the largest reference, then every wave
  // adds a share of the dims, a block of rows at a time.
#pragma unroll
  for (int b = 0; b < RB; b++) {
    l[b] += __shfl_xor(l[b], 16, 64);
    l[b] += __shfl_xor(l[b], 32, 64);
    if (lane < 16) lds.refs[wave][16 * b + lane] = float2{m[b], l[b]};
  }
  __syncthreads();
  typedef __attribute__((address_space(3))) float4_t* f4p;
  static_assert(4 * TB >= 2 * ND * 1024, "the tiles hold two blocks of the waves' results");
#pragma unroll
  for (int b = 0; b < RB; b++) {
    float M = lds.refs[0][16 * b + l16].x, L = 0.f;
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) M = fmaxf(M, lds.refs[w][16 * b + l16].x);
#pragma unroll
    for (int w = 0; w < kFewWaves; w++) {
      const float2 r = lds.refs[w][16 * b + l16];
      L += r.y * __builtin_amdgcn_exp2f(r.x - M);
    }
    const lds_t buf = (lds_t)tiles + (b & 1) * (kFewWaves * ND * 1024) + lane * 16;
    const float own = __builtin_amdgcn_exp2f(m[b] - M);
#pragma unroll
    for (int d = 0; d < ND; d++) *(f4p)(buf + (wave * ND + d) * 1024) = o[b][d] * own;
    __syncthreads();
    const int r = 16 * b + l16;
    const bool live = r < it.nr, part = it.part >= 0;
    const int row = it.r0 + r, t = row / a.G, head = it.kvh * a.G + row % a.G;
    if (part && live && wave == 0 && g == 0)
      *(float4_t*)(a.part_ml + ((int64_t)it.part + r) * 4) = float4_t{M, 0.f, L, 0.f};
    const float mul = part ? 1.f : L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int x = 0; x < ND / kFewWaves; x++) {
      const int d = wave * (ND / kFewWaves) + x;
      float4_t v = float4_t{};
#pragma unroll
      for (int w = 0; w < kFewWaves; w++) v += *(f4p)(buf + (w * ND + d) * 1024);
      if (!live) continue;
      v *= mul;
      if (part) *(float4_t*)(a.part_o + ((int64_t)it.part + r) * D + 16 * d + 4 * g) = v;
      else cache_out4(a, (int64_t)(it.q0 + t) * a.out_row + head * D + 16 * d + 4 * g, v);
    }
  }
}

// Up to kFewRows rows: 16 or 32, two workgroups a CU.
template <int D, bool QF16, bool F8>
__global__ __launch_bounds__(64 * kFewWaves, 2) void cache_few_kernel(CacheAttnArgs a) {
  __shared__ CacheLds<D> lds;
  if (a.items[blockIdx.x].nr <= 16) cache_rows_body<D, QF16, F8, 1>(a, lds);
  else cache_rows_body<D, QF16, F8, 2>(a, lds);
}
// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

void cache_build_plan(int B, const int32_t* extents, const int32_t* lengths, const uint8_t* tree, int H, int Hkv, int D,
                      bool q_f16, int ncu, CachePlan& plan) {
  plan = CachePlan();
  plan.H = H;
  const int G = H / Hkv;
  std::vector<PackedItem> whole, cut;
  int64_t q0 = 0;
  for (int s = 0; s < B; s++) {
    const int64_t rows = (int64_t)extents[s] * G;
    const int shift = lengths[s] - extents[s];
    for (int64_t r0 = 0; r0 < rows; r0 += kFewRows) {
      const int nr = (int)std::min<int64_t>(kFewRows, rows - r0);
      const int hi = (int)std::min<int64_t>(lengths[s], (r0 + nr - 1) / G + shift + 1);
      for (int h = 0; h < Hkv; h++)  // k0: the sequence
        whole.push_back(PackedItem{(int32_t)q0, s, lengths[s], shift, (int32_t)r0, nr, 0, hi, h, -1});
    }
    q0 += extents[s];
  }
  plan.tq = q0;
  PackedPlan merges;
  pack_cut(whole, kFewTile * kFewWaves, 2, ncu, PackRate{1.8 * D / 128.0, 0.7}, cut, merges);
  plan.merges = std::move(merges.merges);
  plan.part_rows = merges.part_rows;
  plan.items.reserve(cut.size());
  for (const PackedItem& p : cut)
    plan.items.push_back(CacheItem{p.q0, p.k0, p.nk, p.shift, p.r0, p.nr, p.kv_lo, p.kv_hi, p.kvh, p.part,
                                   tree && tree[p.k0] ? 1 : 0, 0});
}

template <int D, bool QF16, bool F8>
static void cache_attention_launch(CacheAttnArgs a, hipStream_t st) {
  if (a.few) hipLaunchKernelGGL((cache_few_kernel<D, QF16, F8>), dim3(a.few), dim3(64 * kFewWaves), 0, st, a);
}
template <int D>
static void cache_attention_form(const CacheAttnArgs& a, hipStream_t st) {
  if (a.q_f16) a.c.f8 ? cache_attention_launch<D, true, true>(a, st) : cache_attention_launch<D, true, false>(a, st);
  else a.c.f8 ? cache_attention_launch<D, false, true>(a, st) : cache_attention_launch<D, false, false>(a, st);
}

int cache_attention_enqueue(const CacheAttnArgs& a, hipStream_t st) {
  if (a.c.d == 128) cache_attention_form<128>(a, st);
  else cache_attention_form<64>(a, st);
  if (a.nmerges) {
    PackedArgs p{};
    p.out = a.out;
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.merges = a.merges;
    p.out_row = a.out_row;
    p.out_lo = a.out_lo;
    p.G = a.G;
    p.out_form = a.out_form;
    packed_merge_enqueue(p, a.c.d, a.nmerges, st);
  }
  TGOHIP_HIP(hipGetLastError());
  return 0;
}

}  // namespace tgohip
