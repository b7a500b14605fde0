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
//
// What bounds it: few rows read the codes once, at HBM's rate; with many a wave's products and its
// exponentials take turns, the matrix unit and the VALU each busy 41 to 52% of the time. Measured (32
// heads over 8 of 128 dims, us a call among others, merges in it, from card to card): one f32 token over 8192 int8
// keys 11.4 (two launches and chains of dependent loads; 1.2 more where 36 layers take turns and the
// keys come from HBM); 128 over 16 to 8192 keys 64, the kernel 61, 5.7 TB/s (a plain read here 6.6); 32 trees
// of 16 to 64 tokens over 285 to 4030 keys 92 to 95, of f16 queries 69 to 75; four f32 chunks of 187 to 405 over
// 2616 to 5417 e4m3 keys 133 to 141, f16 111 to 115; 128 tokens over 256 to 4096 keys and two chunks of 512 in one call 154 to
// 159, f16 129 to 133; 2048 f16 tokens, the last of 32768, 1126 to 1177, 0.91 to 0.95 PFLOP/s (a large f16
// matrix product here 1.27).
#include "pack_rows.h"

#include <algorithm>
#include <type_traits>

namespace tgohip {

constexpr int kNonTemporal = 2;  // the nt bit: a context's rows are read once
// The reference starts at kCacheNoMax; where a term passes it by more than 2^kCacheTop (f16
// ends at 2^16) it moves to the row's largest, kCacheLift less, so that small terms
// keep an absolute error of 2^(-25 - kCacheLift) of that one's. Past kCacheFar a step of f32
// is more than 1/4: the reference is then the largest itself, and terms are taken from scores rounded to
// f32 as it was (a multiply-add's would differ from it by what it lacks, at 2^28 up to 16). Whether a term
// passes it is asked of their difference: of scores 16 apart at 2^24, where steps are 2, m + 15 may round to
// m + 16.
constexpr float kCacheNoMax = kPackLeast, kCacheFar = 4194304.f, kCacheLift = 7.f, kCacheTop = 15.f;
// Scales as the store writes them: kept within these, so that a key's probability is lost
// from the sum only where it is below 2^-46 of the largest (126 bits of f32's exponent
// less the 80 between two scales).
constexpr float kScaleLeast = 0x1p-40f, kScaleMost = 0x1p40f;

constexpr int kFewTile = 32;   // keys of a wave's tile
constexpr int kFewWaves = 4;
constexpr int kFewRows = 32;   // rows of an item
// Up to so many rows at the end of a (sequence, head)'s go as such items. Up to 32 / 64 / 96 / 256,
// us: 32 trees of 64 to 256 rows 97.6 / 94.4 / 95.0 / 100.8, four chunks of 748 to 1620
// 141.5 / 141.5 / 141.4 / 144.1.
constexpr int kFewLast = 64;

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

// What a key's scales are in the softmax: a_k, b_k / a_k and 1 / v_scale_k. The products
// accumulate onto b_k / a_k, so that one product makes a score of them, or one multiply-add a
// term's exponent, a_k (b_k / a_k + S_k) - m. A row that stands for NaN makes its key's start NaN, not a_k:
// a masked score, -inf by then, stays so.
struct KeyScales {
  float a, start, inv;
};
__device__ __forceinline__ KeyScales cache_scales(float ks, float vs, float qscale) {
  KeyScales r;
  const float v = fminf(fmaxf(vs, kScaleLeast), kScaleMost);
  r.a = fminf(fmaxf(ks, kScaleLeast), kScaleMost) * qscale;
  r.start = ks == ks && vs == vs ? __builtin_amdgcn_logf(v) * __builtin_amdgcn_rcpf(r.a) : NAN;
  r.inv = __builtin_amdgcn_rcpf(v);
  return r;
}

// What two terms lack as f16: an exact difference each (one instruction that reads the half
// as it is; the compiler makes it a conversion and a subtraction), rounded.
typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ half2_t cache_rest2(float2_t p, half2_t h) {
  float2_t r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r[0]) : "v"(h), "v"(p[0]));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r[1]) : "v"(h), "v"(p[1]));
  return __builtin_convertvector(r, half2_t);
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
// 16 db + 4g + i. A tile stays 8 bits in LDS and is converted by the wave that uses it, V by
// the transposing read of bytes. Probabilities are pairs for f16 queries too: 128 tokens 62.7 us, with f16
// ones 62.1 and 1.1e-4 from the definition beside the output's rounding. Single tokens (4 rows of 16 used) by items of 16 / 32 rows, us: 128 of
// 16 to 8192 keys 65 / 81, one of 8192 11.6 / 13.3. The next tile's loads before the wait for this
// one (twice the bytes in flight): no faster, 64.7 beside 64.0.
template <int D, bool QF16, bool F8, int RB>
__device__ __forceinline__ void cache_rows_body(const CacheAttnArgs& a, const CacheItem& it, lds_t K0, lds_t V0, lds_t K1,
                                                lds_t V1, float* scales, float2* refs) {
  constexpr int TB = kFewTile * D, RPI = 1024 / D, NI = kFewTile / RPI, NS = D / 32, ND = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const lds_t Kw[2] = {K0 + wave * TB, K1 + wave * TB}, Vw[2] = {V0 + wave * TB, V1 + wave * TB};
  float* mine = scales + wave * 3 * kFewTile;
  const uint32_t* table = a.pages + (int64_t)it.seq * a.max_pages;
  const uint32_t head_row = (uint32_t)it.kvh << a.c.bshift;
  const int first = it.kv_lo + wave * kFewTile, step = kFewWaves * kFewTile;

  // The row of the lane's key (lane % 32) of the tile at t0; past the item's keys its last one.
  const auto key_page = [&](int t0) { return table[min(t0 + (lane & 31), it.kv_hi - 1) >> a.c.bshift]; };
  const auto key_row = [&](int t0, uint32_t page) {
    const int p = min(t0 + (lane & 31), it.kv_hi - 1);
    return (int)(page + head_row + (uint32_t)(p & ((1 << a.c.bshift) - 1)));
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
    dma(row, Kw[0], Vw[0]);
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
      pack_load_q<QF16>(a.q, at + 64 * (s / 2) + 16 * g + 8 * (s % 2), qh[b][s], ql[b][QF16 ? 0 : s]);
    m[b] = kCacheNoMax;
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; d++) o[b][d] = float4_t{};
  }
  // from here on a tile is seen in part by some row
  const int partly = it.tree ? it.shift : it.r0 / a.G + it.shift + 1;

  const auto tile = [&](int t0, lds_t K, lds_t V, lds_t Kn, lds_t Vn) {
#pragma clang fp contract(off)  // a product fused into the subtraction would not be the score that m came from
    pack_wait();  // the tile has landed, and what was read of the other buffer has returned
    const KeyScales sk = cache_scales(ks, vs, a.qscale);
    if (lane < 32) {
      mine[lane] = sk.a;
      mine[kFewTile + lane] = sk.start;
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
      for (int b = 0; b < RB; b++) sc[b][kb] = *(const float4_t*)(mine + kFewTile + 16 * kb + 4 * g);
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
      float4_t ka[2];
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        ka[kb] = *(const float4_t*)(mine + 16 * kb + 4 * g);
        sc[b][kb] *= ka[kb];
      }
      if (masked) {
        const uint32_t vis = cache_visible(it, tok[b], mask[b], t0) >> (4 * g);
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (!(vis >> (16 * kb + i) & 1)) sc[b][kb][i] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, sc[b][kb][i]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const bool need = top - m[b] > kCacheTop;
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
        for (int i = 0; i < 4; i += 2) {
          const float2_t p = {__builtin_amdgcn_exp2f(sc[b][kb][i] - m[b]), __builtin_amdgcn_exp2f(sc[b][kb][i + 1] - m[b])};
          const half2_t h = __builtin_convertvector(p, half2_t);
          ph[b][4 * kb + i] = h[0];
          ph[b][4 * kb + i + 1] = h[1];
          const half2_t r = cache_rest2(p, h);
          pl[b][4 * kb + i] = r[0];
          pl[b][4 * kb + i + 1] = r[1];
          l[b] = fmaf(p[0], inv[i], l[b]);
          l[b] = fmaf(p[1], inv[i + 1], l[b]);
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
        o[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[b], o[b][d], 0, 0, 0);
      }
    }
  };
  for (int t0 = first; t0 < it.kv_hi; t0 += 2 * step) {
    tile(t0, Kw[0], Vw[0], Kw[1], Vw[1]);
    if (t0 + step < it.kv_hi) tile(t0 + step, Kw[1], Vw[1], Kw[0], Vw[0]);
  }

  // The waves' rows meet: each brings its own to the largest reference, then every wave
  // adds a share of the dims, a block of rows at a time.
#pragma unroll
  for (int b = 0; b < RB; b++) {
    l[b] += __shfl_xor(l[b], 16, 64);
    l[b] += __shfl_xor(l[b], 32, 64);
    if (lane < 16) refs[wave * kFewRows + 16 * b + lane] = float2{m[b], l[b]};
  }
  __syncthreads();
  typedef __attribute__((address_space(3))) float4_t* f4p;
  static_assert(2 * TB == ND * 1024, "a K and a V tile hold a block of a wave's results");
  const auto merge = [&](auto block) {
    constexpr int b = decltype(block)::value;
    float M = refs[16 * b + l16].x, L = 0.f;
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) M = fmaxf(M, refs[w * kFewRows + 16 * b + l16].x);
#pragma unroll
    for (int w = 0; w < kFewWaves; w++) {
      const float2 r = refs[w * kFewRows + 16 * b + l16];
      L += r.y * __builtin_amdgcn_exp2f(r.x - M);
    }
    const lds_t lo = b ? K1 : K0, hi = b ? V1 : V0;
    const auto at = [&](int w, int d) { return (d < ND / 2 ? lo : hi) + w * TB + d % (ND / 2) * 1024 + lane * 16; };
    const float own = __builtin_amdgcn_exp2f(m[b] - M);
#pragma unroll
    for (int d = 0; d < ND; d++) *(f4p)at(wave, d) = o[b][d] * own;
    __syncthreads();
    const int r = 16 * b + l16;
    const bool live = r < it.nr, part = it.part >= 0;
    const int row = it.r0 + r, t = row / a.G, head = it.kvh * a.G + row % a.G;
    // A sum of 0 is a row's whose scores are all -inf, which is NaN, or of a part that shows it no key. (A
    // part of a tree's shows each row some: it holds more keys than a tree.)
    const bool blank = L == 0.f && t + it.shift >= it.kv_lo;
    if (part && live && wave == 0 && g == 0)
      *(float4_t*)(a.part_ml + ((int64_t)it.part + r) * 4) = float4_t{blank ? NAN : M, 0.f, L, 0.f};
    const float mul = part ? 1.f : blank ? NAN : 1.f / L;
#pragma unroll
    for (int x = 0; x < ND / kFewWaves; x++) {
      const int d = wave * (ND / kFewWaves) + x;
      float4_t v = float4_t{};
#pragma unroll
      for (int w = 0; w < kFewWaves; w++) v += *(f4p)at(w, d);
      if (!live) continue;
      v *= mul;
      if (part) *(float4_t*)(a.part_o + ((int64_t)it.part + r) * D + 16 * d + 4 * g) = v;
      else pack_store4(a, (int64_t)(it.q0 + t) * a.out_row + head * D + 16 * d + 4 * g, v);
    }
  };
  static_assert(RB <= 2, "a pair of buffers for each block");
  merge(std::integral_constant<int, 0>{});
  if constexpr (RB == 2) merge(std::integral_constant<int, 1>{});
}

// Items of up to 32 WAVES rows, 32 a wave: chunks, and trees of more rows. Tiles of 64 keys as
// f16 in LDS, converted once for all rows: the next tile's codes come through registers while
// this one is used, and go into the other buffer behind it. Products as packed_kernel's. By
// items of 32 rows alone (each converts for itself): 2048 f16 tokens behind 30720 positions 1941 us
// beside 1235.
template <int D, bool QF16, bool F8, int WAVES>
__device__ __forceinline__ void cache_tile_body(const CacheAttnArgs& a, const CacheItem& it, lds_t K0, lds_t V0, lds_t K1,
                                                lds_t V1, float* S0, float* S1) {
  constexpr int TB = kPackTile * D * 2, CH = D / 16, ROWS = 64 * WAVES / CH;
  constexpr int RPI = ROWS < kPackTile ? ROWS : kPackTile, NI = kPackTile / RPI;  // with D 64 and 8 waves some idle
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kh = lane >> 5, w0 = 32 * wave;
  PackedArgs pa{};
  pa.q = a.q;
  pa.out = a.out;
  pa.part_o = a.part_o;
  pa.part_ml = a.part_ml;
  pa.q_row = a.q_row;
  pa.out_row = a.out_row;
  pa.out_lo = a.out_lo;
  pa.G = a.G;
  pa.out_form = a.out_form;
  const PackedItem pit{it.q0, 0, it.nk, it.shift, it.r0, it.nr, it.kv_lo, it.kv_hi, it.kvh, it.part};
  const uint32_t* table = a.pages + (int64_t)it.seq * a.max_pages;
  const uint32_t head_row = (uint32_t)it.kvh << a.c.bshift;
  const int kat = pack_k_at<D>(lane & 31, kh), vat = pack_v_at<D>(lane);

  // A thread's chunk of 16 codes of rows p, p + RPI of a tile; the first wave's key for scales.
  const int p = min(tid / CH, kPackTile - 1), c = tid % CH;
  u4 rk[NI], rv[NI];
  uint32_t page[NI], key_page = 0;
  float ks = 0.f, vs = 1.f;
  const auto row_of = [&](int pos, uint32_t pg) {
    return (int64_t)(pg + head_row + (uint32_t)(pos & ((1 << a.c.bshift) - 1)));
  };
  const auto pages = [&](int t0) {
#pragma unroll
    for (int n = 0; n < NI; n++) page[n] = table[min(t0 + n * RPI + p, it.kv_hi - 1) >> a.c.bshift];
    if (tid < kPackTile) key_page = table[min(t0 + tid, it.kv_hi - 1) >> a.c.bshift];
  };
  // Past the item's keys: its last one.
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int n = 0; n < NI; n++) {
      const int64_t at = row_of(min(t0 + n * RPI + p, it.kv_hi - 1), page[n]) * D + 16 * c;
      rk[n] = *(const u4*)(a.c.k + at);
      rv[n] = *(const u4*)(a.c.v + at);
    }
    if (tid < kPackTile) {
      const int64_t at = row_of(min(t0 + tid, it.kv_hi - 1), key_page);
      ks = a.c.ks[at];
      vs = a.c.vs[at];
    }
  };
  const auto put = [&](lds_t K, lds_t V, float* S) {
    typedef __attribute__((address_space(3))) half8_t* h8;
#pragma unroll
    for (int n = 0; n < NI; n++) {
      const int r = n * RPI + p;
      *(h8)(K + r * 2 * D + 16 * ((2 * c) ^ pack_k_swz<D>(r))) = cache_half8<F8>(rk[n][0], rk[n][1]);
      *(h8)(K + r * 2 * D + 16 * ((2 * c + 1) ^ pack_k_swz<D>(r))) = cache_half8<F8>(rk[n][2], rk[n][3]);
      *(h8)(V + r * 2 * D + 16 * ((2 * c) ^ pack_v_swz<D>(r))) = cache_half8<F8>(rv[n][0], rv[n][1]);
      *(h8)(V + r * 2 * D + 16 * ((2 * c + 1) ^ pack_v_swz<D>(r))) = cache_half8<F8>(rv[n][2], rv[n][3]);
    }
    if (tid < kPackTile) {
      const KeyScales s = cache_scales(ks, vs, a.qscale);
      S[tid] = s.a;
      S[kPackTile + tid] = s.start;
      S[2 * kPackTile + tid] = s.inv;
    }
  };
  pages(it.kv_lo);
  fetch(it.kv_lo);
  if (it.kv_lo + kPackTile < it.kv_hi) pages(it.kv_lo + kPackTile);
  PackRows<D, QF16> w;
  w.init(pa, pit, w0, lane);
  w.m = kCacheNoMax;
  const int tok = (it.r0 + (w.r < it.nr ? w.r : 0)) / a.G;
  const uint64_t mask = it.tree ? a.masks[it.q0 + tok] : 0;
  // the first position that some row of the wave may not see, the last that some row may
  const int partly = it.tree ? it.shift : (it.r0 + w0) / a.G + it.shift + 1;
  const int whi = w0 < it.nr ? (it.r0 + min(w0 + 32, it.nr) - 1) / a.G + it.shift : -1;
  // f16 queries: above this a term has passed its range, 2^kCacheTop; below 0 where the row's reference is far
  float limit = 32768.f;
  put(K0, V0, S0);
  __syncthreads();

  const auto tile = [&](int t0, lds_t K, lds_t V, const float* S, lds_t Kn, lds_t Vn, float* Sn) {
    const bool more = t0 + kPackTile < it.kv_hi;
    if (more) {
      fetch(t0 + kPackTile);
      if (t0 + 2 * kPackTile < it.kv_hi) pages(t0 + 2 * kPackTile);
    }
    if (t0 <= whi) {
      // S^T onto where each key's starts, in the lane's order of keys: 32 pb + 8 (i / 4) + 4 kh + i % 4
      float16_t sc[2];
      const auto scores = [&] {
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const float4_t st = *(const float4_t*)(S + kPackTile + 8 * x + 4 * kh);
#pragma unroll
          for (int e = 0; e < 4; e++) sc[x >> 2][4 * (x & 3) + e] = st[e];
        }
#pragma unroll
        for (int s = 0; s < D / 16; s++) {
          half8_t ka[2];
#pragma unroll
          for (int pb = 0; pb < 2; pb++) ka[pb] = pack_k_frag(K, (kat ^ (32 * s)) + 64 * D * pb);
#pragma unroll
          for (int pb = 0; pb < 2; pb++) sc[pb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[pb], w.qh[s], sc[pb], 0, 0, 0);
          if (!QF16) {
#pragma unroll
            for (int pb = 0; pb < 2; pb++)
              sc[pb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[pb], w.ql[QF16 ? 0 : s], sc[pb], 0, 0, 0);
            if (s % 2) __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (t0 + kPackTile > partly || t0 + kPackTile > it.kv_hi) {
#pragma unroll
          for (int pb = 0; pb < 2; pb++) {
            const uint32_t vis = cache_visible(it, tok, mask, t0 + 32 * pb) >> (4 * kh);
#pragma unroll
            for (int i = 0; i < 16; i++)
              if (!(vis >> (8 * (i >> 2) + (i & 3)) & 1)) sc[pb][i] = -INFINITY;
          }
        }
      };
      scores();
      __builtin_amdgcn_sched_barrier(0);
      // The scores as f32 rounds them, in place, and the row's largest.
      const auto scale = [&] {
#pragma clang fp contract(off)  // a product fused into what comes after would not be the score that m came from
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const float4_t ka = *(const float4_t*)(S + 8 * x + 4 * kh);
#pragma unroll
          for (int e = 0; e < 4; e++) sc[x >> 2][4 * (x & 3) + e] *= ka[e];
        }
      };
      const auto largest = [&](bool scaled) {
#pragma clang fp contract(off)
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const float4_t ka = *(const float4_t*)(S + 8 * x + 4 * kh);
#pragma unroll
          for (int e = 0; e < 4; e++) top = fmaxf(top, sc[x >> 2][4 * (x & 3) + e] * (scaled ? 1.f : ka[e]));
        }
        return fmaxf(top, __shfl_xor(top, 32, 64));
      };
      const auto raise = [&](float top, bool need) {
        const float mnew = need ? (fabsf(top) > kCacheFar ? top : top - kCacheLift) : w.m;
        const float alpha = __builtin_amdgcn_exp2f(w.m - mnew);
        w.l *= alpha;
#pragma unroll
        for (int db = 0; db < D / 32; db++) w.o[db] *= alpha;
        w.m = mnew;
      };
      // Step u's eight terms, their share of the sum on l; scaled: sc holds rounded scores.
      const auto terms = [&](bool scaled, int u, half8_t& ph, half8_t& pl, float& l, float& most) {
#pragma clang fp contract(off)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const float4_t ka = *(const float4_t*)(S + 16 * u + 8 * y + 4 * kh);
          const float4_t inv = *(const float4_t*)(S + 2 * kPackTile + 16 * u + 8 * y + 4 * kh);
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int i = 8 * (u & 1) + 4 * y + e;
            float2_t x;
#pragma unroll
            for (int f = 0; f < 2; f++)
              x[f] = __builtin_amdgcn_exp2f(fmaf(sc[u >> 1][i + f], scaled ? 1.f : ka[e + f], -w.m));
            const half2_t h = __builtin_convertvector(x, half2_t);
            ph[4 * y + e] = h[0];
            ph[4 * y + e + 1] = h[1];
            if (QF16) {
              most = fmaxf(fmaxf(most, x[0]), x[1]);
            } else {
              const half2_t r = cache_rest2(x, h);
              pl[4 * y + e] = r[0];
              pl[4 * y + e + 1] = r[1];
            }
            l = fmaf(x[0], inv[e], l);
            l = fmaf(x[1], inv[e + 1], l);
          }
        }
      };
      if constexpr (QF16) {
        // All terms by the reference as it is; only where one of a row's has passed f16's range (its
        // first tile, or a key far above the ones before), or its reference is far, is its largest looked
        // for. Each row by itself: no bit of it depends on the wave's others. Scores rounded in every
        // tile, as f32 queries' are: 1210 us beside 1177 for 2048 tokens behind 30720 positions. f16
        // probabilities are within 2^-11 each, 1e-4 of the result beside the 2.1e-4 that an f16 output is rounded by;
        // as pairs (in f32 queries' order of steps) that call takes 1519 us beside 1165, a prompt of 2048 88 beside
        // 76, 32 trees 82 beside 74.
        half8_t ph[4], none;
        float l[4] = {}, most = 0.f;
#pragma unroll
        for (int u = 0; u < 4; u++) terms(false, u, ph[u], none, l[u], most);
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_amdgcn_ballot_w64(most > limit)) {
          const bool passed = fmaxf(most, __shfl_xor(most, 32, 64)) > limit;
          const float top = largest(false);
          raise(top, limit < 0.f ? top - w.m > kCacheTop : passed);
          const bool scaled = fabsf(w.m) > kCacheFar && w.m != kCacheNoMax;
          if (scaled) scale();
          limit = scaled ? -1.f : 32768.f;
#pragma unroll
          for (int u = 0; u < 4; u++) {
            l[u] = 0.f;
            terms(scaled, u, ph[u], none, l[u], most);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
          for (int db = 0; db < D / 32; db++)
            w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pack_v_frag<D>(V, (vat ^ (64 * db)) + 32 * D * u), ph[u], w.o[db], 0, 0, 0);
        w.l += (l[0] + l[1]) + (l[2] + l[3]);
      } else {
        scale();
        const float top = largest(true);
        const bool need = top - w.m > kCacheTop;
        if (__builtin_amdgcn_ballot_w64(need)) raise(top, need);
        // pairs go step by step: all at once would not fit the registers beside the queries'
        float l[2] = {}, most;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          half8_t ph, pl;
          terms(true, u, ph, pl, l[u & 1], most);
          half8_t va[D / 32];
#pragma unroll
          for (int db = 0; db < D / 32; db++) va[db] = pack_v_frag<D>(V, (vat ^ (64 * db)) + 32 * D * u);
#pragma unroll
          for (int db = 0; db < D / 32; db++) w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[db], ph, w.o[db], 0, 0, 0);
#pragma unroll
          for (int db = 0; db < D / 32; db++) w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[db], pl, w.o[db], 0, 0, 0);
        }
        w.l += l[0] + l[1];
      }
    }
    if (more) put(Kn, Vn, Sn);
    __syncthreads();
  };
  for (int t0 = it.kv_lo; t0 < it.kv_hi; t0 += 2 * kPackTile) {
    tile(t0, K0, V0, S0, K1, V1, S1);
    if (t0 + kPackTile < it.kv_hi) tile(t0 + kPackTile, K1, V1, S1, K0, V0, S0);
  }
  static_assert(TB == 128 * D, "a tile holds a wave's rows");
  const int turn = wave % 4;
  const lds_t buf = turn == 0 ? K0 : turn == 1 ? V0 : turn == 2 ? K1 : V1;
  if (wave < 4) w.write(pa, pit, lane, buf);
  if (WAVES > 4) {
    __syncthreads();
    if (wave >= 4) w.write(pa, pit, lane, buf);
  }
}

// Items of all kinds, two workgroups a CU: chunks, trees and single tokens of a batch run
// beside each other. Registers end at 256 for that: with 128 dims the tile body spills 10 or 11 of them for
// f16 queries (40 bytes a lane), none or 2 for f32.
template <int D, bool QF16, bool F8>
__global__ __launch_bounds__(256, 2) void cache_attention_kernel(CacheAttnArgs a) {
  // an array for each buffer: a read of one does not wait for the DMA into another
  __shared__ __attribute__((aligned(1024))) char K0[128 * D], V0[128 * D], K1[128 * D], V1[128 * D];
  __shared__ __attribute__((aligned(16))) float S0[kFewWaves * 3 * kFewTile], S1[kFewWaves * 2 * kFewRows];
  static_assert(kFewWaves * kFewTile == 128 && 2 * kPackTile == 128, "buffers of either body");
  static_assert(3 * kPackTile <= kFewWaves * 2 * kFewRows && 3 * kPackTile <= kFewWaves * 3 * kFewTile, "scales of either");
  const CacheItem it = a.items[blockIdx.x];
  const lds_t k0 = (lds_t)K0, v0 = (lds_t)V0, k1 = (lds_t)K1, v1 = (lds_t)V1;
  if (it.nr > kFewRows) cache_tile_body<D, QF16, F8, 4>(a, it, k0, v0, k1, v1, S0, S1);
  else if (it.nr > 16) cache_rows_body<D, QF16, F8, 2>(a, it, k0, v0, k1, v1, S0, (float2*)S1);
  else cache_rows_body<D, QF16, F8, 1>(a, it, k0, v0, k1, v1, S0, (float2*)S1);
}
// Items of 256 rows, one workgroup a CU.
template <int D, bool F8>
__global__ __launch_bounds__(512, 1) void cache_wide_kernel(CacheAttnArgs a) {
  __shared__ __attribute__((aligned(1024))) char K0[128 * D], V0[128 * D], K1[128 * D], V1[128 * D];
  __shared__ __attribute__((aligned(16))) float S0[3 * kPackTile], S1[3 * kPackTile];
  const CacheItem it = a.items[blockIdx.x];
  cache_tile_body<D, true, F8, 8>(a, it, (lds_t)K0, (lds_t)V0, (lds_t)K1, (lds_t)V1, S0, S1);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Host time of a plan, its upload and the binding: 18 to 24 us for one sequence or a few, 76 for 128 single tokens,
// 131 for 512, 78 for 32 trees; once for all layers of a step.
void cache_build_plan(int B, const int32_t* extents, const int32_t* lengths, const uint8_t* tree, int H, int Hkv, int D,
                      bool q_f16, int ncu, CachePlan& plan) {
  plan = CachePlan();
  plan.H = H;
  const int G = H / Hkv;
  std::vector<PackedItem> whole[2], cut[2];  // tiles, few rows
  const double dims = D / 128.0;
  const PackRate tiles = q_f16 ? PackRate{1.6 * dims, 0.6} : PackRate{2.2 * dims, 0.55};
  // f16 queries in blocks of 256 rows (one workgroup a CU, half the tiles to convert) where that pads
  // little. Of 128 / 256, us: 2048 tokens behind 30720 positions 1232 / 1134; the padding weighs
  // as much as rows do. f32 queries' pairs leave no registers for it. Where few rows follow, they
  // are a launch of their own behind it, which ends and starts for some 20 us of a CU's time: then
  // only where blocks of 128 would take kWideLeast. 512 tokens behind 1536 and 64 decoders of 1024 to
  // 4096 positions 84 / 106, a prompt of 2048 and 32 of 512 to 2048 74 / 97, 2048 behind 16384 and 128
  // of 2048 to 8192 867 / 821.
  constexpr double kWideLeast = 250.;  // us
  int64_t narrow = 0, wide = 0;
  bool others = false;
  for (int s = 0; s < B; s++) {
    const int64_t rows = (int64_t)extents[s] * G;
    others = others || (rows && (rows - 1) % 256 < kFewLast);
    if (rows <= kFewRows) continue;
    narrow += (rows + 127) / 128 * 128 * lengths[s];
    wide += (rows + 255) / 256 * 256 * lengths[s];
  }
  const double time = (double)narrow / (128 * kPackTile) * Hkv * tiles.tile / tiles.shared / (2 * ncu);
  const int most = q_f16 && 10 * wide <= 11 * narrow && (!others || time > kWideLeast) ? 256 : 128;  // rows of an item
  int64_t q0 = 0;
  for (int s = 0; s < B; s++) {
    const int64_t rows = (int64_t)extents[s] * G;
    const int shift = lengths[s] - extents[s];
    for (int64_t r0 = 0, nr; r0 < rows; r0 += nr) {
      const int64_t left = rows - r0;
      nr = std::min<int64_t>(left, left <= kFewLast ? kFewRows : most);
      const int hi = (int)std::min<int64_t>(lengths[s], (r0 + nr - 1) / G + shift + 1);
      for (int h = 0; h < Hkv; h++)  // k0: the sequence
        whole[nr <= kFewRows].push_back(PackedItem{(int32_t)q0, s, lengths[s], shift, (int32_t)r0, (int)nr, 0, hi, h, -1});
    }
    q0 += extents[s];
  }
  plan.tq = q0;
  // Each kind is cut for its share of the CUs, by what it costs (key: us of an item's key). Both in
  // one launch / one behind the other: 32 trees whose last rows are few 94 / 112 us. Pieces of many
  // rows hold more keys than a tree has tokens, so that each row sees one of them; at least
  // 8 / 12 / 20 tiles: 95.6 / 92.2 / 107.
  const PackRate rate[2] = {most == 256 ? PackRate{2.2 * dims, 0.5} : tiles, PackRate{1.8 * dims, 0.7}};
  const int tile[2] = {kPackTile, kFewTile * kFewWaves}, least[2] = {12, 2};
  double cost[2] = {}, key[2];
  for (int f = 0; f < 2; f++) {
    key[f] = rate[f].tile / rate[f].shared / tile[f];
    for (const PackedItem& it : whole[f]) cost[f] += it.kv_hi * key[f];
  }
  PackedPlan merges;
  for (int f = 0; f < 2; f++) {
    const double share = most == 256 ? 1.0 : cost[f] / std::max(cost[0] + cost[1], 1e-9);
    pack_cut(whole[f], tile[f], least[f], std::max(1, (int)(ncu * share + 0.5)), rate[f], cut[f], merges);
  }
  plan.merges = std::move(merges.merges);
  plan.part_rows = merges.part_rows;
  plan.wide = most == 256 ? (int)cut[0].size() : 0;
  plan.items.reserve(cut[0].size() + cut[1].size());
  const auto take = [&](const PackedItem& p) {
    plan.items.push_back(CacheItem{p.q0, p.k0, p.nk, p.shift, p.r0, p.nr, p.kv_lo, p.kv_hi, p.kvh, p.part,
                                   tree && tree[p.k0] ? 1 : 0, 0});
  };
  // longest first, both kinds together where one kernel takes them
  size_t f = 0;
  for (const PackedItem& p : cut[0]) {
    while (!plan.wide && f < cut[1].size() && (cut[1][f].kv_hi - cut[1][f].kv_lo) * key[1] > (p.kv_hi - p.kv_lo) * key[0])
      take(cut[1][f++]);
    take(p);
  }
  while (f < cut[1].size()) take(cut[1][f++]);
}

template <int D, bool QF16, bool F8>
static void cache_attention_launch(CacheAttnArgs a, hipStream_t st) {
  if constexpr (QF16)
    if (a.wide) hipLaunchKernelGGL((cache_wide_kernel<D, F8>), dim3(a.wide), dim3(512), 0, st, a);
  a.items += a.wide;
  if (a.nitems > a.wide)
    hipLaunchKernelGGL((cache_attention_kernel<D, QF16, F8>), dim3(a.nitems - a.wide), dim3(256), 0, st, a);
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
