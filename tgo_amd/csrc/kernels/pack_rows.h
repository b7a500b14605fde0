// pack_rows.h -- what the attention kernels over tiles of 64 f16 keys in LDS share
// (packed_attention.hip, cache_attention.hip): how a tile lies there, and a wave's block of
// 32 rows: its queries, running sums and results.
#pragma once

#include "operators.h"
#include "waits.h"

namespace tgohip {

constexpr int kPackTile = 64;            // keys staged in LDS per iteration
constexpr float kPackNoMax = -1.0e30f;  // where a row's reference starts
constexpr float kPackLeast = -3.0e38f;  // below every reference: the 8-bit cache's scores reach 2^105

// A tile of kPackTile keys in LDS: rows of D f16, their 16-byte chunks XOR-swizzled.
// K's chunks by the row, so that 32 lanes reading one chunk of 32 rows touch
// distinct banks; V's 64-byte quarters by the row's last two bits (D = 64: halves
// by the next to last), for transposing reads of four rows x 64 bytes. Both
// swizzles repeat every 16 rows and leave the chunk's bits to an XOR, so a lane
// keeps one byte address for each and the rest are constants.
template <int D>
__device__ __forceinline__ int pack_k_swz(int p) {
  return D == 128 ? (p & 15) : ((p >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int pack_v_swz(int p) {
  return D == 128 ? (p & 3) << 2 : ((p >> 1) & 1) << 2;
}
// Byte address of the lane's K operand (row l32, dims 8kh + [0,8)); step s is at
// that XOR 32s, 32 rows on at that + 64 D.
template <int D>
__device__ __forceinline__ int pack_k_at(int l32, int kh) {
  return l32 * 2 * D + 16 * (kh ^ pack_k_swz<D>(l32));
}
// Byte address of the lane's V^T operand: in each 16-lane group lane j names 8
// bytes of row 4kh + j/4 at dim d0 + 4(j%4) and receives dim d0 + j of the four
// rows; dims 32db + .. at that XOR 64db, rows p0 on at that + 2 D p0.
template <int D>
__device__ __forceinline__ int pack_v_at(int lane) {
  const int j = lane & 15, p = 4 * (lane >> 5) + (j >> 2), c = 2 * ((lane >> 4) & 1) + ((j & 3) >> 1);
  return p * 2 * D + 16 * (c ^ pack_v_swz<D>(p)) + 8 * (j & 1);
}
typedef __attribute__((address_space(3))) char* lds_t;
__device__ __forceinline__ half8_t pack_k_frag(lds_t K, int at) {
  return *(__attribute__((address_space(3))) half8_t*)(K + at);
}
// Eight values of one dim: tile rows p0 + 4kh + [0,4) and those + 8.
template <int D>
__device__ __forceinline__ half8_t pack_v_frag(lds_t V, int at) {
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t* lds4;
  const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(V + at));
  const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(V + at + 16 * D));
  return __builtin_bit_cast(half8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <bool QF16>
__device__ __forceinline__ void pack_load_q(const void* q, int64_t off, half8_t& hi, half8_t& lo) {
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

// Four neighbouring values of a result, `off` elements from its start. A: PackedArgs, CacheAttnArgs.
template <typename A>
__device__ __forceinline__ void pack_store4(const A& a, int64_t off, float4_t v) {
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

// One 32-row block of a wave: where its rows are, what they have seen. Lane (r, kh)
// = (lane % 32, lane / 32) holds row r: its query's dims 16s + 8kh + [0,8), its
// reference and (its half of the keys') sum, and of O^T dims 32db + 8g + 4kh + [0,4),
// db below NB.
template <int D, bool QF16, int NB = D / 32>
struct PackRows {
  int r, lim;  // row of the item and its last visible key
  half8_t qh[D / 16], ql[QF16 ? 1 : D / 16];
  float m, e, l;
  float16_t o[NB];

  // Rows past the item's repeat its first one; nothing of them is stored.
  __device__ __forceinline__ void init(const PackedArgs& a, const PackedItem& it, int r0, int lane) {
    r = r0 + (lane & 31);
    const int row = it.r0 + (r < it.nr ? r : 0), tok = row / a.G, head = it.kvh * a.G + row % a.G;
    lim = min(tok + it.shift, it.nk - 1);
#pragma unroll
    for (int s = 0; s < D / 16; s++)
      pack_load_q<QF16>(a.q, (it.q0 + tok) * a.q_row + head * D + 16 * s + 8 * (lane >> 5), qh[s], ql[QF16 ? 0 : s]);
    clear();
  }
  __device__ __forceinline__ void clear() {
    m = kPackNoMax;
    e = 0.f;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < NB; db++) o[db] = float16_t{};
  }
  // 1 over a row's sum, and what a sum of 0 gives: 0 where the row sees no key, NaN where
  // its scores are all -inf. A part keeps its sum, and says the latter in m's place.
  __device__ __forceinline__ float2 finish(const PackedArgs& a, const PackedItem& it, int lane) {
    l += __shfl_xor(l, 32, 64);
    const bool part = it.part >= 0, blank = l == 0.f && lim >= it.kv_lo;
    if (part && lane < 32 && r < it.nr)
      *(float4_t*)(a.part_ml + ((int64_t)it.part + r) * 4) = float4_t{blank ? NAN : m, e, l, 0.f};
    return float2{part ? 1.f : 1.f / l, blank && !part ? NAN : 0.f};
  }
  // The rows' results, through 128 D bytes of LDS that are the wave's own: a lane
  // holds four dims of its row at a time, and stores leave in whole rows. Stored as
  // they lay, 16 bytes of each row per instruction, an item cost 18 us beside 2 us
  // a tile (8192 items of 128 rows, f16).
  __device__ __forceinline__ void write(const PackedArgs& a, const PackedItem& it, int lane, lds_t buf) {
    typedef __attribute__((address_space(3))) float4_t* f4;
    const float2 fin = finish(a, it, lane);
    const int l32 = lane & 31, kh = lane >> 5;
    const bool part = it.part >= 0;
#pragma unroll
    for (int db = 0; db < D / 32; db++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float4_t v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = l == 0.f ? fin.y : o[db][4 * g + e] * fin.x;
        const int c = db * 8 + 2 * g + kh;  // chunk of four dims
        *(f4)(buf + l32 * 4 * D + 16 * (c ^ (l32 & 7))) = v;
      }
    pack_wave_sync();
    const int r0 = r - l32;
    if (part || a.out_form == OUT_F32) {
      constexpr int PL = D / 4;  // lanes per row
#pragma unroll 4
      for (int i = 0; i < 32 * PL / 64; i++) {
        const int x = i * (64 / PL) + lane / PL, c = lane % PL;
        const float4_t v = *(f4)(buf + x * 4 * D + 16 * (c ^ (x & 7)));
        if (r0 + x >= it.nr) continue;
        const int row = it.r0 + r0 + x;
        float* dst = part ? a.part_o + ((int64_t)it.part + r0 + x) * D
                          : (float*)a.out + (it.q0 + row / a.G) * a.out_row + (it.kvh * a.G + row % a.G) * D;
        *(float4_t*)(dst + 4 * c) = v;
      }
    } else {
      constexpr int PL = D / 8;
#pragma unroll 4
      for (int i = 0; i < 32 * PL / 64; i++) {
        const int x = i * (64 / PL) + lane / PL, c = lane % PL;
        const float4_t u = *(f4)(buf + x * 4 * D + 16 * ((2 * c) ^ (x & 7)));
        const float4_t v = *(f4)(buf + x * 4 * D + 16 * ((2 * c + 1) ^ (x & 7)));
        if (r0 + x >= it.nr) continue;
        const int row = it.r0 + r0 + x;
        half_t* dst = (half_t*)a.out + (it.q0 + row / a.G) * a.out_row + (it.kvh * a.G + row % a.G) * D + 8 * c;
        half8_t hv, lv;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float f = e < 4 ? u[e & 3] : v[e & 3];
          hv[e] = (half_t)f;
          lv[e] = (half_t)(f - (float)hv[e]);
        }
        *(half8_t*)dst = hv;
        if (a.out_form == OUT_X2) *(half8_t*)(dst + a.out_lo) = lv;
      }
    }
    pack_wave_sync();
  }
};

// S^T = K . Q^T on v_mfma_f32_32x32x16_f16: lane (r, kh) gets row r's scores at keys
// 32pb + 8(i/4) + 4kh + i%4 of the tile.
template <int D, bool QF16, int NB>
__device__ __forceinline__ void pack_scores(const PackRows<D, QF16, NB>& w, lds_t K, int at, float16_t (&sc)[2]) {
  sc[0] = sc[1] = float16_t{};
#pragma unroll
  for (int s = 0; s < D / 16; s++)
#pragma unroll
    for (int pb = 0; pb < 2; pb++) {
      const half8_t ka = pack_k_frag(K, (at ^ (32 * s)) + 64 * D * pb);
      sc[pb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, w.qh[s], sc[pb], 0, 0, 0);
      if (!QF16) sc[pb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, w.ql[QF16 ? 0 : s], sc[pb], 0, 0, 0);
      if (!QF16 && pb && s % 2) __builtin_amdgcn_sched_barrier(0);
    }
}

}  // namespace tgohip
