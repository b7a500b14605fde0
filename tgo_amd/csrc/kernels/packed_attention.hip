// packed_attention.hip -- attention over packed sequences of different lengths
// whose K and V are plain f16 rows (no pool, no page table): whole prompts,
// chunks of new tokens, single tokens; causal or full; grouped heads.
#include "operators.h"

#include <algorithm>
#include <climits>

namespace tgohip {

constexpr int kPackTile = 64;   // keys staged in LDS per iteration
constexpr int kPackRows = 128;  // rows per workgroup
// Online softmax with a lazy reference m (log2 units): it starts at kPackNoMax, a
// row's probabilities are 2^(s - m), and m moves to the row's maximum - kPackLift
// once that passes m + kPackTop. They so stay below 2^kPackTop (f16 ends at 2^16),
// and the largest is at least 2^kPackLift: an f16 probability keeps an absolute
// error of 2^(-25 - kPackLift) of it, its normal range reaching 2^-21 of it.
constexpr float kPackNoMax = -1.0e30f;
constexpr float kPackLift = 7.f;
constexpr float kPackTop = 15.f;

// ---------------------------------------------------------------------------
// decomposition (host)
// ---------------------------------------------------------------------------

void packed_build_plan(int B, const int32_t* nq, const int32_t* nk, int H, int Hkv, int D, bool causal,
                       bool q_f16, int ncu, PackedPlan& plan) {
  plan = PackedPlan();
  plan.H = H;
  plan.Hkv = Hkv;
  plan.D = D;
  plan.q_f16 = q_f16;
  const int G = H / Hkv;
  std::vector<PackedItem> base;
  double total = 0;
  int64_t q0 = 0, k0 = 0;
  for (int s = 0; s < B; s++) {
    const int64_t rows = (int64_t)nq[s] * G;
    const int shift = causal ? nk[s] - nq[s] : INT_MAX / 2;
    for (int64_t r0 = 0; r0 < rows; r0 += kPackRows) {
      const int nr = (int)std::min<int64_t>(kPackRows, rows - r0);
      const int64_t last = (r0 + nr - 1) / G;
      const int hi = (int)std::max<int64_t>(0, std::min<int64_t>(nk[s], last + shift + 1));
      for (int h = 0; h < Hkv; h++) {
        base.push_back(PackedItem{(int32_t)q0, (int32_t)k0, nk[s], shift, (int32_t)r0, nr, 0, hi, h, -1});
        total += hi;
      }
    }
    q0 += nq[s];
    k0 += nk[s];
  }
  plan.tq = q0;
  plan.tk = k0;
  // Parts long enough that every workgroup slot gets about one.
  const double slots = 2.0 * ncu;
  const int part = std::max(512, (int)std::min(1.0e9, total / slots + kPackTile) / kPackTile * kPackTile);
  for (PackedItem it : base) {
    const int parts = (it.kv_hi + part - 1) / part;
    if (parts <= 1) {
      plan.items.push_back(it);
      continue;
    }
    const int tiles = (it.kv_hi + kPackTile - 1) / kPackTile;
    const int hi = it.kv_hi;
    for (int p = 0; p < parts; p++) {
      it.kv_lo = (int)((int64_t)tiles * p / parts) * kPackTile;
      it.kv_hi = std::min(hi, (int)((int64_t)tiles * (p + 1) / parts) * kPackTile);
      it.part = (int32_t)(plan.part_rows + (int64_t)p * it.nr);
      plan.items.push_back(it);
    }
    for (int i = 0; i < it.nr; i += 8)
      plan.merges.push_back(PackedMerge{it.q0, it.r0 + i, std::min(8, it.nr - i), it.kvh,
                                        (int32_t)plan.part_rows + i, parts, it.nr});
    plan.part_rows += (int64_t)parts * it.nr;
  }
  std::stable_sort(plan.items.begin(), plan.items.end(), [](const PackedItem& a, const PackedItem& b) {
    return a.kv_hi - a.kv_lo > b.kv_hi - b.kv_lo;
  });
}

// ---------------------------------------------------------------------------
// kernels
// ---------------------------------------------------------------------------

// 16-byte chunk c of tile row p: K rows are read whole by 32 lanes at one chunk,
// V by transposing reads of 4 rows x 64 bytes; both orders touch distinct banks.
template <int D>
__device__ __forceinline__ int pack_k_slot(int p, int c) {
  return p * (D / 8) + (c ^ (D == 128 ? (p & 15) : ((p >> 1) & 7)));
}
template <int D>
__device__ __forceinline__ int pack_v_slot(int p, int c) {
  return p * (D / 8) + (c ^ (D == 128 ? (p & 3) << 2 : ((p >> 1) & 1) << 2));
}

// Eight V^T operand values of one dim: tile rows p0 + [0,4) and p0 + 8 + [0,4).
// In each 16-lane group lane j names 8 bytes of row p0 + j/4 at dim d0 + 4(j%4)
// and receives dim d0 + j of the four rows.
template <int D>
__device__ __forceinline__ half8_t pack_v_frag(const half_t* Vs, int p0, int d0, int j) {
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t* lds4;
  const int c = (d0 >> 3) + ((j & 3) >> 1), r = p0 + (j >> 2);
  const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(Vs + pack_v_slot<D>(r, c) * 8 + 4 * (j & 1)));
  const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(Vs + pack_v_slot<D>(r + 8, c) * 8 + 4 * (j & 1)));
  return __builtin_bit_cast(half8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ bool half8_nonfinite(half8_t v) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 w = __builtin_bit_cast(u4, v);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++)
    bad |= (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
  return bad;
}

template <bool QF16>
__device__ __forceinline__ void pack_load_q(const void* q, int64_t off, bool valid, half8_t& hi, half8_t& lo) {
#pragma unroll
  for (int j = 0; j < 8; j++) hi[j] = lo[j] = (half_t)0.f;
  if (!valid) return;
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

// S^T = K . Q^T and O^T += V^T . P^T on v_mfma_f32_32x32x16_f16: lane (r, kh) =
// (lane % 32, lane / 32) holds row r's scores at keys 8(i/4) + 4kh + i%4 of each
// 32-key block, which are the B operand of the second product as they stand.
template <int D, bool QF16>
__global__ __launch_bounds__(256, 2) void packed_kernel(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) half_t Ks[kPackTile * D], Vs[kPackTile * D];
  constexpr int CH = D / 8, NL = kPackTile * CH / 256, KS = D / 16, DB = D / 32;
  const PackedItem it = a.items[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, kh = lane >> 5;
  const int r = wave * 32 + l32;
  const bool valid = r < it.nr;
  const int row = it.r0 + (valid ? r : 0), tok = row / a.G, head = it.kvh * a.G + row % a.G;
  const int lim = min(tok + it.shift, it.nk - 1);
  // first and last key limit of the wave's rows
  const int w0 = wave * 32, w1 = min(w0 + 32, it.nr) - 1;
  const int wlo = min((it.r0 + w0) / a.G + it.shift, it.nk - 1);
  const int whi = w0 < it.nr ? min((it.r0 + w1) / a.G + it.shift, it.nk - 1) : -1;

  half8_t qh[KS], ql[KS];
#pragma unroll
  for (int s = 0; s < KS; s++)
    pack_load_q<QF16>(a.q, (it.q0 + tok) * a.q_row + head * D + 16 * s + 8 * kh, valid, qh[s], ql[s]);

  float m = kPackNoMax, l = 0.f;
  float16_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; db++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[db][i] = 0.f;
  const float qs = a.qscale;
  const int j16 = lane & 15, dgrp = 16 * ((lane >> 4) & 1);

  for (int t0 = it.kv_lo; t0 < it.kv_hi; t0 += kPackTile) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NL; i++) {
      const int s = i * 256 + tid, p = s / CH, c = s % CH;
      const int64_t kr = it.k0 + min(t0 + p, it.kv_hi - 1);
      *(half8_t*)(Ks + pack_k_slot<D>(p, c) * 8) = *(const half8_t*)(a.k + kr * a.k_row + it.kvh * D + c * 8);
      *(half8_t*)(Vs + pack_v_slot<D>(p, c) * 8) = *(const half8_t*)(a.v + kr * a.v_row + it.kvh * D + c * 8);
    }
    __syncthreads();
    if (t0 > whi) continue;  // no row of this wave sees the tile
    const bool masked = t0 + kPackTile - 1 > wlo || t0 + kPackTile > it.kv_hi;
    float16_t sc[2] = {};
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int pb = 0; pb < 2; pb++) {
        const half8_t ka = *(const half8_t*)(Ks + pack_k_slot<D>(pb * 32 + l32, 2 * s + kh) * 8);
        sc[pb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qh[s], sc[pb], 0, 0, 0);
        if (!QF16) sc[pb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, ql[s], sc[pb], 0, 0, 0);
      }
    auto visible = [&](int pb, int i) {
      const int p = t0 + pb * 32 + 8 * (i >> 2) + 4 * kh + (i & 3);
      return p <= lim && p < it.kv_hi;
    };
    if (masked) {
#pragma unroll
      for (int pb = 0; pb < 2; pb++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (!visible(pb, i)) sc[pb][i] = -INFINITY;
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int pb = 0; pb < 2; pb++)
#pragma unroll
      for (int i = 0; i < 16; i++) tmax = fmaxf(tmax, sc[pb][i]);
    tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64)) * qs;
    const bool grow = tmax > m + kPackTop;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float mnew = grow ? tmax - kPackLift : m;
      const float alpha = __builtin_amdgcn_exp2f(m - mnew);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; db++) o[db] *= alpha;
      m = mnew;
    }
    half8_t pf[2][2], pl[2][2];
#pragma unroll
    for (int pb = 0; pb < 2; pb++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float p = __builtin_amdgcn_exp2f(fmaf(sc[pb][i], qs, -m));
        l += p;
        pf[pb][i >> 3][i & 7] = (half_t)p;
        pl[pb][i >> 3][i & 7] = (half_t)(p - (float)(half_t)p);
      }
    bool bad = false;
    if (masked) {
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int db = 0; db < DB; db++)
          bad |= half8_nonfinite(pack_v_frag<D>(Vs, 16 * u + 4 * kh, db * 32 + dgrp, j16));
    }
    if (__builtin_amdgcn_ballot_w64(bad)) {
      // A masked key's probability is 0, but 0 times an infinite or NaN value is
      // not: the finite values go through the product, and what a row sees of
      // NaN, +inf and -inf is counted with products of its visibility.
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int db = 0; db < DB; db++) {
          half8_t va = pack_v_frag<D>(Vs, 16 * u + 4 * kh, db * 32 + dgrp, j16);
#pragma unroll
          for (int e = 0; e < 8; e++) va[e] = __builtin_isfinite((float)va[e]) ? va[e] : (half_t)0.f;
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pf[u >> 1][u & 1], o[db], 0, 0, 0);
          if (!QF16) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[u >> 1][u & 1], o[db], 0, 0, 0);
        }
#pragma unroll 1
      for (int kind = 0; kind < 3; kind++) {
        const float add = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
#pragma unroll
        for (int db = 0; db < DB; db++) {
          float16_t seen = {};
#pragma unroll
          for (int u = 0; u < 4; u++) {
            half8_t va = pack_v_frag<D>(Vs, 16 * u + 4 * kh, db * 32 + dgrp, j16), vis;
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float f = (float)va[e];
              va[e] = (half_t)((kind == 0 ? f != f : f == add) ? 1.f : 0.f);
              vis[e] = (half_t)(visible(u >> 1, (u & 1) * 8 + e) ? 1.f : 0.f);
            }
            seen = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, vis, seen, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 16; i++) o[db][i] += seen[i] > 0.f ? add : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int db = 0; db < DB; db++) {
          const half8_t va = pack_v_frag<D>(Vs, 16 * u + 4 * kh, db * 32 + dgrp, j16);
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pf[u >> 1][u & 1], o[db], 0, 0, 0);
          if (!QF16) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[u >> 1][u & 1], o[db], 0, 0, 0);
        }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (!valid) return;
  // Lane (r, kh) holds dims 32db + 8g + 4kh + [0,4) of row r, g = 0..3.
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int db = 0; db < DB; db++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      float4_t v = {o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
      const int d = db * 32 + 8 * g + 4 * kh;
      if (it.part >= 0) {
        *(float4_t*)(a.part_o + (int64_t)(it.part + r) * D + d) = v;
        continue;
      }
      const int64_t off = (it.q0 + tok) * a.out_row + head * D + d;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = inv == 0.f ? 0.f : v[e] * inv;
      if (a.out_form == OUT_F32) {
        *(float4_t*)((float*)a.out + off) = v;
        continue;
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
  if (it.part >= 0 && kh == 0) {
    a.part_ml[(int64_t)(it.part + r) * 2] = m;
    a.part_ml[(int64_t)(it.part + r) * 2 + 1] = l;
  }
}

// Merges the parts of up to eight rows: sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p,
// four dims per thread.
template <int D>
__global__ __launch_bounds__(256) void packed_merge_kernel(PackedArgs a) {
  const PackedMerge g = a.merges[blockIdx.x];
  const int i = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  if (i >= g.nr) return;
  float M = kPackNoMax;
  for (int p = 0; p < g.parts; p++) M = fmaxf(M, a.part_ml[((int64_t)g.part + i + (int64_t)p * g.step) * 2]);
  float4_t v = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int p = 0; p < g.parts; p++) {
    const int64_t pr = (int64_t)g.part + i + (int64_t)p * g.step;
    const float lp = a.part_ml[pr * 2 + 1];
    if (lp == 0.f) continue;  // the part shows this row no key
    const float w = __builtin_amdgcn_exp2f(a.part_ml[pr * 2] - M);
    l += w * lp;
    const float4_t po = *(const float4_t*)(a.part_o + pr * D + d);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += w * po[e];
  }
  const int row = g.r0 + i, tok = row / a.G, head = g.kvh * a.G + row % a.G;
  const int64_t off = (g.q0 + tok) * a.out_row + head * D + d;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = l == 0.f ? 0.f : v[e] / l;
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

template <int D>
static void packed_launch(const PackedArgs& a, int q_f16, int items, int merges, hipStream_t st) {
  if (items) {
    if (q_f16) hipLaunchKernelGGL((packed_kernel<D, true>), dim3(items), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((packed_kernel<D, false>), dim3(items), dim3(256), 0, st, a);
  }
  if (merges) hipLaunchKernelGGL((packed_merge_kernel<D>), dim3(merges), dim3(256), 0, st, a);
}

int packed_enqueue(const PackedArgs& a, int D, int q_f16, int items, int merges, hipStream_t st) {
  if (D == 128) packed_launch<128>(a, q_f16, items, merges, st);
  else packed_launch<64>(a, q_f16, items, merges, st);
  TGOHIP_HIP(hipGetLastError());
  return 0;
}

}  // namespace tgohip
