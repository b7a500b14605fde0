// packed_attention.hip -- attention over packed sequences of different lengths
// whose K and V are plain f16 rows (no pool, no page table): whole prompts,
// chunks of new tokens, single tokens; causal or full; grouped heads.
//
// o = sum_k 2^(s_k - m) v_k / sum_k 2^(s_k - m), s = scale log2(e) q . k, in one pass
// over the keys: m and the sums move along with the tiles (online softmax), and m only
// when a probability would leave its range. Both products run transposed (S^T = K Q^T,
// O^T = V^T P^T) on v_mfma_f32_32x32x16_f16, so that a lane holds scores of one row and
// its own probabilities are the second product's operand: P never leaves registers.
// f32 queries go as f16 hi + lo pairs, and so do their probabilities, two MFMAs per
// product; f16 queries take f16 probabilities (2^-11 of each, as their outputs). Scores,
// sums, maxima and partial results are f32.
//   packed_kernel        128 rows of a sequence and kv head (token by token, the
//                        group's heads side by side), tiles of 64 keys: MFMA-bound
//   packed_few_kernel    up to 32 such rows (decoding): bound by the keys' bytes
//   packed_merge_kernel  rows whose keys were cut into pieces
// Measured (us a call, averages back to back, 32 heads over 8 of 128 dims unless said):
//   one causal prompt of 16384 f16 rows           2190 (2120 to 2230 by the card), 1.00
//       PFLOP/s, the matrix unit busy 53% at 1.90 GHz (all four SIMDs' power holds the
//       clock), VALU 40%
//   16 f16 prompts of 1 to 1384 rows              54, 0.63 PFLOP/s
//   4 f32 chunks of 82 to 354 rows, 2116 to 8176 keys   125, 0.41 PFLOP/s, twice that executed
//   32 full f32 sequences of 22 to 763 rows, 16 heads of 64   52, 0.30 PFLOP/s
//   64 decoders of 16 to 8192 keys                73, 5.3 TB/s
//   64 decoders of 4096 keys                      165, 6.5 TB/s
// Tried and slower or no faster in packed_kernel, for that prompt (2240 us then): the
// next tile's scores beside this one's softmax 2252; eight waves on four LDS buffers
// 2666; the waves' priorities by phase 2240. 64 rows a wave spilled, with packed_redo's
// registers in the kernel, more than now: not tried since.
#include "operators.h"

#include <algorithm>
#include <climits>
#include <functional>
#include <type_traits>

namespace tgohip {

constexpr int kPackTile = 64;   // keys staged in LDS per iteration
constexpr int kPackFew = 32;    // rows of a sequence and kv head up to which packed_few_kernel takes them
constexpr int kFewTile = 32;    // keys of a wave's tile there
constexpr int kFewWaves = 2;
constexpr int kPackWaves = 4;
static_assert(kPackRows == 32 * kPackWaves, "packed_kernel takes an item's rows");
// Online softmax with a lazy reference m + e (log2 units): it starts at kPackNoMax, a
// row's probabilities are 2^(s - m - e), and it moves to the row's maximum - kPackLift
// once that passes it by more than kPackTop. They so stay below 2^kPackTop (f16 ends at
// 2^16), and the largest is at least about 2^kPackLift: an f16 probability keeps an
// absolute error of 2^(-25 - kPackLift) of it, its normal range reaching 2^-21 of it.
// The multiply-add that scales a score subtracts m in the same rounding, so the one thing
// lost in m is its distance from the maximum: half a step of f32, up to 1/4 while |m| is
// at most kPackFar, and there e is 0. Past that (a step is 16 at 2^28, and probabilities
// would pass f16 or all be 0) m is the rounded maximum and e what it lacks, kPackLift
// less; the lift itself is lost in e from 2^48 on, where two scores are equal or a step
// of 2^25 apart. The kernels' loops keep no e, nor its check in every tile: where a row's
// reference goes past kPackFar, its workgroup takes its keys again with one, as it does
// for values that are not finite.
constexpr float kPackNoMax = -1.0e30f;
constexpr float kPackFar = 4194304.f;  // 2^22
constexpr float kPackLift = 7.f;
constexpr float kPackTop = 15.f;
constexpr float kPackSum = 32768.f;  // 2^kPackTop

// ---------------------------------------------------------------------------
// decomposition (host)
// ---------------------------------------------------------------------------

// How items are cut along their keys: the pieces of each, and their tiles, item by item.
struct PackCut {
  std::vector<int> pieces, tiles;
};

// The order of lengths, longest first and equal ones as they stand: 11 bits at a time
// (a plan is made for every batch: of 512 decoders, 4096 items, it takes 0.4 ms, and
// took 0.2 more with a comparing sort).
static std::vector<int> pack_order(const std::vector<int>& lengths) {
  std::vector<int> order(lengths.size()), from(lengths.size());
  for (size_t i = 0; i < order.size(); i++) order[i] = (int)i;
  const int longest = lengths.empty() ? 0 : *std::max_element(lengths.begin(), lengths.end());
  for (int shift = 0; shift < 31 && longest >> shift; shift += 11) {
    size_t at[2049] = {};
    const auto digit = [&](int i) { return 2047 - ((lengths[i] >> shift) & 2047); };
    for (int i : order) at[digit(i) + 1]++;
    for (int d = 0; d < 2048; d++) at[d + 1] += at[d];
    from.swap(order);
    for (int i : from) order[at[digit(i)]++] = i;
  }
  return order;
}

// What a kernel's tiles of 64 keys cost: us of one whose workgroup has its CU alone, and
// the part of that rate each of two workgroups on a CU reaches.
struct PackRate {
  double tile, shared;
};
constexpr int kPackFixed = 3;  // tiles that a piece costs beside its own: its start and its result

// us until the last piece has ended and the rows of cut items are merged. Pieces are
// dispatched longest first, two workgroups to a CU; merging costs a launch and, for each
// row of a partial result, its way to memory and back. Within 15% of what the kernels
// measure for 18 batches in each of these cuts, but for batches of short pieces.
static double pack_time(const std::vector<PackedItem>& whole, const PackCut& c, int ncu, const PackRate& rate) {
  std::vector<int> tiles;
  tiles.reserve(c.tiles.size());
  for (int i : pack_order(c.tiles)) tiles.push_back(c.tiles[i]);
  struct Cu {
    double now = 0, a = 0, b = 0;  // its clock, and what is left of its two pieces, a <= b
  };
  std::vector<Cu> cus(std::min<size_t>(tiles.size(), ncu));
  size_t next = 0;
  for (; next < tiles.size() && next < 2 * cus.size(); next++) {
    Cu& u = cus[next % cus.size()];
    (next < cus.size() ? u.b : u.a) = tiles[next] + kPackFixed;
  }
  // the next end on a CU: of the shorter piece while there are two
  const auto end = [&](const Cu& u) { return u.now + (u.a > 0 ? u.a / rate.shared : u.b); };
  typedef std::pair<double, int> Event;
  std::vector<Event> ends;  // a heap, the soonest first
  for (size_t i = 0; i < cus.size(); i++) ends.push_back({end(cus[i]), (int)i});
  std::make_heap(ends.begin(), ends.end(), std::greater<Event>());
  double last = 0;
  while (!ends.empty()) {
    const int cu = ends[0].second;
    Cu& u = cus[cu];
    last = u.now = ends[0].first;
    u.b = u.a > 0 ? u.b - u.a : 0;
    u.a = 0;
    if (next < tiles.size()) {
      u.a = tiles[next++] + kPackFixed;
      if (u.a > u.b) std::swap(u.a, u.b);
    }
    // the CU's next end in the place of this one, or the heap's last
    Event e = {end(u), cu};
    if (u.b <= 0) {
      e = ends.back();
      ends.pop_back();
    }
    for (size_t i = 0, k; i < ends.size(); i = k) {
      k = 2 * i + 1;
      if (k + 1 < ends.size() && ends[k + 1].first < ends[k].first) k++;
      if (k >= ends.size() || ends[k].first >= e.first) {
        ends[i] = e;
        break;
      }
      ends[i] = ends[k];
    }
  }
  int64_t rows = 0;
  for (size_t i = 0; i < whole.size(); i++)
    if (c.pieces[i] > 1) rows += (int64_t)c.pieces[i] * whole[i].nr;
  return last * rate.tile + (rows ? 4.5 + 0.35e-3 * (double)rows : 0.0);
}

// Pieces that fill the shares of `slots` workgroups one after the other, ending where a
// share does, at least `least` tiles long.
static PackCut pack_shares(const std::vector<int>& tiles, int slots, int least) {
  PackCut c;
  int64_t total = 0;
  for (int t : tiles) total += t + kPackFixed;
  const int64_t share = std::max<int64_t>((total + slots - 1) / slots, least + kPackFixed);
  // the pieces' own fixed costs, about one more per slot
  const int64_t room = share + (share > least + kPackFixed ? kPackFixed : 0);
  int64_t left = room;
  for (int t : tiles) {
    int n = 0, at = 0;
    do {
      if (left < least + kPackFixed) left = room;
      int take = (int)std::min<int64_t>(t - at, left - kPackFixed);
      const int rest = t - at - take;
      if (rest > 0 && rest < least) take = t - at >= 2 * least ? t - at - least : t - at;
      at += take;
      left -= take + kPackFixed;
      c.tiles.push_back(take);
      n++;
    } while (at < t);
    c.pieces.push_back(n);
  }
  return c;
}

// No more pieces than slots, an item's of one size, the longest as short as that allows.
static PackCut pack_even(const std::vector<int>& tiles, int slots, int longest, int least) {
  const auto pieces = [](int t, int most) { return t ? (t + most - 1) / most : 1; };
  int lo = least, hi = std::max(longest, least);
  while (lo < hi) {
    const int most = (lo + hi) / 2;
    int64_t n = 0;
    for (int t : tiles) n += pieces(t, most);
    if (n <= slots) hi = most;
    else lo = most + 1;
  }
  PackCut c;
  for (int t : tiles) {
    const int n = pieces(t, lo);
    c.pieces.push_back(n);
    for (int i = 0; i < n; i++) c.tiles.push_back((int)((int64_t)t * (i + 1) / n - (int64_t)t * i / n));
  }
  return c;
}

// Orders items longest first and cuts them along their keys in the way that ends
// soonest: not at all, in even pieces (one or two workgroups a CU) or in shares (two).
// Measured, us for these four: 64 decoders of 16 to 8192 keys 187, -, -, 74; 66 of 4096
// keys 249, -, -, 175; 4 chunks of 82 to 354 f32 queries over 2116 to 8176 keys 237, 226,
// 130, 136; 2 of 23 and 114 over 2300 and 2700 87, 39, 41, 43; one prompt of 2048 f16
// queries 61, -, -, 68; 3 prompts of 600 to 900 f32 queries 52, -, -, 59.
static void pack_cut(const std::vector<PackedItem>& whole, int tile, int least, int ncu, const PackRate& rate,
                     std::vector<PackedItem>& out, PackedPlan& plan) {
  PackCut cut;
  cut.pieces.assign(whole.size(), 1);
  cut.tiles.reserve(whole.size());
  int64_t total = 0;
  int longest = 0;
  for (const PackedItem& it : whole) {
    const int t = (it.kv_hi + tile - 1) / tile;
    cut.tiles.push_back(t);
    total += t + kPackFixed;
    longest = std::max(longest, t);
  }
  // Nothing to gain where whole items, longest first, end within a tenth of even shares,
  // or the longest is a quarter of a workgroup's share. A cut has to win by 5%: the
  // estimates are no closer.
  const double even = (double)total / ncu * rate.tile / (2 * rate.shared);
  if (longest > least && 8.0 * longest * ncu > (double)total) {
    double best = pack_time(whole, cut, ncu, rate);
    if (best > 1.1 * even) {
      const std::vector<int> tiles = cut.tiles;
      const auto take = [&](PackCut other) {
        const double time = pack_time(whole, other, ncu, rate);
        if (time >= 0.95 * best) return;
        best = time;
        cut = std::move(other);
      };
      if ((int64_t)whole.size() < ncu) take(pack_even(tiles, ncu, longest, least));
      if ((int64_t)whole.size() < 2 * ncu) take(pack_even(tiles, 2 * ncu, longest, least));
      take(pack_shares(tiles, 2 * ncu, least));
    }
  }
  std::vector<PackedItem> cuts;
  size_t at = 0;
  for (size_t i = 0; i < whole.size() && cut.tiles.size() > whole.size(); i++) {
    PackedItem it = whole[i];
    const int parts = cut.pieces[i], hi = it.kv_hi;
    if (parts == 1) {
      at++;
      cuts.push_back(it);
      continue;
    }
    int end = 0;
    for (int p = 0; p < parts; p++) {
      it.kv_lo = end * tile;
      end += cut.tiles[at++];
      it.kv_hi = std::min(hi, end * tile);
      it.part = (int32_t)(plan.part_rows + (int64_t)p * it.nr);
      cuts.push_back(it);
    }
    // rows of a merge: few where there are many parts, whose rows then share its threads (4
    // chunks of up to 5 parts: 130 us with 8 rows, 134 with 2)
    const int rows = parts > 64 ? 1 : parts > 16 ? 2 : 8;
    for (int r = 0; r < it.nr; r += rows)
      plan.merges.push_back(PackedMerge{it.q0, it.r0 + r, std::min(rows, it.nr - r), it.kvh,
                                        (int32_t)plan.part_rows + r, parts, it.nr});
    plan.part_rows += (int64_t)parts * it.nr;
  }
  const std::vector<PackedItem>& all = cuts.empty() ? whole : cuts;
  std::vector<int> keys;
  keys.reserve(all.size());
  for (const PackedItem& it : all) keys.push_back(it.kv_hi - it.kv_lo);
  out.reserve(all.size());
  for (int i : pack_order(keys)) out.push_back(all[i]);
}

void packed_build_plan(int B, const int32_t* nq, const int32_t* nk, int H, int Hkv, int D, bool causal,
                       bool q_f16, int ncu, PackedPlan& plan) {
  plan = PackedPlan();
  plan.H = H;
  plan.Hkv = Hkv;
  plan.D = D;
  plan.q_f16 = q_f16;
  const int G = H / Hkv;
  // Sequences of up to kPackFew rows per kv head go to the few-row kernel where they
  // hold most of the keys (64 decoders of 16 to 8192 keys 73 us, 84 without); beside longer
  // prompts they are not worth a launch of their own (16 prompts, eight of a few tokens:
  // 60 us, 65 with it).
  int64_t few_keys = 0, keys = 0;
  for (int s = 0; s < B; s++) {
    keys += nk[s];
    if ((int64_t)nq[s] * G <= kPackFew) few_keys += nk[s];
  }
  const int64_t few_rows = 2 * few_keys > keys ? kPackFew : 0;
  std::vector<PackedItem> whole[2];  // tiles of rows, few rows
  int64_t items = 0;
  for (int s = 0; s < B; s++) items += ((int64_t)nq[s] * G + kPackRows - 1) / kPackRows * Hkv;
  whole[few_rows ? 1 : 0].reserve((size_t)items);
  int64_t q0 = 0, k0 = 0;
  for (int s = 0; s < B; s++) {
    const int64_t rows = (int64_t)nq[s] * G;
    const int shift = causal ? nk[s] - nq[s] : INT_MAX / 2;
    for (int64_t r0 = 0; r0 < rows; r0 += kPackRows) {
      const int nr = (int)std::min<int64_t>(kPackRows, rows - r0);
      const int64_t last = (r0 + nr - 1) / G;
      const int hi = (int)std::max<int64_t>(0, std::min<int64_t>(nk[s], last + shift + 1));
      for (int h = 0; h < Hkv; h++)
        whole[rows <= few_rows].push_back(
            PackedItem{(int32_t)q0, (int32_t)k0, nk[s], shift, (int32_t)r0, nr, 0, hi, h, -1});
    }
    q0 += nq[s];
    k0 += nk[s];
  }
  plan.tq = q0;
  plan.tk = k0;
  const double dims = D / 128.0;
  const PackRate rate = q_f16 ? PackRate{1.31 * dims, 0.64} : PackRate{1.8 * dims, 0.53};
  pack_cut(whole[0], kPackTile, 4, ncu, rate, plan.items, plan);
  pack_cut(whole[1], kFewTile * kFewWaves, 2, ncu, PackRate{1.8 * dims, 0.7}, plan.few, plan);
}

// ---------------------------------------------------------------------------
// kernels
// ---------------------------------------------------------------------------

// s_waitcnt vmcnt(0) lgkmcnt(0), and no memory access moves across it: the wave's DMA has
// landed, and its LDS reads have returned, before other data goes where they read.
__device__ __forceinline__ void pack_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
}
// A barrier without a memory fence, which would wait for every DMA in flight; no
// memory access moves across it.
__device__ __forceinline__ void pack_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Orders a wave's own LDS writes before its other lanes' reads (and back).
__device__ __forceinline__ void pack_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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

// Four neighbouring values of a result, `off` elements from its start.
__device__ __forceinline__ void pack_store4(const PackedArgs& a, int64_t off, float4_t v) {
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
// Whether the lane's row sees the key of its score (pb, i); left: the row's last
// visible key, counted from the lane's first of the tile (4kh on).
__device__ __forceinline__ bool pack_visible(int left, int pb, int i) {
  return pb * 32 + 8 * (i >> 2) + (i & 3) <= left;
}
// A row's largest score of a tile, not scaled.
__device__ __forceinline__ float pack_top(const float16_t (&sc)[2]) {
  // one chain: the compiler makes it 16 three-way maxima (of pairs, it quiets every
  // score first, 32 instructions more)
  float t = -INFINITY;
#pragma unroll
  for (int pb = 0; pb < 2; pb++)
#pragma unroll
    for (int i = 0; i < 16; i++) t = fmaxf(t, sc[pb][i]);
  return fmaxf(t, __shfl_xor(t, 32, 64));
}
// Moves the reference of the rows that need it to their tile's largest score `top`. A
// row's own scores alone decide: its result does not depend on the rows beside it. Without
// an e (FAR false), past: a row's reference should have one.
template <bool FAR, int D, bool QF16, int NB>
__device__ __forceinline__ void pack_raise(PackRows<D, QF16, NB>& w, float top, float qs, bool need, bool& past) {
#pragma clang fp contract(off)  // the same bits in every kernel
  const float t = top * qs;
  const bool far = fabsf(t) > kPackFar;
  const float mnew = need ? (FAR && far ? t : fmaf(top, qs, -kPackLift)) : w.m;
  float alpha = w.m - mnew;
  if constexpr (FAR) {
    const float enew = need ? (far ? fmaf(top, qs, -t) - kPackLift : 0.f) : w.e;
    alpha += w.e - enew;
    w.e = enew;
  } else {
    past |= need && far;
  }
  alpha = __builtin_amdgcn_exp2f(alpha);
  w.l *= alpha;
#pragma unroll
  for (int db = 0; db < NB; db++) w.o[db] *= alpha;
  w.m = mnew;
}
// Scores 8u .. 8u + 7 of the lane to probabilities, their sum on l, as f16 (or a
// pair) where the second product's B operand wants them: its k index 8kh + e of
// step u is key 16u + (e < 4 ? 4kh + e : 8 + 4kh + e - 4), the lane's own score e.
// f16 probabilities are summed as rounded, two to an instruction, in f32.
template <bool QF16, bool FAR>
__device__ __forceinline__ void pack_probs(const float16_t (&sc)[2], int u, float qs, float m, float& l, half8_t& ph,
                                           half8_t& pl, float below) {
  typedef float float2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float2_t p;
#pragma unroll
    for (int g = 0; g < 2; g++) {
      const float x = fmaf(sc[u >> 1][8 * (u & 1) + e + g], qs, -m);
      p[g] = __builtin_amdgcn_exp2f(FAR ? x - below : x);
    }
    const half2_t h = __builtin_convertvector(p, half2_t);
    ph[e] = h[0];
    ph[e + 1] = h[1];
    if (QF16) {
      l = __builtin_amdgcn_fdot2(h, half2_t{(half_t)1.f, (half_t)1.f}, l, false);
    } else {
      l += p[0] + p[1];
      const float2_t r = {fmaf((float)h[0], -1.f, p[0]), fmaf((float)h[1], -1.f, p[1])};
      const half2_t g = __builtin_convertvector(r, half2_t);
      pl[e] = g[0];
      pl[e + 1] = g[1];
    }
  }
}
// A tile of f16 probabilities. They are taken with the reference maximum as it is
// and their sum tells whether one may have passed f16 (the row's first tile, or a
// key far above the ones before): only then is the tile's maximum looked for, and
// the probabilities taken again. That saves the search, 25 of 165 VALU
// instructions a tile.
template <bool FAR, int D, int NB>
__device__ __forceinline__ void pack_probs_f16(PackRows<D, true, NB>& w, const float16_t (&sc)[2], float qs,
                                               half8_t (&ph)[4], bool& past) {
  float l[4] = {};
  half8_t none;
#pragma unroll
  for (int u = 0; u < 4; u++) pack_probs<true, FAR>(sc, u, qs, w.m, l[u], ph[u], none, w.e);
  const bool over = (l[0] + l[1]) + (l[2] + l[3]) > kPackSum;
  if (__builtin_amdgcn_ballot_w64(over)) {  // uniform across the wave
    const bool other = __shfl_xor((int)over, 32, 64);  // the row's other half of the keys
    pack_raise<FAR>(w, pack_top(sc), qs, over | other, past);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      l[u] = 0.f;
      pack_probs<true, FAR>(sc, u, qs, w.m, l[u], ph[u], none, w.e);
    }
  }
  w.l += (l[0] + l[1]) + (l[2] + l[3]);
}
// A tile's maximum, before its pairs of probabilities.
template <bool FAR, int D, bool QF16, int NB>
__device__ __forceinline__ void pack_maximum(PackRows<D, QF16, NB>& w, const float16_t (&sc)[2], float qs, bool& past) {
  const float top = pack_top(sc);
  bool grow = top * qs > w.m + kPackTop;  // as without an e where the row has none
  if (FAR && fabsf(w.m) > kPackFar + kPackLift) grow = fmaf(top, qs, -w.m) - w.e > kPackTop;
  if (__builtin_amdgcn_ballot_w64(grow)) pack_raise<FAR>(w, top, qs, grow, past);
}
// A tile's probabilities and O^T += V^T . P^T. f16 probabilities all come first: the
// other wave of the SIMD fills the matrix unit meanwhile. Pairs come step by step,
// or they would not fit the registers beside q's pairs.
template <int D, bool QF16>
__device__ __forceinline__ void pack_values(PackRows<D, QF16>& w, const float16_t (&sc)[2], float qs, lds_t V, int at,
                                            bool& past) {
  half8_t ph[4], pl, first[D / 32];
  if (QF16) {
    // the first products' operands come from LDS under the exponentials
#pragma unroll
    for (int db = 0; db < D / 32; db++) first[db] = pack_v_frag<D>(V, at ^ (64 * db));
  }
  if constexpr (QF16) pack_probs_f16<false>(w, sc, qs, ph, past);
  else pack_maximum<false>(w, sc, qs, past);
  float l[4] = {};  // a chain of adds per step
#pragma unroll
  for (int u = 0; u < 4; u++) {
    if (!QF16) pack_probs<QF16, false>(sc, u, qs, w.m, l[u], ph[u], pl, 0.f);
#pragma unroll
    for (int db = 0; db < D / 32; db++) {
      const half8_t va = QF16 && u == 0 ? first[db] : pack_v_frag<D>(V, (at ^ (64 * db)) + 32 * D * u);
      w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[u], w.o[db], 0, 0, 0);
      if (!QF16) w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl, w.o[db], 0, 0, 0);
    }
    if (!QF16) __builtin_amdgcn_sched_barrier(0);
  }
  if (!QF16) w.l += (l[0] + l[1]) + (l[2] + l[3]);
}

// Rows [w0, w0 + 32) of an item again, for a workgroup whose references need an e or that
// met an infinite or NaN value in a tile some of its rows see only part of: a masked key's
// probability is 0, but 0 times such a value is not. The products take those
// values as 0 (the same sums, to the bit, where none is seen); a product of
// visibility and occurrence then tells which outputs see +inf and which -inf, NaN
// being both. Rare: a plain loop behind the kernel's own, 32 dims of the result at a
// time where there are 128, so that the kernel keeps next to none of its registers in
// memory around it (with all dims 102 to 111, with 64 of them 30 and 83, 1% on the kernel's
// own time). Measured, us: 4 f32 chunks of 2116 to 8176 keys 125, an infinity in the last
// value 1570, scores of 2^28 927; 32 full f32 sequences, 16 heads of 64, 52, 156, 156.
template <int D, bool QF16>
__device__ __forceinline__ void packed_redo(const PackedArgs* ap, int item, int w0, lds_t K, lds_t V) {
  const PackedArgs& a = *ap;
  const PackedItem it = a.items[item];
  const int tid = threadIdx.x, lane = tid & 63, kh = lane >> 5;
  const int kat = pack_k_at<D>(lane & 31, kh);
  constexpr int NB = D == 64 ? 2 : 1;  // blocks of 32 dims at a time
  PackRows<D, QF16, NB> w;
#pragma unroll 1
  for (int d0 = 0; d0 < D; d0 += 32 * NB) {
    const int vat = pack_v_at<D>(lane) ^ (2 * d0);
    w.init(a, it, w0, lane);
    bool past = false, odd = false;
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
      if (pass == 1 && !__syncthreads_or(odd)) break;  // every value is finite
      float16_t seen[NB] = {};
#pragma unroll 1
      for (int t0 = it.kv_lo; t0 < it.kv_hi; t0 += kPackTile) {
        __syncthreads();
        for (int i = tid; i < kPackTile * (D / 8); i += blockDim.x) {
          const int p = i / (D / 8), c = i % (D / 8);
          const int64_t row = it.k0 + min(t0 + p, it.kv_hi - 1);
          if (pass == 0)
            *(__attribute__((address_space(3))) half8_t*)(K + p * 2 * D + 16 * (c ^ pack_k_swz<D>(p))) =
                *(const half8_t*)(a.k + row * a.k_row + it.kvh * D + c * 8);
          const half8_t vv = *(const half8_t*)(a.v + row * a.v_row + it.kvh * D + c * 8);
          *(__attribute__((address_space(3))) half8_t*)(V + p * 2 * D + 16 * (c ^ pack_v_swz<D>(p))) = vv;
          odd |= half8_nonfinite(vv);
        }
        __syncthreads();
        float16_t sc[2];
        half8_t ps[4];
        const int left = min(w.lim, it.kv_hi - 1) - t0 - 4 * kh;
        if (pass == 0) {
          pack_scores(w, K, kat, sc);
          bool any = false;
#pragma unroll
          for (int pb = 0; pb < 2; pb++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const bool vis = pack_visible(left, pb, i);
              any |= vis;
              if (!vis) sc[pb][i] = -INFINITY;
            }
          if (!__builtin_amdgcn_ballot_w64(any)) continue;  // as the kernel skips it
          if constexpr (QF16) pack_probs_f16<true>(w, sc, a.qscale, ps, past);
          else pack_maximum<true>(w, sc, a.qscale, past);
        }
        float l[4] = {};
#pragma unroll
        for (int u = 0; u < 4; u++) {
          half8_t ph = ps[u], pl;
          if (pass == 0) {
            if (!QF16) pack_probs<QF16, true>(sc, u, a.qscale, w.m, l[u], ph, pl, w.e);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
              ph[e] = (half_t)(pack_visible(left, u >> 1, (u & 1) * 8 + e) ? 1.f : 0.f);
          }
#pragma unroll
          for (int db = 0; db < NB; db++) {
            half8_t va = pack_v_frag<D>(V, (vat ^ (64 * db)) + 32 * D * u);
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float f = (float)va[e];
              if (pass == 0) va[e] = fabsf(f) < INFINITY ? va[e] : (half_t)0.f;
              else va[e] = (half_t)(f != f || f == (pass == 1 ? INFINITY : -INFINITY) ? 1.f : 0.f);
            }
            if (pass == 0) {
              w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph, w.o[db], 0, 0, 0);
              if (!QF16) w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl, w.o[db], 0, 0, 0);
            } else {
              seen[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph, seen[db], 0, 0, 0);
            }
          }
        }
        w.l += (l[0] + l[1]) + (l[2] + l[3]);
      }
#pragma unroll
      for (int db = 0; db < NB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (seen[db][i] > 0.f) w.o[db][i] += pass == 1 ? INFINITY : -INFINITY;
    }
    const float2 fin = w.finish(a, it, lane);
    const int row = it.r0 + w.r;
#pragma unroll
    for (int db = 0; db < NB; db++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float4_t v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = w.l == 0.f ? fin.y : w.o[db][4 * g + e] * fin.x;
        const int d = d0 + 32 * db + 8 * g + 4 * kh;
        if (w.r < it.nr) {
          if (it.part >= 0) *(float4_t*)(a.part_o + ((int64_t)it.part + w.r) * D + d) = v;
          else pack_store4(a, (it.q0 + row / a.G) * a.out_row + (it.kvh * a.G + row % a.G) * D + d, v);
        }
      }
  }
}

// The workgroup's share of a tile by DMA (global_load_lds_dwordx4): lane i of wave v's
// instruction n writes the 16-byte slot 64 (WAVES n + v) + i of the tile, and reads
// the chunk that the swizzle keeps there. `off`: the lane's byte offset from the
// tile's first row, the same for every n but for whole rows.
template <int D, int WAVES>
__device__ __forceinline__ void pack_dma(const char* base, uint32_t off, int64_t row_bytes, lds_t tile, int wave) {
  constexpr int RPI = 64 * WAVES / (D / 8);  // rows per instruction of the workgroup
#pragma unroll
  for (int n = 0; n < kPackTile / RPI; n++)
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(base + n * RPI * row_bytes + off),
        (__attribute__((address_space(3))) void*)(tile + 1024 * (WAVES * n + wave)), 16, 0, 0);
}
// The same where the tile ends behind the item's keys: rows from `rows` on repeat the
// last one (no row sees them; a value there that is not finite is packed_redo's).
template <int D, int WAVES>
__device__ __forceinline__ void pack_dma_end(const char* base, int p, int c, int rows, int64_t row_bytes, lds_t tile,
                                             int wave) {
  constexpr int RPI = 64 * WAVES / (D / 8);
#pragma unroll
  for (int n = 0; n < kPackTile / RPI; n++)
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(base + min(n * RPI + p, rows - 1) * row_bytes + 16 * c),
        (__attribute__((address_space(3))) void*)(tile + 1024 * (WAVES * n + wave)), 16, 0, 0);
}

// WAVES waves of 32 rows each; tiles of 64 keys go through two LDS buffers, the next
// one's DMA in flight while one is used. Two workgroups a CU (128 dims: 64 KiB of LDS and
// 251 or 256 registers each; 64 dims: 33 KiB, and 221 or 244 registers, of which the loop
// alone would leave room for a third workgroup and packed_redo does not), so that one's products run under the other's softmax: without the
// softmax the 16384-row prompt took 12% less, without the DMA 14%.
template <int D, bool QF16, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void packed_kernel(PackedArgs a) {
  constexpr int TB = kPackTile * D * 2;  // bytes of a tile
  __shared__ __attribute__((aligned(1024))) char K0[TB], V0[TB], K1[TB], V1[TB];
  const PackedItem it = a.items[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kh = lane >> 5, w0 = 32 * wave;
  // first and last key limit of the wave's rows
  const int wlo = min((it.r0 + w0) / a.G + it.shift, it.nk - 1);
  const int whi = w0 < it.nr ? min((it.r0 + min(w0 + 32, it.nr) - 1) / a.G + it.shift, it.nk - 1) : -1;
  const int kat = pack_k_at<D>(lane & 31, kh), vat = pack_v_at<D>(lane);

  const int p = (64 * wave + lane) / (D / 8), c = lane % (D / 8);
  const int kc = c ^ pack_k_swz<D>(p), vc = c ^ pack_v_swz<D>(p);
  const int64_t kb = a.k_row * 2, vb = a.v_row * 2;
  const uint32_t koff = (uint32_t)(p * kb + 16 * kc), voff = (uint32_t)(p * vb + 16 * vc);
  const char* kp = (const char*)(a.k + it.k0 * a.k_row + it.kvh * D);
  const char* vp = (const char*)(a.v + it.k0 * a.v_row + it.kvh * D);
  auto dma = [&](int t0, lds_t K, lds_t V) {
    if (t0 + kPackTile <= it.kv_hi) {
      pack_dma<D, WAVES>(kp + t0 * kb, koff, kb, K, wave);
      pack_dma<D, WAVES>(vp + t0 * vb, voff, vb, V, wave);
    } else if (t0 < it.kv_hi) {
      pack_dma_end<D, WAVES>(kp + t0 * kb, p, kc, it.kv_hi - t0, kb, K, wave);
      pack_dma_end<D, WAVES>(vp + t0 * vb, p, vc, it.kv_hi - t0, vb, V, wave);
    }
  };
  dma(it.kv_lo, (lds_t)K0, (lds_t)V0);
  PackRows<D, QF16> w;
  w.init(a, it, w0, lane);
  bool bad = false;
  auto tile = [&](int t0, lds_t K, lds_t V, lds_t Kn, lds_t Vn) {
    // this wave's DMA of the tile has landed, every wave's has, and every wave is
    // done with the other buffer
    pack_wait();
    pack_barrier();
    dma(t0 + kPackTile, Kn, Vn);
    if (t0 > whi) return;  // no row of this wave sees the tile
    float16_t sc[2];
    pack_scores(w, K, kat, sc);
    if (t0 + kPackTile - 1 > wlo || t0 + kPackTile > it.kv_hi) {
      const int left = min(w.lim, it.kv_hi - 1) - t0 - 4 * kh;
#pragma unroll
      for (int pb = 0; pb < 2; pb++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (!pack_visible(left, pb, i)) sc[pb][i] = -INFINITY;
#pragma unroll 1
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int db = 0; db < D / 32; db++) bad |= half8_nonfinite(pack_v_frag<D>(V, (vat ^ (64 * db)) + 32 * D * u));
    }
    pack_values<D, QF16>(w, sc, a.qscale, V, vat, bad);
  };
  for (int t0 = it.kv_lo; t0 < it.kv_hi; t0 += 2 * kPackTile) {
    tile(t0, (lds_t)K0, (lds_t)V0, (lds_t)K1, (lds_t)V1);
    if (t0 + kPackTile < it.kv_hi) tile(t0 + kPackTile, (lds_t)K1, (lds_t)V1, (lds_t)K0, (lds_t)V0);
  }
  // a wave's own 32 rows of f32 in the tiles' place
  static_assert(4 * TB >= WAVES * 128 * D, "the tiles hold the rows");
  const int per = TB / (128 * D);
  lds_t buf = (lds_t)(wave < per ? K0 : wave < 2 * per ? V0 : wave < 3 * per ? K1 : V1) + wave % per * 128 * D;
  if (__syncthreads_or(bad)) {
    packed_redo<D, QF16>((const PackedArgs*)__builtin_amdgcn_kernarg_segment_ptr(), blockIdx.x, w0, (lds_t)K0, (lds_t)V0);
    return;
  }
  w.write(a, it, lane, buf);
}

constexpr int kNonTemporal = 2;  // the nt bit: keys of few rows are read once

// Items of up to 32 rows (single tokens, a few of them): bound by the bytes of their
// keys. Two waves take tiles of 32 keys in turn, each through two LDS buffers of its
// own, so that nothing but its own DMA holds a wave up; their results meet in LDS.
// 64 KiB and two waves a workgroup, two workgroups a CU: at any time about 64 KiB of
// K and V are on their way to each CU, and one workgroup's start and end lie under
// the other's stream.
// 64 decoders of 4096 keys: 165 us, 6.5 TB/s of the 7.0 that a plain read reaches here,
// 190 in packed_kernel; of 16 to 8192 keys 73 us, 5.3 TB/s, and 84.
template <int D, bool QF16>
__global__ __launch_bounds__(64 * kFewWaves, 1) void packed_few_kernel(PackedArgs a) {
  constexpr int TB = kFewTile * D * 2, CH = D / 8, RPI = 64 / CH, NI = kFewTile / RPI;
  __shared__ __attribute__((aligned(1024))) char K0[kFewWaves * TB], V0[kFewWaves * TB];
  __shared__ __attribute__((aligned(1024))) char K1[kFewWaves * TB], V1[kFewWaves * TB];
  const PackedItem it = a.items[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kh = lane >> 5;
  const int kat = pack_k_at<D>(lane & 31, kh), vat = pack_v_at<D>(lane);
  const lds_t Kw[2] = {(lds_t)K0 + wave * TB, (lds_t)K1 + wave * TB};
  const lds_t Vw[2] = {(lds_t)V0 + wave * TB, (lds_t)V1 + wave * TB};

  const int p = lane / CH, c = lane % CH;
  const int64_t kb = a.k_row * 2, vb = a.v_row * 2;
  const char* kp = (const char*)(a.k + it.k0 * a.k_row + it.kvh * D);
  const char* vp = (const char*)(a.v + it.k0 * a.v_row + it.kvh * D);
  // Rows past the item's keys repeat its last one.
  auto dma = [&](int t0, lds_t K, lds_t V) {
    if (t0 >= it.kv_hi) return;
    const int rows = it.kv_hi - t0;
#pragma unroll
    for (int n = 0; n < NI; n++) {
      const int r = n * RPI + p, x = min(r, rows - 1);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(kp + (t0 + x) * kb + 16 * (c ^ pack_k_swz<D>(r))),
          (__attribute__((address_space(3))) void*)(K + 1024 * n), 16, 0, kNonTemporal);
    }
#pragma unroll
    for (int n = 0; n < NI; n++) {
      const int r = n * RPI + p, x = min(r, rows - 1);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(vp + (t0 + x) * vb + 16 * (c ^ pack_v_swz<D>(r))),
          (__attribute__((address_space(3))) void*)(V + 1024 * n), 16, 0, kNonTemporal);
    }
  };
  const int first = it.kv_lo + wave * kFewTile, step = kFewWaves * kFewTile;
  dma(first, Kw[0], Vw[0]);
  PackRows<D, QF16> w;
  w.init(a, it, 0, lane);
  const int wlo = min(it.r0 / a.G + it.shift, it.nk - 1);
  const int whi = min((it.r0 + it.nr - 1) / a.G + it.shift, it.nk - 1);

  // MODE 0: the attention. Where a masked tile holds a value that is not finite, or a
  // reference needs its e, the keys run again as packed_redo does: MODE 1 with one and
  // such values as 0, then 2 and 3 for what the rows see of +inf and -inf.
  bool bad = false;
  float16_t seen[D / 32];
  auto run = [&](auto mode) {
    constexpr int MODE = decltype(mode)::value;
    auto tile = [&](int t0, lds_t K, lds_t V, lds_t Kn, lds_t Vn) {
      pack_wait();
      dma(t0 + step, Kn, Vn);
      if (t0 > whi) return;
      const int left = min(w.lim, it.kv_hi - 1) - t0 - 4 * kh;
      const bool masked = t0 + kFewTile - 1 > wlo || t0 + kFewTile > it.kv_hi;
      half8_t ph[2], pl[2];
      if constexpr (MODE < 2) {
        float16_t sc[2] = {};
#pragma unroll
        for (int s = 0; s < D / 16; s++) {
          const half8_t ka = pack_k_frag(K, kat ^ (32 * s));
          sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, w.qh[s], sc[0], 0, 0, 0);
          if (!QF16) sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, w.ql[QF16 ? 0 : s], sc[0], 0, 0, 0);
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (!pack_visible(left, 0, i)) sc[0][i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) sc[1][i] = -INFINITY;
        pack_maximum<MODE == 1>(w, sc, a.qscale, bad);
        float l[2] = {};
#pragma unroll
        for (int u = 0; u < 2; u++)
          pack_probs<QF16, MODE == 1>(sc, u, a.qscale, w.m, l[u], ph[u], pl[u], w.e);
        w.l += l[0] + l[1];
      } else {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) ph[u][e] = (half_t)(pack_visible(left, 0, u * 8 + e) ? 1.f : 0.f);
      }
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int db = 0; db < D / 32; db++) {
          half8_t va = pack_v_frag<D>(V, (vat ^ (64 * db)) + 32 * D * u);
          if constexpr (MODE == 0) {
            if (masked) bad |= half8_nonfinite(va);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float f = (float)va[e];
              if (MODE == 1) va[e] = fabsf(f) < INFINITY ? va[e] : (half_t)0.f;
              else va[e] = (half_t)(f != f || f == (MODE == 2 ? INFINITY : -INFINITY) ? 1.f : 0.f);
            }
          }
          if constexpr (MODE < 2) {
            w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[u], w.o[db], 0, 0, 0);
            if (!QF16) w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[u], w.o[db], 0, 0, 0);
          } else {
            seen[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[u], seen[db], 0, 0, 0);
          }
        }
    };
    if (MODE != 0) {
      pack_wait();  // the run before may still be reading the buffer
      dma(first, Kw[0], Vw[0]);
    }
    for (int t0 = first; t0 < it.kv_hi; t0 += 2 * step) {
      tile(t0, Kw[0], Vw[0], Kw[1], Vw[1]);
      if (t0 + step < it.kv_hi) tile(t0 + step, Kw[1], Vw[1], Kw[0], Vw[0]);
    }
  };
  run(std::integral_constant<int, 0>{});
  if (__syncthreads_or(bad)) {
    w.clear();
    run(std::integral_constant<int, 1>{});
    auto add = [&](float v) {
#pragma unroll
      for (int db = 0; db < D / 32; db++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (seen[db][i] > 0.f) w.o[db][i] += v;
    };
    auto none = [&] {
#pragma unroll
      for (int db = 0; db < D / 32; db++) seen[db] = float16_t{};
    };
    none();
    run(std::integral_constant<int, 2>{});
    add(INFINITY);
    none();
    run(std::integral_constant<int, 3>{});
    add(-INFINITY);
    __syncthreads();
  }
  // The two waves' rows to the higher one's reference, through LDS.
  static_assert(kFewWaves == 2 && 2 * TB >= 128 * D, "a buffer holds a wave's rows");
  typedef __attribute__((address_space(3))) float16_t* f16p;
  typedef __attribute__((address_space(3))) float4_t* f4;
  if (wave == 1) {
#pragma unroll
    for (int db = 0; db < D / 32; db++) *(f16p)((lds_t)K0 + (db * 64 + lane) * 64) = w.o[db];
    *(f4)((lds_t)V0 + lane * 16) = float4_t{w.m, w.e, w.l, 0.f};
  }
  __syncthreads();
  if (wave == 1) return;
  const float4_t other = *(f4)((lds_t)V0 + lane * 16);
  const float up = (other[0] - w.m) + (other[1] - w.e);
  const bool higher = up > 0.f;
  const float x0 = higher ? __builtin_amdgcn_exp2f(-up) : 1.f, x1 = higher ? 1.f : __builtin_amdgcn_exp2f(up);
  w.l = x0 * w.l + x1 * other[2];
  w.m = higher ? other[0] : w.m;
  w.e = higher ? other[1] : w.e;
#pragma unroll
  for (int db = 0; db < D / 32; db++) {
    const float16_t o1 = *(f16p)((lds_t)K0 + (db * 64 + lane) * 64);
#pragma unroll
    for (int i = 0; i < 16; i++) w.o[db][i] = x0 * w.o[db][i] + x1 * o1[i];
  }
  w.write(a, it, lane, (lds_t)K1);
}

// Merges the parts of up to eight rows: sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p, m_p
// and M being references, m + e.
// D / 4 lanes hold a row, four dims each; with fewer rows the lane groups share a
// row's parts and meet in LDS, in their order.
template <int D>
__global__ __launch_bounds__(256) void packed_merge_kernel(PackedArgs a) {
  constexpr int LR = D / 4, GR = 256 / LR;  // lanes per row, groups of them
  __shared__ float4_t so[GR][LR];
  __shared__ float sl[GR], sm[GR], se[GR];
  const PackedMerge g = a.merges[blockIdx.x];
  const int grp = threadIdx.x / LR, d = threadIdx.x % LR * 4;
  const int slices = GR / (g.nr > 4 ? 8 : g.nr > 2 ? 4 : g.nr), i = grp / slices, sl0 = grp % slices;
  float4_t v = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f, M = kPackNoMax, E = 0.f;
  bool blank = false;  // a part with a sum of 0 whose keys all score -inf
  if (i < g.nr) {
    // eight parts' loads in flight, the reference moving with them
    for (int p0 = sl0; p0 < g.parts; p0 += 8 * slices) {
      float3 ml[8];
      float4_t po[8];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int p = min(p0 + u * slices, g.parts - 1);
        const int64_t pr = (int64_t)g.part + i + (int64_t)p * g.step;
        ml[u] = *(const float3*)(a.part_ml + pr * 4);
        po[u] = *(const float4_t*)(a.part_o + pr * D + d);
      }
      float tm = M, te = E;
#pragma unroll
      for (int u = 0; u < 8; u++) {
        blank |= ml[u].z == 0.f && ml[u].x != ml[u].x;  // past the parts: the last one again
        if (p0 + u * slices >= g.parts) ml[u].z = 0.f;
        if (ml[u].z != 0.f && (ml[u].x - tm) + (ml[u].y - te) > 0.f) tm = ml[u].x, te = ml[u].y;
      }
      const float old = __builtin_amdgcn_exp2f((M - tm) + (E - te));
      M = tm;
      E = te;
      l *= old;
      v *= old;
#pragma unroll
      for (int u = 0; u < 8; u++) {
        if (ml[u].z == 0.f) continue;  // the part shows this row no key, or none that counts
        const float w = __builtin_amdgcn_exp2f((ml[u].x - M) + (ml[u].y - E));
        l += w * ml[u].z;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += w * po[u][e];
      }
    }
  }
  if (slices > 1) {
    so[grp][d / 4] = v;
    if (d == 0) {
      sl[grp] = l;
      sm[grp] = l == 0.f && blank ? NAN : M;
      se[grp] = E;
    }
    __syncthreads();
    if (sl0 == 0) {
      float tm = M, te = E;
      for (int s = 1; s < slices; s++) {
        if (sl[grp + s] == 0.f) blank |= sm[grp + s] != sm[grp + s];
        else if ((sm[grp + s] - tm) + (se[grp + s] - te) > 0.f) tm = sm[grp + s], te = se[grp + s];
      }
      float w = __builtin_amdgcn_exp2f((M - tm) + (E - te));
      l *= w;
      v *= w;
      for (int s = 1; s < slices; s++) {
        if (sl[grp + s] == 0.f) continue;
        w = __builtin_amdgcn_exp2f((sm[grp + s] - tm) + (se[grp + s] - te));
        l += w * sl[grp + s];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += w * so[grp + s][d / 4][e];
      }
    }
  }
  if (i >= g.nr || sl0) return;
  const int row = g.r0 + i, tok = row / a.G, head = g.kvh * a.G + row % a.G;
  const int64_t off = (g.q0 + tok) * a.out_row + head * D + d;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = l == 0.f ? (blank ? NAN : 0.f) : v[e] / l;
  pack_store4(a, off, v);
}

template <int D, bool QF16>
static void packed_launch(PackedArgs a, const PackedCounts& n, hipStream_t st) {
  if (n.items) hipLaunchKernelGGL((packed_kernel<D, QF16, kPackWaves>), dim3(n.items), dim3(64 * kPackWaves), 0, st, a);
  a.items += n.items;
  if (n.few) hipLaunchKernelGGL((packed_few_kernel<D, QF16>), dim3(n.few), dim3(64 * kFewWaves), 0, st, a);
  if (n.merges) hipLaunchKernelGGL((packed_merge_kernel<D>), dim3(n.merges), dim3(256), 0, st, a);
}

int packed_enqueue(const PackedArgs& a, int D, int q_f16, const PackedCounts& n, hipStream_t st) {
  if (D == 128) q_f16 ? packed_launch<128, true>(a, n, st) : packed_launch<128, false>(a, n, st);
  else q_f16 ? packed_launch<64, true>(a, n, st) : packed_launch<64, false>(a, n, st);
  TGOHIP_HIP(hipGetLastError());
  return 0;
}

}  // namespace tgohip
