// operators.h -- the op-level operators beside the projections and paged
// attention: rotary positions, packed attention, the adapters of many requests.
// Arguments and launches of kernels/rope.hip, packed_attention.hip, adapters.hip.
#pragma once

#include "../common.h"

#include <algorithm>

namespace tgohip {

// ---- rotary positions (rope.hip) -------------------------------------------
constexpr int kRopeGroups = 3;      // tensors of heads per call
constexpr int kRopeMaxHeadDim = 256;
struct RopeGroup {
  const void* x;
  void* y;
  int64_t x_row, x_head, y_row, y_head;  // elements
  int32_t heads, x_f16, y_f16, rotate;
  uint64_t magic;  // set by launch_rope
};
struct RopeArgs {
  const int32_t* positions;
  const double* inv_freq;  // [rotary_dim / 2], turns per position (angle / 2 pi)
  float attention;         // cos and sin are multiplied by it
  int T, d, rd, half;      // half: pairs (i, i + rd/2), else (2i, 2i + 1)
  int rows;  // of a workgroup, set by launch_rope
  int n;
  RopeGroup g[kRopeGroups];
};
void launch_rope(const RopeArgs& a, int ncu, hipStream_t st);

// ---- packed attention (packed_attention.hip) --------------------------------
// A work item: rows [r0, r0 + nr) of one sequence and kv head against its keys
// [kv_lo, kv_hi). Row r is query head kvh * G + r % G of token r / G.
struct PackedItem {
  int32_t q0, k0;   // the sequence's first packed query and key row
  int32_t nk;       // its keys
  int32_t shift;    // token t sees keys 0 .. min(t + shift, nk - 1)
  int32_t r0, nr;
  int32_t kv_lo, kv_hi;
  int32_t kvh;
  int32_t part;     // first row of its partial result, -1 when it writes out
};
// Rows [r0, r0 + nr) of a (sequence, kv head): `parts` partial results, row i of
// part p at partial row part + p * step + i.
struct PackedMerge {
  int32_t q0, r0, nr, kvh, part, parts, step;
};
struct PackedPlan {
  int H = 0, Hkv = 0, D = 0, q_f16 = 0;
  int64_t tq = 0, tk = 0;  // packed query and key rows
  std::vector<PackedItem> items;  // of the tile kernel
  std::vector<PackedItem> few;    // of the few-row kernel
  std::vector<PackedMerge> merges;
  int64_t part_rows = 0;
};
constexpr int kPackRows = 128;  // the most rows of an item
// Decomposes a call (host only). nq, nk: [B], checked by the caller.
void packed_build_plan(int B, const int32_t* nq, const int32_t* nk, int H, int Hkv, int D, bool causal,
                       bool q_f16, int ncu, PackedPlan& plan);
// Key rows at most this many elements apart: offsets in a tile fit 32 bits.
constexpr int64_t kPackMaxRow = (int64_t)1 << 24;
struct PackedArgs {
  const void* q;
  const half_t* k;
  const half_t* v;
  void* out;
  float* part_o;   // [part_rows][D]
  float* part_ml;  // [part_rows][4]: the reference m, e (log2) and the sum
  const PackedItem* items;
  const PackedMerge* merges;
  int64_t q_row, k_row, v_row, out_row, out_lo;  // elements
  int G, out_form;                               // OUT_F32, OUT_F16, OUT_X2 (lo plane out_lo on)
  float qscale;                                  // scale * log2(e)
};
// a.items: the tile kernel's, then the few-row kernel's.
struct PackedCounts {
  int items = 0, few = 0, merges = 0;
};
int packed_enqueue(const PackedArgs& a, int D, int q_f16, const PackedCounts& n, hipStream_t st);

// ---- adapters (adapters.hip) --------------------------------------------------
constexpr int kAdapterMaxRank = 128;
// Rows up to which a batch's tiles hold 16 rows, 64 beyond. Tiles of 16 / of 64, us:
//   [4096, 6144], rank 16, 8 adapters: 128 rows 7.5 / 11.2, 512 11.8 / 16.9, 1024 18.8 /
//       21.9, 2048 31.5 / 31.9; 256 adapters: 256 rows 29.2 / 27.6, 1024 33.3 / 32.9
//   [4096, 4096], rank 64, 8 adapters: 256 rows 11.6 / 17.0, 512 17.0 / 21.6, 768 22.2 /
//       24.6, 1024 28.0 / 25.8; 256 adapters: 256 rows 64.1 / 55.5, 1024 78.2 / 70.7
// Rows alone decide: with many rows of a small rank 16 would do a little longer, with
// many adapters of a large one less long.
constexpr int kAdapterFewRows = 512;
struct AdapterEntry {
  const half_t* down;  // [rank_pad][K]
  const half_t* up;    // [N][rank_pad]
  int32_t rank_pad;    // 16, 32, 64 or 128; 0: no adapter at this index
  float scale;
};
// Rows perm[start .. start + n) carry the adapter (-1: none).
struct AdapterTile {
  int32_t adapter, start, n;
};
struct AdapterArgs {
  const AdapterEntry* table;
  const AdapterTile* tiles;
  const int32_t* perm;
  int ntiles, T, K, N;
  const void* x;
  int xk;  // XK_F16, XK_F32, XK_X2
  const void* base;
  void* y;
  int y_f16;
  int splits;  // shares of K
  int cols;    // columns per workgroup of the second kernel (set by launch_adapters)
  int rank_pad;  // the set's largest
  float* u;      // [splits][T][kAdapterMaxRank]: x . down^T of the permuted rows, by share
  half_t* pair;  // [T][2][kAdapterMaxRank]: their sums as scaled hi + lo pairs
  float* pair_scale;  // [T]
};
// The shares of K for a batch of `tiles` tiles (their planes are the workspace): up to
// two workgroups a CU, all on the chip at once. With 1, 2, 3 or 4 per CU, us: 8000 f16
// rows of [12288, 4096] 86, 81, 92, 86; 1152 pairs of [4096, 24576] 104, 103, 107, 106.
// Tiles without an adapter count too, though their workgroups return at once. Counting
// all / only those with one, us: an adapter for 1000 of 8000 f32 rows of [12288, 4096] 53 /
// 32, for half of 1056 of [4096, 24576] 57 / 55, for a third of 48 tiles of [12288, 4096]
// 35 / 37.
constexpr int kAdapterMaxSplits = 16;
inline int adapter_splits(int tiles, int ncu) {
  return tiles > 0 ? std::min(kAdapterMaxSplits, std::max(1, 2 * ncu / tiles)) : 1;
}
// tile_rows: 16 or 64, the most rows of a tile.
void launch_adapters(const AdapterArgs& a, int tile_rows, int ncu, hipStream_t st);

}  // namespace tgohip
