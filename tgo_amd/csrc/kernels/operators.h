// operators.h -- the op-level operators beside the projections and paged
// attention: rotary positions, packed attention, the adapters of many requests, the
// 8-bit cache. Arguments and launches of kernels/rope.hip, packed_attention.hip,
// adapters.hip, cache_rows.hip, cache_attention.hip.
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
// What a kernel's tiles of 64 keys cost: us of one whose workgroup has its CU alone, and
// the part of that rate each of two workgroups on a CU reaches.
struct PackRate {
  double tile, shared;
};
// Items, longest first, cut along their keys at multiples of `tile` (pieces of at least
// `least` tiles) as ends soonest; plan gets the merges and rows of partial results.
void pack_cut(const std::vector<PackedItem>& whole, int tile, int least, int ncu, const PackRate& rate,
              std::vector<PackedItem>& out, PackedPlan& plan);
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
// The merges alone, of partial results that other kernels left (a.q, k, v and items unused).
void packed_merge_enqueue(const PackedArgs& a, int D, int merges, hipStream_t st);

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

// ---- 8-bit cache (cache_rows.hip, cache_attention.hip) ------------------------------
// One layer: codes [pages][kv_heads][block][d], scales [pages][kv_heads][block]. A row is
// one position of one kv head; the rows of a layer number below 2^31.
struct CacheLayer {
  uint8_t *k, *v;
  float *ks, *vs;
  int32_t capacity, bshift, Hkv, d, f8;  // pages * block; log2(block)
  // the row of a slot and head
  __host__ __device__ int64_t row(int32_t slot, int h) const {
    return ((((int64_t)(slot >> bshift) * Hkv) + h) << bshift) + (slot & ((1 << bshift) - 1));
  }
};
constexpr int kCacheMaxHeads = 4096;
struct CacheStoreArgs {
  CacheLayer c;
  const int32_t *positions, *slots;
  const double* inv_freq;  // as RopeArgs's
  float attention;
  int T, rd, half;  // rd 0: nothing is rotated
  const void *q, *k, *v;
  void* q_out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  const float *q_gain, *k_gain;  // null: not normed
  float eps;
  int H, x_f16, out_f16;
  int rows, slice;  // rows and heads of a workgroup, set by launch_cache_store
};
void launch_cache_store(const CacheStoreArgs& a, int ncu, hipStream_t st);
struct CacheReadArgs {
  CacheLayer c;
  const int32_t* slots;
  int T, f16;
  void* out[2];  // k's, v's; null: not read
  int64_t row[2], head[2];
};
void launch_cache_read(const CacheReadArgs& a, hipStream_t st);
// Rows src[i] to dst[i] (slots) of every layer and head; a workgroup takes moves
// [start, start + n) of one (layer, head), kCacheMoveSeg of them read before any is written.
constexpr int kCacheMoveSeg = 64;
struct CacheMoveBatch {
  int32_t start, n;
};
struct CacheMoveArgs {
  CacheLayer c;  // of layer 0
  int layers, batches;
  int64_t layer_rows;
  const int32_t *src, *dst;
  const CacheMoveBatch* batch;
};
// Up to this many moves and batches go with the kernel's arguments, which end at 4 KB; more are
// fetched to the device first. By arguments / fetched, us a call: 448 moves of 36 layers
// and 8 heads 16.2 / 25.0, 4 moves 5.2 / 12.
constexpr int kCacheMoveFew = 480, kCacheMoveFewBatches = 16;
struct CacheMoveFew {
  int32_t n;  // 0: CacheMoveArgs's
  CacheMoveBatch batch[kCacheMoveFewBatches];
  int32_t src[kCacheMoveFew], dst[kCacheMoveFew];
};
static_assert(sizeof(CacheMoveArgs) + sizeof(CacheMoveFew) <= 4096, "a kernel's arguments");
void launch_cache_move(const CacheMoveArgs& a, const CacheMoveFew& f, hipStream_t st);

// A work item: rows [r0, r0 + nr) of a sequence and kv head (as PackedItem's) against
// positions [kv_lo, kv_hi). tree 0: token t sees positions up to t + shift; 1: those
// below shift, and shift + j where bit j of its mask is set.
struct CacheItem {
  int32_t q0, seq, nk, shift, r0, nr, kv_lo, kv_hi, kvh, part, tree, pad;
};
struct CachePlan {
  int H = 0;
  int64_t tq = 0;
  std::vector<CacheItem> items;
  int wide = 0;       // those of the kernel of 256 rows, which come first
  std::vector<PackedMerge> merges;
  int64_t part_rows = 0;
};
constexpr int kCacheMaxTree = 64;  // tokens of a tree: the bits of a mask
// tree: [B], whether a sequence's new tokens are one (null: none is).
void cache_build_plan(int B, const int32_t* extents, const int32_t* lengths, const uint8_t* tree, int H, int Hkv, int D,
                      bool q_f16, int ncu, CachePlan& plan);
struct CacheAttnArgs {
  CacheLayer c;
  const void* q;
  void* out;
  const CacheItem* items;
  const PackedMerge* merges;
  const uint32_t* pages;  // the row of a page's first position (head 0)
  const uint64_t* masks;
  float *part_o, *part_ml;
  int64_t q_row, out_row, out_lo;
  int max_pages, G, out_form, q_f16;
  int nitems, wide, nmerges;
  float qscale;  // scale * log2(e)
};
int cache_attention_enqueue(const CacheAttnArgs& a, hipStream_t st);

}  // namespace tgohip
