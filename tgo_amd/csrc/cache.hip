// cache.hip -- C ABI of the 8-bit paged cache's operators: store, read, move, attention.
#include "operators_abi.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <unordered_map>

namespace {

// Beyond any tensor. Bytes from an operand's first row to its last stay in 64 bits: a stride of at most
// kTopStride elements times fewer than 2^24 rows, or rows times their stride at most kTopReach.
constexpr int64_t kTopStride = (int64_t)1 << 36, kTopReach = (int64_t)1 << 60;

std::string str(int64_t v) { return std::to_string(v); }

// The cache's geometry, or why it is refused.
int check_geometry(const char* what, const tgohip_cache* c) {
  const auto bad = [what](const std::string& m) { return refuse(std::string(what) + ": " + m); };
  if (!c) return bad("the cache is missing");
  if (c->form != TGOHIP_CACHE_I8 && c->form != TGOHIP_CACHE_F8)
    return bad("form is " + str(c->form) + ", neither int8 nor e4m3");
  if (c->head_dim != 64 && c->head_dim != 128)
    return bad("head_dim is " + str(c->head_dim) + "; the kernels are built for 64 and 128");
  if (c->block < 1 || c->block > 1024 || (c->block & (c->block - 1)))
    return bad("block is " + str(c->block) + "; a power of two up to 1024");
  if (c->kv_heads < 1 || c->kv_heads > kCacheMaxHeads)
    return bad(str(c->kv_heads) + " kv heads; 1 to " + str(kCacheMaxHeads));
  if (c->layers < 1 || c->layers > 65535 || (int64_t)c->layers * c->kv_heads > 65535)
    return bad(str(c->layers) + " layers of " + str(c->kv_heads) + " kv heads; layers times heads is 1 to 65535");
  if (c->pages < 1 || (int64_t)c->pages * c->block * c->kv_heads > INT_MAX)
    return bad(str(c->pages) + " pages of " + str(c->block) + " positions and " + str(c->kv_heads) +
               " heads; at least one, and rows of a layer stay below 2^31");
  return 0;
}

int64_t layer_rows(const tgohip_cache* c) { return (int64_t)c->pages * c->block * c->kv_heads; }

// The cache's buffers, all of them: codes and scales.
void cache_spans(const tgohip_cache* c, Span (&s)[4]) {
  const int64_t rows = layer_rows(c) * c->layers;
  s[0] = Span{(const char*)c->k, 1, 1, 0, 0, rows * c->head_dim};
  s[1] = Span{(const char*)c->v, 1, 1, 0, 0, rows * c->head_dim};
  s[2] = Span{(const char*)c->k_scale, 1, 1, 0, 0, rows * 4};
  s[3] = Span{(const char*)c->v_scale, 1, 1, 0, 0, rows * 4};
}
const char* const kSpanNames[4] = {"k", "v", "k_scale", "v_scale"};

int check_cache(const char* what, const tgohip_cache* c, int layer) {
  if (const int rc = check_geometry(what, c)) return rc;
  const auto bad = [what](const std::string& m) { return refuse(std::string(what) + ": " + m); };
  if (layer < 0 || layer >= c->layers) return bad("layer " + str(layer) + " of " + str(c->layers));
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return bad("the cache's codes and scales are device buffers");
  if (misaligned(c->k) || misaligned(c->v) || (uintptr_t)c->k_scale % 4 || (uintptr_t)c->v_scale % 4)
    return bad("codes start on 16-byte boundaries, scales on 4-byte ones");
  Span s[4];
  cache_spans(c, s);
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < i; j++)
      if (meet(s[i], s[j])) return bad(std::string("the cache's ") + kSpanNames[j] + " and " + kSpanNames[i] + " meet in memory");
  return 0;
}
// Refuses an operand that lies in the cache.
int check_apart(const char* what, const tgohip_cache* c, const Span& x, const char* name) {
  Span s[4];
  cache_spans(c, s);
  for (int i = 0; i < 4; i++)
    if (meet(x, s[i])) return refuse(std::string(what) + ": " + name + " meets the cache's " + kSpanNames[i] + " in memory");
  return 0;
}

CacheLayer layer_of(const tgohip_cache* c, int layer) {
  const int64_t first = layer_rows(c) * layer;
  CacheLayer l{};
  l.k = (uint8_t*)c->k + first * c->head_dim;
  l.v = (uint8_t*)c->v + first * c->head_dim;
  l.ks = c->k_scale + first;
  l.vs = c->v_scale + first;
  l.capacity = c->pages * c->block;
  while (1 << l.bshift < c->block) l.bshift++;
  l.Hkv = c->kv_heads;
  l.d = c->head_dim;
  l.f8 = c->form == TGOHIP_CACHE_F8;
  return l;
}

bool bad_type(int t) { return t != TGOHIP_F32 && t != TGOHIP_F16; }
bool bad_stride(int64_t s) { return s < 0 || s > kTopStride; }

// Whether rows of heads of d elements share an element.
bool overlap(int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t d) {
  int64_t s0 = rows > 1 ? row : 0, n0 = rows, s1 = heads > 1 ? head : 0, n1 = heads;
  if (s0 > s1) {
    std::swap(s0, s1);
    std::swap(n0, n1);
  }
  int64_t need = d;
  if (n0 > 1) {
    if (s0 < need) return true;
    need = (n0 - 1) * s0 + d;
  }
  return n1 > 1 && s1 < need;
}

// What a slot is written by: open addressing over a power of two of at least twice the moves.
struct Writers {
  std::vector<int32_t> slot, move;
  uint32_t mask;
  explicit Writers(int n) {
    uint32_t size = 16;
    while (size < 2 * (uint32_t)n) size *= 2;
    mask = size - 1;
    slot.assign(size, -1);
    move.resize(size);
  }
  uint32_t at(int32_t s) const {  // the slot's place, or the free one it would take
    uint32_t i = (uint32_t)s * 0x9e3779b1u >> 7 & mask;
    while (slot[i] >= 0 && slot[i] != s) i = (i + 1) & mask;
    return i;
  }
};

// One component's moves in an order in which a row is read before, or in the same 64 as, it
// is written over; p: its moves, more than 64.
int order_component(const int32_t* p, int n, const std::vector<int>& next, std::vector<int>& sorted) {
  std::unordered_map<int, int> before;  // moves that come before one
  for (int i = 0; i < n; i++)
    if (next[p[i]] >= 0) before[next[p[i]]]++;
  const auto waits = [&](int i) {
    const auto b = before.find(i);
    return b != before.end() && b->second > 0;
  };
  sorted.clear();
  for (int i = 0; i < n; i++)
    if (!waits(p[i])) sorted.push_back(p[i]);
  for (size_t k = 0; k < sorted.size(); k++) {
    const int m = next[sorted[k]];
    if (m >= 0 && --before[m] == 0) sorted.push_back(m);
  }
  // What is left is the component's one cycle: it goes last, whole, in a segment of its
  // own when it does not fit behind the others.
  std::vector<int> cycle;
  for (int i = 0; i < n; i++)
    if (waits(p[i])) cycle.push_back(p[i]);
  if (cycle.size() > (size_t)kCacheMoveSeg)
    return refuse("cache_move: a cycle of " + str((int64_t)cycle.size()) + " slots; up to " + str(kCacheMoveSeg));
  if (!cycle.empty())
    while (sorted.size() % kCacheMoveSeg + cycle.size() > (size_t)kCacheMoveSeg)
      sorted.push_back(sorted.back());  // again: reads what it read, writes what it wrote
  sorted.insert(sorted.end(), cycle.begin(), cycle.end());
  return 0;
}

// The moves without those onto themselves, in batches for a workgroup each: moves that
// depend on each other stay in one. Up to 64 of a batch are all read before any is
// written, in whatever order they stand.
int order_moves(const int32_t* from, const int32_t* to, int n, std::vector<int32_t>& src, std::vector<int32_t>& dst,
                std::vector<CacheMoveBatch>& batches) {
  Writers w(n);
  std::vector<int32_t> kept;
  kept.reserve((size_t)n);
  for (int i = 0; i < n; i++) {
    const uint32_t at = w.at(to[i]);
    if (w.slot[at] >= 0) return refuse("cache_move: two rows go to slot " + str(to[i]));
    w.slot[at] = to[i];
    w.move[at] = i;
    if (from[i] != to[i]) kept.push_back(i);
  }
  if (kept.empty()) return 0;
  src.reserve(kept.size());
  dst.reserve(kept.size());
  const auto put = [&](const int32_t* p, int count) {
    if (batches.empty() || batches.back().n + count > kCacheMoveSeg)
      batches.push_back(CacheMoveBatch{(int32_t)src.size(), 0});
    batches.back().n += count;
    for (int i = 0; i < count; i++) {
      src.push_back(from[p[i]]);
      dst.push_back(to[p[i]]);
    }
  };
  if (kept.size() <= (size_t)kCacheMoveSeg) {
    put(kept.data(), (int)kept.size());
    return 0;
  }
  // next[i]: the move that writes what i reads, which i comes before. Its graph's components:
  // root[i] is never behind i, so a component's root is its first move.
  std::vector<int> next((size_t)n, -1), root((size_t)n);
  for (const int i : kept) {
    root[i] = i;
    const uint32_t at = w.at(from[i]);
    if (w.slot[at] < 0) continue;
    const int m = w.move[at];
    if (from[m] != to[m]) next[i] = m;
  }
  const auto find_root = [&](int i) {
    while (root[i] != i) i = root[i] = root[root[i]];
    return i;
  };
  for (const int i : kept) {
    if (next[i] < 0) continue;
    const int a = find_root(i), b = find_root(next[i]);
    root[std::max(a, b)] = std::min(a, b);
  }
  // sorted by component, components as their first moves stand
  std::vector<int32_t> count((size_t)n, 0), part(kept.size());
  for (const int i : kept) count[find_root(i)]++;
  int32_t sum = 0;
  for (const int i : kept)
    if (root[i] == i) {
      const int32_t c = count[i];
      count[i] = sum;
      sum += c;
    }
  for (const int i : kept) part[count[find_root(i)]++] = i;
  std::vector<int> sorted;
  for (size_t i = 0; i < part.size();) {
    const size_t end = count[find_root(part[i])];
    if (end - i <= (size_t)kCacheMoveSeg) {
      put(&part[i], (int)(end - i));
    } else {
      const int rc = order_component(&part[i], (int)(end - i), next, sorted);
      if (rc) return rc;
      put(sorted.data(), (int)sorted.size());
    }
    i = end;
  }
  return 0;
}

}  // namespace

extern "C" {

int tgohip_cache_store(tgohip_ctx* c, const tgohip_cache* cache, int layer, int rope, const int32_t* positions,
                       const int32_t* slots, int T, const tgohip_cache_rows* rows) {
  return guarded([&]() -> int {
    int rc = check_cache("cache_store", cache, layer);
    if (rc) return rc;
    if (!rows) return refuse("cache_store: the rows are missing");
    const tgohip_cache_rows& r = *rows;
    const int d = cache->head_dim;
    if (T < 0 || T >= 1 << 24) return refuse("cache_store: " + str(T) + " rows; 0 to 2^24 - 1");
    if (r.heads < 0 || r.heads > kCacheMaxHeads)
      return refuse("cache_store: " + str(r.heads) + " query heads; 0 to " + str(kCacheMaxHeads));
    if (bad_type(r.x_dtype) || (r.heads && bad_type(r.out_dtype)))
      return refuse("cache_store: x_dtype and out_dtype are f32 or f16");
    if ((r.q_gain || r.k_gain) && !(r.eps >= 0.f && std::isfinite(r.eps)))
      return refuse("cache_store: eps is " + num(r.eps) + "; a finite number, not negative");
    if (T == 0) return c ? 0 : no_ctx("cache_store");
    if (!r.k || !r.v || !slots || (r.heads && (!r.q || !r.q_out)))
      return refuse("cache_store: q, k, v, q_out and slots are device buffers");
    if (rope && !positions) return refuse("cache_store: positions is a device buffer of int32");
    const int64_t xb = elt(r.x_dtype == TGOHIP_F16), ob = elt(r.out_dtype == TGOHIP_F16);
    if ((uintptr_t)r.k % xb || (uintptr_t)r.v % xb || (r.heads && ((uintptr_t)r.q % xb || (uintptr_t)r.q_out % ob)) ||
        (uintptr_t)slots % 4 || (uintptr_t)positions % 4 || (uintptr_t)r.q_gain % 4 || (uintptr_t)r.k_gain % 4)
      return refuse("cache_store: an operand is not aligned to its type");
    if (bad_stride(r.k_row) || bad_stride(r.k_head) || bad_stride(r.v_row) || bad_stride(r.v_head) ||
        (r.heads && (bad_stride(r.q_row) || bad_stride(r.q_head) || bad_stride(r.out_row) || bad_stride(r.out_head))))
      return refuse("cache_store: strides are not negative, and at most 2^36 elements");
    if (r.heads && overlap(T, r.out_row, r.heads, r.out_head, d))
      return refuse("cache_store: heads of q_out overlap (strides " + str(r.out_row) + ", " + str(r.out_head) + ")");
    if (!c) return no_ctx("cache_store");
    CacheStoreArgs a{};
    if (rope) {
      RopeTable* t = find(c->ops.ropes, rope, "cache_store: rope");
      if (!t) return TGOHIP_EINVAL;
      if (t->d != d)
        return refuse("cache_store: the rotary handle is of heads of " + str(t->d) + ", the cache of " + str(d));
      a.inv_freq = (const double*)t->inv_freq.p;
      a.attention = t->attention;
      a.rd = t->rd;
      a.half = t->half;
    }
    const int Hkv = cache->kv_heads;
    const Span sq{(const char*)r.q, r.heads ? T : 0, r.heads, r.q_row * xb, r.q_head * xb, d * xb};
    const Span so{(const char*)r.q_out, r.heads ? T : 0, r.heads, r.out_row * ob, r.out_head * ob, d * ob};
    const Span sk{(const char*)r.k, T, Hkv, r.k_row * xb, r.k_head * xb, d * xb};
    const Span sv{(const char*)r.v, T, Hkv, r.v_row * xb, r.v_head * xb, d * xb};
    const Span sp{(const char*)positions, rope ? 1 : 0, 1, 0, 0, (int64_t)T * 4};
    const Span ss{(const char*)slots, 1, 1, 0, 0, (int64_t)T * 4};
    const Span gq{(const char*)r.q_gain, r.q_gain ? 1 : 0, 1, 0, 0, (int64_t)d * 4};
    const Span gk{(const char*)r.k_gain, r.k_gain ? 1 : 0, 1, 0, 0, (int64_t)d * 4};
    const struct {
      const Span& s;
      const char* name;
    } all[] = {{so, "q_out"}, {sq, "q"}, {sk, "k"}, {sv, "v"}, {sp, "positions"}, {ss, "slots"}, {gq, "q_gain"}, {gk, "k_gain"}};
    for (const auto& x : all) {
      if ((rc = check_apart("cache_store", cache, x.s, x.name))) return rc;
      if (&x.s == &so || !meet(so, x.s)) continue;
      if (&x.s == &sq && r.x_dtype == r.out_dtype && same(so, sq)) continue;
      return refuse(std::string("cache_store: q_out meets ") + x.name +
                    " in memory; it is q itself (same type and strides) or apart");
    }
    a.c = layer_of(cache, layer);
    a.positions = positions;
    a.slots = slots;
    a.T = T;
    a.q = r.q;
    a.k = r.k;
    a.v = r.v;
    a.q_out = r.q_out;
    a.q_row = r.q_row;
    a.q_head = r.q_head;
    a.k_row = r.k_row;
    a.k_head = r.k_head;
    a.v_row = r.v_row;
    a.v_head = r.v_head;
    a.out_row = r.out_row;
    a.out_head = r.out_head;
    a.q_gain = r.q_gain;
    a.k_gain = r.k_gain;
    a.eps = r.eps;
    a.H = r.heads;
    a.x_f16 = r.x_dtype == TGOHIP_F16;
    a.out_f16 = r.out_dtype == TGOHIP_F16;
    OnDevice on(c->device);
    launch_cache_store(a, c->ncu, c->stream);
    TGOHIP_HIP(hipGetLastError());
    return 0;
  });
}

int tgohip_cache_read(tgohip_ctx* c, const tgohip_cache* cache, int layer, const int32_t* slots, int T, void* k_out,
                      int64_t k_row, int64_t k_head, void* v_out, int64_t v_row, int64_t v_head, int out_dtype) {
  return guarded([&]() -> int {
    int rc = check_cache("cache_read", cache, layer);
    if (rc) return rc;
    if (T < 0 || (int64_t)T * cache->kv_heads >= 1 << 29)  // threads of a launch stay below 2^32
      return refuse("cache_read: " + str(T) + " rows of " + str(cache->kv_heads) + " heads; heads of rows stay below 2^29");
    if (bad_type(out_dtype)) return refuse("cache_read: out_dtype is " + str(out_dtype) + "; f32 or f16");
    if (T == 0 || (!k_out && !v_out)) return c ? 0 : no_ctx("cache_read");
    if (!slots || (uintptr_t)slots % 4) return refuse("cache_read: slots is a device buffer of int32");
    const int64_t ob = elt(out_dtype == TGOHIP_F16), d = cache->head_dim, Hkv = cache->kv_heads;
    void* const out[2] = {k_out, v_out};
    const int64_t row[2] = {k_row, v_row}, head[2] = {k_head, v_head};
    const char* const names[2] = {"k_out", "v_out"};
    const Span ss{(const char*)slots, 1, 1, 0, 0, (int64_t)T * 4};
    Span so[2];
    CacheReadArgs a{};
    for (int i = 0; i < 2; i++) {
      so[i] = Span{(const char*)out[i], out[i] ? T : 0, Hkv, row[i] * ob, head[i] * ob, d * ob};
      if (!out[i]) continue;
      if ((uintptr_t)out[i] % ob) return refuse(std::string("cache_read: ") + names[i] + " is not aligned to its type");
      if (bad_stride(row[i]) || bad_stride(head[i]))
        return refuse("cache_read: strides are not negative, and at most 2^36 elements");
      if (row[i] > kTopReach / T)
        return refuse(std::string("cache_read: ") + names[i] + "'s " + str(T) + " rows are " + str(row[i]) +
                      " elements apart; rows times their stride is at most 2^60");
      if (overlap(T, row[i], Hkv, head[i], d))
        return refuse(std::string("cache_read: heads of ") + names[i] + " overlap (strides " + str(row[i]) + ", " +
                      str(head[i]) + ")");
      if ((rc = check_apart("cache_read", cache, so[i], names[i]))) return rc;
      if (meet(so[i], ss)) return refuse(std::string("cache_read: ") + names[i] + " meets slots in memory");
      a.out[i] = out[i];
      a.row[i] = row[i];
      a.head[i] = head[i];
    }
    if (k_out && v_out && meet(so[0], so[1])) return refuse("cache_read: k_out and v_out meet in memory");
    if (!c) return no_ctx("cache_read");
    a.c = layer_of(cache, layer);
    a.slots = slots;
    a.T = T;
    a.f16 = out_dtype == TGOHIP_F16;
    OnDevice on(c->device);
    launch_cache_read(a, c->stream);
    TGOHIP_HIP(hipGetLastError());
    return 0;
  });
}

int tgohip_cache_move(tgohip_ctx* c, const tgohip_cache* cache, const int32_t* from, const int32_t* to, int n) {
  return guarded([&]() -> int {
    int rc = check_cache("cache_move", cache, 0);
    if (rc) return rc;
    if (n < 0 || n >= 1 << 24) return refuse("cache_move: " + str(n) + " rows; 0 to 2^24 - 1");
    if (n && (!from || !to)) return refuse("cache_move: from and to are host arrays");
    const int64_t capacity = (int64_t)cache->pages * cache->block;
    for (int i = 0; i < n; i++)
      if (from[i] < 0 || from[i] >= capacity || to[i] < 0 || to[i] >= capacity)
        return refuse("cache_move: row " + str(i) + " goes from slot " + str(from[i]) + " to slot " + str(to[i]) +
                      " of a pool of " + str(capacity));
    std::vector<int32_t> src, dst;
    std::vector<CacheMoveBatch> batches;
    if ((rc = order_moves(from, to, n, src, dst, batches))) return rc;
    if (!c) return no_ctx("cache_move");
    OnDevice on(c->device);
    if ((rc = no_capture(c, "cache_move"))) return rc;
    if (batches.empty()) return 0;
    CacheMoveArgs a{};
    a.c = layer_of(cache, 0);
    a.layers = cache->layers;
    a.batches = (int)batches.size();
    a.layer_rows = layer_rows(cache);
    CacheMoveFew few;
    few.n = 0;
    if (src.size() <= (size_t)kCacheMoveFew && batches.size() <= (size_t)kCacheMoveFewBatches) {
      std::copy(batches.begin(), batches.end(), few.batch);
      few.n = (int32_t)src.size();
      std::copy(src.begin(), src.end(), few.src);
      std::copy(dst.begin(), dst.end(), few.dst);
    } else {
      Stager sg;
      const size_t o0 = sg.add(src.data(), src.size() * 4), o1 = sg.add(dst.data(), dst.size() * 4);
      const size_t o2 = sg.add(batches.data(), batches.size() * sizeof(CacheMoveBatch));
      if ((rc = sg.upload(c))) return rc;
      a.src = sg.dev<int32_t>(c, o0);
      a.dst = sg.dev<int32_t>(c, o1);
      a.batch = sg.dev<CacheMoveBatch>(c, o2);
    }
    launch_cache_move(a, few, c->stream);
    TGOHIP_HIP(hipGetLastError());
    return 0;
  });
}

int tgohip_cache_plan(tgohip_ctx* c, const tgohip_cache* cache, int B, const int32_t* extents, const int32_t* lengths,
                      const uint32_t* pages, int max_pages, const int32_t* parents, int H, int q_dtype, int* handle) {
  return guarded([&]() -> int {
    int rc = check_geometry("cache_plan", cache);
    if (rc) return rc;
    const auto bad = [](const std::string& m) { return refuse("cache_plan: " + m); };
    if (B < 0) return bad(str(B) + " sequences");
    if (B && (!extents || !lengths || !pages)) return bad("extents, lengths and pages are host arrays");
    if (max_pages < 0 || (int64_t)B * max_pages > INT_MAX) return bad(str(max_pages) + " pages a sequence");
    const int Hkv = cache->kv_heads;
    if (H <= 0 || H > 65536 || H % Hkv)
      return bad(str(H) + " query heads over " + str(Hkv) + " kv heads; each kv head serves the same number, H at most 65536");
    if (bad_type(q_dtype)) return bad("q_dtype is " + str(q_dtype) + "; queries are f32 or f16");
    int64_t tq = 0, blocks = 0;
    for (int b = 0; b < B; b++) {
      const auto seq = [b](const std::string& m) { return refuse("cache_plan: sequence " + str(b) + m); };
      if (extents[b] < 0 || lengths[b] < extents[b])
        return seq(" has " + str(extents[b]) + " new tokens of " + str(lengths[b]) + " positions");
      if (lengths[b] > (int64_t)max_pages * cache->block || lengths[b] > INT_MAX - 256)
        return seq(" has " + str(lengths[b]) + " positions and " + str(max_pages) + " pages of " + str(cache->block));
      for (int64_t p = 0; extents[b] && p * cache->block < lengths[b]; p++)
        if (pages[(int64_t)b * max_pages + p] >= (uint32_t)cache->pages)
          return seq(": page " + str(p) + " is " + str(pages[(int64_t)b * max_pages + p]) + " of a pool of " + str(cache->pages));
      tq += extents[b];
      blocks += ((int64_t)extents[b] * (H / Hkv) + 15) / 16 * Hkv;
    }
    if (tq * H >= (int64_t)1 << 30) return bad(str(tq) + " new tokens of " + str(H) + " heads; heads of rows stay below 2^30");
    if (blocks > INT_MAX / 256) return bad("the batch needs " + str(blocks) + " workgroups, more than one launch takes");
    std::vector<uint64_t> masks;
    std::vector<uint8_t> tree;
    if (parents) {
      tree.assign((size_t)B, 0);
      int64_t at = 0;
      for (int b = 0; b < B; at += extents[b++]) {
        for (int i = 0; i < extents[b]; i++) {
          const int p = parents[at + i];
          if (p < -1 || p >= i)
            return bad("sequence " + str(b) + ": token " + str(i) + " has parent " + str(p) +
                       "; an earlier token of its sequence, or -1");
          tree[b] |= p != i - 1;
        }
        if (tree[b] && extents[b] > kCacheMaxTree)
          return bad("sequence " + str(b) + ": a tree of " + str(extents[b]) + " tokens; up to " + str(kCacheMaxTree));
      }
      masks.assign((size_t)tq, 0);
      at = 0;
      for (int b = 0; b < B; at += extents[b++])
        for (int i = 0; tree[b] && i < extents[b]; i++) {
          const int p = parents[at + i];
          masks[at + i] = (p < 0 ? 0 : masks[at + p]) | 1ull << i;
        }
    }
    if (!c) return no_ctx("cache_plan");
    if (!handle) return bad("handle is missing");
    if (*handle && !find(c->ops.caches, *handle, "cache_plan")) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if ((rc = no_capture(c, "cache_plan"))) return rc;
    CachePlan plan;
    cache_build_plan(B, extents, lengths, parents ? tree.data() : nullptr, H, Hkv, cache->head_dim,
                     q_dtype == TGOHIP_F16, c->ncu, plan);
    if (plan.part_rows > INT_MAX) return bad("the batch has more rows of partial results than 2^31 - 1");
    if (std::max(plan.items.size(), plan.merges.size()) > (size_t)INT_MAX / 256)
      return bad("the batch needs more workgroups than one launch takes");
    const bool fresh = *handle == 0;
    const int h = fresh ? c->ops.next++ : *handle;
    CacheHandle& p = c->ops.caches[h];
    p.D = 0;
    Stager sg;
    sg.add(plan.items.data(), plan.items.size() * sizeof(CacheItem));
    p.merges_off = sg.add(plan.merges.data(), plan.merges.size() * sizeof(PackedMerge));
    // the kernels' table: the row, in a layer, of a page's first position of head 0
    std::vector<uint32_t> rows(pages, pages + (size_t)B * max_pages);
    for (uint32_t& x : rows) x *= (uint32_t)(Hkv * cache->block);
    p.pages_off = sg.add(rows.data(), rows.size() * sizeof(uint32_t));
    p.masks_off = sg.add(masks.data(), masks.size() * sizeof(uint64_t));
    if (plan.part_rows) rc = p.part.ensure((size_t)plan.part_rows * (cache->head_dim + 4) * sizeof(float));
    if (!rc) rc = sg.upload(c, p.meta);
    if (rc) {
      if (fresh) {
        p.meta.release();
        p.part.release();
        c->ops.caches.erase(h);
      }
      return rc;
    }
    p.items = (int)plan.items.size();
    p.nmerges = (int)plan.merges.size();
    p.max_pages = max_pages;
    p.q_f16 = q_dtype == TGOHIP_F16;
    p.pages = cache->pages;
    p.Hkv = Hkv;
    p.block = cache->block;
    p.D = cache->head_dim;
    plan.items.clear();
    plan.merges.clear();
    p.plan = plan;
    *handle = h;
    return 0;
  });
}

int tgohip_cache_plan_free(tgohip_ctx* c, int handle) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("cache_plan_free");
    CacheHandle* p = find(c->ops.caches, handle, "cache_plan_free");
    if (!p) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "cache_plan_free")) return rc;
    TGOHIP_HIP(hipStreamSynchronize(c->stream));
    p->meta.release();
    p->part.release();
    c->ops.caches.erase(handle);
    return 0;
  });
}

int tgohip_cache_attention(tgohip_ctx* c, int handle, const tgohip_cache* cache, int layer, const void* q, int64_t q_row,
                           float scale, void* out, int64_t out_row, int out_dtype) {
  return guarded([&]() -> int {
    int rc = check_cache("cache_attention", cache, layer);
    if (rc) return rc;
    const auto bad = [](const std::string& m) { return refuse("cache_attention: " + m); };
    // a key's scale times it, and log2 of a value's over that, stay in f32's range
    if (!(scale >= 0x1p-64f && scale <= 0x1p32f)) return bad("scale is " + num(scale) + "; at least 2^-64 and at most 2^32");
    if (out_dtype != TGOHIP_F32 && out_dtype != TGOHIP_F16 && out_dtype != TGOHIP_F16X2)
      return bad("out_dtype is " + str(out_dtype) + "; f32, f16 or a pair");
    if (!c) return no_ctx("cache_attention");
    CacheHandle* p = find(c->ops.caches, handle, "cache_attention");
    if (!p) return TGOHIP_EINVAL;
    if (!p->D) return fail(TGOHIP_ESTATE, "cache_attention: the plan was not made again after a failure");
    if (p->pages != cache->pages || p->Hkv != cache->kv_heads || p->block != cache->block || p->D != cache->head_dim)
      return bad("the plan is of " + str(p->pages) + " pages of " + str(p->block) + " positions, " + str(p->Hkv) +
                 " kv heads of " + str(p->D) + "; the cache has " + str(cache->pages) + " of " + str(cache->block) + ", " +
                 str(cache->kv_heads) + " of " + str(cache->head_dim));
    const CachePlan& pl = p->plan;
    if (pl.tq == 0) return 0;
    if (!q || !out) return bad("q and out are device buffers");
    const int64_t w = (int64_t)pl.H * p->D, top = (int64_t)1 << 30, qb = elt(p->q_f16);
    const int64_t ob = out_dtype == TGOHIP_F32 ? 4 : 2, planes = out_dtype == TGOHIP_F16X2 ? 2 : 1;
    if (pl.tq > 1 && (q_row < w || q_row > top || out_row < w || out_row > top))
      return bad("rows are " + str(q_row) + " and " + str(out_row) + " elements apart and hold " + str(w) +
                 "; at most 2^30 apart");
    if (misaligned(q) || misaligned(out) || (pl.tq > 1 && (q_row * qb % 16 || out_row * ob % 16)))
      return bad("rows of q and out start on 16-byte boundaries");
    if (planes == 2 && pl.tq > 1 && out_row != w)
      return bad("a pair's rows are dense (out_row " + str(out_row) + ", not " + str(w) + ")");
    const Span sq{(const char*)q, pl.tq, 1, q_row * qb, 0, w * qb};
    const Span so{(const char*)out, planes * pl.tq, 1, (pl.tq > 1 ? out_row : w) * ob, 0, w * ob};
    if (meet(so, sq)) return bad("out meets q in memory");
    if ((rc = check_apart("cache_attention", cache, so, "out"))) return rc;
    CacheAttnArgs a{};
    a.c = layer_of(cache, layer);
    a.q = q;
    a.out = out;
    const char* meta = (const char*)p->meta.p;
    a.items = (const CacheItem*)meta;
    a.merges = (const PackedMerge*)(meta + p->merges_off);
    a.pages = (const uint32_t*)(meta + p->pages_off);
    a.masks = (const uint64_t*)(meta + p->masks_off);
    a.part_o = (float*)p->part.p;
    a.part_ml = (float*)p->part.p + (size_t)pl.part_rows * p->D;
    a.q_row = q_row;
    a.out_row = out_row;
    a.out_lo = pl.tq * w;
    a.max_pages = p->max_pages;
    a.G = pl.H / p->Hkv;
    a.out_form = out_dtype == TGOHIP_F32 ? OUT_F32 : out_dtype == TGOHIP_F16 ? OUT_F16 : OUT_X2;
    a.q_f16 = p->q_f16;
    a.nitems = p->items;
    a.wide = pl.wide;
    a.nmerges = p->nmerges;
    a.qscale = scale * 1.4426950408889634f;
    OnDevice on(c->device);
    return cache_attention_enqueue(a, c->stream);
  });
}

}  // extern "C"
