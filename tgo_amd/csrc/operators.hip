// operators.hip -- C ABI of the op-level operators beside the projections and
// paged attention: rotary positions, packed attention, the adapters of many
// requests. A program makes their handles once (per model, per batch) and each
// call then only launches kernels on the context's stream.
#include "runtime.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

namespace tgohip {

void OpHandles::release() {
  for (auto& r : ropes) r.second.inv_freq.release();
  for (auto& p : packed) {
    p.second.meta.release();
    p.second.part.release();
  }
  for (auto& s : sets) {
    for (AdapterEntry& e : s.second.table) (void)hipFree((void*)e.down);
    s.second.table_dev.release();
  }
  for (auto& r : rows) {
    r.second.meta.release();
    r.second.u.release();
  }
  ropes.clear();
  packed.clear();
  sets.clear();
  rows.clear();
}

}  // namespace tgohip

namespace {

// Entry points do not throw across the C ABI, and a refused call leaves no error behind
// that the next launch would report as its own.
template <typename F>
int guarded(F f) {
  try {
    const int rc = f();
    if (rc) (void)hipGetLastError();
    return rc;
  } catch (const std::bad_alloc&) {
    return fail(TGOHIP_ENOMEM, "host allocation failed");
  } catch (const std::exception& e) {
    return fail(TGOHIP_EDEVICE, std::string("internal: ") + e.what());
  }
}

// Makes the context's device current for a call, and the caller's again after it.
struct OnDevice {
  int prev = -1;
  bool moved = false;
  explicit OnDevice(int device) {
    if (hipGetDevice(&prev) == hipSuccess && prev != device) moved = hipSetDevice(device) == hipSuccess;
  }
  ~OnDevice() {
    if (moved) (void)hipSetDevice(prev);
  }
};

int refuse(const std::string& why) { return fail(TGOHIP_EINVAL, why); }
int no_ctx(const char* what) { return refuse(std::string(what) + ": the context is missing"); }

// Making, changing or freeing a handle copies, allocates and waits, which a graph
// cannot hold.
int no_capture(tgohip_ctx* c, const char* what) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  const hipError_t e = hipStreamIsCapturing(c->stream, &st);
  if (e != hipSuccess) return fail(TGOHIP_EDEVICE, hip_message(e, what));
  if (st == hipStreamCaptureStatusNone) return 0;
  return fail(TGOHIP_ESTATE, std::string(what) + ": the context's stream is being captured");
}

template <typename T>
T* find(std::map<int, T>& m, int handle, const char* what) {
  auto it = m.find(handle);
  if (it != m.end()) return &it->second;
  refuse(std::string(what) + ": no handle " + std::to_string(handle));
  return nullptr;
}

bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
int64_t elt(int f16) { return f16 ? 2 : 4; }

// A device operand: `rows` rows of `heads` heads of d elements, strides in bytes.
struct Span {
  const char* p;
  int64_t rows, heads, row, head, d;
  int64_t width() const { return (heads - 1) * head + d; }  // of one row
  int64_t end() const { return rows ? (rows - 1) * row + width() : 0; }
};
// Whether two operands may share memory: apart, or columns of the same rows that
// do not meet.
bool meet(const Span& a, const Span& b) {
  if (!a.rows || !b.rows) return false;
  if (a.p + a.end() <= b.p || b.p + b.end() <= a.p) return false;
  if (a.row == b.row && a.row > 0 && a.width() <= a.row && b.width() <= a.row) {
    int64_t off = (b.p - a.p) % a.row;
    if (off < 0) off += a.row;
    if (off >= a.width() && off + b.width() <= a.row) return false;
  }
  return true;
}
bool same(const Span& a, const Span& b) {
  return a.p == b.p && a.d == b.d && (a.rows <= 1 || a.row == b.row) && (a.heads <= 1 || a.head == b.head);
}

// Rounds to the nearest f16 (ties to even), subnormal ones included: an adapter's
// values sit near the bottom of f16's range, where the loader's rule
// (tgohip_to_f16) flushes to 0. Both ranges are computed and one is taken, so that
// the loop vectorises (a conversion by the compiler's function takes 5 ns a value).
// False if a finite value is past f16's range.
bool to_half(const float* src, uint16_t* dst, size_t n) {
  uint32_t past = 0;
  for (size_t i = 0; i < n; i++) {
    uint32_t w;
    memcpy(&w, src + i, 4);
    const uint32_t mag = w & 0x7fffffffu;
    float f;
    memcpy(&f, &mag, 4);
    f += 0.5f;  // of 2^-24 an ulp, f16's subnormal step
    uint32_t small;
    memcpy(&small, &f, 4);
    small -= 0x3f000000u;
    const uint32_t normal = (mag + 0xfffu + ((mag >> 13) & 1) - (112u << 23)) >> 13;
    uint32_t h = mag < (113u << 23) ? small : normal;
    const uint32_t over = mag < 0x7f800000u && mag >= 0x477ff000u;  // 65520 rounds to 2^16
    past |= over;
    h = mag >= 0x7f800000u ? (mag > 0x7f800000u ? 0x7e00u : 0x7c00u) : h;
    dst[i] = (uint16_t)(h | ((w >> 16) & 0x8000u));
  }
  return !past;
}

std::string num(double v) {
  char b[64];
  snprintf(b, sizeof b, "%g", v);
  return b;
}

int check_rope(const tgohip_rope_cfg* c) {
  if (!c) return refuse("rope: the configuration is missing");
  if (c->head_dim < 2 || c->head_dim > kRopeMaxHeadDim || c->head_dim % 2)
    return refuse("rope: head_dim is " + std::to_string(c->head_dim) + "; an even number from 2 to " +
                  std::to_string(kRopeMaxHeadDim));
  if (c->rotary_dim < 2 || c->rotary_dim > c->head_dim || c->rotary_dim % 2)
    return refuse("rope: rotary_dim is " + std::to_string(c->rotary_dim) + " of head_dim " +
                  std::to_string(c->head_dim) + "; an even number from 2 to head_dim");
  if (c->layout != TGOHIP_ROPE_INTERLEAVED && c->layout != TGOHIP_ROPE_HALF)
    return refuse("rope: layout is " + std::to_string(c->layout) + ", neither interleaved nor half");
  if (c->scaling < TGOHIP_ROPE_UNSCALED || c->scaling > TGOHIP_ROPE_BANDS)
    return refuse("rope: scaling is " + std::to_string(c->scaling) + ", not a TGOHIP_ROPE_* kind");
  if (!(c->base > 1.0) || !std::isfinite(c->base))
    return refuse("rope: base is " + num(c->base) + "; a finite number above 1");
  if (!(c->attention >= 0.0) || !std::isfinite((float)c->attention))
    return refuse("rope: attention is " + num(c->attention) + "; a finite factor of f32, 0 for the scaling's own");
  if (c->scaling == TGOHIP_ROPE_UNSCALED) return 0;
  if (!(c->factor >= 1.0) || !std::isfinite(c->factor))
    return refuse("rope: factor is " + num(c->factor) + "; a finite number of at least 1");
  if (c->scaling == TGOHIP_ROPE_LINEAR) return 0;
  if (!(c->original > 0.0) || !std::isfinite(c->original))
    return refuse("rope: original is " + num(c->original) + "; the positions trained on, above 0");
  if (!(c->slow > 0.0) || !(c->fast > c->slow) || !std::isfinite(c->fast))
    return refuse("rope: fast is " + num(c->fast) + " and slow " + num(c->slow) +
                  " turns over the original positions; fast is above slow and slow above 0");
  return 0;
}

void rope_freqs(const tgohip_rope_cfg& c, double* w, double* attention) {
  const int rd = c.rotary_dim, pairs = rd / 2;
  const double turn = 2.0 * M_PI;
  double lo = 0, hi = 0;
  if (c.scaling == TGOHIP_ROPE_YARN) {
    auto edge = [&](double turns) { return rd * std::log(c.original / (turns * turn)) / (2.0 * std::log(c.base)); };
    lo = std::max(std::floor(edge(c.fast)), 0.0);
    hi = std::min(std::ceil(edge(c.slow)), (double)(rd - 1));
  }
  for (int i = 0; i < pairs; i++) {
    double f = std::pow(c.base, -2.0 * i / rd), kept = 1.0;
    if (c.scaling == TGOHIP_ROPE_LINEAR) kept = 0.0;
    if (c.scaling == TGOHIP_ROPE_YARN) kept = 1.0 - std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 1e-3)));
    if (c.scaling == TGOHIP_ROPE_BANDS)
      kept = std::min(1.0, std::max(0.0, (c.original * f / turn - c.slow) / (c.fast - c.slow)));
    w[i] = c.scaling == TGOHIP_ROPE_UNSCALED ? f : f * kept + f / c.factor * (1.0 - kept);
  }
  *attention = c.attention != 0.0                    ? c.attention
               : c.scaling == TGOHIP_ROPE_YARN ? 0.1 * std::log(c.factor) + 1.0
                                                     : 1.0;
}

// Packed rows and head counts stay below this, so that every index fits 32 bits.
constexpr int64_t kMaxIndex = (int64_t)1 << 30;

// Items and merges are one launch each, of at most 256 threads a workgroup.
int packed_fits(int64_t items, int64_t merges) {
  const int64_t most = INT_MAX / 256, n = std::max(items, merges);
  if (n <= most) return 0;
  return refuse("packed_plan: the batch needs " + std::to_string(n) + " workgroups, more than one launch takes");
}

int check_packed(int B, const int32_t* nq, const int32_t* nk, int H, int Hkv, int D, int q_dtype) {
  if (B < 0) return refuse("packed_plan: " + std::to_string(B) + " sequences");
  if (B > 0 && (!nq || !nk)) return refuse("packed_plan: q_lengths and kv_lengths are host arrays");
  if (D != 64 && D != 128)
    return refuse("packed_plan: head_dim is " + std::to_string(D) + "; the kernels are built for 64 and 128");
  if (H <= 0 || Hkv <= 0 || H % Hkv != 0)
    return refuse("packed_plan: " + std::to_string(H) + " query heads over " + std::to_string(Hkv) +
                  " kv heads; each kv head serves the same number of query heads");
  if (H > 65536) return refuse("packed_plan: " + std::to_string(H) + " query heads; at most 65536");
  if (q_dtype != TGOHIP_F32 && q_dtype != TGOHIP_F16)
    return refuse("packed_plan: q_dtype is " + std::to_string(q_dtype) + "; queries are f32 or f16");
  int64_t tq = 0, tk = 0, blocks = 0;
  for (int s = 0; s < B; s++) {
    if (nq[s] < 0 || nk[s] < 0)
      return refuse("packed_plan: sequence " + std::to_string(s) + " has " + std::to_string(nq[s]) +
                    " queries and " + std::to_string(nk[s]) + " keys");
    tq += nq[s];
    tk += nk[s];
    blocks += ((int64_t)nq[s] * (H / Hkv) + kPackRows - 1) / kPackRows * Hkv;
  }
  if (tq * H >= kMaxIndex || tk >= kMaxIndex)
    return refuse("packed_plan: " + std::to_string(tq) + " query rows of " + std::to_string(H) +
                  " heads and " + std::to_string(tk) + " key rows; heads of rows, and key rows, stay below 2^30");
  return packed_fits(blocks, blocks);
}

// A checked batch's decomposition on `ncu` compute units.
int packed_decompose(int B, const int32_t* nq, const int32_t* nk, int H, int Hkv, int D, int causal, int q_dtype, int ncu,
                     PackedPlan& plan) {
  packed_build_plan(B, nq, nk, H, Hkv, D, causal != 0, q_dtype == TGOHIP_F16, ncu, plan);
  if (plan.part_rows > INT_MAX) return refuse("packed_plan: the batch has more rows of partial results than 2^31 - 1");
  return packed_fits((int64_t)(plan.items.size() + plan.few.size()), (int64_t)plan.merges.size());
}

}  // namespace

extern "C" {

// ---- rotary positions ---------------------------------------------------------

int tgohip_rope_freqs(const tgohip_rope_cfg* cfg, double* inv_freq, double* attention) {
  return guarded([&]() -> int {
    const int rc = check_rope(cfg);
    if (rc) return rc;
    if (!inv_freq || !attention) return refuse("rope_freqs: inv_freq and attention are host buffers");
    rope_freqs(*cfg, inv_freq, attention);
    return 0;
  });
}

int tgohip_rope_new(tgohip_ctx* c, const tgohip_rope_cfg* cfg, int* handle) {
  return guarded([&]() -> int {
    int rc = check_rope(cfg);
    if (rc) return rc;
    if (!c) return no_ctx("rope_new");
    if (!handle) return refuse("rope_new: handle is missing");
    OnDevice on(c->device);
    if ((rc = no_capture(c, "rope_new"))) return rc;
    double w[kRopeMaxHeadDim / 2], attention;
    rope_freqs(*cfg, w, &attention);
    for (int i = 0; i < cfg->rotary_dim / 2; i++) w[i] /= 2.0 * M_PI;
    RopeTable t;
    t.d = cfg->head_dim;
    t.rd = cfg->rotary_dim;
    t.half = cfg->layout == TGOHIP_ROPE_HALF;
    t.attention = (float)attention;
    Stager sg;
    sg.add(w, (size_t)t.rd / 2 * sizeof(double));
    if ((rc = sg.upload(c, t.inv_freq))) {
      t.inv_freq.release();
      return rc;
    }
    const int h = c->ops.next++;
    c->ops.ropes[h] = t;
    *handle = h;
    return 0;
  });
}

int tgohip_rope_free(tgohip_ctx* c, int handle) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("rope_free");
    RopeTable* t = find(c->ops.ropes, handle, "rope_free");
    if (!t) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "rope_free")) return rc;
    TGOHIP_HIP(hipStreamSynchronize(c->stream));
    t->inv_freq.release();
    c->ops.ropes.erase(handle);
    return 0;
  });
}

int tgohip_rope(tgohip_ctx* c, int handle, const int32_t* positions, int T, const tgohip_rope_heads* heads, int n) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("rope");
    RopeTable* t = find(c->ops.ropes, handle, "rope");
    if (!t) return TGOHIP_EINVAL;
    if (T < 0 || T >= 1 << 24) return refuse("rope: " + std::to_string(T) + " rows; 0 to 2^24 - 1");
    if (n < 1 || n > kRopeGroups || !heads)
      return refuse("rope: " + std::to_string(n) + " tensors of heads; 1 to " + std::to_string(kRopeGroups));
    if (T == 0) return 0;
    if (!positions || (uintptr_t)positions % 4) return refuse("rope: positions is a device buffer of int32");
    const Span at{(const char*)positions, 1, 1, 0, 0, (int64_t)T * 4};
    RopeArgs a{};
    Span xs[kRopeGroups], ys[kRopeGroups];
    for (int i = 0; i < n; i++) {
      const tgohip_rope_heads& g = heads[i];
      auto bad = [i](const std::string& m) { return refuse("rope: tensor " + std::to_string(i) + ": " + m); };
      if (!g.x || !g.y) return bad("x and y are device buffers");
      if (g.heads < 1 || g.heads > 65536) return bad(std::to_string(g.heads) + " heads; 1 to 65536");
      if ((g.x_dtype != TGOHIP_F32 && g.x_dtype != TGOHIP_F16) || (g.y_dtype != TGOHIP_F32 && g.y_dtype != TGOHIP_F16))
        return bad("x_dtype and y_dtype are f32 or f16");
      const int xf = g.x_dtype == TGOHIP_F16, yf = g.y_dtype == TGOHIP_F16;
      if (((uintptr_t)g.x & (elt(xf) - 1)) || ((uintptr_t)g.y & (elt(yf) - 1)))
        return bad("x or y is not aligned to its type");
      const int64_t top = (int64_t)1 << 36;  // beyond any tensor; the products below stay in 64 bits
      if (g.x_row < 0 || g.x_head < 0 || g.x_row > top || g.x_head > top || g.y_row > top || g.y_head > top)
        return bad("strides are not negative, and at most 2^36 elements");
      // no two heads of y share an element
      int64_t s0 = g.y_row, n0 = T, s1 = g.y_head, n1 = g.heads;
      if (n0 == 1) s0 = 0;
      if (n1 == 1) s1 = 0;
      if (s0 > s1) {
        std::swap(s0, s1);
        std::swap(n0, n1);
      }
      int64_t need = t->d;
      if (n0 > 1) {
        if (s0 < need)
          return bad("heads of y overlap (strides " + std::to_string(g.y_row) + ", " + std::to_string(g.y_head) + ")");
        need = (n0 - 1) * s0 + t->d;
      }
      if (n1 > 1 && s1 < need)
        return bad("heads of y overlap (strides " + std::to_string(g.y_row) + ", " + std::to_string(g.y_head) + ")");
      xs[i] = Span{(const char*)g.x, T, g.heads, g.x_row * elt(xf), g.x_head * elt(xf), t->d * elt(xf)};
      ys[i] = Span{(const char*)g.y, T, g.heads, g.y_row * elt(yf), g.y_head * elt(yf), t->d * elt(yf)};
      a.g[i] = RopeGroup{g.x, g.y, g.x_row, g.x_head, g.y_row, g.y_head, g.heads, xf, yf, g.rotate != 0, 0};
    }
    for (int i = 0; i < n; i++) {
      if (meet(ys[i], at))
        return refuse("rope: y of tensor " + std::to_string(i) + " meets positions in memory");
      for (int j = 0; j < n; j++) {
        if (meet(ys[i], xs[j]) && !(i == j && a.g[i].x_f16 == a.g[i].y_f16 && same(ys[i], xs[i])))
          return refuse("rope: y of tensor " + std::to_string(i) + " meets x of tensor " + std::to_string(j) +
                        " in memory; y is its own x (same type and strides) or apart");
        if (i < j && meet(ys[i], ys[j]))
          return refuse("rope: y of tensors " + std::to_string(i) + " and " + std::to_string(j) + " meet in memory");
      }
    }
    a.positions = positions;
    a.inv_freq = (const double*)t->inv_freq.p;
    a.attention = t->attention;
    a.T = T;
    a.d = t->d;
    a.rd = t->rd;
    a.half = t->half;
    a.n = n;
    OnDevice on(c->device);
    launch_rope(a, c->ncu, c->stream);
    TGOHIP_HIP(hipGetLastError());
    return 0;
  });
}

// ---- packed attention -----------------------------------------------------------

int tgohip_packed_plan(tgohip_ctx* c, int B, const int32_t* q_lengths, const int32_t* kv_lengths, int H, int H_kv,
                       int head_dim, int causal, int q_dtype, int* handle) {
  return guarded([&]() -> int {
    int rc = check_packed(B, q_lengths, kv_lengths, H, H_kv, head_dim, q_dtype);
    if (rc) return rc;
    if (!c) return no_ctx("packed_plan");
    if (!handle) return refuse("packed_plan: handle is missing");
    if (*handle && !find(c->ops.packed, *handle, "packed_plan")) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if ((rc = no_capture(c, "packed_plan"))) return rc;
    PackedPlan plan;
    if ((rc = packed_decompose(B, q_lengths, kv_lengths, H, H_kv, head_dim, causal, q_dtype, c->ncu, plan))) return rc;
    const size_t items = plan.items.size();
    plan.items.insert(plan.items.end(), plan.few.begin(), plan.few.end());
    const bool fresh = *handle == 0;
    const int h = fresh ? c->ops.next++ : *handle;
    PackedHandle& p = c->ops.packed[h];
    p.n = PackedCounts{};
    p.plan = PackedPlan();
    Stager sg;
    sg.add(plan.items.data(), plan.items.size() * sizeof(PackedItem));
    const size_t off = sg.add(plan.merges.data(), plan.merges.size() * sizeof(PackedMerge));
    if (plan.part_rows) rc = p.part.ensure((size_t)plan.part_rows * (head_dim + 4) * sizeof(float));
    if (!rc) rc = sg.upload(c, p.meta);
    if (rc) {
      if (fresh) {
        p.meta.release();
        p.part.release();
        c->ops.packed.erase(h);
      }
      return rc;
    }
    p.n = PackedCounts{(int)items, (int)plan.few.size(), (int)plan.merges.size()};
    p.merges_off = off;
    plan.items.clear();
    plan.few.clear();
    plan.merges.clear();
    p.plan = plan;
    *handle = h;
    return 0;
  });
}

int tgohip_packed_describe(int B, const int32_t* q_lengths, const int32_t* kv_lengths, int H, int H_kv, int head_dim,
                           int causal, int q_dtype, int ncu, tgohip_packed_plan_t* out) {
  return guarded([&]() -> int {
    int rc = check_packed(B, q_lengths, kv_lengths, H, H_kv, head_dim, q_dtype);
    if (rc) return rc;
    if (ncu < 1 || ncu > 65536 || !out) return refuse("packed_describe: ncu (1 to 65536) and plan");
    PackedPlan plan;
    if ((rc = packed_decompose(B, q_lengths, kv_lengths, H, H_kv, head_dim, causal, q_dtype, ncu, plan))) return rc;
    *out = tgohip_packed_plan_t{(int32_t)plan.items.size(), (int32_t)plan.few.size(), 0, 0, plan.part_rows, 0};
    for (const PackedItem& it : plan.items) out->longest_tile = std::max(out->longest_tile, it.kv_hi - it.kv_lo);
    for (const PackedItem& it : plan.few) out->longest_few = std::max(out->longest_few, it.kv_hi - it.kv_lo);
    for (const PackedMerge& m : plan.merges) out->merged_rows += m.nr;
    return 0;
  });
}

int tgohip_packed_pieces(int B, const int32_t* q_lengths, const int32_t* kv_lengths, int H, int H_kv, int head_dim,
                         int causal, int q_dtype, int ncu, tgohip_packed_piece_t* pieces, int* n_pieces,
                         tgohip_packed_merge_t* merges, int* n_merges) {
  return guarded([&]() -> int {
    int rc = check_packed(B, q_lengths, kv_lengths, H, H_kv, head_dim, q_dtype);
    if (rc) return rc;
    if (ncu < 1 || ncu > 65536 || !n_pieces || !n_merges)
      return refuse("packed_pieces: ncu (1 to 65536), n_pieces and n_merges");
    PackedPlan plan;
    if ((rc = packed_decompose(B, q_lengths, kv_lengths, H, H_kv, head_dim, causal, q_dtype, ncu, plan))) return rc;
    plan.items.insert(plan.items.end(), plan.few.begin(), plan.few.end());
    const int np = (int)plan.items.size(), nm = (int)plan.merges.size(), mp = *n_pieces, mm = *n_merges;
    *n_pieces = np;
    *n_merges = nm;
    if (mp == 0 && mm == 0) return 0;
    if (mp < np || mm < nm || (np && !pieces) || (nm && !merges))
      return refuse("packed_pieces: the arrays hold " + std::to_string(mp) + " pieces and " + std::to_string(mm) +
                    " merges; the batch has " + std::to_string(np) + " and " + std::to_string(nm));
    for (int i = 0; i < np; i++) {
      const PackedItem& it = plan.items[i];
      pieces[i] = tgohip_packed_piece_t{it.q0, it.k0, it.kvh, it.r0, it.nr, it.kv_lo, it.kv_hi, it.shift, it.part};
    }
    for (int i = 0; i < nm; i++) {
      const PackedMerge& m = plan.merges[i];
      merges[i] = tgohip_packed_merge_t{m.q0, m.kvh, m.r0, m.nr, m.part, m.parts, m.step};
    }
    return 0;
  });
}

int tgohip_packed_free(tgohip_ctx* c, int handle) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("packed_free");
    PackedHandle* p = find(c->ops.packed, handle, "packed_free");
    if (!p) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "packed_free")) return rc;
    TGOHIP_HIP(hipStreamSynchronize(c->stream));
    p->meta.release();
    p->part.release();
    c->ops.packed.erase(handle);
    return 0;
  });
}

int tgohip_packed_attention(tgohip_ctx* c, int handle, const void* q, int64_t q_row, const void* k, int64_t k_row,
                            const void* v, int64_t v_row, float scale, void* out, int64_t out_row, int out_dtype) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("packed_attention");
    PackedHandle* p = find(c->ops.packed, handle, "packed_attention");
    if (!p) return TGOHIP_EINVAL;
    const PackedPlan& pl = p->plan;
    if (!pl.D) return fail(TGOHIP_ESTATE, "packed_attention: the plan was not made again after a failure");
    if (!(scale > 0.f) || scale > 0x1p32f)  // scores stay below 2^72, and above kPackNoMax
      return refuse("packed_attention: scale is " + num(scale) + "; a number above 0, at most 2^32");
    if (out_dtype != TGOHIP_F32 && out_dtype != TGOHIP_F16 && out_dtype != TGOHIP_F16X2)
      return refuse("packed_attention: out_dtype is " + std::to_string(out_dtype) + "; f32, f16 or a pair");
    if (pl.tq == 0) return 0;
    if (!q || !out) return refuse("packed_attention: q and out are device buffers");
    if (pl.tk && (!k || !v)) return refuse("packed_attention: k and v are device buffers");
    const int64_t qw = (int64_t)pl.H * pl.D, kw = (int64_t)pl.Hkv * pl.D, top = (int64_t)1 << 30;
    struct {
      const char* name;
      const void* p;
      int64_t row, width, rows, unit, most;
    } ops[] = {{"q", q, q_row, qw, pl.tq, pl.q_f16 ? 8 : 4, top},
               {"k", k, k_row, kw, pl.tk, 8, kPackMaxRow},
               {"v", v, v_row, kw, pl.tk, 8, kPackMaxRow},
               {"out", out, out_row, qw, pl.tq, out_dtype == TGOHIP_F32 ? 4 : 8, top}};
    for (auto& o : ops) {
      if (o.rows > 1 && (o.row < o.width || o.row > o.most))
        return refuse(std::string("packed_attention: ") + o.name + " rows are " + std::to_string(o.row) +
                      " elements apart and hold " + std::to_string(o.width) + "; at most " +
                      std::to_string(o.most) + " apart");
      if (misaligned(o.p) || (o.rows > 1 && o.row % o.unit))
        return refuse(std::string("packed_attention: ") + o.name + " rows start on 16-byte boundaries");
    }
    if (out_dtype == TGOHIP_F16X2 && pl.tq > 1 && out_row != qw)
      return refuse("packed_attention: a pair's rows are dense (out_row " + std::to_string(out_row) + ", not " +
                    std::to_string(qw) + ")");
    const int64_t ob = out_dtype == TGOHIP_F32 ? 4 : 2, planes = out_dtype == TGOHIP_F16X2 ? 2 : 1;
    const Span so{(const char*)out, planes * pl.tq, 1, (pl.tq > 1 ? out_row : qw) * ob, 0, qw * ob};
    const Span in[] = {{(const char*)q, pl.tq, 1, q_row * elt(pl.q_f16), 0, qw * elt(pl.q_f16)},
                       {(const char*)k, pl.tk, 1, k_row * 2, 0, kw * 2},
                       {(const char*)v, pl.tk, 1, v_row * 2, 0, kw * 2}};
    for (int i = 0; i < 3; i++)
      if (meet(so, in[i])) return refuse(std::string("packed_attention: out meets ") + ops[i].name + " in memory");
    PackedArgs a{};
    a.q = q;
    a.k = (const half_t*)k;
    a.v = (const half_t*)v;
    a.out = out;
    a.part_o = (float*)p->part.p;
    a.part_ml = (float*)p->part.p + (size_t)pl.part_rows * pl.D;
    a.items = (const PackedItem*)p->meta.p;
    a.merges = (const PackedMerge*)((const char*)p->meta.p + p->merges_off);
    a.q_row = q_row;
    a.k_row = k_row;
    a.v_row = v_row;
    a.out_row = out_row;
    a.out_lo = pl.tq * qw;
    a.G = pl.H / pl.Hkv;
    a.out_form = out_dtype == TGOHIP_F32 ? OUT_F32 : out_dtype == TGOHIP_F16 ? OUT_F16 : OUT_X2;
    a.qscale = scale * 1.4426950408889634f;
    OnDevice on(c->device);
    return packed_enqueue(a, pl.D, pl.q_f16, p->n, c->stream);
  });
}

// ---- adapters ---------------------------------------------------------------------

int tgohip_adapters_new(tgohip_ctx* c, int K, int N, int capacity, int* handle) {
  return guarded([&]() -> int {
    if (K <= 0 || N <= 0 || K % 64 != 0 || N % 32 != 0 || K > 1 << 22 || N > 1 << 22)
      return refuse("adapters_new: the projection is [" + std::to_string(K) + "," + std::to_string(N) +
                    "]; this library takes K a multiple of 64 and N a multiple of 32, up to 2^22");
    if (capacity < 1 || capacity > 65536)
      return refuse("adapters_new: capacity is " + std::to_string(capacity) + "; 1 to 65536 adapters");
    if (!c) return no_ctx("adapters_new");
    if (!handle) return refuse("adapters_new: handle is missing");
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "adapters_new")) return rc;
    AdapterSet s;
    s.K = K;
    s.N = N;
    s.table.assign((size_t)capacity, AdapterEntry{nullptr, nullptr, 0, 0.f});
    int rc = s.table_dev.ensure(s.table.size() * sizeof(AdapterEntry));
    if (!rc) {
      const hipError_t e = hipMemcpy(s.table_dev.p, s.table.data(), s.table.size() * sizeof(AdapterEntry),
                                     hipMemcpyHostToDevice);
      if (e != hipSuccess) rc = fail(TGOHIP_EDEVICE, hip_message(e, "adapter table"));
    }
    if (rc) {
      s.table_dev.release();
      return rc;
    }
    const int h = c->ops.next++;
    c->ops.sets[h] = s;
    *handle = h;
    return 0;
  });
}

// Puts entry e at index of the set and frees what was there, the context's stream drained first.
static int adapter_set(tgohip_ctx* c, AdapterSet* s, int index, const AdapterEntry& e) {
  TGOHIP_HIP(hipStreamSynchronize(c->stream));
  TGOHIP_HIP(hipMemcpy((AdapterEntry*)s->table_dev.p + index, &e, sizeof e, hipMemcpyHostToDevice));
  (void)hipFree((void*)s->table[index].down);
  s->table[index] = e;
  s->rank_pad = 0;
  for (const AdapterEntry& a : s->table) s->rank_pad = std::max(s->rank_pad, a.rank_pad);
  return 0;
}

int tgohip_adapters_put(tgohip_ctx* c, int handle, int index, int rank, int dtype, const void* down, const void* up,
                        float scale) {
  return guarded([&]() -> int {
    if (rank < 1 || rank > kAdapterMaxRank)
      return refuse("adapters_put: rank is " + std::to_string(rank) + "; 1 to " + std::to_string(kAdapterMaxRank));
    if (dtype != TGOHIP_F32 && dtype != TGOHIP_F16)
      return refuse("adapters_put: dtype is " + std::to_string(dtype) + "; host planes are f32 or f16");
    if (!down || !up) return refuse("adapters_put: down and up are host planes");
    if (!std::isfinite(scale)) return refuse("adapters_put: scale is " + num(scale) + ", not a finite number");
    if (!c) return no_ctx("adapters_put");
    AdapterSet* s = find(c->ops.sets, handle, "adapters_put");
    if (!s) return TGOHIP_EINVAL;
    if (index < 0 || index >= (int)s->table.size())
      return refuse("adapters_put: index " + std::to_string(index) + " of a set of " + std::to_string(s->table.size()));
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "adapters_put")) return rc;
    // down [rank][K] with rows of zeros, up [N][rank] with columns of zeros, to a
    // rank the kernels' products take whole; one allocation
    const int rp = rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128;
    const size_t nd = (size_t)rp * s->K, nu = (size_t)s->N * rp;
    std::vector<uint16_t> h(nd + nu, 0), tmp;
    const uint16_t *d16 = (const uint16_t*)down, *u16 = (const uint16_t*)up;
    if (dtype == TGOHIP_F32) {
      tmp.resize((size_t)rank * (s->K + (size_t)s->N));
      if (!to_half((const float*)down, tmp.data(), (size_t)rank * s->K) ||
          !to_half((const float*)up, tmp.data() + (size_t)rank * s->K, (size_t)rank * s->N))
        return refuse("adapters_put: a value is past f16's range (65504)");
      d16 = tmp.data();
      u16 = tmp.data() + (size_t)rank * s->K;
    }
    memcpy(h.data(), d16, (size_t)rank * s->K * 2);
    for (int n = 0; n < s->N; n++) memcpy(&h[nd + (size_t)n * rp], u16 + (size_t)n * rank, (size_t)rank * 2);
    void* dev = nullptr;
    hipError_t e = hipMalloc(&dev, h.size() * 2);
    if (e != hipSuccess)
      return fail(TGOHIP_ENOMEM,
                  "device allocation of " + std::to_string(h.size() * 2) + " bytes: " + hipGetErrorString(e));
    e = hipMemcpy(dev, h.data(), h.size() * 2, hipMemcpyHostToDevice);
    int rc = e == hipSuccess ? 0 : fail(TGOHIP_EDEVICE, hip_message(e, "adapter planes"));
    if (!rc) rc = adapter_set(c, s, index, AdapterEntry{(const half_t*)dev, (const half_t*)dev + nd, rp, scale});
    if (rc) (void)hipFree(dev);
    return rc;
  });
}

int tgohip_adapters_drop(tgohip_ctx* c, int handle, int index) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("adapters_drop");
    AdapterSet* s = find(c->ops.sets, handle, "adapters_drop");
    if (!s) return TGOHIP_EINVAL;
    if (index < 0 || index >= (int)s->table.size())
      return refuse("adapters_drop: index " + std::to_string(index) + " of a set of " +
                    std::to_string(s->table.size()));
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "adapters_drop")) return rc;
    return adapter_set(c, s, index, AdapterEntry{nullptr, nullptr, 0, 0.f});
  });
}

int tgohip_adapters_free(tgohip_ctx* c, int handle) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("adapters_free");
    AdapterSet* s = find(c->ops.sets, handle, "adapters_free");
    if (!s) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "adapters_free")) return rc;
    TGOHIP_HIP(hipStreamSynchronize(c->stream));
    for (AdapterEntry& e : s->table) (void)hipFree((void*)e.down);
    s->table_dev.release();
    c->ops.sets.erase(handle);
    return 0;
  });
}

int tgohip_adapter_rows(tgohip_ctx* c, int B, const int32_t* extents, const int32_t* adapters, int* handle) {
  return guarded([&]() -> int {
    if (B < 0) return refuse("adapter_rows: " + std::to_string(B) + " requests");
    if (B > 0 && (!extents || !adapters)) return refuse("adapter_rows: extents and adapters are host arrays");
    int64_t T = 0;
    int top = -1;
    for (int b = 0; b < B; b++) {
      const auto bad = [b](const std::string& m) { return refuse("adapter_rows: request " + std::to_string(b) + m); };
      if (extents[b] < 0) return bad(" has " + std::to_string(extents[b]) + " rows");
      if (adapters[b] < -1 || adapters[b] >= 65536)
        return bad(" names adapter " + std::to_string(adapters[b]) + "; -1 (none) to 65535");
      T += extents[b];
      if (extents[b]) top = std::max(top, (int)adapters[b]);
    }
    if (T >= 1 << 20) return refuse("adapter_rows: " + std::to_string(T) + " rows; below 2^20");
    if (!c) return no_ctx("adapter_rows");
    if (!handle) return refuse("adapter_rows: handle is missing");
    if (*handle && !find(c->ops.rows, *handle, "adapter_rows")) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "adapter_rows")) return rc;
    // rows by adapter, in their own order within one, in tiles of 16 (decode batches:
    // most adapters have a few rows) or 64 (prompts: an adapter is read once per tile)
    const size_t tile = T <= kAdapterFewRows ? 16 : 64;
    std::vector<std::vector<int32_t>> by((size_t)top + 2);
    int32_t row = 0;
    for (int b = 0; b < B; b++)
      for (int i = 0; i < extents[b]; i++) by[(size_t)adapters[b] + 1].push_back(row++);
    std::vector<int32_t> perm;
    perm.reserve((size_t)T);
    std::vector<AdapterTile> tiles;
    for (size_t a = 0; a < by.size(); a++)
      for (size_t i = 0; i < by[a].size(); i += tile) {
        const int n = (int)std::min<size_t>(tile, by[a].size() - i);
        tiles.push_back(AdapterTile{(int32_t)a - 1, (int32_t)perm.size(), n});
        perm.insert(perm.end(), by[a].begin() + i, by[a].begin() + i + n);
      }
    const bool fresh = *handle == 0;
    const int h = fresh ? c->ops.next++ : *handle;
    AdapterRows& r = c->ops.rows[h];
    r.T = -1;
    Stager sg;
    sg.add(perm.data(), perm.size() * 4);
    const size_t off = sg.add(tiles.data(), tiles.size() * sizeof(AdapterTile));
    int rc = 0;
    const int splits = adapter_splits((int)tiles.size(), c->ncu);
    if (T) rc = r.u.ensure((size_t)T * ((size_t)(splits + 1) * kAdapterMaxRank + 1) * sizeof(float));
    if (!rc) rc = sg.upload(c, r.meta);
    if (rc) {
      if (fresh) {
        r.meta.release();
        r.u.release();
        c->ops.rows.erase(h);
      }
      return rc;
    }
    r.T = (int)T;
    r.ntiles = (int)tiles.size();
    r.tile_rows = (int)tile;
    r.splits = splits;
    r.max_adapter = top;
    r.tiles_off = off;
    *handle = h;
    return 0;
  });
}

int tgohip_adapter_rows_free(tgohip_ctx* c, int handle) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("adapter_rows_free");
    AdapterRows* r = find(c->ops.rows, handle, "adapter_rows_free");
    if (!r) return TGOHIP_EINVAL;
    OnDevice on(c->device);
    if (const int rc = no_capture(c, "adapter_rows_free")) return rc;
    TGOHIP_HIP(hipStreamSynchronize(c->stream));
    r->meta.release();
    r->u.release();
    c->ops.rows.erase(handle);
    return 0;
  });
}

int tgohip_adapters(tgohip_ctx* c, int set, int rows, const void* x, int x_dtype, const void* base, void* y,
                    int y_dtype) {
  return guarded([&]() -> int {
    if (!c) return no_ctx("adapters");
    AdapterSet* s = find(c->ops.sets, set, "adapters: set");
    if (!s) return TGOHIP_EINVAL;
    AdapterRows* r = find(c->ops.rows, rows, "adapters: rows");
    if (!r) return TGOHIP_EINVAL;
    if (r->T < 0) return fail(TGOHIP_ESTATE, "adapters: the rows were not made again after a failure");
    if (x_dtype != TGOHIP_F32 && x_dtype != TGOHIP_F16 && x_dtype != TGOHIP_F16X2)
      return refuse("adapters: x_dtype is " + std::to_string(x_dtype) + "; f32, f16 or a pair");
    if (y_dtype != TGOHIP_F32 && y_dtype != TGOHIP_F16)
      return refuse("adapters: y_dtype is " + std::to_string(y_dtype) + "; f32 or f16");
    if (r->max_adapter >= (int)s->table.size())
      return refuse("adapters: the rows name adapter " + std::to_string(r->max_adapter) + " and the set holds " +
                    std::to_string(s->table.size()));
    if (r->T == 0) return 0;
    if (!x || !y) return refuse("adapters: x and y are device buffers");
    if (misaligned(x) || misaligned(base) || misaligned(y))
      return refuse("adapters: x, base and y start on 16-byte boundaries");
    const int64_t T = r->T, yb = y_dtype == TGOHIP_F16 ? 2 : 4;
    const Span sx{(const char*)x, 1, 1, 0, 0, T * s->K * (x_dtype == TGOHIP_F16 ? 2 : 4)};
    const Span sy{(const char*)y, 1, 1, 0, 0, T * s->N * yb}, sb{(const char*)base, 1, 1, 0, 0, T * s->N * yb};
    if (meet(sy, sx)) return refuse("adapters: y meets x in memory");
    if (base && base != y && meet(sy, sb)) return refuse("adapters: y meets base in memory; y is base itself or apart");
    AdapterArgs a{};
    a.table = (const AdapterEntry*)s->table_dev.p;
    a.tiles = (const AdapterTile*)((const char*)r->meta.p + r->tiles_off);
    a.perm = (const int32_t*)r->meta.p;
    a.ntiles = r->ntiles;
    a.T = r->T;
    a.K = s->K;
    a.N = s->N;
    a.x = x;
    a.xk = x_dtype == TGOHIP_F32 ? XK_F32 : x_dtype == TGOHIP_F16 ? XK_F16 : XK_X2;
    a.base = base;
    a.y = y;
    a.y_f16 = y_dtype == TGOHIP_F16;
    a.u = (float*)r->u.p;
    OnDevice on(c->device);
    a.splits = r->splits;
    a.rank_pad = s->rank_pad;
    a.pair = (half_t*)(a.u + (size_t)r->splits * T * kAdapterMaxRank);  // as many bytes as a plane
    a.pair_scale = a.u + (size_t)(r->splits + 1) * T * kAdapterMaxRank;
    launch_adapters(a, r->tile_rows, c->ncu, c->stream);
    TGOHIP_HIP(hipGetLastError());
    return 0;
  });
}

}  // extern "C"
