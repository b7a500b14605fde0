// runtime.h -- what the C ABI's entry points share (runtime.hip, operators.hip):
// the context, its grow-only device buffers and the staging of per-call metadata.
#pragma once

#include "common.h"
#include "kernels/operators.h"

#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <utility>
#include <vector>

namespace tgohip {

constexpr size_t kBufAlign = (size_t)2 << 20;

// Grow-only device buffer.
struct DevBuf {
  void* p = nullptr;
  size_t bytes = 0;
  int ensure(size_t n) {
    if (n <= bytes) return 0;
    // Whole 2 MiB pages: each buffer starts on its own page. With sizes as
    // asked, the step's attention ran 4% slower or not depending on how the
    // buffers happened to fall (one process or the other); rounded, it
    // always runs the faster way.
    n = (n + kBufAlign - 1) / kBufAlign * kBufAlign;
    // a step still in flight may read the old buffer (the scheduler's
    // overlap mode): let the device drain before it goes
    if (p) (void)hipDeviceSynchronize();
    if (p) (void)hipFree(p);
    p = nullptr;
    bytes = 0;
    hipError_t e = hipMalloc(&p, n);
    if (e != hipSuccess) {
      p = nullptr;
      return fail(TGOHIP_ENOMEM, "device allocation of " + std::to_string(n) + " bytes: " +
                                     hipGetErrorString(e));
    }
    bytes = n;
    // TGOHIP_DEBUG_NAN_FILL=1: every activation and workspace buffer starts as
    // all-ones bytes (NaN in f32 and f16), so a kernel that reads memory no
    // earlier kernel wrote shows up as NaN logits or changed tokens.
    static const bool nan_fill = [] {
      const char* v = getenv("TGOHIP_DEBUG_NAN_FILL");
      return v && atoi(v) != 0;
    }();
    if (nan_fill) {
      e = hipMemset(p, 0xff, n);
      if (e == hipSuccess) e = hipDeviceSynchronize();
      if (e != hipSuccess) return fail(TGOHIP_EDEVICE, hip_message(e, "debug fill"));
    }
    return 0;
  }
  void release() {
    if (p) (void)hipFree(p);
    p = nullptr;
    bytes = 0;
  }
};

// Sub-ports of a layer's fused projections, one bit each once uploaded.
enum { SUB_WQ = 1, SUB_WK = 2, SUB_WV = 4, SUB_WGATE = 8, SUB_WUP = 16, SUB_ALL = 31 };

struct Layer {
  PackedWeight qkv, wo, gateup, down;
  int bound = 0;  // SUB_* bits of the fused QKV and gate/up sub-ports written
  float* g_attn = nullptr;
  float* g_ffn = nullptr;
  float* g_q = nullptr;
  float* g_k = nullptr;
};

// ---- what a program makes once for the operators of operators.hip ------------
struct RopeTable {
  int d = 0, rd = 0, half = 0;
  float attention = 1.f;
  DevBuf inv_freq;  // [rd / 2] double, turns per position
};
// A batch's decomposition on the device, and the partial results of its calls.
struct PackedHandle {
  PackedPlan plan;  // its vectors empty: they are in meta
  PackedCounts n;
  size_t merges_off = 0;
  DevBuf meta, part;
};
struct AdapterSet {
  int K = 0, N = 0;
  int rank_pad = 0;  // the largest loaded
  std::vector<AdapterEntry> table;
  DevBuf table_dev;
};
struct AdapterRows {
  int T = 0, ntiles = 0, tile_rows = 0, splits = 1, max_adapter = -1;
  size_t tiles_off = 0;
  DevBuf meta, u;
};
struct OpHandles {
  int next = 1;
  std::map<int, RopeTable> ropes;
  std::map<int, PackedHandle> packed;
  std::map<int, AdapterSet> sets;
  std::map<int, AdapterRows> rows;
  void release();  // frees the device memory of every handle
};

}  // namespace tgohip

using namespace tgohip;

constexpr int kPinnedSlots = 4;

struct tgohip_ctx {
  int device = 0;
  hipStream_t own_stream = nullptr;
  hipStream_t stream = nullptr;
  int ncu = 256;
  bool configured = false;
  tgohip_model_cfg cfg{};
  std::vector<Layer> layers;
  void* embed = nullptr;
  uint16_t* embed_scales = nullptr;
  int embed_form = -1;
  PackedWeight lm_head;
  float* g_final = nullptr;
  double* inv_freq = nullptr;
  half_t* kc = nullptr;
  half_t* vc = nullptr;
  int kv_positions = 0;
  int precision = 1;  // 1 (default): tgo's f32 arithmetic (hi+lo pairs), 0: f16 operands
  int cascade = 0;    // minimum sequences sharing a prefix for prefix-shared attention (0: off)
  // activations and workspaces
  DevBuf h, xn, qkv, q, attn, act, lastn, logits, argmax, margin, meta, gemm_ws, part_o, part_ml;
  DevBuf amax_part;  // per-chunk partials of the greedy selection
  DevBuf rows;  // [2][rows]: positions and slots derived on the device
  DevBuf rope;  // [rows][32] float4: the rows' rotary cos and sin (rope_table)
  int rows_cap = 0, batch_cap = 0;
  int last_batch = 0;  // members of the last launched step (its margins are in `margin`)
  // The head of the last launched step ran over the members that worked only:
  // logits row i is member head_rows[i]'s (empty: one row per member).
  std::vector<int32_t> head_rows;
  // pinned staging for per-call metadata: a call writes the next slot while the
  // device still reads the ones before, and waits only for the slot it takes
  struct Pinned {
    void* p = nullptr;
    size_t bytes = 0;
    hipEvent_t read = nullptr;  // the device's last read of it
  };
  Pinned pinned[kPinnedSlots];
  int pinned_next = 0;
  hipEvent_t ev0 = nullptr, ev1 = nullptr;
  std::vector<void*> allocs;  // weight and gain allocations owned by the context
  std::map<int, PackedWeight> handles;
  tgohip::OpHandles ops;
  int next_handle = 1;
  // profiling: HIP events around the launches of the kernels in prof_mask
  // (TGOHIP_PROF_* bits) in every prof_stride-th layer of a step
  bool profile = false;
  int prof_stride = 1;
  int prof_mask = 1 << TGOHIP_PROF_ATTN;
  std::vector<hipEvent_t> prof_ev;  // [2 sets][layers][kinds][begin, end]
  double prof_ms[TGOHIP_PROF_KINDS] = {}, prof_bytes[TGOHIP_PROF_KINDS] = {},
         prof_flops[TGOHIP_PROF_KINDS] = {};
  int64_t prof_launches[TGOHIP_PROF_KINDS] = {};
  void* scratch = nullptr;  // this device's address of the static split-K workspace
};

namespace tgohip {

// The next staging slot, free and of at least `bytes`.
inline int take_pinned(tgohip_ctx* c, size_t bytes, tgohip_ctx::Pinned** out) {
  tgohip_ctx::Pinned& s = c->pinned[c->pinned_next];
  c->pinned_next = (c->pinned_next + 1) % kPinnedSlots;
  TGOHIP_HIP(hipEventSynchronize(s.read));
  if (bytes > s.bytes) {
    if (s.p) (void)hipHostFree(s.p);
    s.p = nullptr;
    s.bytes = 0;
    TGOHIP_HIP(hipHostMalloc(&s.p, bytes, hipHostMallocDefault));
    s.bytes = bytes;
  }
  *out = &s;
  return 0;
}

// Metadata packer: appends arrays into a pinned staging slot at 256-byte
// aligned offsets, then one kernel reads all of them into c->meta, or, above
// kFetchBytes (a page table of some thousand pages for each of hundreds of
// sequences), the copy engine, whose rate across PCIe is higher. Attention over
// 64-position contexts, us a call back to back / alone, kernel : engine:
// 0.03 MB of page table 26-30 / 45 : 35 / 50; 1.0 MB 46 / 85 : 55 / 83; 2.1 MB
// 82 / 144 : 82 / 134; 4.2 MB 135 / 221 : 120 / 199; 8.4 MB 231 / 372 : 196 / 326.
constexpr size_t kFetchBytes = (size_t)3 << 19;
struct Stager {
  std::vector<std::pair<const void*, size_t>> parts;
  std::vector<size_t> offs;
  size_t total = 0;
  size_t add(const void* p, size_t bytes) {
    const size_t o = total;
    parts.push_back({p, bytes});
    offs.push_back(o);
    total += (bytes + 255) / 256 * 256;
    return o;
  }
  int upload(tgohip_ctx* c) { return upload(c, c->meta); }
  int upload(tgohip_ctx* c, DevBuf& dst) {
    if (total == 0) return 0;
    tgohip_ctx::Pinned* s = nullptr;
    int rc = take_pinned(c, total, &s);
    if (rc) return rc;
    rc = dst.ensure(total);
    if (rc) return rc;
    for (size_t i = 0; i < parts.size(); i++)
      if (parts[i].second) memcpy((char*)s->p + offs[i], parts[i].first, parts[i].second);
    if (total <= kFetchBytes) {
      launch_fetch(s->p, dst.p, total, c->stream);
      TGOHIP_HIP(hipGetLastError());
    } else {
      TGOHIP_HIP(hipMemcpyAsync(dst.p, s->p, total, hipMemcpyHostToDevice, c->stream));
    }
    TGOHIP_HIP(hipEventRecord(s->read, c->stream));
    return 0;
  }
  template <class T> T* dev(tgohip_ctx* c, size_t off) { return (T*)((char*)c->meta.p + off); }
};

}  // namespace tgohip
