// rope.hip -- rotary positions over strided heads (nn/attention.go:203-211 for
// the interleaved layout of a whole head): pair i of a head at position p turns
// by p * w_i, (a, b) -> m (a cos - b sin, a sin + b cos).
//
// Bound by the heads' bytes. A workgroup takes some rows of one tensor: its
// threads first put the rows' cos and sin into LDS, once per pair and row
// (computed by every thread that uses them, 72 heads of 16384 rows took 443 us
// instead of 131), then walk the rows' heads in units of 2V elements, V pairs of
// a head's rotated part or 2V elements of the rest, neighbouring threads on
// neighbouring units. Measured: 604 MB of f16 heads (16384 rows) 131 us, 4.6 TB/s, a
// copy of that size 4.8; 52 MB of f32 rows to f16 (1152 rows) 10 us, 5.3 TB/s; one row
// 3.4 us in the kernel, 8 with the call.
#include "heads.h"

#include <algorithm>

namespace tgohip {

// One tensor's heads of the block's rows.
template <int V, bool HALF, bool XF16, bool YF16>
__device__ __forceinline__ void rope_heads(const RopeArgs& a, const RopeGroup& g, int t0, int rows, const float2* cs) {
  const int pairs = a.rd / 2, rot = g.rotate ? pairs / V : 0;
  const int units = g.rotate ? rot + (a.d - a.rd) / (2 * V) : a.d / (2 * V);
  const int slots = 256 / units, u = threadIdx.x % units, slot = threadIdx.x / units;
  if (slot >= slots) return;
  const bool turn = u < rot;
  // where the unit's elements lie in a head: two runs of V, or one of 2V
  const int ja = !turn ? (g.rotate ? a.rd : 0) + 2 * V * (u - rot) : HALF ? V * u : 2 * V * u;
  const int jb = turn && HALF ? ja + pairs : ja + V;
  for (int r = slot; r < rows * g.heads; r += slots) {
    const int t = (int)(((uint64_t)r * g.magic) >> 32), h = r - t * g.heads;
    const int64_t x = (t0 + t) * g.x_row + h * g.x_head, y = (t0 + t) * g.y_row + h * g.y_head;
    float p[2 * V], A[V], B[V];
    if constexpr (HALF) {
      rope_load<V, XF16>(g.x, x + ja, A);
      rope_load<V, XF16>(g.x, x + jb, B);
    } else {
      rope_load<2 * V, XF16>(g.x, x + ja, p);
    }
    if (turn) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float2 w = cs[t * pairs + V * u + i];
        const float e = HALF ? A[i] : p[2 * i], f = HALF ? B[i] : p[2 * i + 1];
        // Written out, and kept apart from the store's rounding (some widths would
        // otherwise round the multiply-add to f16 at once), so that all round alike.
        float e2 = fmaf(e, w.x, -(f * w.y)), f2 = fmaf(e, w.y, f * w.x);
        asm("" : "+v"(e2), "+v"(f2));
        if (HALF) A[i] = e2, B[i] = f2;
        else p[2 * i] = e2, p[2 * i + 1] = f2;
      }
    }
    if constexpr (HALF) {
      rope_store<V, YF16>(g.y, y + ja, A);
      rope_store<V, YF16>(g.y, y + jb, B);
    } else {
      rope_store<2 * V, YF16>(g.y, y + ja, p);
    }
  }
}

template <int V, bool HALF>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  extern __shared__ float2 cs[];  // [rows][pairs]
  const RopeGroup g = a.g[blockIdx.y];
  const int t0 = blockIdx.x * a.rows, rows = min(a.rows, a.T - t0), pairs = a.rd / 2;
  if (g.rotate) {
    for (int i = threadIdx.x; i < rows * pairs; i += 256) {
      const int t = i / pairs;
      cs[i] = rope_angle(a.positions[t0 + t], a.inv_freq[i - t * pairs], a.attention);
    }
    __syncthreads();
  }
  if (g.x_f16) {
    if (g.y_f16) rope_heads<V, HALF, true, true>(a, g, t0, rows, cs);
    else rope_heads<V, HALF, true, false>(a, g, t0, rows, cs);
  } else {
    if (g.y_f16) rope_heads<V, HALF, false, true>(a, g, t0, rows, cs);
    else rope_heads<V, HALF, false, false>(a, g, t0, rows, cs);
  }
}

template <int V, bool HALF>
static void rope_launch(const RopeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((rope_kernel<V, HALF>), dim3((unsigned)((a.T + a.rows - 1) / a.rows), (unsigned)a.n), dim3(256),
                     (size_t)a.rows * (a.rd / 2) * sizeof(float2), st, a);
}

void launch_rope(const RopeArgs& args, int ncu, hipStream_t st) {
  RopeArgs a = args;
  int heads = 0;
  bool aligned = true;  // every head starts on 16 bytes
  for (int i = 0; i < a.n; i++) {
    RopeGroup& g = a.g[i];
    heads = std::max(heads, g.heads);
    // r / heads = r * magic >> 32 for r < 2^16 (rows of a block times heads, below)
    g.magic = (((uint64_t)1 << 32) + g.heads - 1) / g.heads;
    const int xs = g.x_f16 ? 8 : 4, ys = g.y_f16 ? 8 : 4;  // elements in 16 bytes
    aligned = aligned && (uintptr_t)g.x % 16 == 0 && (uintptr_t)g.y % 16 == 0 && g.x_row % xs == 0 &&
              g.x_head % xs == 0 && g.y_row % ys == 0 && g.y_head % ys == 0;
  }
  // Rows per workgroup: enough that its few heads fill it, few enough that the chip is
  // full; a power of two of at most 16, and r below 2^16. At most 1 / 4 / 16 / 64 rows, us,
  // f16 heads of 128 dims: 65536 rows of one head 48.8 / 17.2 / 12.9 / 14.5, 16384 of 8
  // heads 16.9 / 12.3 / 12.4 / 12.3, of 72 heads 108 / 118 / 123 / 123.
  a.rows = 1;
  while (a.rows < 16 && 2 * a.rows * heads <= 65535 && (int64_t)a.n * a.T / (2 * a.rows) >= 4 * ncu) a.rows *= 2;
  // Units of 16 bytes and more: V pairs need runs of V (half) or 2V elements. Such units /
  // single elements, us: 16384 rows of 72 f16 heads 123 / 241, 4096 of 40 14.1 / 22.9,
  // 1152 f32 rows of 40 heads 10.2 / 10.0.
  const auto fits = [&](int v) { return aligned && a.rd % (2 * v) == 0 && a.d % (2 * v) == 0 && a.d / (2 * v) <= 256; };
  if (a.half) {
    if (fits(8)) rope_launch<8, true>(a, st);
    else if (fits(4)) rope_launch<4, true>(a, st);
    else rope_launch<1, true>(a, st);
  } else {
    if (fits(4)) rope_launch<4, false>(a, st);
    else rope_launch<1, false>(a, st);
  }
}

}  // namespace tgohip
