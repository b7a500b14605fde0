// rope.hip -- rotary positions over strided heads (nn/attention.go:203-211 for
// the interleaved layout of a whole head): pair i of a head at position p turns
// by p * w_i, (a, b) -> m (a cos - b sin, a sin + b cos).
#include "operators.h"

namespace tgohip {

__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  __shared__ float cs[kRopeMaxHeadDim / 2], sn[kRopeMaxHeadDim / 2];
  const int t = blockIdx.x;
  const double p = (double)a.positions[t];
  for (int i = threadIdx.x; i < a.rd / 2; i += 256) {
    const double turns = p * a.inv_freq[i];
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    cs[i] = (float)(c * (double)a.attention);
    sn[i] = (float)(s * (double)a.attention);
  }
  __syncthreads();
  for (int gi = 0; gi < a.n; gi++) {
    const RopeGroup g = a.g[gi];
    const int rd = g.rotate ? a.rd : 0;
    auto load = [&](int h, int j) {
      const int64_t o = t * g.x_row + h * g.x_head + j;
      return g.x_f16 ? (float)((const half_t*)g.x)[o] : ((const float*)g.x)[o];
    };
    auto store = [&](int h, int j, float v) {
      const int64_t o = t * g.y_row + h * g.y_head + j;
      if (g.y_f16) ((half_t*)g.y)[o] = (half_t)v;
      else ((float*)g.y)[o] = v;
    };
    const int pairs = rd / 2, units = pairs + (a.d - rd);
    for (int e = threadIdx.x; e < g.heads * units; e += 256) {
      const int h = e / units, u = e - h * units;
      if (u < pairs) {
        const int ja = a.half ? u : 2 * u, jb = a.half ? u + pairs : 2 * u + 1;
        const float x = load(h, ja), y = load(h, jb);
        store(h, ja, x * cs[u] - y * sn[u]);
        store(h, jb, x * sn[u] + y * cs[u]);
      } else {
        store(h, rd + u - pairs, load(h, rd + u - pairs));
      }
    }
  }
}

void launch_rope(const RopeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(rope_kernel, dim3((unsigned)a.T), dim3(256), 0, st, a);
}

}  // namespace tgohip
