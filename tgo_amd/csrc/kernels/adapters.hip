// adapters.hip -- low-rank adapters of many requests beside a shared projection:
// y[t] = base[t] + s (x[t] . down^T) . up^T with the adapter of the request that
// row t belongs to, or y[t] = base[t] where it has none.
#include "operators.h"

namespace tgohip {

__device__ __forceinline__ float adapter_x(const AdapterArgs& a, int64_t row, int k) {
  const int64_t o = row * a.K + k;
  if (a.xk == XK_F32) return ((const float*)a.x)[o];
  const half_t* h = (const half_t*)a.x;
  if (a.xk == XK_F16) return (float)h[o];
  return (float)h[o] + (float)h[(int64_t)a.T * a.K + o];
}

// u[i][r] of the tile's rows, one workgroup per tile.
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a) {
  const AdapterTile t = a.tiles[blockIdx.x];
  if (t.adapter < 0) return;
  const AdapterEntry e = a.table[t.adapter];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = wave; i < t.n * e.rank_pad; i += 4) {
    const int row = i / e.rank_pad, r = i - row * e.rank_pad;
    const int64_t src = a.perm[t.start + row];
    float s = 0.f;
    for (int k = lane; k < a.K; k += 64) s += adapter_x(a, src, k) * (float)e.down[(int64_t)r * a.K + k];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) a.u[(int64_t)(t.start + row) * kAdapterMaxRank + r] = s;
  }
}

__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a) {
  const AdapterTile t = a.tiles[blockIdx.y];
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  AdapterEntry e{};
  if (t.adapter >= 0) e = a.table[t.adapter];
  for (int i = 0; i < t.n; i++) {
    const int64_t o = (int64_t)a.perm[t.start + i] * a.N + n;
    float s = 0.f;
    for (int r = 0; r < e.rank_pad; r++)
      s += a.u[(int64_t)(t.start + i) * kAdapterMaxRank + r] * (float)e.up[(int64_t)n * e.rank_pad + r];
    float b = 0.f;
    if (a.base) b = a.y_f16 ? (float)((const half_t*)a.base)[o] : ((const float*)a.base)[o];
    const float y = b + e.scale * s;
    if (a.y_f16) ((half_t*)a.y)[o] = (half_t)y;
    else ((float*)a.y)[o] = y;
  }
}

void launch_adapters(const AdapterArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(adapter_down_kernel, dim3((unsigned)a.ntiles), dim3(256), 0, st, a);
  hipLaunchKernelGGL(adapter_up_kernel, dim3((unsigned)((a.N + 255) / 256), (unsigned)a.ntiles), dim3(256), 0, st, a);
}

}  // namespace tgohip
