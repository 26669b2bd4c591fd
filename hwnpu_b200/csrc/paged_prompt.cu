// paged_prompt.cu: attention of many new tokens a sequence over a caller's paged 16-bit cache
// (hc_paged_prompt_run).
#include <cuda_bf16.h>

#include "device.cuh"
#include "paged.h"

namespace hc {
namespace {
__device__ __forceinline__ float paged_val(uint16_t b, bool bf16) {
  return bf16 ? __uint_as_float(uint32_t(b) << 16) : __half2float(__ushort_as_half(b));
}
__device__ __forceinline__ uint16_t paged_bits(float v, bool bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// One CTA a (row, kv head), a warp a query head at a time: the lanes share a key's dimensions, the
// softmax runs with its maximum and sum.
template <int HD>
__global__ void __launch_bounds__(256) paged_rows_kernel(PagedView c, PagedQuery a, const int32_t *__restrict__ starts,
                                                         int rows, int max_rows, bool accumulate) {
  constexpr int E = HD / 32;
  __shared__ float sm_m[128], sm_l[128];
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int i = blockIdx.z, row = i, n = paged_len(c, i), p = n - 1;
  if (starts) {
    const int t = blockIdx.x;
    row = starts[i] + t;
    const int cnt = starts[i + 1] - starts[i];
    if (t >= cnt || t >= max_rows || row < 0 || row >= rows) return;
    p = n - cnt + t;
  }
  auto score = [&](const float (&q)[E], int64_t at) {
    float s = 0.f;
    if (at >= 0)
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], paged_val(c.k[at + lane + 32 * e], c.bf16), s);
    return warp_sum(s) * a.scale;
  };
  auto sees = [&](int j) { return a.window == 0 || p - j < a.window || j < a.first; };
  for (int r = warp; r < a.rep; r += 8) {
    const int hq = h * a.rep + r;
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      q[e] = paged_val(a.q[row * a.q_row + hq * a.q_head + lane + 32 * e], c.bf16);
      o[e] = 0.f;
    }
    float m = a.sinks ? a.sinks[hq] : -INFINITY, l = a.sinks ? 1.f : 0.f;
    if (m == -INFINITY) l = 0.f;
    for (int j = 0; j <= p; ++j) {
      if (!sees(j)) continue;
      const int64_t at = paged_row(c, i, h, j);
      const float s = score(q, at);
      const float nm = fmaxf(m, s);
      const float f = m == -INFINITY ? 0.f : expf(m - nm), w = nm == -INFINITY ? 0.f : expf(s - nm);
      l = l * f + w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * f + (at >= 0 ? w * paged_val(c.v[at + lane + 32 * e], c.bf16) : 0.f);
      m = nm;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) a.o[row * a.o_row + hq * a.o_head + lane + 32 * e] = paged_bits(o[e] * inv, c.bf16);
    if (lane == 0) {
      sm_m[r] = m;
      sm_l[r] = inv;
    }
  }
  if (!accumulate) return;
  __syncthreads();
  for (int j = warp; j <= p; j += 8) {
    if (!sees(j)) continue;
    const int64_t at = paged_row(c, i, h, j);
    float w = 0.f;
    for (int r = 0; r < a.rep; ++r) {
      float q[E];
#pragma unroll
      for (int e = 0; e < E; ++e) q[e] = paged_val(a.q[row * a.q_row + (h * a.rep + r) * a.q_head + lane + 32 * e], c.bf16);
      const float s = score(q, at);
      if (sm_m[r] > -INFINITY) w += expf(s - sm_m[r]) * sm_l[r];
    }
    if (lane == 0) c.weights[(int64_t(i) * c.kv_heads + h) * c.cap + j] += w;
  }
}

}  // namespace

size_t paged_prompt_scratch(const PagedView &, int, int, int, int, int, int, int) { return 0; }

cudaError_t paged_prompt(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows, int,
                         void *, int, cudaStream_t st) {
  const dim3 grid(max_rows, c.kv_heads, c.seqs);
  if (c.hd == 128) paged_rows_kernel<128><<<grid, 256, 0, st>>>(c, a, starts, rows, max_rows, false);
  else paged_rows_kernel<64><<<grid, 256, 0, st>>>(c, a, starts, rows, max_rows, false);
  return cudaGetLastError();
}

}  // namespace hc

