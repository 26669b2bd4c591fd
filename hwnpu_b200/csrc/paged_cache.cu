// paged_cache.cu: the rows of a caller's paged 16-bit cache: append (new rows into the pages) and evict
// (the rows with the largest accumulated attention weight, in slot order, into other pages). Both
// move rows and compute nothing: they are bound by the bytes they move.
#include <algorithm>

#include "device.cuh"
#include "kernels.h"
#include "paged.h"

namespace hc {
namespace {

// One thread a 16-byte piece of kAppendRows (row, head)s' keys and of their values, CH pieces a row. All pieces are on
// their way while the rows' places are looked up (row, then block table: two loads that wait for one another).
// Bound by HBM once there are enough rows: 75 MB (9,000 rows of 8 heads of 128) take 16.3 us, 4.6 TB/s; with 1 row a
// thread 17.2, with 4 18.1.
constexpr int kAppendRows = 2;
template <int CH>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedView c, const uint16_t *__restrict__ k,
                                                           const uint16_t *__restrict__ v, int64_t k_row,
                                                           int64_t k_head, int64_t v_row, int64_t v_head,
                                                           const int32_t *__restrict__ seq,
                                                           const int32_t *__restrict__ slot, int rows) {
  const int ch = threadIdx.x % CH;
  const int64_t first = int64_t(blockIdx.x) * (256 / CH * kAppendRows) + threadIdx.x / CH;
  uint4 kk[kAppendRows], vv[kAppendRows];
  int i[kAppendRows], j[kAppendRows], h[kAppendRows];
#pragma unroll
  for (int u = 0; u < kAppendRows; ++u) {
    const int64_t rh = first + u * (256 / CH);
    const bool there = rh < int64_t(rows) * c.kv_heads;
    const int r = there ? int(rh / c.kv_heads) : 0;
    h[u] = there ? int(rh % c.kv_heads) : 0;
    i[u] = there ? seq[r] : -1;
    j[u] = there ? slot[r] : -1;
    kk[u] = vv[u] = make_uint4(0, 0, 0, 0);
    if (there) {
      kk[u] = *reinterpret_cast<const uint4 *>(k + r * k_row + h[u] * k_head + 8 * ch);
      vv[u] = *reinterpret_cast<const uint4 *>(v + r * v_row + h[u] * v_head + 8 * ch);
    }
  }
  int64_t at[kAppendRows];
#pragma unroll
  for (int u = 0; u < kAppendRows; ++u) {
    const bool in = unsigned(i[u]) < unsigned(c.seqs) && unsigned(j[u]) < unsigned(c.cap);
    at[u] = in ? paged_row(c, i[u], h[u], j[u]) : -1;
  }
#pragma unroll
  for (int u = 0; u < kAppendRows; ++u) {
    if (at[u] < 0) continue;
    *reinterpret_cast<uint4 *>(c.k + at[u] + 8 * ch) = kk[u];
    *reinterpret_cast<uint4 *>(c.v + at[u] + 8 * ch) = vv[u];
    if (c.weights && ch == 0) c.weights[(int64_t(i[u]) * c.kv_heads + h[u]) * c.cap + j[u]] = 0.f;
  }
}

// A weight as a key whose unsigned order is the order evict keeps by: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048;
constexpr int kSelAhead = 8;      // weights a thread loads at once
constexpr int kSelCache = 49152;  // keys a CTA can hold in shared memory (192 KB)

// Exclusive prefix sum of v over the CTA's threads.
__device__ __forceinline__ int sel_scan(int v, int *warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += u;
  }
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  static_assert(kSelThreads == 1024, "a lane a warp");
  int upto = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  const int before = __shfl_sync(0xffffffffu, upto, max(warp - 1, 0));
  __syncthreads();
  return (warp > 0 ? before : 0) + x - v;
}

// One CTA a (sequence, kv head): the slots to keep into idx, ascending. The key of the last candidate that stays
// is found by radix selection, 11, 11 and 10 bits at a time, over the candidates' keys in shared
// memory (a row of up to 49,152; longer ones are read again, from the L2 cache); then every thread counts what
// stays of a run of candidates, and writes it behind what the threads before it count.
//
// Bound by the passes over a row by one SM, not by its bytes (64% of the issue slots): 128 rows of up to 32,771 weights
// (10 MB) take 20 us, one CTA an SM; with one weight loaded at a time 29. Adding a warp's equal digits at once (ballots) or several copies of
// the histogram were no faster, and rows of one value are not slower without. A CTA that also copied what it kept
// took longer (136 us against 133 then): the SMs with few rows end early and HBM is not full.
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(PagedView c, int keep, int first, int recent, int cache,
                                                                   int32_t *__restrict__ idx,
                                                                   int32_t *__restrict__ to_lengths) {
  extern __shared__ uint32_t sel_keys[];
  __shared__ int hist[kSelBins];
  __shared__ int warps[kSelThreads / 32];
  __shared__ int sh_digit, sh_above, sh_count;
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.x, i = blockIdx.y, tid = threadIdx.x;
  const int n = paged_len(c, i);
  int32_t *out = idx + (int64_t(i) * c.kv_heads + h) * keep;
  if (h == 0 && tid == 0) to_lengths[i] = min(n, keep);
  if (n <= keep) {
    for (int d = tid; d < keep; d += kSelThreads) out[d] = d < n ? d : -1;
    return;
  }
  const int cand = n - recent - first, want = keep - first - recent;  // more candidates than may stay
  const float *w = c.weights + (int64_t(i) * c.kv_heads + h) * c.cap + first;
  for (int d = tid; d < first; d += kSelThreads) out[d] = d;
  for (int d = tid; d < recent; d += kSelThreads) out[keep - recent + d] = n - recent + d;
  if (want == 0) return;
  const bool cached = cand <= cache;
  uint32_t prefix = 0, known = 0;  // the threshold's bits found so far, and which they are
  int need = want;                 // the need-th largest of the keys with this prefix is the threshold
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int d = tid; d < kSelBins; d += kSelThreads) hist[d] = 0;
    __syncthreads();
    if (pass == 0 || !cached) {
      for (int j0 = 0; j0 < cand; j0 += kSelAhead * kSelThreads) {
        float x[kSelAhead];
#pragma unroll
        for (int u = 0; u < kSelAhead; ++u) x[u] = j0 + u * kSelThreads + tid < cand ? w[j0 + u * kSelThreads + tid] : 0.f;
#pragma unroll
        for (int u = 0; u < kSelAhead; ++u) {
          const int j = j0 + u * kSelThreads + tid;
          if (j >= cand) break;
          const uint32_t key = weight_key(x[u]);
          if (pass == 0 && cached) sel_keys[j] = key;
          if ((key & known) == prefix) atomicAdd(&hist[(key >> shift) & ((1 << bits) - 1)], 1);
        }
      }
    } else {
#pragma unroll 4
      for (int j = tid; j < cand; j += kSelThreads) {
        const uint32_t key = sel_keys[j];
        if ((key & known) == prefix) atomicAdd(&hist[(key >> shift) & ((1 << bits) - 1)], 1);
      }
    }
    __syncthreads();
    // thread t holds bins 2 t and 2 t + 1 from the largest digit down
    const int d0 = kSelBins - 1 - 2 * tid, n0 = hist[d0], n1 = hist[d0 - 1];
    const int above = sel_scan(n0 + n1, warps);
    if (above < need && above + n0 + n1 >= need) {
      const bool upper = above + n0 >= need;
      sh_digit = upper ? d0 : d0 - 1;
      sh_above = above + (upper ? 0 : n0);
      sh_count = upper ? n0 : n1;
    }
    __syncthreads();
    prefix |= uint32_t(sh_digit) << shift;
    known |= ((1u << bits) - 1) << shift;
    need -= sh_above;
    const bool all = sh_count == need;  // every key with this prefix stays: the bits below do not matter
    __syncthreads();
    if (all) break;
  }
  // runs of an odd number of candidates a thread: no two lanes on one bank
  const int run = ((cand + kSelThreads - 1) / kSelThreads) | 1;
  const int j0 = int(min(int64_t(cand), int64_t(tid) * run)), j1 = min(cand, j0 + run);
  int gt = 0, eq = 0;
#pragma unroll 4
  for (int j = j0; j < j1; ++j) {
    const uint32_t key = cached ? sel_keys[j] : weight_key(w[j]);
    gt += key > prefix;
    eq += key == prefix;
  }
  const int over = sel_scan(gt, warps);
  int ties = min(need, sel_scan(eq, warps)), at = first + over + ties;
  for (int j = j0; j < j1; ++j) {
    const uint32_t key = cached ? sel_keys[j] : weight_key(w[j]);
    const bool tie = key == prefix && ties < need;
    if (key > prefix || tie) {
      out[at++] = first + j;
      ties += tie;
    }
  }
}

// Copies the kept rows: a thread has a 16-byte piece of kCopyRows rows, keys and values, all loaded before the
// first is stored. Bound by HBM: 4,096 rows a head of 16 sequences of 8 heads of 128, 270 MB read and as much
// written, take 83 us (6.5 TB/s; 4 rows a thread 93, 1 row 89).
constexpr int kCopyRows = 2;
template <int CH>
__global__ void __launch_bounds__(256) paged_copy_kernel(PagedView c, PagedView to, int keep,
                                                         const int32_t *__restrict__ idx) {
  constexpr int kStep = 256 / CH;
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.y, i = blockIdx.z, ch = threadIdx.x % CH;
  const int d0 = blockIdx.x * (kStep * kCopyRows) + threadIdx.x / CH;
  const int64_t row = int64_t(i) * c.kv_heads + h;
  int j[kCopyRows];
  uint4 kk[kCopyRows], vv[kCopyRows];
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) j[u] = d0 + u * kStep < keep ? idx[row * keep + d0 + u * kStep] : -1;
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) {
    const int64_t src = j[u] >= 0 ? paged_row(c, i, h, j[u]) : -1;
    kk[u] = vv[u] = make_uint4(0, 0, 0, 0);
    if (src >= 0) {
      kk[u] = *reinterpret_cast<const uint4 *>(c.k + src + 8 * ch);
      vv[u] = *reinterpret_cast<const uint4 *>(c.v + src + 8 * ch);
    }
  }
#pragma unroll
  for (int u = 0; u < kCopyRows; ++u) {
    const int d = d0 + u * kStep;
    if (j[u] < 0) continue;
    if (to.weights && ch == 0) to.weights[row * to.cap + d] = c.weights[row * c.cap + j[u]];
    const int64_t dst = paged_row(to, i, h, d);
    if (dst < 0) continue;
    *reinterpret_cast<uint4 *>(to.k + dst + 8 * ch) = kk[u];
    *reinterpret_cast<uint4 *>(to.v + dst + 8 * ch) = vv[u];
  }
}

}  // namespace

cudaError_t paged_append(const PagedView &c, const uint16_t *k, const uint16_t *v, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head, const int32_t *seq, const int32_t *slot, int rows,
                         cudaStream_t st) {
  const int per = 256 / (c.hd / 8) * kAppendRows;
  const int64_t blocks = (int64_t(rows) * c.kv_heads + per - 1) / per;
  if (c.hd == 128)
    paged_append_kernel<16><<<unsigned(blocks), 256, 0, st>>>(c, k, v, k_row, k_head, v_row, v_head, seq, slot, rows);
  else
    paged_append_kernel<8><<<unsigned(blocks), 256, 0, st>>>(c, k, v, k_row, k_head, v_row, v_head, seq, slot, rows);
  return cudaGetLastError();
}

cudaError_t paged_evict(const PagedView &c, const PagedView &to, int keep, int first, int recent, int max_len,
                        int32_t *idx, cudaStream_t st) {
  const int cache = std::min(max_len, kSelCache);
  cudaError_t e = cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kSelCache * int(sizeof(uint32_t)));
  if (e != cudaSuccess) return e;
  launch_pdl(paged_select_kernel, dim3(c.kv_heads, c.seqs), dim3(kSelThreads), size_t(cache) * sizeof(uint32_t), st, c,
             keep, first, recent, cache, idx, to.lengths);
  const int rows = 256 / (c.hd / 8) * kCopyRows;
  const dim3 grid((keep + rows - 1) / rows, c.kv_heads, c.seqs);
  if (c.hd == 128) launch_pdl(paged_copy_kernel<16>, grid, dim3(256), 0, st, c, to, keep, idx);
  else launch_pdl(paged_copy_kernel<8>, grid, dim3(256), 0, st, c, to, keep, idx);
  return cudaGetLastError();
}

}  // namespace hc
