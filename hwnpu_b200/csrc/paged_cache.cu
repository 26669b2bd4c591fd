// paged_cache.cu: the rows of a caller's paged 16-bit cache: append (new rows into the pages) and evict
// (the rows with the largest accumulated attention weight, in slot order, into other pages). Both
// move rows and compute nothing: they are bound by the bytes they move.
#include "device.cuh"
#include "paged.h"

namespace hc {
namespace {

// One thread a 16-byte piece of a row's key and of its value; CH pieces a row.
template <int CH>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedView c, const uint16_t *__restrict__ k,
                                                           const uint16_t *__restrict__ v, int64_t k_row,
                                                           int64_t k_head, int64_t v_row, int64_t v_head,
                                                           const int32_t *__restrict__ seq,
                                                           const int32_t *__restrict__ slot, int rows) {
  const int64_t u = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int ch = int(u % CH);
  const int64_t rh = u / CH;
  if (rh >= int64_t(rows) * c.kv_heads) return;
  const int r = int(rh / c.kv_heads), h = int(rh % c.kv_heads);
  const int i = seq[r], j = slot[r];
  if (unsigned(i) >= unsigned(c.seqs) || unsigned(j) >= unsigned(c.cap)) return;
  const int64_t at = paged_row(c, i, h, j);
  if (at < 0) return;
  const uint4 kk = *reinterpret_cast<const uint4 *>(k + r * k_row + h * k_head + 8 * ch);
  const uint4 vv = *reinterpret_cast<const uint4 *>(v + r * v_row + h * v_head + 8 * ch);
  *reinterpret_cast<uint4 *>(c.k + at + 8 * ch) = kk;
  *reinterpret_cast<uint4 *>(c.v + at + 8 * ch) = vv;
  if (c.weights && ch == 0) c.weights[(int64_t(i) * c.kv_heads + h) * c.cap + j] = 0.f;
}

// A weight as a key whose unsigned order is the order evict keeps by: NaN lowest, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = w == 0.f ? 0u : __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// One CTA a (sequence, kv head): the slots to keep into idx. The key of the last candidate that stays
// is found by radix selection, a histogram of 8 bits at a time; then one pass in slot order writes the
// slots above it and the first ones equal to it.
__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(PagedView c, int keep, int first, int recent,
                                                                   int32_t *__restrict__ idx,
                                                                   int32_t *__restrict__ to_lengths) {
  __shared__ int hist[256];
  __shared__ int sh_digit, sh_above;
  __shared__ int wsum[2][32];
  const int h = blockIdx.x, i = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = paged_len(c, i);
  int32_t *out = idx + (int64_t(i) * c.kv_heads + h) * keep;
  const int n_new = min(n, keep);
  if (h == 0 && tid == 0) to_lengths[i] = n_new;
  if (n <= keep) {
    for (int d = tid; d < keep; d += kSelThreads) out[d] = d < n ? d : -1;
    return;
  }
  const float *w = c.weights + (int64_t(i) * c.kv_heads + h) * c.cap;
  const int lo = first, hi = n - recent;  // candidates; more than `want` of them
  const int want = keep - first - recent;
  for (int d = tid; d < first; d += kSelThreads) out[d] = d;
  for (int d = tid; d < recent; d += kSelThreads) out[keep - recent + d] = n - recent + d;
  if (want == 0) return;
  uint32_t prefix = 0;
  int need = want;  // the need-th largest of the keys with this prefix is the threshold
  for (int b = 24; b >= 0; b -= 8) {
    for (int d = tid; d < 256; d += kSelThreads) hist[d] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kSelThreads) {
      const uint32_t key = weight_key(w[j]);
      if (b == 24 || (key >> (b + 8)) == (prefix >> (b + 8))) atomicAdd(&hist[(key >> b) & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {
      // lane l holds digits 8 l .. 8 l + 7, counted from the largest digit down
      int own = 0;
      for (int d = 0; d < 8; ++d) own += hist[255 - (8 * lane + d)];
      int upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      int above = upto - own;
      if (above < need && upto >= need) {
        for (int d = 0; d < 8; ++d) {
          const int cnt = hist[255 - (8 * lane + d)];
          if (above + cnt >= need) {
            sh_digit = 255 - (8 * lane + d);
            sh_above = above;
            break;
          }
          above += cnt;
        }
      }
    }
    __syncthreads();
    prefix |= uint32_t(sh_digit) << b;
    need -= sh_above;
    __syncthreads();
  }
  // slots whose key is above the threshold, and the first `need` equal to it, in slot order
  int base = first, ties = 0;
  for (int j0 = lo; j0 < hi; j0 += kSelThreads) {
    const int j = j0 + tid;
    const uint32_t key = j < hi ? weight_key(w[j]) : 0u;
    const bool gt = j < hi && key > prefix, eq = j < hi && key == prefix;
    const unsigned beq = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) wsum[0][warp] = __popc(beq);
    __syncthreads();
    int before = ties, total = 0;
    for (int x = 0; x < kSelThreads / 32; ++x) {
      before += x < warp ? wsum[0][x] : 0;
      total += wsum[0][x];
    }
    const bool stay = gt || (eq && before + __popc(beq & ((1u << lane) - 1)) < need);
    ties += total;
    const unsigned bst = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) wsum[1][warp] = __popc(bst);
    __syncthreads();
    int at = base;
    total = 0;
    for (int x = 0; x < kSelThreads / 32; ++x) {
      at += x < warp ? wsum[1][x] : 0;
      total += wsum[1][x];
    }
    base += total;
    if (stay) out[at + __popc(bst & ((1u << lane) - 1))] = j;
    __syncthreads();
  }
}

// Copies the kept rows: one thread a 16-byte piece of a row's key and of its value.
template <int CH>
__global__ void __launch_bounds__(256) paged_copy_kernel(PagedView c, PagedView to, int keep,
                                                         const int32_t *__restrict__ idx) {
  constexpr int kRows = 256 / CH;
  const int h = blockIdx.y, i = blockIdx.z;
  const int d = blockIdx.x * kRows + threadIdx.x / CH, ch = threadIdx.x % CH;
  if (d >= keep) return;
  const int j = idx[(int64_t(i) * c.kv_heads + h) * keep + d];
  if (j < 0) return;
  const int64_t src = paged_row(c, i, h, j), dst = paged_row(to, i, h, d);
  if (to.weights && ch == 0)
    to.weights[(int64_t(i) * c.kv_heads + h) * to.cap + d] = c.weights[(int64_t(i) * c.kv_heads + h) * c.cap + j];
  if (dst < 0) return;
  uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
  if (src >= 0) {
    kk = *reinterpret_cast<const uint4 *>(c.k + src + 8 * ch);
    vv = *reinterpret_cast<const uint4 *>(c.v + src + 8 * ch);
  }
  *reinterpret_cast<uint4 *>(to.k + dst + 8 * ch) = kk;
  *reinterpret_cast<uint4 *>(to.v + dst + 8 * ch) = vv;
}

}  // namespace

cudaError_t paged_append(const PagedView &c, const uint16_t *k, const uint16_t *v, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head, const int32_t *seq, const int32_t *slot, int rows,
                         cudaStream_t st) {
  const int ch = c.hd / 8;
  const int64_t blocks = (int64_t(rows) * c.kv_heads * ch + 255) / 256;
  if (c.hd == 128)
    paged_append_kernel<16><<<unsigned(blocks), 256, 0, st>>>(c, k, v, k_row, k_head, v_row, v_head, seq, slot, rows);
  else
    paged_append_kernel<8><<<unsigned(blocks), 256, 0, st>>>(c, k, v, k_row, k_head, v_row, v_head, seq, slot, rows);
  return cudaGetLastError();
}

cudaError_t paged_evict(const PagedView &c, const PagedView &to, int keep, int first, int recent, int32_t *idx,
                        cudaStream_t st) {
  paged_select_kernel<<<dim3(c.kv_heads, c.seqs), kSelThreads, 0, st>>>(c, keep, first, recent, idx, to.lengths);
  const int rows = 256 / (c.hd / 8);
  const dim3 grid((keep + rows - 1) / rows, c.kv_heads, c.seqs);
  if (c.hd == 128) paged_copy_kernel<16><<<grid, 256, 0, st>>>(c, to, keep, idx);
  else paged_copy_kernel<8><<<grid, 256, 0, st>>>(c, to, keep, idx);
  return cudaGetLastError();
}

}  // namespace hc
