// paged.h: the kernels of a caller's paged 16-bit cache (hc_paged_* of include/hwnpu_cuda.h) and what
// they share: append and evict (paged_cache.cu), decode (paged_decode.cu), prompt (paged_prompt.cu).
#ifndef HWNPU_PAGED_H
#define HWNPU_PAGED_H

#include "common.h"

namespace hc {

// A checked hc_paged_cache, as the kernels take it.
struct PagedView {
  uint16_t *k, *v;
  const int32_t *table;
  int32_t *lengths;
  float *weights;
  int64_t page_stride, head_stride, row_stride, table_stride;
  int seqs, kv_heads, hd, shift, pages, max_pages, cap;  // page_size = 1 << shift; cap in slots
  bool bf16;
};

// A checked hc_paged_attn.
struct PagedQuery {
  const uint16_t *q;
  uint16_t *o;
  int64_t q_row, q_head, o_row, o_head;
  const float *sinks;
  float scale;
  int heads, rep, window, first;  // rep: query heads a kv head
};

#ifdef __CUDACC__
// The slots sequence i uses, held to the capacity.
__device__ __forceinline__ int paged_len(const PagedView &c, int i) {
  const int n = c.lengths[i];
  return n < 0 ? 0 : (n > c.cap ? c.cap : n);
}
// The element offset of the row of slot j (below cap) of sequence i, head h, or -1 where the page id
// is outside the pool.
__device__ __forceinline__ int64_t paged_row(const PagedView &c, int i, int h, int j) {
  const int page = c.table[i * c.table_stride + (j >> c.shift)];
  if (unsigned(page) >= unsigned(c.pages)) return -1;
  return page * c.page_stride + h * c.head_stride + (j & ((1 << c.shift) - 1)) * c.row_stride;
}
#endif

// Each returns the launch's error, if any; sms: the device's multiprocessors.
cudaError_t paged_append(const PagedView &c, const uint16_t *k, const uint16_t *v, int64_t k_row, int64_t k_head,
                         int64_t v_row, int64_t v_head, const int32_t *seq, const int32_t *slot, int rows,
                         cudaStream_t st);
// idx: [seqs][kv_heads][keep] int32, the slots kept (-1 past the new length).
cudaError_t paged_evict(const PagedView &c, const PagedView &to, int keep, int first, int recent, int max_len,
                        int32_t *idx, cudaStream_t st);
size_t paged_decode_scratch(const PagedView &c, int heads, int window, int first, int max_len, bool accumulate, int sms);
cudaError_t paged_decode(const PagedView &c, const PagedQuery &a, int max_len, bool accumulate, void *scratch, int sms,
                         cudaStream_t st);
// Whether a prompt call is one of few rows (tokens times query heads a kv head), which run as decode does.
bool paged_few(const PagedView &c, int heads, int max_rows);
size_t paged_few_scratch(const PagedView &c, int heads, int window, int first, int rows, int max_len, int sms);
cudaError_t paged_few_run(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows,
                          int max_len, void *scratch, int sms, cudaStream_t st);
size_t paged_prompt_scratch(const PagedView &c, int heads, int window, int first, int rows, int max_rows, int max_len,
                            int sms);
cudaError_t paged_prompt(const PagedView &c, const PagedQuery &a, const int32_t *starts, int rows, int max_rows,
                         int max_len, void *scratch, int sms, cudaStream_t st);
// *code: of the first wait of the prompt kernel that ran out on the current device since the last
// call (0: none), cleared.
cudaError_t paged_status_take(int *code);

}  // namespace hc

#endif
