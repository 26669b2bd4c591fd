// paged.cpp: the C entry points of a caller's paged 16-bit cache (include/hwnpu_cuda.h, hc_paged_*):
// the checks of the arguments, then the kernels' launches.
#include "paged.h"

#include <cmath>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <string>

namespace {

// Runs f and turns an exception (an allocation of an error string that failed) into an error string,
// so that none crosses the C boundary.
template <typename F>
char *guarded(F f) {
  try {
    return f();
  } catch (const std::exception &) {
    static const char msg[] = "hc_paged: out of host memory";
    char *p = static_cast<char *>(std::malloc(sizeof msg));
    if (p) std::memcpy(p, msg, sizeof msg);
    return p;
  }
}

char *fail(const char *who, const std::string &what) { return hc::make_error(std::string(who) + ": " + what); }

char *launched(const char *who, cudaError_t e) {
  return e == cudaSuccess ? nullptr : fail(who, cudaGetErrorString(e));
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A stride the kernels' 16-byte loads and the tensor maps can take.
bool good_stride(int64_t s) { return s >= 0 && s % 8 == 0 && s < (int64_t(1) << 38); }

char *view(const char *who, const hc_paged_cache *c, hc::PagedView *out) {
  if (!c) return fail(who, "NULL cache");
  if (!c->k || !c->v || !c->block_table || !c->lengths) return fail(who, "NULL pointer in the cache");
  if (c->type != HC_FMT_F16 && c->type != HC_FMT_BF16) return fail(who, "type must be HC_FMT_F16 or HC_FMT_BF16");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(who, "head_dim must be 64 or 128");
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
    return fail(who, "page_size must be a power of two from 16 to 1024");
  if (c->seqs < 1 || c->seqs > 65535 || c->kv_heads < 1 || c->kv_heads > 1024)
    return fail(who, "seqs must be 1..65535 and kv_heads 1..1024");
  if (c->pages < 1 || c->max_pages < 1 || c->table_stride < c->max_pages)
    return fail(who, "pages and max_pages must be positive and table_stride at least max_pages");
  if (int64_t(c->max_pages) * c->page_size >= (int64_t(1) << 30)) return fail(who, "capacity must be below 2^30 slots");
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(who, "k and v must be 16-byte aligned");
  // a dimension of one has no stride of its own
  const int64_t ps = c->pages == 1 ? 0 : c->page_stride, hs = c->kv_heads == 1 ? 0 : c->head_stride;
  if (!good_stride(ps) || !good_stride(hs) || !good_stride(c->row_stride))
    return fail(who, "strides must be multiples of 8 elements, from 0 to 2^38");
  if (c->row_stride < c->head_dim || (c->kv_heads > 1 && hs < c->head_dim) || (c->pages > 1 && ps < c->head_dim))
    return fail(who, "rows must not overlap: every stride is at least head_dim");
  if (c->device) {
    int current = 0;
    if (char *e = launched(who, cudaGetDevice(&current))) return e;
    if (current != c->device - 1)
      return fail(who, "the cache is on device " + std::to_string(c->device - 1) + ", but device " +
                           std::to_string(current) + " is current");
  }
  int shift = 4;
  while ((1 << shift) < c->page_size) ++shift;
  *out = hc::PagedView{static_cast<uint16_t *>(c->k), static_cast<uint16_t *>(c->v), c->block_table, c->lengths,
                       c->weights, ps, hs, c->row_stride, c->table_stride, c->seqs, c->kv_heads, c->head_dim, shift,
                       c->pages, c->max_pages, c->max_pages * c->page_size, c->type == HC_FMT_BF16};
  return nullptr;
}

char *heads_ok(const char *who, const hc::PagedView &c, int heads, int window, int first, int max_len) {
  if (heads < 1 || heads % c.kv_heads) return fail(who, "heads must be a positive multiple of kv_heads");
  if (heads / c.kv_heads > 128) return fail(who, "at most 128 query heads a kv head");
  if (window < 0 || first < 0) return fail(who, "window and first must not be negative");
  if (max_len < 0) return fail(who, "max_len must not be negative");
  return nullptr;
}

char *query(const char *who, const hc::PagedView &c, const hc_paged_attn *a, int rows, int max_len, hc::PagedQuery *out) {
  if (!a) return fail(who, "NULL attention arguments");
  if (!a->q || !a->o) return fail(who, "NULL q or o");
  if (char *e = heads_ok(who, c, a->heads, a->window, a->first, max_len)) return e;
  if (!aligned16(a->q) || !aligned16(a->o)) return fail(who, "q and o must be 16-byte aligned");
  if (!good_stride(a->q_row) || !good_stride(a->q_head) || !good_stride(a->o_row) || !good_stride(a->o_head))
    return fail(who, "strides must be multiples of 8 elements, from 0 to 2^38");
  if ((rows > 1 && a->o_row < c.hd) || (a->heads > 1 && a->o_head < c.hd))
    return fail(who, "rows of o must not overlap: its strides are at least head_dim");
  if (!std::isfinite(a->scale)) return fail(who, "scale must be finite");
  *out = hc::PagedQuery{static_cast<const uint16_t *>(a->q), static_cast<uint16_t *>(a->o), a->q_row, a->q_head,
                        a->o_row, a->o_head, a->sinks, a->scale, a->heads, a->heads / c.kv_heads, a->window, a->first};
  return nullptr;
}

char *scratch_ok(const char *who, const void *scratch, uint64_t have, uint64_t need) {
  if (have < need || (need && !scratch))
    return fail(who, "scratch of " + std::to_string(have) + " bytes, " + std::to_string(need) + " are needed");
  if (need && !aligned16(scratch)) return fail(who, "scratch must be 16-byte aligned");
  return nullptr;
}

// Multiprocessors of the current device.
char *multiprocessors(const char *who, int *sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  return launched(who, e);
}

int bound_of(const hc::PagedView &c, int max_len) { return max_len < 1 || max_len > c.cap ? c.cap : max_len; }

}  // namespace

extern "C" {

HC_API char *hc_paged_append_run(const hc_paged_cache *cache, const void *k, const void *v, int64_t k_row,
                                 int64_t k_head, int64_t v_row, int64_t v_head, const int32_t *seq,
                                 const int32_t *slot, int32_t rows, void *stream) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_append_run";
    hc::PagedView c;
    if (char *e = view(who, cache, &c)) return e;
    if (rows < 0) return fail(who, "rows must not be negative");
    if (rows == 0) return nullptr;
    if (!k || !v || !seq || !slot) return fail(who, "NULL argument");
    if (!aligned16(k) || !aligned16(v)) return fail(who, "k and v must be 16-byte aligned");
    if (!good_stride(k_row) || !good_stride(k_head) || !good_stride(v_row) || !good_stride(v_head))
      return fail(who, "strides must be multiples of 8 elements, from 0 to 2^38");
    return launched(who, hc::paged_append(c, static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), k_row,
                                          k_head, v_row, v_head, seq, slot, rows, static_cast<cudaStream_t>(stream)));
  });
}

HC_API char *hc_paged_decode_scratch(const hc_paged_cache *cache, int32_t heads, int32_t window, int32_t first,
                                     int32_t max_len, int32_t accumulate, uint64_t *bytes) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_decode_scratch";
    hc::PagedView c;
    int sms = 0;
    if (!bytes) return fail(who, "NULL argument");
    if (char *e = view(who, cache, &c)) return e;
    if (char *e = heads_ok(who, c, heads, window, first, max_len)) return e;
    if (char *e = multiprocessors(who, &sms)) return e;
    *bytes = hc::paged_decode_scratch(c, heads, window, first, bound_of(c, max_len), accumulate != 0, sms);
    return nullptr;
  });
}

HC_API char *hc_paged_decode_run(const hc_paged_cache *cache, const hc_paged_attn *attn, int32_t max_len,
                                 int32_t accumulate, void *scratch, uint64_t scratch_bytes, void *stream) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_decode_run";
    hc::PagedView c;
    hc::PagedQuery a;
    int sms = 0;
    if (char *e = view(who, cache, &c)) return e;
    if (char *e = query(who, c, attn, c.seqs, max_len, &a)) return e;
    if (accumulate && !c.weights) return fail(who, "accumulate needs a cache with weights");
    if (char *e = multiprocessors(who, &sms)) return e;
    const int bound = bound_of(c, max_len);
    if (char *e = scratch_ok(who, scratch, scratch_bytes,
                             hc::paged_decode_scratch(c, a.heads, a.window, a.first, bound, accumulate != 0, sms)))
      return e;
    return launched(who, hc::paged_decode(c, a, bound, accumulate != 0, scratch, sms, static_cast<cudaStream_t>(stream)));
  });
}

HC_API char *hc_paged_prompt_scratch(const hc_paged_cache *cache, int32_t heads, int32_t window, int32_t first,
                                     int32_t rows, int32_t max_rows, int32_t max_len, uint64_t *bytes) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_prompt_scratch";
    hc::PagedView c;
    int sms = 0;
    if (!bytes) return fail(who, "NULL argument");
    if (char *e = view(who, cache, &c)) return e;
    if (char *e = heads_ok(who, c, heads, window, first, max_len)) return e;
    if (rows < 0 || max_rows < 0) return fail(who, "rows and max_rows must not be negative");
    if (char *e = multiprocessors(who, &sms)) return e;
    *bytes = hc::paged_prompt_scratch(c, heads, window, first, rows, max_rows, bound_of(c, max_len), sms);
    return nullptr;
  });
}

HC_API char *hc_paged_prompt_run(const hc_paged_cache *cache, const hc_paged_attn *attn, const int32_t *starts,
                                 int32_t rows, int32_t max_rows, int32_t max_len, void *scratch,
                                 uint64_t scratch_bytes, void *stream) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_prompt_run";
    hc::PagedView c;
    hc::PagedQuery a;
    int sms = 0;
    if (char *e = view(who, cache, &c)) return e;
    if (rows < 0 || max_rows < 0) return fail(who, "rows and max_rows must not be negative");
    if (rows == 0 || max_rows == 0) return nullptr;
    if (!starts) return fail(who, "NULL starts");
    if (char *e = query(who, c, attn, rows, max_len, &a)) return e;
    if (char *e = multiprocessors(who, &sms)) return e;
    const int bound = bound_of(c, max_len), most = max_rows < rows ? max_rows : rows;
    if (char *e = scratch_ok(who, scratch, scratch_bytes,
                             hc::paged_prompt_scratch(c, a.heads, a.window, a.first, rows, most, bound, sms)))
      return e;
    return launched(who, hc::paged_prompt(c, a, starts, rows, most, bound, scratch, sms, static_cast<cudaStream_t>(stream)));
  });
}

HC_API char *hc_paged_check(void) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_check";
    int code = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = hc::paged_status_take(&code);
    if (char *err = launched(who, e)) return err;
    return code ? fail(who, "a wait of the paged prompt attention ran out (code " + std::to_string(code) + ")") : nullptr;
  });
}

HC_API char *hc_paged_evict_scratch(const hc_paged_cache *cache, int32_t keep, int32_t max_len, uint64_t *bytes) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_evict_scratch";
    hc::PagedView c;
    if (!bytes) return fail(who, "NULL argument");
    if (char *e = view(who, cache, &c)) return e;
    if (keep < 1 || max_len < 0) return fail(who, "keep must be positive and max_len not negative");
    *bytes = uint64_t(c.seqs) * c.kv_heads * keep * sizeof(int32_t);
    return nullptr;
  });
}

HC_API char *hc_paged_evict_run(const hc_paged_cache *cache, const hc_paged_cache *into, int32_t keep, int32_t first,
                                int32_t recent, int32_t max_len, int32_t *kept, void *scratch, uint64_t scratch_bytes,
                                void *stream) {
  return guarded([&]() -> char * {
    const char *who = "hc_paged_evict_run";
    hc::PagedView c, to;
    if (char *e = view(who, cache, &c)) return e;
    if (char *e = view(who, into, &to)) return e;
    if (!c.weights) return fail(who, "the cache has no weights");
    if (c.seqs != to.seqs || c.kv_heads != to.kv_heads || c.hd != to.hd || c.bf16 != to.bf16)
      return fail(who, "both caches must have the same type, seqs, kv_heads and head_dim");
    if (keep < 1 || first < 0 || recent < 0 || int64_t(first) + recent > keep)
      return fail(who, "keep must be positive and at least first + recent, neither negative");
    if (max_len < 0) return fail(who, "max_len must not be negative");
    if (keep > to.cap) return fail(who, "keep is above the capacity of the cache it copies into");
    if (c.lengths == to.lengths || c.table == to.table || c.weights == to.weights)
      return fail(who, "the cache it copies into needs a block table, lengths and weights of its own");
    // the kept slots are written to `kept` or, without it, to the scratch
    const uint64_t need = kept ? 0 : uint64_t(c.seqs) * c.kv_heads * keep * sizeof(int32_t);
    if (char *e = scratch_ok(who, scratch, scratch_bytes, need)) return e;
    return launched(who, hc::paged_evict(c, to, keep, first, recent, bound_of(c, max_len),
                                         kept ? kept : static_cast<int32_t *>(scratch), static_cast<cudaStream_t>(stream)));
  });
}

}  // extern "C"
