"""Attention over a caller's paged 16-bit key-value cache (include/hwnpu_cuda.h, hc_paged_*).

The cache and every operand are device tensors of the caller: objects with data_ptr(), shape, stride()
and dtype, such as torch's. Nothing is allocated or copied; a call enqueues its kernels on `stream` (a
cudaStream_t as an integer; None: torch's current stream, or the default one for other objects than
torch's tensors) and returns. Wrong arguments raise HcError, torch's tensors among them when they are not on
the cache's GPU or that is not the current one (where other objects are is the caller's to know).
"""

import ctypes as C
import sys

from . import _abi as A

_TYPES = {"torch.float16": A.HC_FMT_F16, "torch.bfloat16": A.HC_FMT_BF16, "float16": A.HC_FMT_F16}


def _need(ok, what):
    if not ok:
        raise A.HcError(what)


class PagedCache:
    """One layer's cache of `seqs` sequences.

    k, v: [pages][kv_heads][page_size][head_dim], fp16 or bf16, the last dimension contiguous (a
    [pages][page_size][kv_heads][head_dim] pool goes in as its permute(0, 2, 1, 3));
    block_table: int32 [seqs][max_pages]; lengths: int32 [seqs], the slots in use, read by the device at
    each call; weights: float32 [seqs][kv_heads][max_pages * page_size] accumulated attention weights,
    or None."""

    def __init__(self, k, v, block_table, lengths, weights=None):
        _need(len(k.shape) == 4 and tuple(k.shape) == tuple(v.shape) and k.stride() == v.stride(),
              "PagedCache: k and v must have one 4-dimensional shape and the same strides")
        _need(str(k.dtype) in _TYPES and k.dtype == v.dtype, "PagedCache: k and v must both be fp16 or bf16")
        _need(k.stride(3) == 1, "PagedCache: the last dimension of k and v must be contiguous")
        pages, heads, page, dim = k.shape
        _need(str(block_table.dtype).endswith("int32") and len(block_table.shape) == 2 and block_table.stride(1) == 1,
              "PagedCache: block_table must be int32 [seqs][max_pages]")
        seqs, width = block_table.shape
        _need(str(lengths.dtype).endswith("int32") and tuple(lengths.shape) == (seqs,) and lengths.is_contiguous(),
              "PagedCache: lengths must be int32 [seqs]")
        if weights is not None:
            _need(str(weights.dtype).endswith("float32") and tuple(weights.shape) == (seqs, heads, width * page)
                  and weights.is_contiguous(), "PagedCache: weights must be float32 [seqs][kv_heads][max_pages * page_size]")
        torch = sys.modules.get("torch")
        self._gpu = None  # the GPU of torch's tensors; -2, which no get_device() gives: they are elsewhere
        if torch is not None and isinstance(k, torch.Tensor):
            self._gpu = -2
            if k.is_cuda:
                self._gpu = k.get_device()
                # the current stream in 0.06 us; torch.cuda.current_stream().cuda_stream takes 1.3 to 3
                self._current = torch._C._cuda_getCurrentRawStream
            _need(all(t is None or t.device == k.device for t in (v, block_table, lengths, weights)),
                  "PagedCache: the cache's tensors must be on one device")
        self.k, self.v, self.block_table, self.lengths, self.weights = k, v, block_table, lengths, weights
        self.seqs, self.kv_heads, self.head_dim, self.dtype = seqs, heads, dim, k.dtype
        self.desc = A.PagedCacheDesc(k.data_ptr(), v.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
                                     weights.data_ptr() if weights is not None else None, k.stride(0), k.stride(1),
                                     k.stride(2), block_table.stride(0), _TYPES[str(k.dtype)], seqs, heads, dim, page,
                                     pages, width, 0 if self._gpu is None or self._gpu < 0 else self._gpu + 1)
        self._ref = C.addressof(self.desc)
        self._int32 = block_table.dtype

    def _misplaced(self, *operands):
        """Raises if a kernel would see an address of the host or of another GPU than the cache's, which the library
        holds against the current one. (The short calls test their own operands first: this costs 0.3 us.)"""
        _need(self._gpu >= 0, "PagedCache: the cache must be on a GPU")
        _need(all(t is None or t.get_device() == self._gpu for t in operands),
              "PagedCache: every tensor must be on the cache's GPU")

    def _attn(self, q, out, scale, window, first, sinks):
        rows, heads, dim = q.shape
        dtype = self.dtype
        if q.dtype != dtype or out.dtype != dtype:
            raise A.HcError("PagedCache: q and out must have the cache's type")
        if out.shape != q.shape or dim != self.head_dim:
            raise A.HcError("PagedCache: q and out must be [rows][heads][head_dim]")
        qs, os = q.stride(), out.stride()
        if qs[2] != 1 or os[2] != 1:
            raise A.HcError("PagedCache: the last dimension of q and out must be contiguous")
        if sinks is not None:
            _need(str(sinks.dtype).endswith("float32") and sinks.shape == (heads,) and sinks.is_contiguous(),
                  "PagedCache: sinks must be float32 [heads]")
            sinks = sinks.data_ptr()
        return A.PagedAttn(q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], sinks, scale, heads, window, first)

    @staticmethod
    def _scratch(scratch):
        if scratch is None:
            return None, 0
        _need(scratch.is_contiguous(), "PagedCache: scratch must be contiguous")
        return scratch.data_ptr(), scratch.nbytes

    def append(self, k, v, seq, slot, stream=None):
        """Writes rows k, v [rows][kv_heads][head_dim] into slot[r] of sequence seq[r] (int32 [rows]);
        a negative slot leaves its row out. Lengths are the caller's to move."""
        rows = k.shape[0]
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise A.HcError("PagedCache.append: k and v must have the cache's type")
        if k.shape != (rows, self.kv_heads, self.head_dim) or v.shape != k.shape:
            raise A.HcError("PagedCache.append: k and v must be [rows][kv_heads][head_dim]")
        ks, vs = k.stride(), v.stride()
        if ks[2] != 1 or vs[2] != 1:
            raise A.HcError("PagedCache.append: the last dimension of k and v must be contiguous")
        for t in (seq, slot):
            if t.dtype != self._int32 or t.shape != (rows,) or not t.is_contiguous():
                raise A.HcError("PagedCache.append: seq and slot must be int32 [rows]")
        if self._gpu is not None and not (k.get_device() == v.get_device() == seq.get_device() == slot.get_device()
                                          == self._gpu):
            self._misplaced(k, v, seq, slot)
        if stream is None and self._gpu is not None:
            stream = self._current(self._gpu)
        A.check(A.lib().hc_paged_append_run(self._ref, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1],
                                            seq.data_ptr(), slot.data_ptr(), rows, stream))

    def decode(self, q, out, scale, window=0, first=0, sinks=None, accumulate=False, max_len=0, scratch=None,
               stream=None):
        """Attention of one new token a sequence: q, out [seqs][heads][head_dim], row i the token in slot
        lengths[i] - 1. It sees the last `window` slots (0: all) and the `first` first ones. With
        accumulate the visible slots' weights grow by what its heads gave them. scratch: device bytes
        (decode_scratch; with accumulate 4 a sequence, head and visible slot of the capacity)."""
        _need(len(q.shape) == 3 and q.shape[0] == self.seqs, "PagedCache.decode: q must be [seqs][heads][head_dim]")
        a = self._attn(q, out, scale, window, first, sinks)
        p, n = self._scratch(scratch)
        if self._gpu is not None and not (q.get_device() == out.get_device() == self._gpu
                                          and (sinks is None or sinks.get_device() == self._gpu)
                                          and (scratch is None or scratch.get_device() == self._gpu)):
            self._misplaced(q, out, sinks, scratch)
        if stream is None and self._gpu is not None:
            stream = self._current(self._gpu)
        A.check(A.lib().hc_paged_decode_run(self._ref, C.addressof(a), max_len, 1 if accumulate else 0, p, n, stream))

    def decode_scratch(self, heads, max_len=0, window=0, first=0, accumulate=False):
        """Bytes of scratch decode needs with these arguments."""
        n = C.c_uint64()
        A.check(A.lib().hc_paged_decode_scratch(self._ref, heads, window, first, max_len, 1 if accumulate else 0,
                                                C.byref(n)))
        return n.value

    def prompt(self, q, out, starts, max_rows, scale, window=0, first=0, sinks=None, max_len=0, scratch=None,
               stream=None):
        """Attention of many new tokens a sequence, whose keys and values are in the pages: rows
        starts[i] .. starts[i + 1] - 1 of q, out [rows][heads][head_dim] are sequence i's last slots
        (starts int32 [seqs + 1]; no sequence has more than max_rows of them)."""
        _need(len(q.shape) == 3, "PagedCache.prompt: q must be [rows][heads][head_dim]")
        if starts.dtype != self._int32 or starts.shape != (self.seqs + 1,) or not starts.is_contiguous():
            raise A.HcError("PagedCache.prompt: starts must be int32 [seqs + 1]")
        a = self._attn(q, out, scale, window, first, sinks)
        p, n = self._scratch(scratch)
        if self._gpu is not None:
            self._misplaced(q, out, starts, sinks, scratch)
            stream = self._current(self._gpu) if stream is None else stream
        A.check(A.lib().hc_paged_prompt_run(self._ref, C.addressof(a), starts.data_ptr(), q.shape[0], max_rows, max_len,
                                            p, n, stream))

    def prompt_scratch(self, heads, rows, max_rows, max_len=0, window=0, first=0):
        """Bytes of scratch prompt needs with these arguments."""
        n = C.c_uint64()
        A.check(A.lib().hc_paged_prompt_scratch(self._ref, heads, window, first, rows, max_rows, max_len, C.byref(n)))
        return n.value

    @staticmethod
    def check():
        """Waits for the current device's work and raises HcError if a bounded wait inside a prompt call ran out since
        the last check: that call's output is not to be trusted. Nothing else reports it, so a caller polls it
        where a result matters more than its latency."""
        A.check(A.lib().hc_paged_check())

    def evict(self, to, keep, first=0, recent=0, kept=None, max_len=0, scratch=None, stream=None):
        """Copies at most `keep` slots a head of every sequence into the pages of `to`, in slot order: the
        `first` first, the `recent` last and the heaviest between. Only decode gathers weights: straight after a
        prompt all are 0 and the oldest slots stay; a cache read through a window needs recent >= window. Writes to.lengths, to.weights and
        kept (int32 [seqs][kv_heads][keep], the slots they came from, -1 past the new length)."""
        _need(isinstance(to, PagedCache), "PagedCache.evict: `to` must be a PagedCache")
        if kept is not None:
            _need(kept.dtype == self._int32 and kept.shape == (self.seqs, self.kv_heads, keep) and kept.is_contiguous(),
                  "PagedCache.evict: kept must be int32 [seqs][kv_heads][keep]")
        p, n = self._scratch(scratch)
        if self._gpu is not None:
            self._misplaced(to.k, kept, scratch)
            stream = self._current(self._gpu) if stream is None else stream
        A.check(A.lib().hc_paged_evict_run(self._ref, to._ref, keep, first, recent, max_len,
                                           kept.data_ptr() if kept is not None else None, p, n, stream))

    def evict_scratch(self, keep, max_len=0):
        """Bytes of scratch evict needs with these arguments and without `kept` (with it, none)."""
        n = C.c_uint64()
        A.check(A.lib().hc_paged_evict_scratch(self._ref, keep, max_len, C.byref(n)))
        return n.value
