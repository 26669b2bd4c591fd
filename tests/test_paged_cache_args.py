"""The refusals of the paged-cache entry points (hc_paged_*): wrong arguments come back as error strings
before anything is launched, so they need no GPU."""

import ctypes as C

import pytest

import hwnpu_b200 as hb
from hwnpu_b200 import _abi as A

P = 1 << 20  # an aligned address that no refused call reads


def cache(**kw):
    d = dict(k=P, v=P, block_table=P, lengths=P, weights=P, page_stride=8 * 16 * 128, head_stride=16 * 128,
             row_stride=128, table_stride=8, type=A.HC_FMT_BF16, seqs=2, kv_heads=8, head_dim=128, page_size=16,
             pages=20, max_pages=8)
    d.update(kw)
    return A.PagedCacheDesc(**d)


def attn(**kw):
    d = dict(q=P, o=P, q_row=2048, q_head=128, o_row=2048, o_head=128, sinks=None, scale=0.1, heads=16, window=0, first=0)
    d.update(kw)
    return A.PagedAttn(**d)


def calls(c, a):
    L, c, a = A.lib(), C.byref(c), C.byref(a)
    yield lambda: A.check(L.hc_paged_decode_run(c, a, 0, 0, P, 1 << 40, None))
    yield lambda: A.check(L.hc_paged_prompt_run(c, a, P, 4, 2, 0, P, 1 << 40, None))


@pytest.mark.parametrize("kw,why", [
    (dict(k=None), "NULL pointer"), (dict(lengths=None), "NULL pointer"), (dict(block_table=None), "NULL pointer"),
    (dict(type=A.HC_FMT_INT8_ROW), "type"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=2048), "page_size"),
    (dict(seqs=0), "seqs"), (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "pages"), (dict(max_pages=-1), "max_pages"),
    (dict(table_stride=7), "table_stride"), (dict(max_pages=1 << 27, table_stride=1 << 27), "capacity"),
    (dict(k=P + 8), "aligned"), (dict(v=P + 2), "aligned"), (dict(page_stride=16388), "multiples of 8"),
    (dict(row_stride=-128), "strides"), (dict(row_stride=64), "overlap"), (dict(head_stride=8), "overlap")])
def test_cache_refusals(kw, why):
    c = cache(**kw)
    n = C.c_uint64()
    for call in calls(c, attn()):
        with pytest.raises(hb.HcError, match=why):
            call()
    for f in (lambda: A.lib().hc_paged_append_run(C.byref(c), P, P, 1024, 128, 1024, 128, P, P, 3, None),
              lambda: A.lib().hc_paged_evict_run(C.byref(c), C.byref(cache(lengths=2 * P, block_table=2 * P, weights=2 * P)),
                                                 32, 0, 0, 0, None, P, 1 << 40, None),
              lambda: A.lib().hc_paged_evict_run(C.byref(cache(lengths=2 * P, block_table=2 * P, weights=2 * P)), C.byref(c),
                                                 32, 0, 0, 0, None, P, 1 << 40, None),
              lambda: A.lib().hc_paged_evict_scratch(C.byref(c), 32, 0, C.byref(n)),
              lambda: A.lib().hc_paged_decode_scratch(C.byref(c), 16, 0, 0, 0, 0, C.byref(n)),
              lambda: A.lib().hc_paged_prompt_scratch(C.byref(c), 16, 0, 0, 4, 2, 0, C.byref(n))):
        with pytest.raises(hb.HcError, match=why):
            A.check(f())


@pytest.mark.parametrize("kw,why", [
    (dict(q=None), "NULL"), (dict(o=None), "NULL"), (dict(q=P + 4), "aligned"), (dict(o=P + 8), "aligned"),
    (dict(heads=0), "heads"), (dict(heads=12), "multiple of kv_heads"), (dict(heads=8 * 129), "128 query heads"),
    (dict(window=-1), "window"), (dict(first=-1), "first"), (dict(q_row=2044), "strides"), (dict(o_head=-128), "strides"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")])
def test_query_refusals(kw, why):
    for call in calls(cache(), attn(**kw)):
        with pytest.raises(hb.HcError, match=why):
            call()


def test_null_descriptors_and_negative_counts():
    L, c, a = A.lib(), cache(), attn()
    pc, pa = C.byref(c), C.byref(a)
    for f, why in ((lambda: L.hc_paged_decode_run(None, pa, 0, 0, P, 1, None), "NULL cache"),
                   (lambda: L.hc_paged_decode_run(pc, None, 0, 0, P, 1, None), "NULL attention"),
                   (lambda: L.hc_paged_decode_run(pc, pa, -1, 0, P, 1, None), "max_len"),
                   (lambda: L.hc_paged_prompt_run(pc, pa, None, 4, 2, 0, P, 1, None), "NULL starts"),
                   (lambda: L.hc_paged_prompt_run(pc, pa, P, -4, 2, 0, P, 1, None), "rows"),
                   (lambda: L.hc_paged_prompt_run(pc, pa, P, 4, -2, 0, P, 1, None), "rows"),
                   (lambda: L.hc_paged_append_run(pc, None, P, 1024, 128, 1024, 128, P, P, 3, None), "NULL"),
                   (lambda: L.hc_paged_append_run(pc, P, P, 1024, 128, 1024, 128, P, None, 3, None), "NULL"),
                   (lambda: L.hc_paged_append_run(pc, P + 8, P, 1024, 128, 1024, 128, P, P, 3, None), "aligned"),
                   (lambda: L.hc_paged_append_run(pc, P, P, 1023, 128, 1024, 128, P, P, 3, None), "strides"),
                   (lambda: L.hc_paged_append_run(pc, P, P, 1024, 128, 1024, 128, P, P, -3, None), "rows"),
                   (lambda: L.hc_paged_decode_scratch(pc, 16, 0, 0, 0, 0, None), "NULL"),
                   (lambda: L.hc_paged_prompt_scratch(pc, 16, 0, 0, 4, 2, 0, None), "NULL"),
                   (lambda: L.hc_paged_evict_scratch(pc, 16, 0, None), "NULL")):
        with pytest.raises(hb.HcError, match=why):
            A.check(f())
    # accumulating needs weights; no rows are no work
    with pytest.raises(hb.HcError, match="weights"):
        A.check(L.hc_paged_decode_run(C.byref(cache(weights=None)), pa, 0, 1, P, 1 << 40, None))
    A.check(L.hc_paged_append_run(pc, None, None, 0, 0, 0, 0, None, None, 0, None))
    A.check(L.hc_paged_prompt_run(pc, pa, None, 0, 0, 0, None, 0, None))


@pytest.mark.parametrize("keep,first,recent,max_len,why", [
    (0, 0, 0, 0, "keep"), (-1, 0, 0, 0, "keep"), (32, -1, 0, 0, "keep"), (32, 0, -1, 0, "keep"), (32, 20, 13, 0, "keep"),
    (32, 2 ** 31 - 1, 2 ** 31 - 1, 0, "keep"), (32, 0, 0, -1, "max_len"), (129, 0, 0, 0, "capacity")])
def test_evict_refusals(keep, first, recent, max_len, why):
    c, to = cache(), cache(lengths=2 * P, block_table=2 * P, weights=2 * P)
    with pytest.raises(hb.HcError, match=why):
        A.check(A.lib().hc_paged_evict_run(C.byref(c), C.byref(to), keep, first, recent, max_len, None, P, 1 << 40, None))


@pytest.mark.parametrize("kw,why", [
    (dict(weights=2 * P, lengths=2 * P), "block table"), (dict(block_table=2 * P, weights=2 * P), "lengths"),
    (dict(seqs=3), "same"), (dict(kv_heads=4), "same"), (dict(type=A.HC_FMT_F16), "same"),
    (dict(head_dim=64), "same")])
def test_evict_needs_a_cache_of_its_own(kw, why):
    with pytest.raises(hb.HcError, match=why):
        A.check(A.lib().hc_paged_evict_run(C.byref(cache()), C.byref(cache(**kw)), 32, 0, 0, 0, None, P, 1 << 40, None))
    with pytest.raises(hb.HcError, match="no weights"):
        A.check(A.lib().hc_paged_evict_run(C.byref(cache(weights=None)),
                                           C.byref(cache(lengths=2 * P, block_table=2 * P)), 32, 0, 0, 0, None, P, 1 << 40, None))
    with pytest.raises(hb.HcError, match="scratch"):
        A.check(A.lib().hc_paged_evict_run(C.byref(cache()), C.byref(cache(lengths=2 * P, block_table=2 * P, weights=2 * P)),
                                           32, 0, 0, 0, None, P, 16, None))


def test_python_checks():
    torch = pytest.importorskip("torch")
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    t, n = torch.zeros((1, 3), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    ok = hb.PagedCache(k, k.clone(), t, n)
    for bad, why in ((lambda: hb.PagedCache(k, k[:2], t, n), "shape"),
                     (lambda: hb.PagedCache(k.float(), k.float(), t, n), "fp16 or bf16"),
                     (lambda: hb.PagedCache(k.transpose(2, 3), k.transpose(2, 3), t, n), "contiguous"),
                     (lambda: hb.PagedCache(k, k, t.long(), n), "int32"),
                     (lambda: hb.PagedCache(k, k, t, n.float()), "lengths"),
                     (lambda: hb.PagedCache(k, k, t, n, weights=torch.zeros(1, 2, 47)), "weights"),
                     (lambda: ok.decode(torch.zeros(2, 4, 64, dtype=k.dtype), None, 1.0), "seqs"),
                     (lambda: ok.decode(torch.zeros(1, 4, 64), torch.zeros(1, 4, 64), 1.0), "type"),
                     (lambda: ok.decode(torch.zeros(1, 4, 32, dtype=k.dtype), torch.zeros(1, 4, 32, dtype=k.dtype), 1.0), "head_dim"),
                     (lambda: ok.prompt(torch.zeros(1, 4, 64, dtype=k.dtype), torch.zeros(1, 4, 64, dtype=k.dtype), t[0], 1, 1.0), "starts"),
                     (lambda: ok.append(k[0, :, :3], k[0, :, :3], n, n), "rows"),
                     (lambda: ok.evict(None, 4), "PagedCache"),
                     (lambda: ok.evict(ok, 4, kept=torch.zeros(1, 2, 5, dtype=torch.int32)), "kept")):
        with pytest.raises(hb.HcError, match=why):
            bad()


@pytest.mark.parametrize("kw", [dict(o_row=0), dict(o_head=0), dict(o_row=120), dict(o_head=64)])
def test_an_output_that_overlaps_itself_is_refused(kw):
    for call in calls(cache(), attn(**kw)):
        with pytest.raises(hb.HcError, match="overlap"):
            call()


def test_tensors_that_are_not_on_the_gpu_are_refused():
    torch = pytest.importorskip("torch")
    bf = torch.bfloat16
    k = torch.zeros((4, 2, 16, 64), dtype=bf)
    t, n, w = torch.zeros((1, 3), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2, 48))
    c = hb.PagedCache(k, k.clone(), t, n, weights=w)
    to = hb.PagedCache(k.clone(), k.clone(), t.clone(), n.clone(), weights=w.clone())
    q, new, starts = torch.zeros((1, 4, 64), dtype=bf), torch.zeros((1, 2, 64), dtype=bf), torch.zeros(2, dtype=torch.int32)
    scratch = torch.zeros(1 << 16, dtype=torch.uint8)
    for call in (lambda: c.decode(q, q.clone(), 1.0, scratch=scratch), lambda: c.append(new, new, n, n),
                 lambda: c.prompt(q, q.clone(), starts, 1, 1.0, scratch=scratch), lambda: c.evict(to, 4, scratch=scratch)):
        with pytest.raises(hb.HcError, match="on a GPU"):
            call()
    with pytest.raises(hb.HcError, match="one device"):
        hb.PagedCache(k, torch.zeros((4, 2, 16, 64), dtype=bf, device="meta"), t, n)


@pytest.mark.gpu
def test_tensors_of_another_place_are_refused():
    # refused by the binding: no kernel sees any of these addresses
    torch = pytest.importorskip("torch")
    bf, dev = torch.bfloat16, "cuda"
    k = torch.zeros((4, 2, 16, 64), dtype=bf, device=dev)
    t, n = torch.zeros((1, 3), dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    w = torch.zeros((1, 2, 48), device=dev)
    c = hb.PagedCache(k, k.clone(), t, n, weights=w)
    to = hb.PagedCache(k.clone(), k.clone(), t.clone(), n.clone(), weights=w.clone())
    q, new, starts = torch.zeros((1, 4, 64), dtype=bf, device=dev), torch.zeros((1, 2, 64), dtype=bf, device=dev), n.new_tensor([0, 1])
    sinks, scratch = torch.zeros(4, device=dev), torch.zeros(1 << 16, dtype=torch.uint8, device=dev)
    kept = torch.zeros((1, 2, 4), dtype=torch.int32, device=dev)
    calls = {"decode": (lambda q, out, sinks, scratch: c.decode(q, out, 1.0, sinks=sinks, scratch=scratch), [q, q.clone(), sinks, scratch]),
             "prompt": (lambda q, out, starts, sinks, scratch: c.prompt(q, out, starts, 1, 1.0, sinks=sinks, scratch=scratch),
                        [q, q.clone(), starts, sinks, scratch]),
             "append": (c.append, [new, new.clone(), n - 1, n - 1]),
             "evict": (lambda kept, scratch: c.evict(to, 4, kept=kept, scratch=scratch), [kept, scratch])}
    for f, good in calls.values():
        f(*good)
        for i in range(len(good)):
            with pytest.raises(hb.HcError, match="cache's GPU"):
                f(*[x.cpu() if i == j else x for j, x in enumerate(good)])
        for held in {c, to} if f is calls["evict"][0] else {c}:
            held.desc.device = 2  # as if it were on another GPU than the current one
            with pytest.raises(hb.HcError, match="device 0 is current"):
                f(*good)
            held.desc.device = 1
    torch.cuda.synchronize()
    for bad in ({"v": k.cpu()}, {"block_table": t.cpu()}, {"lengths": n.cpu()}, {"weights": w.cpu()}):
        with pytest.raises(hb.HcError, match="one device"):
            hb.PagedCache(**{**dict(k=k, v=k, block_table=t, lengths=n, weights=w), **bad})
