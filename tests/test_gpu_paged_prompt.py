"""The tensor-core prompt kernel of a caller's paged 16-bit cache (hc_paged_prompt_run with more than 16 rows a kv head:
fewer run as decode does), where test_gpu_paged_cache.py leaves off. Same plain implementation, same bounds."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import hwnpu_b200 as hb
from hwnpu_b200 import _abi as A
from test_gpu_paged_cache import BF, FP, U, Case, check_out, ref_rows, run_prompt

pytestmark = pytest.mark.gpu


def starts_of(rows):
    return torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")


def prompt(cache, q, rows, scale=0.1, max_len=0, out=None, scratch=None, stream=None, starts=None, **kw):
    out = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype) if out is None else out
    if scratch is None:
        n = cache.prompt_scratch(q.shape[1], q.shape[0], max(rows), max_len, kw.get("window", 0), kw.get("first", 0))
        scratch = torch.full((max(16, n),), 255, dtype=torch.uint8, device="cuda")
    cache.prompt(q, out, starts_of(rows) if starts is None else starts, max(rows), scale, max_len=max_len, scratch=scratch,
                 stream=stream, **kw)
    return out


def check(c, q, out, rows, scale=0.1, lens=None):
    """out against the plain form in float64, at the lengths given (Case's own if none)."""
    torch.cuda.synchronize()
    at, held = 0, c.lens
    c.lens = held if lens is None else lens
    for i, r in enumerate(rows):
        p = torch.arange(c.lens[i] - r, c.lens[i], device="cuda")
        o, mag, _ = ref_rows(c, i, q[at : at + r].double(), p, scale, 0, 0, None)
        check_out(out[at : at + r], o, mag, c.dtype)
        at += r
    c.lens = held


@pytest.mark.parametrize("dtype,heads,hd", [(BF, 8, 128), (FP, 32, 128), (BF, 32, 64)])
def test_many_blocks_a_cta(device, dtype, heads, hd):
    # Each CTA walks 7 to 17 blocks of 1 to 6 half tiles, odd and even numbers of them one behind the other: a block's
    # scores must not overtake the softmax of the one before. The results repeat bit for bit, and no wait runs out.
    lens = [1 + (37 * i) % 330 for i in range(96)]
    outs = []
    for _ in range(3):
        outs.append(run_prompt(Case(lens, heads, 8, hd, 16, dtype, seed=5), lens))
        A.check(A.lib().hc_device_check(device.h))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("scale", [-0.1, 0.0, -3.0])
@pytest.mark.parametrize("heads,kv,hd,dtype", [(16, 8, 128, BF), (16, 4, 64, FP)])
@pytest.mark.parametrize("rows", [[3, 1, 2], [300, 40, 129]])
def test_negative_and_zero_scale(scale, heads, kv, hd, dtype, rows):
    # 0: the mean of the visible values. -3: one key takes nearly everything, and a float32 score is too coarse for the
    # bounds on weights, so the bits of +3 with every key's sign turned
    c = Case([300, 57, 1130], heads, kv, hd, 32, dtype)
    q = c.queries(sum(rows))
    out = prompt(c.cache(), q, rows, scale)
    if scale == -3.0:
        big = Case([300, 57, 1130], heads, kv, hd, 32, dtype)
        big.k.neg_()
        assert torch.equal(out, prompt(big.cache(), big.queries(sum(rows)), rows, 3.0))
    else:
        check(c, q, out, rows, scale)


@pytest.mark.parametrize("hd,ps", [(64, 16), (64, 64), (128, 16), (128, 128), (128, 1024)])
@pytest.mark.parametrize("rows", [[40, 9], [300, 129]])
def test_page_ids_outside_the_pool_read_as_zeros(hd, ps, rows):
    n = 6 * ps + 5 if ps < 1024 else 2 * ps + 5
    outs = []
    for broken in (True, False):
        c = Case([max(n, 320), max(n, 140)], 16, 8, hd, ps)
        for i, bad in ((0, 1 << 30), (1, -5)):
            page = 1 if ps < 1024 else i  # in the middle of what the rows see
            slots = torch.arange(page * ps, min(c.lens[i], (page + 1) * ps), device="cuda")
            c.put(i, slots, torch.zeros(len(slots), 8, hd, device="cuda"), torch.zeros(len(slots), 8, hd, device="cuda"))
            if broken:
                c.put(i, slots, torch.ones(len(slots), 8, hd, device="cuda"), torch.ones(len(slots), 8, hd, device="cuda"))
                c.table[i, page] = bad
        if broken:
            c.table[1, -1] = c.k.shape[0]  # past the sequence's end: never read
        outs.append(prompt(c.cache(), c.queries(sum(rows)), rows))
    assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("hd,pages", [(64, 8400), (128, 4200)])
def test_offsets_past_32_bits(hd, pages):
    # pools of more than 2^32 elements; the sequence's pages are the last ones
    ps, kv = 1024, 8
    k, v = (torch.empty((pages, kv, ps, hd), device="cuda", dtype=BF) for _ in range(2))
    small = Case([1500], 16, kv, hd, ps)
    table = torch.tensor([[pages - 1, pages - 2, 0]], dtype=torch.int32, device="cuda")
    for new, old in zip(table[0].tolist(), small.table[0].tolist()):
        k[new], v[new] = small.k[old], small.v[old]
    big = hb.PagedCache(k, v, table, small.lengths)
    q = small.queries(700)
    assert torch.equal(prompt(small.cache(), q, [700]), prompt(big, q, [700]))


@pytest.mark.parametrize("hd", [64, 128])
def test_on_another_stream_and_in_a_graph(hd):
    rows = [300, 40]
    c = Case([700, 90], 16, 8, hd)
    a, starts, q = c.cache(), starts_of(rows), c.queries(sum(rows))
    outs = [torch.zeros(q.shape, device="cuda", dtype=BF) for _ in range(3)]
    scratch = torch.zeros(max(16, a.prompt_scratch(16, 340, 300, 1000)), dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    prompt(a, q, rows, max_len=1000, out=outs[0], scratch=scratch, starts=starts, stream=st.cuda_stream)
    st.synchronize()
    check(c, q, outs[0], rows)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        prompt(a, q, rows, max_len=1000, out=outs[1], scratch=scratch, starts=starts,
               stream=torch.cuda.current_stream().cuda_stream)
    c.put(0, torch.arange(700, 703, device="cuda"), c.randn(3, 8, hd), c.randn(3, 8, hd))
    for lens in ([700, 90], [305, 3], [703, 0], [700, 90]):  # the graph reads the lengths of the moment
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        check(c, q, outs[1], rows, lens=lens)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("heads,kv,hd", [(16, 8, 128), (64, 8, 64)])
def test_longer_than_the_bound(heads, kv, hd):
    # max_len only plans the cut: sequences beyond it are still read whole
    for rows in ([40, 700, 300], [1, 90, 17]):
        for bound in (1, 64, 2000):
            run_prompt(Case([40, 3000, 900], heads, kv, hd), rows, max_len=bound)


@pytest.mark.parametrize("hd", [64, 128])
def test_lengths_outside_the_capacity_are_held_to_it(hd):
    c = Case([640, 20], 16, 8, hd, spare=0)
    c.lengths.copy_(torch.tensor([1 << 20, -3], dtype=torch.int32))
    rows = [200, 20]
    q = c.queries(220)
    out = prompt(c.cache(), q, rows)
    check(c, q, out, rows, lens=[640, 0])
    assert float(out[200:].abs().max()) == 0.0


@pytest.mark.parametrize("heads,kv,hd,dtype", [(16, 8, 128, BF), (64, 8, 64, BF), (8, 8, 128, FP)])
def test_last_rows_agree_with_decode(heads, kv, hd, dtype):
    c = Case([41, 77, 1500, 4001], heads, kv, hd, 16, dtype)
    rows = [41, 60, 1, 300]
    q = c.queries(sum(rows))
    a = c.cache()
    last = torch.tensor(np.cumsum(rows) - 1, device="cuda")
    dec = torch.zeros((4, heads, hd), device="cuda", dtype=dtype)
    a.decode(q[last].contiguous(), dec, 0.09,
             scratch=torch.zeros(max(16, a.decode_scratch(heads)), dtype=torch.uint8, device="cuda"))
    # two roundings of weights and results, each at most the type's unit of values below 4
    assert float((prompt(a, q, rows, 0.09)[last].double() - dec.double()).abs().max()) <= 2 * U[dtype] * 4


def test_a_wait_that_ran_out_is_reported_without_a_device_handle(device):
    c = Case([300], 16, 8, 64)
    rows = [300]
    q = c.queries(300)
    out = prompt(c.cache(), q, rows)
    hb.PagedCache.check()
    check(c, q, out, rows)
    A.check(A.lib().hc_set_fault(b"wait:1"))  # on the host: no wait on the GPU runs out
    with pytest.raises(hb.HcError, match="prompt attention ran out"):
        c.cache().check()
    hb.PagedCache.check()  # cleared
    A.check(A.lib().hc_set_fault(b"wait:1"))
    with pytest.raises(hb.HcError, match="prompt attention ran out"):
        A.check(A.lib().hc_device_check(device.h))
    A.check(A.lib().hc_device_check(device.h))
