"""The operators of a caller's paged 16-bit cache (hc_paged_*, hwnpu_b200.PagedCache) against a plain
implementation in float64 (this file's ref_*), at the lengths, layouts and masks where they can go
wrong. Slots that no query sees hold NaN throughout.

Bounds, from the arithmetic: a kernel reads 16-bit values exactly, sums in float32 and rounds the result
once to the output's type (by at most u = 2^-8 of it for bf16, 2^-11 for fp16), and may round each
softmax weight to that type too. A float32 score
of up to 128 products is off by less than 128 * 2^-24 * sum|q k| * scale, below 1e-4 for the inputs
here, which moves a weight by as much relatively (and its sum by no more). So
  |o - ref| <= u |ref| + (u + 2e-4) sum_j w_j |v_j| + 1e-7
and an accumulated weight w0 + dw is within 2e-4 dw + 2^-22 (w0 + dw) + 1e-9."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import hwnpu_b200 as hb

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, FP = torch.bfloat16, torch.float16


class Case:
    """A cache of sequences with the given lengths over shuffled pages; every unused slot is NaN."""

    def __init__(self, lens, heads=16, kv=8, hd=128, ps=16, dtype=BF, layout="hnd", seed=0, spare=1, mean=0.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.lens, self.heads, self.kv, self.hd, self.ps, self.dtype = g, list(lens), heads, kv, hd, ps, dtype
        S = len(lens)
        self.width = max(1, -(-max(lens) // ps)) + spare
        pages = S * self.width + 2
        shape = (pages, kv, ps, hd) if layout == "hnd" else (pages, ps, kv, hd)
        self.k, self.v = (torch.full(shape, float("nan"), device="cuda", dtype=dtype) for _ in range(2))
        if layout == "nhd":
            self.k, self.v = self.k.permute(0, 2, 1, 3), self.v.permute(0, 2, 1, 3)
        self.table = torch.randperm(pages, device="cuda", generator=g)[: S * self.width].to(torch.int32).view(S, -1)
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.weights = torch.rand((S, kv, self.width * ps), device="cuda", generator=g)
        for i, n in enumerate(self.lens):
            if n:
                self.put(i, torch.arange(n, device="cuda"), self.randn(n, kv, hd), self.randn(n, kv, hd) + mean)

    def randn(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.g)

    def where(self, i, slots):
        return self.table[i].long()[slots // self.ps], slots % self.ps

    def put(self, i, slots, k, v):
        page, r = self.where(i, slots)
        self.k[page, :, r] = k.to(self.dtype)
        self.v[page, :, r] = v.to(self.dtype)

    def hide(self, i, slots):
        page, r = self.where(i, slots)
        self.k[page, :, r] = float("nan")
        self.v[page, :, r] = float("inf")

    def rows(self, i, h):
        """Keys and values of sequence i's slots, float64 [n][hd]."""
        page, r = self.where(i, torch.arange(self.lens[i], device="cuda"))
        return self.k[page, h, r].double(), self.v[page, h, r].double()

    def cache(self, weights=True):
        return hb.PagedCache(self.k, self.v, self.table, self.lengths, weights=self.weights if weights else None)

    def queries(self, n):
        """A strided view of a fused q|k|v projection."""
        return self.randn(n, self.heads + 2 * self.kv, self.hd).to(self.dtype)[:, : self.heads]


def ref_rows(c, i, q, p, scale, window, first, sinks):
    """q float64 [rows][heads][hd] at slots p of sequence i: (o, sum w|v|) [rows][heads][hd] and the
    weights summed over the rows and the kv head's heads [kv][n], all float64."""
    rep = c.heads // c.kv
    o, mag = torch.zeros_like(q), torch.zeros_like(q)
    acc = torch.zeros((c.kv, c.lens[i]), dtype=torch.float64, device="cuda")
    if not c.lens[i]:
        return o, mag, acc
    j = torch.arange(c.lens[i], device="cuda").view(1, -1)
    p = p.view(-1, 1)
    see = (j <= p) & (((p - j) < window) | (j < first) if window else torch.ones_like(j <= p))
    for h in range(c.kv):
        k, v = c.rows(i, h)
        for r in range(rep):
            x = h * rep + r
            s = torch.where(see, (q[:, x].unsqueeze(1) * k.nan_to_num(0.0)).sum(-1) * scale, -math.inf) \
                if q.shape[0] * c.lens[i] < 20000 else torch.where(see, q[:, x] @ k.nan_to_num(0.0).T * scale, -math.inf)
            m = s.amax(1, keepdim=True)
            if sinks is not None:
                m = torch.clamp(m, min=float(sinks[x]))
            m = torch.where(m == -math.inf, torch.zeros_like(m), m)
            e = torch.exp(s - m)
            l = e.sum(1, keepdim=True) + (torch.exp(sinks[x].double() - m) if sinks is not None else 0.0)
            w = torch.where(l > 0, e / l, torch.zeros_like(e))
            fv = torch.where(see.any(0).view(-1, 1), v, torch.zeros_like(v))
            o[:, x], mag[:, x] = w @ fv, w @ fv.abs()
            acc[h] += w.sum(0)
    return o, mag, acc


def check_out(got, o, mag, dtype):
    u = U[dtype]
    err = (got.double() - o).abs()
    bound = u * o.abs() + (u + 2e-4) * mag + 1e-7
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), float((err / bound).max())


def run_decode(c, window=0, first=0, sinks=False, accumulate=False, max_len=None, stream=None, scale=None):
    S = len(c.lens)
    scale = scale or c.hd ** -0.5
    for i, n in enumerate(c.lens):  # what the mask hides may hold anything
        if window and n > window:
            lo = max(first, 0)
            if n - window > lo:
                c.hide(i, torch.arange(lo, n - window, device="cuda"))
    q = c.queries(S)
    out = torch.full((S, c.heads, c.hd), 7.0, device="cuda", dtype=c.dtype)
    sk = c.randn(c.heads) if sinks else None
    cache = c.cache()
    max_len = max(c.lens) if max_len is None else max_len
    scratch = torch.full((max(16, cache.decode_scratch(c.heads, max_len, window, first, accumulate)),), 255,
                         device="cuda", dtype=torch.uint8)
    before = c.weights.double()
    cache.decode(q, out, scale, window=window, first=first, sinks=sk, accumulate=accumulate, max_len=max_len,
                 scratch=scratch, stream=stream)
    torch.cuda.synchronize()
    for i in range(S):
        o, mag, acc = ref_rows(c, i, q[i : i + 1].double(), torch.tensor([c.lens[i] - 1], device="cuda"), scale, window,
                               first, sk)
        check_out(out[i : i + 1], o, mag, c.dtype)
        if accumulate:
            n = c.lens[i]
            got, want = c.weights[i].double(), before[i].clone()
            want[:, :n] += acc
            bound = torch.full_like(want, 0.0)
            bound[:, :n] = 2e-4 * acc + 2.0 ** -22 * want[:, :n] + 1e-9
            assert bool(((got - want).abs() <= bound).all())
    if not accumulate:
        assert torch.equal(c.weights.double(), before)
    return out


RAGGED = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 1023, 1025]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,heads,kv,hd,ps,layout", [
    (BF, 16, 8, 128, 16, "hnd"), (FP, 16, 8, 128, 32, "nhd"), (BF, 64, 8, 64, 16, "nhd"), (FP, 16, 4, 64, 128, "hnd"),
    (BF, 5, 1, 128, 64, "hnd"), (FP, 3, 3, 64, 16, "hnd"), (BF, 24, 2, 128, 16, "nhd"), (FP, 40, 2, 64, 256, "hnd")])
def test_decode_lengths(dtype, heads, kv, hd, ps, layout, accumulate):
    run_decode(Case(RAGGED, heads, kv, hd, ps, dtype, layout), accumulate=accumulate)


@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (16, 4), (33, 17), (128, 4), (128, 200), (5000, 64)])
@pytest.mark.parametrize("sinks", [False, True])
def test_decode_window_and_first(window, first, sinks):
    run_decode(Case(RAGGED, 64, 8, 64, 16), window, first, sinks, accumulate=True)
    run_decode(Case(RAGGED[::2] + [3001], 16, 8, 128, 32, FP, "nhd", seed=1), window, first, sinks)


@pytest.mark.parametrize("n", [1, 700, 4096, 20011, 70003])
@pytest.mark.parametrize("accumulate", [False, True])
def test_decode_one_long(n, accumulate):
    run_decode(Case([n], 32, 8, 128, 64, seed=n), accumulate=accumulate)


def test_decode_longer_than_the_bound():
    # max_len only plans the split: sequences beyond it are still read whole
    run_decode(Case([40, 3000, 900]), max_len=64, accumulate=True)
    run_decode(Case([40, 3000, 900], 64, 8, 64), max_len=1)


def test_decode_large_scores_and_equal_keys():
    c = Case([300, 4000], mean=1.0)
    run_decode(c, scale=40.0)  # one key takes nearly everything
    run_decode(Case([300, 4000], dtype=FP, mean=1.0), scale=1e-6)  # all weights alike


def test_decode_same_result_twice():
    c = Case([5000, 100, 2500], 32, 8, 128)
    a = c.cache()
    q, scratch = c.queries(3), torch.zeros(a.decode_scratch(32, 5000, accumulate=True) + 16, dtype=torch.uint8, device="cuda")
    w0, outs = c.weights.clone(), []
    for _ in range(3):
        c.weights.copy_(w0)
        out = torch.zeros((3, 32, 128), device="cuda", dtype=BF)
        a.decode(q, out, 0.1, accumulate=True, max_len=5000, scratch=scratch)
        outs.append((out, c.weights.clone()))
    assert all(torch.equal(outs[0][0], o) and torch.equal(outs[0][1], w) for o, w in outs[1:])


def run_prompt(c, rows, window=0, first=0, sinks=False, max_rows=None, max_len=None, scale=None, pad=0):
    S, T = len(c.lens), sum(rows)
    scale = scale or c.hd ** -0.5
    for i, n in enumerate(c.lens):
        p0 = n - rows[i]
        if window and p0 - window + 1 > first:
            c.hide(i, torch.arange(first, p0 - window + 1, device="cuda"))
    q = c.queries(T + pad)[pad:] if pad else c.queries(T)
    out = torch.full((T, c.heads, c.hd), 7.0, device="cuda", dtype=c.dtype)
    sk = c.randn(c.heads) if sinks else None
    starts = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    cache = c.cache(weights=False)
    max_rows = max(rows) if max_rows is None else max_rows
    max_len = max(c.lens) if max_len is None else max_len
    scratch = torch.full((max(16, cache.prompt_scratch(c.heads, T, max_rows, max_len, window, first)),), 255,
                         device="cuda", dtype=torch.uint8)
    cache.prompt(q, out, starts, max_rows, scale, window=window, first=first, sinks=sk, max_len=max_len, scratch=scratch)
    torch.cuda.synchronize()
    at = 0
    for i in range(S):
        r = rows[i]
        p = torch.arange(c.lens[i] - r, c.lens[i], device="cuda")
        o, mag, _ = ref_rows(c, i, q[at : at + r].double(), p, scale, window, first, sk)
        check_out(out[at : at + r], o, mag, c.dtype)
        at += r
    return out


LENS = [0, 1, 16, 17, 100, 127, 128, 129, 300, 700]


@pytest.mark.parametrize("dtype,heads,kv,hd,ps,layout", [
    (BF, 16, 8, 128, 16, "hnd"), (FP, 16, 8, 128, 32, "nhd"), (BF, 64, 8, 64, 16, "nhd"), (FP, 16, 4, 64, 128, "hnd"),
    (BF, 5, 1, 128, 64, "hnd"), (FP, 3, 3, 64, 16, "hnd"), (BF, 24, 2, 128, 1024, "nhd"), (FP, 20, 4, 128, 16, "hnd")])
def test_prompt_whole(dtype, heads, kv, hd, ps, layout):
    run_prompt(Case(LENS, heads, kv, hd, ps, dtype, layout), LENS)


@pytest.mark.parametrize("window,first", [(1, 0), (7, 3), (16, 16), (128, 4), (100, 130), (129, 1), (4096, 64)])
@pytest.mark.parametrize("sinks", [False, True])
def test_prompt_window_and_first(window, first, sinks):
    run_prompt(Case(LENS, 64, 8, 64, 16), LENS, window, first, sinks)
    run_prompt(Case([900, 40], 16, 8, 128, 32, FP, "nhd", seed=2), [500, 40], window, first, sinks)


@pytest.mark.parametrize("rows", [1, 2, 5, 31, 64, 130])
def test_prompt_few_rows_over_a_long_cache(rows):
    run_prompt(Case([9001, 200], 16, 8, 128, 16, seed=rows), [rows, rows])
    run_prompt(Case([5003], 32, 8, 128, 64, FP, seed=rows), [rows], window=1000, first=20)


def test_prompt_rows_that_see_nothing():
    # more rows than slots: the first ones lie before the cache and see nothing
    out = run_prompt(Case([3, 0, 200]), [10, 4, 7])
    assert float(out[:7].abs().max()) == 0.0 and float(out[10:14].abs().max()) == 0.0
    run_prompt(Case([3, 0, 200], 64, 8, 64), [10, 4, 7], window=4, sinks=True)


def test_prompt_sequences_without_rows():
    run_prompt(Case([50, 300, 20, 0, 128]), [0, 40, 0, 0, 128])


def test_prompt_max_rows_bounds_what_is_written():
    c = Case([100, 300])
    q, out = c.queries(340), torch.full((340, 16, 128), 7.0, device="cuda", dtype=BF)
    starts = torch.tensor([0, 40, 340], dtype=torch.int32, device="cuda")
    a = c.cache()
    scratch = torch.zeros(a.prompt_scratch(16, 340, 64, 300) + 16, dtype=torch.uint8, device="cuda")
    a.prompt(q, out, starts, 64, 0.1, max_len=300, scratch=scratch)
    torch.cuda.synchronize()
    assert bool((out[40 + 64 :] == 7.0).all())
    o, mag, _ = ref_rows(c, 1, q[40:104].double(), torch.arange(0, 64, device="cuda"), 0.1, 0, 0, None)
    check_out(out[40:104], o, mag, BF)


def test_prompt_large_scores():
    run_prompt(Case([500], mean=1.0), [500], scale=20.0)
    run_prompt(Case([500], dtype=FP, mean=1.0), [500], scale=20.0)
    run_prompt(Case([2500], dtype=FP, mean=1.0), [300], scale=1e-6)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_prompt_maximum_that_moves_at_every_half_tile(hd, dtype):
    # keys along one direction, 8 nats of score a 64 slots for a query of unit length along it, up or down: the running
    # maximum is passed by more than 2^8 again and again, at the first and last half of tiles too. Scores stay
    # below 300, so that a float32 score is off by less than 300 * 2^-22 < 1e-4 of a weight.
    lens = [64, 65, 128, 129, 192, 193, 257, 330]
    c = Case(lens, 8, 4, hd, 16, dtype)
    u = c.randn(c.kv, hd)
    for i, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        c.put(i, j, (j / 8.0).view(-1, 1, 1) * u + c.randn(n, c.kv, hd), c.randn(n, c.kv, hd))
    run_prompt(c, lens)
    run_prompt(c, [min(n, 70) for n in lens])


@pytest.mark.parametrize("heads,kv,hd,dtype", [(8, 4, 128, BF), (16, 4, 64, FP), (10, 2, 128, FP), (4, 4, 64, BF)])
@pytest.mark.parametrize("window", [0, 900])
@pytest.mark.parametrize("sinks", [False, True])
def test_decode_of_few_sequences_is_split_and_joined(heads, kv, hd, dtype, window, sinks):
    # few enough for one cluster a row; sequences of one group and of none among long ones
    for accumulate in (False, True):
        run_decode(Case([0, 7, 1500, 300, 2047], heads, kv, hd, 16, dtype), window, 5, sinks, accumulate)
    if heads // kv <= 3:
        run_prompt(Case([1500, 5, 300, 2047], heads, kv, hd, 32, dtype), [5, 3, 0, 1], window, 5, sinks)


def test_prompt_and_decode_agree_on_one_row():
    c = Case([1, 77, 1500, 4001], 16, 8, 128, 16)
    q = c.queries(4)
    outs = []
    a = c.cache()
    for prompt in (False, True):
        out = torch.zeros((4, 16, 128), device="cuda", dtype=BF)
        if prompt:
            n = a.prompt_scratch(16, 4, 1, 4001)
            a.prompt(q, out, torch.arange(5, dtype=torch.int32, device="cuda"), 1, 0.09, max_len=4001,
                     scratch=torch.zeros(n + 16, dtype=torch.uint8, device="cuda"))
        else:
            n = a.decode_scratch(16, 4001)
            a.decode(q, out, 0.09, max_len=4001, scratch=torch.zeros(n + 16, dtype=torch.uint8, device="cuda"))
        outs.append(out.double())
    # two roundings of weights and results, each at most the type's unit of values below 4
    assert float((outs[0] - outs[1]).abs().max()) <= 2 * U[BF] * 4


def test_offsets_past_32_bits():
    # pools of more than 2^32 elements; the sequence's pages are the last ones
    ps, kv, hd, pages = 1024, 8, 128, 4200
    k, v = (torch.empty((pages, kv, ps, hd), device="cuda", dtype=BF) for _ in range(2))
    small = Case([1500], 16, kv, hd, ps)
    table = torch.tensor([[pages - 1, pages - 2, 0]], dtype=torch.int32, device="cuda")
    for new, old in zip(table[0].tolist(), small.table[0].tolist()):
        k[new], v[new] = small.k[old], small.v[old]
    big = hb.PagedCache(k, v, table, small.lengths, weights=small.weights)
    q = small.queries(1)
    scratch = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    outs = []
    for cache in (small.cache(), big):
        o1, o2 = (torch.zeros((1, 16, hd), device="cuda", dtype=BF) for _ in range(2))
        cache.decode(q, o1, 0.1, scratch=scratch)
        cache.prompt(q, o2, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1, 0.1, scratch=scratch)
        outs.append((o1, o2))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    new = small.randn(1, kv, hd).to(BF)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    big.append(new, new, one, one + 1499)
    assert torch.equal(k[pages - 2, :, 1499 - 1024], new[0]) and torch.equal(v[pages - 2, :, 1499 - 1024], new[0])


@pytest.mark.parametrize("hd", [64, 128])
def test_page_ids_outside_the_pool_read_as_zeros(hd):
    c = Case([40, 40], 16, 8, hd)
    zero = Case([40, 40], 16, 8, hd)
    zero.put(0, torch.arange(16, 32, device="cuda"), torch.zeros(16, 8, hd, device="cuda"), torch.zeros(16, 8, hd, device="cuda"))
    c.table[0, 1] = 1 << 30
    c.table[1, 3] = -5  # past the sequence's end: never read
    q = c.queries(2)
    outs = []
    for x in (c, zero):
        a = x.cache()
        o1, o2 = (torch.zeros((2, 16, hd), device="cuda", dtype=BF) for _ in range(2))
        scratch = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
        a.decode(q, o1, 0.1, scratch=scratch)
        a.prompt(q, o2, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), 1, 0.1, scratch=scratch)
        outs += [o1, o2]
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_lengths_outside_the_capacity_are_held_to_it():
    c = Case([64, 20], spare=0)
    want = Case([64, 0], spare=0)
    want.k, want.v, want.table = c.k, c.v, c.table
    c.lengths.copy_(torch.tensor([1 << 20, -3], dtype=torch.int32))
    q = c.queries(2)
    scratch = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    outs = []
    for x in (c, want):
        out = torch.full((2, 16, 128), 7.0, device="cuda", dtype=BF)
        x.cache().decode(q, out, 0.1, scratch=scratch)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and float(outs[0][1].abs().max()) == 0.0


# ---- evict ------------------------------------------------------------------------------------


def ref_kept(w, n, keep, first, recent):
    """The slots that stay, from the rule: numpy float32 weights of one head."""
    if n <= keep:
        return np.arange(n)
    body = np.arange(first, n - recent)
    key = np.where(np.isnan(w[body]), -np.inf, w[body].astype(np.float64))
    nan = np.isnan(w[body])
    order = np.lexsort((body, nan, -key))[: keep - first - recent]
    return np.concatenate([np.arange(first), np.sort(body[order]), np.arange(n - recent, n)])


def run_evict(c, keep, first, recent, to=None, kept=True):
    S = len(c.lens)
    to = to or Case([keep] * S, c.heads, c.kv, c.hd, c.ps, c.dtype, seed=9)
    to.lengths.fill_(-1)
    kp = torch.full((S, c.kv, keep), 77, dtype=torch.int32, device="cuda") if kept else None
    a = c.cache()
    scratch = torch.full((a.evict_scratch(keep),), 255, dtype=torch.uint8, device="cuda")
    a.evict(to.cache(), keep, first=first, recent=recent, kept=kp, scratch=scratch)
    torch.cuda.synchronize()
    w = c.weights.cpu().numpy()
    for i, n in enumerate(c.lens):
        assert int(to.lengths[i]) == min(n, keep)
        for h in range(c.kv):
            want = ref_kept(w[i, h, :n], n, keep, first, recent)
            if kept:
                got = kp[i, h].cpu().numpy()
                assert np.array_equal(got[: len(want)], want), (i, h)
                assert (got[len(want) :] == -1).all()
            src, dst = torch.from_numpy(want).cuda(), torch.arange(len(want), device="cuda")
            for x, y in ((c.k, to.k), (c.v, to.v)):
                page, r = c.where(i, src)
                tp, tr = to.where(i, dst)
                assert torch.equal(x[page, h, r].view(torch.int16), y[tp, h, tr].view(torch.int16))
            assert np.array_equal(to.weights[i, h, : len(want)].cpu().numpy().view(np.int32), w[i, h, want].view(np.int32))


@pytest.mark.parametrize("dtype,kv,hd,ps,layout", [(BF, 8, 128, 16, "hnd"), (FP, 8, 64, 32, "nhd"), (FP, 1, 128, 128, "hnd")])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (64, 4, 16), (64, 0, 64), (100, 1, 0), (257, 7, 100), (1000, 0, 0)])
def test_evict(dtype, kv, hd, ps, layout, keep, first, recent):
    run_evict(Case([0, 1, 63, 64, 65, 256, 257, 258, 999, 1001, 2500], 2 * kv, kv, hd, ps, dtype, layout), keep, first, recent)


def test_evict_ties_zeros_and_nan():
    c = Case([3000, 3000, 3000, 3000], 8, 8, 64)
    c.weights[0] = 0.0  # all alike: the lowest slots stay
    c.weights[1] = torch.where(c.weights[1] < 0.5, torch.zeros_like(c.weights[1]), -torch.zeros_like(c.weights[1]))
    c.weights[2] = torch.floor(c.weights[2] * 4)  # many equal ones at the threshold
    c.weights[3, :, ::3] = float("nan")
    c.weights[3, :, 1::7] = float("inf")
    c.weights[3, :, 2::7] = -float("inf")
    run_evict(c, 500, 3, 20)
    run_evict(c, 2990, 3, 20)
    run_evict(c, 2999, 0, 0)


@pytest.mark.parametrize("n", [33000, 131072 + 17])
def test_evict_long(n):
    c = Case([n, 100], 4, 2, 64, 64)
    c.weights.pow_(8)
    run_evict(c, 4000, 4, 256)
    run_evict(c, 20000, 0, 1, kept=False)


def test_evict_into_pages_of_the_same_pool():
    c = Case([200, 150, 40], spare=6)
    to = Case([64] * 3)
    free = c.table[:, -6:].contiguous()
    keep_k, keep_v = c.k.clone(), c.v.clone()
    to.k, to.v, to.table, to.width = c.k, c.v, free, 6
    to.weights = torch.zeros((3, 8, 96), device="cuda")
    run_evict(c, 64, 4, 8, to=to)
    used = c.table[:, :-6].reshape(-1).long()
    assert torch.equal(c.k[used].view(torch.int16), keep_k[used].view(torch.int16))
    assert torch.equal(c.v[used].view(torch.int16), keep_v[used].view(torch.int16))


# ---- append, streams, graphs ------------------------------------------------------------------


@pytest.mark.parametrize("dtype,kv,hd,ps,layout", [(BF, 8, 128, 16, "hnd"), (FP, 4, 64, 32, "nhd"), (BF, 1, 128, 64, "nhd")])
def test_append(dtype, kv, hd, ps, layout):
    c = Case([40, 0, 100], 2 * kv, kv, hd, ps, dtype, layout)
    fused = c.randn(9, 4 * kv, hd).to(dtype)
    nk, nv = fused[:, 2 * kv : 3 * kv], fused[:, 3 * kv :]
    seq = torch.tensor([0, 0, 1, 2, 2, 0, 3, -1, 1], dtype=torch.int32, device="cuda")
    slot = torch.tensor([40, 41, 0, 100, 17, -1, 0, 5, 1 << 29], dtype=torch.int32, device="cuda")
    k, v, w = c.k.clone(), c.v.clone(), c.weights.clone()
    c.cache().append(nk, nv, seq, slot)
    torch.cuda.synchronize()
    for r in range(5):  # the other rows are out of range
        i, j = int(seq[r]), int(slot[r])
        page = int(c.table[i, j // ps])
        k[page, :, j % ps], v[page, :, j % ps] = nk[r], nv[r]
        w[i, :, j] = 0.0
    assert torch.equal(c.k.view(torch.int16), k.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), v.view(torch.int16))
    assert torch.equal(c.weights, w)


def test_on_another_stream_and_in_a_graph():
    c = Case([700, 90], 16, 8, 128)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    a = c.cache()
    scratch = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q, outs = c.queries(2), [torch.zeros((2, 16, 128), device="cuda", dtype=BF) for _ in range(4)]
    torch.cuda.synchronize()

    def calls(o1, o2, stream):
        a.decode(q, o1, 0.1, max_len=2000, scratch=scratch, stream=stream)
        a.prompt(q, o2, starts, 1, 0.1, max_len=2000, scratch=scratch, stream=stream)

    with torch.cuda.stream(st):
        calls(outs[0], outs[1], st.cuda_stream)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        calls(outs[2], outs[3], torch.cuda.current_stream().cuda_stream)
    for lens in ([700, 90], [650, 3]):  # the graph reads the lengths of the moment
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        c.lens = lens
        g.replay()
        torch.cuda.synchronize()
        for out in outs[2:]:
            for i in range(2):
                o, mag, _ = ref_rows(c, i, q[i : i + 1].double(), torch.tensor([lens[i] - 1], device="cuda"), 0.1, 0, 0, None)
                check_out(out[i : i + 1], o, mag, BF)
        if lens[0] == 700:
            assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_a_loop_of_all_four():
    """A prompt, then steps that append and decode, and evictions when the budget is passed: the output
    of every step against the float64 attention over the rows that should be there."""
    kv, heads, hd, ps, budget, keep = 2, 4, 64, 16, 80, 48
    c = [Case([1], heads, kv, hd, ps, FP, spare=8), Case([1], heads, kv, hd, ps, FP, spare=8, seed=1)]
    caches = [x.cache() for x in c]
    for x in c:
        x.lengths.zero_()
        x.weights.zero_()
    rows = [[[], []] for _ in range(kv)]  # the rows each head should hold, keys and values
    scratch = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    kept = torch.zeros((1, kv, keep), dtype=torch.int32, device="cuda")
    cur, n = 0, 0
    for step in range(70):
        x, r = c[cur], 30 if step == 0 else 1
        new = x.randn(r, heads + 2 * kv, hd).to(FP)
        seq = torch.zeros(r, dtype=torch.int32, device="cuda")
        caches[cur].append(new[:, heads : heads + kv], new[:, heads + kv :], seq, torch.arange(n, n + r, dtype=torch.int32, device="cuda"))
        for h in range(kv):
            rows[h][0] += list(new[:, heads + h].double())
            rows[h][1] += list(new[:, heads + kv + h].double())
        n += r
        x.lengths.fill_(n)
        out = torch.zeros((r, heads, hd), device="cuda", dtype=FP)
        if step == 0:
            caches[cur].prompt(new[:, :heads], out, torch.tensor([0, r], dtype=torch.int32, device="cuda"), r, 0.125, scratch=scratch)
        else:
            caches[cur].decode(new[:, :heads], out, 0.125, accumulate=True, scratch=scratch)
        for h in range(kv):
            k, v = torch.stack(rows[h][0]), torch.stack(rows[h][1])
            for y in range(2 * h, 2 * h + 2):
                s = new[:, y].double() @ k.T * 0.125
                s = s.masked_fill(torch.arange(n, device="cuda") > torch.arange(n - r, n, device="cuda").view(-1, 1), -math.inf)
                w = torch.softmax(s, 1)
                check_out(out[:, y], w @ v, w @ v.abs(), FP)
        if n >= budget:
            caches[cur].evict(caches[1 - cur], keep, first=2, recent=8, kept=kept, scratch=scratch)
            for h in range(kv):
                at = kept[0, h].tolist()
                rows[h] = [[rows[h][z][j] for j in at] for z in range(2)]
            cur, n = 1 - cur, keep


def test_evict_needs_no_scratch_beside_kept():
    c = Case([300, 40], 8, 4, 64)
    kept = [torch.zeros((2, 4, 64), dtype=torch.int32, device="cuda") for _ in range(2)]
    to = [Case([64, 64], 8, 4, 64, seed=9) for _ in range(2)]
    a = c.cache()
    a.evict(to[0].cache(), 64, recent=8, kept=kept[0], scratch=torch.zeros(a.evict_scratch(64), dtype=torch.uint8, device="cuda"))
    a.evict(to[1].cache(), 64, recent=8, kept=kept[1])
    torch.cuda.synchronize()
    assert torch.equal(kept[0], kept[1]) and torch.equal(to[0].lengths, to[1].lengths)
    with pytest.raises(hb.HcError, match="scratch"):
        a.evict(to[1].cache(), 64, recent=8)
