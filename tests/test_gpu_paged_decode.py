"""Decode over a caller's paged 16-bit cache where test_gpu_paged_cache.py leaves off."""

import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged_cache import BF, FP, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads,kv,hd", [(16, 8, 128), (40, 4, 64)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_infinite_values_come_out_as_the_formula_says(dtype, heads, kv, hd, accumulate):
    # A visible value of +-infinity has a weight above 0 here (scores stay within +-10), so its column of the output is
    # infinite, NaN where both signs meet, and the other columns are what they were.
    lens = [1, 5, 70, 700, 4000]
    c = Case(lens, heads, kv, hd, 16, dtype)
    outs = []
    for broken in (False, True):
        if broken:
            for i, n in enumerate(lens):
                page, r = c.where(i, torch.tensor([0, n // 2, n - 1], device="cuda"))
                c.v[page[0], :, r[0], 3] = math.inf
                c.v[page[1], :, r[1], 8] = -math.inf
                c.v[page[0], :, r[0], 21] = math.inf
                c.v[page[2], :, r[2], 21] = -math.inf if n > 1 else math.inf
        c.g.manual_seed(4)
        q = c.queries(len(lens))
        out = torch.zeros((len(lens), heads, hd), device="cuda", dtype=dtype)
        a = c.cache()
        scratch = torch.zeros(max(16, a.decode_scratch(heads, 4000, accumulate=accumulate)), dtype=torch.uint8, device="cuda")
        a.decode(q, out, hd ** -0.5, max_len=4000, accumulate=accumulate, scratch=scratch)
        outs.append(out)
    sound, out = outs
    want = sound.clone()
    want[:, :, 3], want[:, :, 8] = math.inf, -math.inf
    want[:, :, 21] = math.nan
    want[0, :, 21] = math.inf
    torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True)
