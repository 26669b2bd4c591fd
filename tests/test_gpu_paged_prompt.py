"""The tensor-core prompt kernel of a caller's paged 16-bit cache (hc_paged_prompt_run with more than 16 rows a kv head:
fewer run as decode does), where test_gpu_paged_cache.py leaves off. Same plain implementation, same bounds."""

import pytest

torch = pytest.importorskip("torch")

from hwnpu_b200 import _abi as A
from test_gpu_paged_cache import BF, FP, Case, run_prompt

pytestmark = pytest.mark.gpu


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
