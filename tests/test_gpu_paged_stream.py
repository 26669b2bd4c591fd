"""Calls of PagedCache without a stream run where their tensors' own work runs: on torch's current stream."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged_cache import BF, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("side", [False, True])
def test_without_a_stream_calls_follow_the_current_one(side):
    results = []
    for delayed in (False, True):
        c, to = Case([300], 16, 8, 128), Case([64], 16, 8, 128, seed=1)
        c.weights.zero_()
        new, q0 = c.queries(40).new_zeros(1, 32, 128), c.queries(40).contiguous()
        source = c.randn(1, 32, 128).to(BF)
        q = torch.zeros_like(q0)
        outs = [torch.zeros((r, 16, 128), device="cuda", dtype=BF) for r in (1, 40)]
        kept = torch.zeros((1, 8, 64), dtype=torch.int32, device="cuda")
        scratch = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
        starts = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
        one = torch.zeros(1, dtype=torch.int32, device="cuda")
        a, b = c.cache(), to.cache()
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.default_stream()):
            if delayed:
                torch.cuda._sleep(20_000_000)  # about 10 ms: the operands are written after the calls were made
            new.copy_(source)
            q.copy_(q0)
            a.append(new[:, 16:24], new[:, 24:], one, one + 299)
            a.decode(q[:1], outs[0], 0.1, accumulate=True, scratch=scratch)
            a.prompt(q, outs[1], starts, 40, 0.1, scratch=scratch)
            a.evict(b, 64, recent=8, kept=kept, scratch=scratch)
        torch.cuda.synchronize()
        results.append([*outs, kept, c.weights])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    assert float(results[0][0].abs().max()) > 0 and int(results[0][2].max()) == 299


def test_captured_without_a_stream():
    c = Case([300], 16, 8, 64)
    a, q = c.cache(), c.queries(1)
    out, scratch = torch.zeros((1, 16, 64), device="cuda", dtype=BF), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    a.decode(q, out, 0.1, scratch=scratch)
    want = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.decode(q, out, 0.1, scratch=scratch)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
