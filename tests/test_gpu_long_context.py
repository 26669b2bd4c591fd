"""examples/long_context.py as a user runs it, at small sizes: the loop holds its budget, does not depend on
how the prompt was cut, and without evictions gives what a plain implementation of its layers gives."""

import os
import sys

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
pytestmark = pytest.mark.gpu


def test_holds_its_budget():
    import long_context as L

    x, held, _ = L.run(3, 300, 60, 256)
    assert torch.isfinite(x).all()
    assert 192 <= held <= 256
    y, full, _ = L.run(3, 300, 60, 256, evicting=False)
    assert full == 360 and torch.isfinite(y).all()


def test_does_not_depend_on_the_chunks():
    import long_context as L

    # the same rows in other blocks: the weights' roundings (2^-8 of each) move the outputs, no more. Rows have
    # unit mean square; four layers of a relative 2^-8 and a factor of 4 for the random walk's tails
    x, _, _ = L.run(2, 260, 8, 1000, chunk=512)
    y, _, _ = L.run(2, 260, 8, 1000, chunk=100)
    assert float((x - y).float().square().mean().sqrt()) < 4 * 4 * 2.0 ** -8


def plain(seqs, prompt, steps, layers, window, seed):
    """long_context.run without evictions, in plain torch: whole sequences through every layer in float32 (weights
    and inputs as run makes them), one new row a step."""
    import long_context as L

    dtype = torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(seed)
    stack = [L.Layer(seqs, prompt + steps, 192, window if n % 2 == 0 else 0, gen, dtype) for n in range(layers)]
    x = torch.randn((seqs, prompt, L.HEADS * L.DIM), device="cuda", generator=gen).to(dtype).float()
    rep = L.HEADS // L.KV
    kv = [[None, None] for _ in stack]

    def step(x, at):
        n = x.shape[1]
        pos = at + torch.arange(n, device="cuda")
        for ly, c in zip(stack, kv):
            y = (x @ ly.qkv.float().T).view(seqs, n, L.HEADS + 2 * L.KV, L.DIM)
            turn = lambda z: torch.stack([L.rope(s, pos) for s in z])  # noqa: E731
            q, k, v = turn(y[:, :, : L.HEADS]), turn(y[:, :, L.HEADS : L.HEADS + L.KV]), y[:, :, L.HEADS + L.KV :]
            c[0] = k if c[0] is None else torch.cat([c[0], k], 1)
            c[1] = v if c[1] is None else torch.cat([c[1], v], 1)
            s = torch.einsum("snhd,smhd->shnm", q, c[0].repeat_interleave(rep, 2)) * L.DIM ** -0.5
            j = torch.arange(at + n, device="cuda")
            see = j <= pos.view(-1, 1)
            if ly.window:
                see = see & ((pos.view(-1, 1) - j < ly.window) | (j < L.FIRST))
            s = s.masked_fill(~see, -float("inf"))
            if ly.sinks is not None:
                s = torch.cat([s, ly.sinks.view(1, -1, 1, 1).expand(seqs, -1, n, 1)], -1)
            p = torch.softmax(s, -1)[..., : at + n]
            o = torch.einsum("shnm,smhd->snhd", p, c[1].repeat_interleave(rep, 2)).reshape(seqs, n, -1)
            x = x + o @ ly.out.float().T
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        return x

    x = step(x, 0)[:, -1:]
    for s in range(steps):
        x = step(x, prompt + s)
    return x[:, 0]


def test_equals_plain_layers():
    import long_context as L

    got, _, _ = L.run(2, 200, 6, 1000, seed=3)
    want = plain(2, 200, 6, 4, 128, 3)
    # bf16 rows of unit mean square through four layers and up to 7 tokens that feed one another: a rounding is at
    # most 2^-8 of a value, with six of them a layer, summed as a walk and doubled for its tails
    err = float((got.float() - want).square().mean().sqrt())
    assert err < 2 * 2.0 ** -8 * (6 * 4 * 7) ** 0.5, err


def rows_held(layer, seq, n):
    """The marks (key column 0) of the rows sequence seq of a layer's cache holds, head by head."""
    c = layer.caches[0]
    slots = torch.arange(n, device="cuda")
    return [c.k[c.block_table[seq].long()[slots // c.k.shape[2]], h, slots % c.k.shape[2], 0].tolist() for h in range(c.kv_heads)]


@pytest.mark.parametrize("n,keep", [(300, 192), (300, 132), (1000, 300)])
def test_sliding_layers_keep_their_window(n, keep):
    import long_context as L

    layer = L.Layer(2, n, keep, 128, torch.Generator(device="cuda").manual_seed(0), torch.float16)
    c, slots = layer.caches[0], torch.arange(n, dtype=torch.int32, device="cuda")
    rows = slots.half().view(-1, 1, 1).expand(n, L.KV, L.DIM).contiguous()  # whole numbers below 2,048: exact in fp16
    for seq in range(2):
        c.append(rows, rows, torch.full_like(slots, seq), slots)
    c.lengths.fill_(n)
    layer.evict(keep)
    torch.cuda.synchronize()
    assert layer.caches[0].lengths.tolist() == [keep] * 2
    # all the model can see of it: the first rows and the window, here with the newest of what lies between
    want = [float(j) for j in [*range(L.FIRST), *range(n - keep + L.FIRST, n)]]
    for seq in range(2):
        assert all(held == want for held in rows_held(layer, seq, keep))


def test_sliding_layers_do_not_feel_the_evictions():
    import long_context as L

    # one sliding layer alone: what its mask shows is always held, so only the order of sums differs. fp16 rows of unit
    # mean square, 20 tokens that feed one another, six roundings of 2^-11 each, summed as a walk and doubled
    x, held, _ = L.run(3, 300, 20, 256, layers=1, dtype=torch.float16)
    y, full, _ = L.run(3, 300, 20, 256, layers=1, dtype=torch.float16, evicting=False)
    assert held < full
    err = float((x - y).float().square().mean().sqrt())
    assert err < 2 * 2.0 ** -11 * (6 * 20) ** 0.5, err


def test_a_budget_below_the_window_is_refused():
    import long_context as L

    with pytest.raises(ValueError, match="window"):
        L.run(1, 200, 2, 160)
