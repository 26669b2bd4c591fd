"""The operators of a paged 16-bit key-value cache as a long-context serving loop calls them:
append (new rows into the pages), decode (one new token a sequence), prompt (many new tokens a
sequence, with a sliding window and first tokens that stay visible) and evict (the rows with the
largest accumulated attention weight are kept, in order, in other pages).

Shapes come from the configurations of hwnpu_b200/synth.py: 16 query heads over 8 key-value heads of
128 (C2), 64 over 8 of 64 with a window of 128 and sink logits (C3), 64 ragged sequences as in the
C5 batch; 32 over 8 of 128 is the generic long-context shape.

The cache: k, v [pages][kv_heads][page_size][head_dim] (or, layout "nhd", the same view of
[pages][page_size][kv_heads][head_dim]), table int32 [seqs][max_pages], lengths int32 [seqs],
weights float32 [seqs][kv_heads][max_pages * page_size]. Slot j of sequence i is row j % page_size
of page table[i][j // page_size]. A query at slot p sees the slots j <= p with p - j < window
(window 0: all) or j < first.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, **kw):
    c = {"name": name, "op": op, "type": "bf16", "heads": 16, "kv_heads": 8, "head_dim": 128, "page_size": 16,
         "layout": "hnd", "seqs": 1, "lo": 1, "hi": 1}
    c.update(kw)
    return c


def listed():
    return [
        # one conversation early on: the smallest decode call, all latency
        _case("decode one short", "decode", type="fp16", lo=333, hi=333, window=0, first=0, sinks=False,
              accumulate=False),
        # a continuous batch of 64 ragged sequences that gathers the weights its evictions will need
        _case("decode ragged batch", "decode", seqs=64, lo=0, hi=8200, window=0, first=0, sinks=False,
              accumulate=True),
        # one very long document: few rows, the cache's length is what there is to split
        _case("decode one long", "decode", heads=32, page_size=64, lo=131071, hi=131071, window=0, first=0,
              sinks=False, accumulate=False, layout="nhd"),
        # a gpt-oss sliding layer at batch 128: short windows in long caches, 4 first tokens kept
        _case("decode window batch", "decode", heads=64, head_dim=64, seqs=128, lo=5, hi=4099, window=128, first=4,
              sinks=True, accumulate=False),
        # a speculative verify: a handful of rows a sequence over cached context
        _case("prompt verify", "prompt", type="fp16", seqs=8, lo=500, hi=2100, rows_lo=5, rows_hi=5, window=0,
              first=0, sinks=False),
        # the last chunk of a long prompt read in pieces of 512: few rows over a long cache
        _case("prompt chunk", "prompt", heads=32, page_size=64, lo=16901, hi=16901, rows_lo=512, rows_hi=512, window=0,
              first=0, sinks=False, layout="nhd"),
        # a batch of ragged prompts on a gpt-oss sliding layer
        _case("prompt window ragged", "prompt", heads=64, head_dim=64, seqs=16, lo=3, hi=2050, rows_lo=0, rows_hi=0,
              window=128, first=4, sinks=True),
        # a whole long prompt, with a window of 4,096 and 64 first tokens that stay visible
        _case("prompt long", "prompt", page_size=32, lo=16384, hi=16384, rows_lo=0, rows_hi=0, window=4096, first=64,
              sinks=False),
        # one conversation that passes its budget
        _case("evict one", "evict", type="fp16", lo=1500, hi=1500, keep=1024, first=4, recent=128),
        # a batch of long documents cut to 4,096 rows a head after their prompts
        _case("evict long batch", "evict", heads=32, seqs=16, lo=3000, hi=32771, keep=4096, first=4, recent=256,
              page_size=32),
        # one new row for each sequence of a decode batch
        _case("append step", "append", seqs=64, lo=1, hi=8200, rows_lo=1, rows_hi=1),
        # a prompt's rows
        _case("append prompt", "append", seqs=4, lo=700, hi=4100, rows_lo=0, rows_hi=0, page_size=32, layout="nhd",
              type="fp16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (64, 8, 64), (32, 8, 128), (16, 4, 64), (8, 8, 128),
                                            (20, 4, 128)])
    op = rng.choice(["decode", "decode", "prompt", "prompt", "evict", "append"])
    c = {"op": op, "type": rng.choice(["fp16", "bf16"]), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "page_size": rng.choice([16, 16, 32, 64, 128]), "layout": rng.choice(["hnd", "nhd"])}
    if op in ("decode", "prompt"):
        windowed = rng.random() < 0.5
        c["window"] = _log_int(rng, 16, 4096) if windowed else 0
        c["first"] = rng.choice([0, 1, 4, 17, 64]) if windowed else 0
        c["sinks"] = rng.random() < 0.3
    if op == "decode":
        c["seqs"] = _log_int(rng, 1, 128)
        c["hi"] = _log_int(rng, 1, max(2, min(131071, 64 * 4000 // c["seqs"])))
        c["lo"] = rng.choice([0, 1, max(1, c["hi"] // 2), c["hi"]])
        c["accumulate"] = rng.random() < 0.5
    elif op == "prompt":
        c["seqs"] = _log_int(rng, 1, 16)
        c["hi"] = _log_int(rng, 1, 8192)
        c["lo"] = rng.choice([1, max(1, c["hi"] // 2), c["hi"]])
        # the plain form holds every score of the padded batch at once: at most 8 GB of them
        most = max(1, min(c["lo"], 8 * 10 ** 9 // (4 * c["seqs"] * heads * c["hi"])))
        c["rows_hi"] = _log_int(rng, 1, most)
        c["rows_lo"] = rng.choice([1, c["rows_hi"]])
    elif op == "evict":
        c["seqs"] = _log_int(rng, 1, 32)
        c["hi"] = _log_int(rng, 40, max(50, min(65536, 300000 // c["seqs"])))
        c["lo"] = rng.choice([1, c["hi"] // 2, c["hi"]])
        c["keep"] = _log_int(rng, 16, max(17, min(4096, c["hi"])))
        c["first"] = rng.choice([0, 1, 4])
        c["recent"] = rng.randint(0, c["keep"] - 4)
    else:
        c["seqs"] = _log_int(rng, 1, 64)
        c["hi"] = _log_int(rng, 1, 8200)
        c["lo"] = rng.choice([1, max(1, c["hi"] // 2), c["hi"]])
        most = max(1, min(c["lo"], 8000 // c["seqs"]))
        c["rows_hi"] = _log_int(rng, 1, most)
        c["rows_lo"] = c["rows_hi"]
    return c


def _spread(lo, hi, n):
    """n whole numbers over lo..hi in a ragged order (multiples of the golden ratio), hi among them."""
    f = np.modf(np.arange(n) * 0.6180339887498949 + 1e-9)[0]
    v = lo + np.floor(f * (hi - lo + 1)).astype(np.int64)
    v[-1] = hi
    return v


def _lengths(case):
    return _spread(case["lo"], case["hi"], case["seqs"])


def _rows(case):
    """New rows of each sequence: rows_hi 0 means the whole sequence."""
    if case["rows_hi"] == 0:
        return _lengths(case)
    return _spread(case["rows_lo"], case["rows_hi"], case["seqs"])


def _visible(case, p):
    """How many slots a query at each slot of p sees."""
    if not case["window"]:
        return p + 1
    return np.minimum(p + 1, case["window"]) + np.clip(p + 1 - case["window"], 0, case["first"])


def work(case):
    n = _lengths(case)
    h, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "decode":
        seen = int(_visible(case, n - 1)[n > 0].sum())
        by = seen * h * d * 4 + 2 * case["seqs"] * case["heads"] * d * 2 + (seen * h * 8 if case["accumulate"] else 0)
        return {"bytes": by, "flops": 4 * seen * case["heads"] * d}
    if case["op"] == "prompt":
        r = _rows(case)
        pairs = sum(int(_visible(case, np.arange(a - b, a)).sum()) for a, b in zip(n, r))
        reach = [a - max(0, a - b - case["window"] + 1) + min(case["first"], max(0, a - b - case["window"] + 1))
                 if case["window"] else a for a, b in zip(n, r)]
        return {"bytes": int(sum(reach)) * h * d * 4 + 2 * int(r.sum()) * case["heads"] * d * 2,
                "flops": 4 * pairs * case["heads"] * d}
    if case["op"] == "evict":
        kept = int(np.minimum(n, case["keep"]).sum())
        return {"bytes": int(n.sum()) * h * 4 + kept * h * (d * 8 + 8), "flops": int(n.sum()) * h}
    return {"bytes": int(_rows(case).sum()) * h * d * 8, "flops": 0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, dev = TYPES[case["type"]], "cuda"
    S, H, D, ps = case["seqs"], case["kv_heads"], case["head_dim"], case["page_size"]
    lengths = _lengths(case)
    max_len = int(lengths.max())
    width = max(1, -(-max_len // ps)) + 1  # pages a sequence may hold: one more than it needs
    pages = S * width + 3

    def pool(fill, n):
        shape = (n, H, ps, D) if case["layout"] == "hnd" else (n, ps, H, D)
        x = torch.randn(shape, device=dev, dtype=dt, generator=g) if fill else torch.zeros(shape, device=dev, dtype=dt)
        return x if case["layout"] == "hnd" else x.permute(0, 2, 1, 3)

    def table(n, w):
        return torch.randperm(n, device=dev, generator=g)[: S * w].to(torch.int32).view(S, w).contiguous()

    s = {"case": case, "max_len": max_len, "scale": D ** -0.5, "k": pool(True, pages), "v": pool(True, pages),
         "table": table(pages, width), "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev)}
    # what earlier steps have given each slot: a few heavy rows, many light ones, zeros of rows just appended
    w = torch.rand((S, H, width * ps), device=dev, generator=g).pow_(8).mul_(4)
    s["weights"] = torch.where(w < 1e-6, torch.zeros_like(w), w)
    if case["op"] in ("decode", "prompt"):
        T = S if case["op"] == "decode" else int(_rows(case).sum())
        # the rows of a fused q|k|v projection: q is a strided view of them
        qkv = torch.randn((T, case["heads"] + 2 * H, D), device=dev, dtype=dt, generator=g)
        s["q"] = qkv[:, : case["heads"]]
        s["out"] = torch.zeros((T, case["heads"], D), device=dev, dtype=dt)
        s["sinks"] = torch.randn(case["heads"], device=dev, generator=g) if case["sinks"] else None
    if case["op"] == "prompt":
        r = _rows(case)
        s["max_rows"] = int(r.max())
        s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(r)]), dtype=torch.int32, device=dev)
    if case["op"] == "append":
        r = _rows(case)
        qkv = torch.randn((int(r.sum()), case["heads"] + 2 * H, D), device=dev, dtype=dt, generator=g)
        s["new_k"], s["new_v"] = qkv[:, case["heads"] : case["heads"] + H], qkv[:, case["heads"] + H :]
        seq = np.repeat(np.arange(S), r)
        slot = np.concatenate([np.arange(a - b, a) for a, b in zip(lengths, r)])
        s["seq"] = torch.tensor(seq, dtype=torch.int32, device=dev)
        s["slot"] = torch.tensor(slot, dtype=torch.int32, device=dev)
    if case["op"] == "evict":
        w2 = -(-case["keep"] // ps)
        s["to_k"], s["to_v"] = pool(False, S * w2 + 1), pool(False, S * w2 + 1)
        s["to_table"] = table(S * w2 + 1, w2)
        s["to_lengths"] = torch.zeros(S, dtype=torch.int32, device=dev)
        s["to_weights"] = torch.zeros((S, H, w2 * ps), device=dev)
        s["kept"] = torch.zeros((S, H, case["keep"]), dtype=torch.int32, device=dev)
    if own:
        from hwnpu_b200 import PagedCache

        s["cache"] = PagedCache(s["k"], s["v"], s["table"], s["lengths"], weights=s["weights"])
        n = 0
        if case["op"] == "decode":
            n = s["cache"].decode_scratch(case["heads"], max_len, window=case["window"], first=case["first"],
                                          accumulate=case["accumulate"])
        elif case["op"] == "prompt":
            n = s["cache"].prompt_scratch(case["heads"], s["q"].shape[0], s["max_rows"], max_len,
                                          window=case["window"], first=case["first"])
        elif case["op"] == "evict":
            s["to"] = PagedCache(s["to_k"], s["to_v"], s["to_table"], s["to_lengths"], weights=s["to_weights"])
            n = s["cache"].evict_scratch(case["keep"], max_len)
        s["scratch"] = torch.zeros(max(1, n), dtype=torch.uint8, device=dev)
    return s


# ---- the plain forms --------------------------------------------------------------------------


def _gather(s, x):
    """The sequences' rows in slot order, float32 [seqs][kv_heads][slots][head_dim]."""
    c = s["case"]
    t = s["table"][:, : max(1, -(-s["max_len"] // c["page_size"]))].long()
    y = x[t].permute(0, 2, 1, 3, 4)
    return y.reshape(y.shape[0], y.shape[1], -1, y.shape[4]).float()


def _softmax(scores, see, sinks):
    """exp(score - max) over the visible slots, divided by their sum (and the sink's); rows that see
    nothing are zeros. Works on scores in place; sinks is broadcast over [..][1] or None."""
    scores.masked_fill_(~see, -math.inf)
    m = scores.amax(-1, keepdim=True)
    if sinks is not None:
        m = torch.maximum(m, sinks)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    scores.sub_(m).exp_()
    total = scores.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - m)
    return scores.div_(torch.where(total == 0, torch.ones_like(total), total))


def _decode(s):
    c = s["case"]
    S, H, D, R = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    k, v = _gather(s, s["k"]), _gather(s, s["v"])
    n = s["lengths"].long().view(S, 1, 1, 1)
    j = torch.arange(k.shape[2], device=k.device).view(1, 1, 1, -1)
    see = j < n
    if c["window"]:
        see = see & ((n - 1 - j < c["window"]) | (j < c["first"]))
    scores = torch.matmul(s["q"].float().reshape(S, H, R, D), k.transpose(2, 3)) * s["scale"]
    sinks = None if s["sinks"] is None else s["sinks"].view(1, H, R, 1)
    p = _softmax(scores, see, sinks)
    out = torch.matmul(p, v.masked_fill_(~see.view(S, 1, -1, 1), 0.0))
    s["out"].copy_(out.view(S, c["heads"], D))
    if not c["accumulate"]:
        return {"out": s["out"]}
    s["weights"][:, :, : k.shape[2]] += p.sum(2)
    return {"out": s["out"], "weights": s["weights"]}


def _prompt(s):
    c = s["case"]
    S, H, D, R, N = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], s["max_rows"]
    k, v = _gather(s, s["k"]), _gather(s, s["v"])
    C, T = k.shape[2], s["q"].shape[0]
    start = s["starts"].long()
    n, rows = s["lengths"].long().view(S, 1, 1), (start[1:] - start[:-1]).view(S, 1, 1)
    at = (start[:-1, None] + torch.arange(N, device=k.device)).clamp_(max=T - 1)
    q = s["q"][at].float().reshape(S, N, H, R, D).permute(0, 2, 3, 1, 4).reshape(S, H, R * N, D)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(S, H, R, N, C)
    j = torch.arange(C, device=k.device).view(1, 1, C)
    p = n - rows + torch.arange(N, device=k.device).view(1, N, 1)
    see = (j <= p) & (j < n)
    if c["window"]:
        see = see & ((p - j < c["window"]) | (j < c["first"]))
    sinks = None if s["sinks"] is None else s["sinks"].view(1, H, R, 1, 1)
    _softmax(scores, see.view(S, 1, 1, N, C), sinks)
    v.masked_fill_((j >= n).view(S, 1, C, 1), 0.0)
    out = torch.matmul(scores.view(S, H, R * N, C), v).view(S, H, R, N, D).permute(0, 3, 1, 2, 4)
    token = torch.arange(T, device=k.device)
    seq = torch.searchsorted(start[1:].contiguous(), token, right=True)
    s["out"].copy_(out.reshape(S, N, c["heads"], D)[seq, token - start[seq]])
    return {"out": s["out"]}


def _evict(s):
    c = s["case"]
    S, H, ps, keep = c["seqs"], c["kv_heads"], c["page_size"], c["keep"]
    n = s["lengths"].long().view(S, 1, 1)
    C = s["weights"].shape[2]
    j = torch.arange(C, device=n.device).view(1, 1, C)
    fixed = (j < c["first"]) | ((j >= n - c["recent"]) & (j < n))
    free = (j < n) & ~fixed
    order = torch.where(free, s["weights"], torch.full_like(s["weights"], -1.0)).sort(dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(2, order, j.expand(S, H, C).contiguous())
    stays = torch.where(n <= keep, j < n, fixed | (free & (rank < keep - c["first"] - c["recent"])))
    slots = torch.where(stays, j, torch.full_like(j, 1 << 40)).sort(-1)[0][:, :, :keep]
    slots = torch.nn.functional.pad(slots, (0, keep - slots.shape[2]), value=1 << 40)
    there = slots < C
    src = torch.where(there, slots, torch.zeros_like(slots))
    d = torch.arange(keep, device=n.device)
    seq = torch.arange(S, device=n.device).view(S, 1, 1)
    head = torch.arange(H, device=n.device).view(1, H, 1)
    sp, dp = s["table"].long()[seq, src // ps], s["to_table"].long()[seq, (d // ps).view(1, 1, keep)].expand(S, H, keep)
    old = (dp, head.expand(S, H, keep), (d % ps).view(1, 1, keep).expand(S, H, keep))
    s["to_k"][old] = torch.where(there.unsqueeze(-1), s["k"][sp, head, src % ps], s["to_k"][old])
    s["to_v"][old] = torch.where(there.unsqueeze(-1), s["v"][sp, head, src % ps], s["to_v"][old])
    w = s["weights"].gather(2, src)
    s["to_weights"][:, :, :keep] = torch.where(there, w, s["to_weights"][:, :, :keep])
    s["to_lengths"].copy_(s["lengths"].clamp(max=keep))
    s["kept"].copy_(torch.where(there, slots, torch.full_like(slots, -1)))
    return {"k": s["to_k"], "v": s["to_v"], "weights": s["to_weights"], "lengths": s["to_lengths"], "kept": s["kept"]}


def _append(s):
    ps = s["case"]["page_size"]
    seq, slot = s["seq"].long(), s["slot"].long()
    page = s["table"].long()[seq, slot // ps]
    s["k"][page, :, slot % ps] = s["new_k"]
    s["v"][page, :, slot % ps] = s["new_v"]
    s["weights"][seq, :, slot] = 0.0
    return {"k": s["k"], "v": s["v"], "weights": s["weights"]}


def run(s):
    c = s["case"]
    if not own:
        return {"decode": _decode, "prompt": _prompt, "evict": _evict, "append": _append}[c["op"]](s)
    cache = s["cache"]
    if c["op"] == "decode":
        cache.decode(s["q"], s["out"], s["scale"], window=c["window"], first=c["first"], sinks=s["sinks"],
                     accumulate=c["accumulate"], max_len=s["max_len"], scratch=s["scratch"])
        return {"out": s["out"], "weights": s["weights"]} if c["accumulate"] else {"out": s["out"]}
    if c["op"] == "prompt":
        cache.prompt(s["q"], s["out"], s["starts"], s["max_rows"], s["scale"], window=c["window"], first=c["first"],
                     sinks=s["sinks"], max_len=s["max_len"], scratch=s["scratch"])
        return {"out": s["out"]}
    if c["op"] == "evict":
        cache.evict(s["to"], c["keep"], first=c["first"], recent=c["recent"], kept=s["kept"], max_len=s["max_len"],
                    scratch=s["scratch"])
        return {"k": s["to_k"], "v": s["to_v"], "weights": s["to_weights"], "lengths": s["to_lengths"],
                "kept": s["kept"]}
    cache.append(s["new_k"], s["new_v"], s["seq"], s["slot"])
    return {"k": s["k"], "v": s["v"], "weights": s["weights"]}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    S, H, D, ps, R = case["seqs"], case["kv_heads"], case["head_dim"], case["page_size"], case["heads"] // case["kv_heads"]
    n = [int(x) for x in _lengths(case)]
    if case["op"] == "append":
        k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
        at, table = 0, s["table"].cpu()
        for i, r in enumerate(_rows(case)):
            for slot in range(n[i] - int(r), n[i]):
                page = int(table[i, slot // ps])
                k[page, :, slot % ps] = s["new_k"][at].double()
                v[page, :, slot % ps] = s["new_v"][at].double()
                w[i, :, slot] = 0
                at += 1
        return {"k": k, "v": v, "weights": w}
    if case["op"] == "evict":
        k, v, w = s["to_k"].double(), s["to_v"].double(), s["to_weights"].double()
        for i in range(S):
            new = torch.arange(min(n[i], case["keep"]), device="cuda")
            page = s["to_table"][i].long()[new // ps]
            for h in range(H):
                have = s["weights"][i, h, : n[i]].cpu().numpy()
                if n[i] <= case["keep"]:
                    slots = np.arange(n[i])
                else:
                    body = np.arange(case["first"], n[i] - case["recent"])
                    heavy = body[np.lexsort((body, -have[body].astype(np.float64)))]
                    heavy = np.sort(heavy[: case["keep"] - case["first"] - case["recent"]])
                    slots = np.concatenate([np.arange(case["first"]), heavy, np.arange(n[i] - case["recent"], n[i])])
                slots = torch.from_numpy(slots.astype(np.int64)).cuda()
                old = s["table"][i].long()[slots // ps]
                k[page, h, new % ps] = s["k"][old, h, slots % ps].double()
                v[page, h, new % ps] = s["v"][old, h, slots % ps].double()
                w[i, h, : len(new)] = s["weights"][i, h, slots].double()
        return {"k": k, "v": v, "weights": w, "lengths": None, "kept": None}
    out = torch.zeros(tuple(s["out"].shape), dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    rows = np.ones(S, np.int64) if case["op"] == "decode" else _rows(case)
    at = 0
    for i in range(S):
        r = int(rows[i])
        if n[i]:
            slot = torch.arange(n[i], device="cuda")
            page = s["table"][i].long()[slot // ps]
            for h in range(H):
                k, v = s["k"][page, h, slot % ps].double(), s["v"][page, h, slot % ps].double()
                for b in range(0, r, 2048):
                    e = min(r, b + 2048)
                    p = torch.arange(n[i] - r + b, n[i] - r + e, device="cuda").unsqueeze(1)
                    hidden = slot.unsqueeze(0) > p
                    if case["window"]:
                        hidden |= (p - slot.unsqueeze(0) >= case["window"]) & (slot.unsqueeze(0) >= case["first"])
                    for x in range(h * R, (h + 1) * R):
                        z = (s["q"][at + b : at + e, x].double() @ k.T) / math.sqrt(D)
                        z[hidden] = -math.inf
                        if s["sinks"] is not None:
                            z = torch.cat([z, s["sinks"][x].double().expand(e - b, 1)], 1)
                        z = torch.softmax(z, 1)[:, : n[i]]
                        out[at + b : at + e, x] = z @ v
                        if case["op"] == "decode":
                            weights[i, h, : n[i]] += z[0]
        at += r
    if case["op"] == "decode" and case["accumulate"]:
        return {"out": out, "weights": weights}
    return {"out": out}
