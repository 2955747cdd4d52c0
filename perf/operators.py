"""Timed cases of the packed-batch operators: page tables and slot maps built
on the GPU, rotary positions with several axes fused with the cache write, and
attention over packed prompts.

``own`` selects the side: False computes each operator in elementary torch
operations (32 bits, 64 where angles need them, rounded once at the end), True
calls the framework's operators through ``memopt_C``.
"""
import os
import random
import sys

import torch

own = False
_C = None


def _ops():
    global _C
    if _C is None:
        pkg = os.path.join(os.getcwd(), "memopt-transformer-runtime_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import memopt_C

        _C = memopt_C
    return _C


_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_LIMIT = 4.3e9  # padded scores of the plain attention: sequences * heads * longest^2


def listed():
    return [
        # Chat turns that arrive together: a few dozen tokens each, one-token and empty ones among them.
        {"name": "attention chat turns", "op": "attention", "seqs": 24, "low": 0, "high": 96, "mix": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "fp16", "causal": True, "window": -1, "fused": True},
        # A batch of ordinary prompts of very different lengths, grouped heads.
        {"name": "attention ragged prompts", "op": "attention", "seqs": 12, "low": 100, "high": 2048, "mix": 2,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "fp16", "causal": True, "window": -1, "fused": True},
        # Documents under a sliding window, bf16, 64-wide heads.
        {"name": "attention window", "op": "attention", "seqs": 5, "low": 500, "high": 4096, "mix": 3, "heads": 32,
         "kv_heads": 32, "dim": 64, "dtype": "bf16", "causal": True, "window": 1000, "fused": False},
        # Bidirectional encoding of a batch (the framework's non-causal default), bf16, 128-wide heads.
        {"name": "attention non-causal", "op": "attention", "seqs": 6, "low": 1, "high": 2500, "mix": 4, "heads": 16,
         "kv_heads": 4, "dim": 128, "dtype": "bf16", "causal": False, "window": -1, "fused": True},
        # The framework's long-prefill shape (8192 tokens, 32 heads of 128), two prompts, causal: the largest.
        {"name": "attention long prompts", "op": "attention", "seqs": 2, "low": 8100, "high": 8192, "mix": 5,
         "heads": 32, "kv_heads": 32, "dim": 128, "dtype": "fp16", "causal": True, "window": -1, "fused": False},
        # One decode step of 32 sequences far into their contexts.
        {"name": "rotary decode step", "op": "rotary", "tokens": 32, "axes": 1, "pairs": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "fp16", "interleaved": False, "far": 131072, "cache": True,
         "block": 16},
        # A packed prompt with image and video tokens: time, height and width positions, bf16.
        {"name": "rotary three axes", "op": "rotary", "tokens": 4099, "axes": 3, "pairs": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "interleaved": False, "far": 32768, "cache": True, "block": 16},
        # Half of a 64-wide head rotated in neighbouring pairs, no cache behind it.
        {"name": "rotary partial pairs", "op": "rotary", "tokens": 10007, "axes": 2, "pairs": 16, "heads": 16,
         "kv_heads": 16, "dim": 64, "dtype": "bf16", "interleaved": True, "far": 8192, "cache": False, "block": 16},
        # Four prompts of 8192 tokens, 32 full heads, into the pool.
        {"name": "rotary long prompts", "op": "rotary", "tokens": 32768, "axes": 1, "pairs": 64, "heads": 32,
         "kv_heads": 32, "dim": 128, "dtype": "fp16", "interleaved": False, "far": 8192, "cache": True, "block": 32},
        # A speculative step: a few draft tokens for each of 64 running sequences, all rejected.
        {"name": "pages draft and reject", "op": "pages", "rows": 64, "low": 1, "high": 5, "old": 4000, "mix": 6,
         "block": 16, "width": 512, "pad": 0},
        # Requests of up to 4096 tokens admitted together, and finished.
        {"name": "pages admit prompts", "op": "pages", "rows": 32, "low": 1, "high": 4096, "old": 0, "mix": 7,
         "block": 16, "width": 512, "pad": 100},
        # A thousand requests at once.
        {"name": "pages admit a thousand", "op": "pages", "rows": 1000, "low": 1, "high": 1500, "old": 300, "mix": 8,
         "block": 32, "width": 256, "pad": 0},
    ]


def _log_int(rng, low, high):
    """A whole number in [low, high], even in its logarithm."""
    low, high = max(low, 1), max(high, 1)
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "pages"])
    mix = rng.randrange(1, 1 << 30)
    if op == "attention":
        dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        high = _log_int(rng, 8, min(8192, int((_LIMIT / 2 / heads) ** 0.5)))
        seqs = _log_int(rng, 1, max(1, min(48, int(_LIMIT / 2 / (heads * high * high)))))
        causal = rng.random() < 0.75
        window = _log_int(rng, 1, high) if rng.random() < 0.3 else -1
        return {"op": op, "seqs": seqs, "low": rng.choice([0, 1, max(1, high // 3)]), "high": high, "mix": mix,
                "heads": heads, "kv_heads": kv, "dim": dim, "dtype": rng.choice(["fp16", "bf16"]), "causal": causal,
                "window": window, "fused": rng.random() < 0.5}
    if op == "rotary":
        dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8, 32])
        heads = kv * rng.choice([1, 2, 4, 5]) if kv < 32 else 32
        return {"op": op, "tokens": _log_int(rng, 1, 32768), "axes": rng.choice([1, 2, 3]), "heads": heads,
                "kv_heads": kv, "pairs": 8 * rng.randrange(3, dim // 16 + 1), "dim": dim,
                "dtype": rng.choice(["fp16", "bf16"]), "interleaved": rng.random() < 0.4,
                "far": _log_int(rng, 64, 1 << 20), "cache": rng.random() < 0.7, "block": rng.choice([16, 32]),
                "mix": mix}
    block = rng.choice([16, 32])
    high = _log_int(rng, 1, 4096)
    old = rng.choice([0, _log_int(rng, 1, 4000)])
    rows = _log_int(rng, 1, min(1000, max(1, 700000 // high)))
    return {"op": op, "rows": rows, "low": 1, "high": high, "old": old, "mix": mix, "block": block,
            "width": -(-(high + old) // block) + rng.randrange(0, 9), "pad": rng.choice([0, 0, 37])}


def _lengths(case, count):
    """The case's own sequence lengths: even in their logarithm, the first as long as any may be."""
    rng = random.Random(case["mix"])
    low, high = case["low"], case["high"]
    got = [high] + [_log_int(rng, max(low, 1), high) for _ in range(count - 1)]
    if low == 0:  # empty and one-token sequences among them
        for i in range(1, count):
            if i % 5 == 2:
                got[i] = 0
            elif i % 5 == 4:
                got[i] = 1
    return got


def _old_lengths(case):
    rng = random.Random(case["mix"] + 1)
    return [rng.randrange(case["old"] // 2, case["old"] + 1) for _ in range(case["rows"])]


def _sections(case):
    """How the pairs are shared out among the axes: the last axis takes what is left."""
    each = case["pairs"] // case["axes"]
    return [each] * (case["axes"] - 1) + [case["pairs"] - each * (case["axes"] - 1)]


def _pages_needed(case):
    old, new, bs = _old_lengths(case), _lengths(case, case["rows"]), case["block"]
    before = sum(-(-o // bs) for o in old)
    return before, sum(-(-(o + n) // bs) for o, n in zip(old, new)) - before


def _visible(case):
    """Pairs of a query and a key that it sees, over the sequences."""
    total = 0
    for n in _lengths(case, case["seqs"]):
        w = case["window"] if 0 < case["window"] < n else n
        total += w * (w + 1) // 2 + (n - w) * w if case["causal"] else n * w
    return total


def work(case):
    if case["op"] == "attention":
        t, d = sum(_lengths(case, case["seqs"])), case["dim"]
        return {"bytes": t * d * 2 * 2 * (case["heads"] + case["kv_heads"]) + 4 * (case["seqs"] + 1),
                "flops": 4 * d * case["heads"] * _visible(case)}
    if case["op"] == "rotary":
        t, d, h, kv = case["tokens"], case["dim"], case["heads"], case["kv_heads"]
        moved = 2 * h + 2 * kv + (3 * kv if case["cache"] else 0)
        return {"bytes": t * d * 2 * moved + 4 * t * (case["axes"] + int(case["cache"])) + 8 * case["pairs"],
                "flops": 3 * 2 * case["pairs"] * (h + kv) * t}
    new = sum(_lengths(case, case["rows"]))
    _, pages = _pages_needed(case)
    b = case["rows"]
    # reserve: lengths in, slots and positions out, rows of the table copied out, pages from the ring to the
    # table; truncate: the pages back to the ring and out of the table.
    return {"bytes": 8 * (new + case["pad"]) + 2 * 4 * b * case["width"] + 2 * 4 * pages + 3 * 4 * pages + 4 * 9 * b,
            "flops": 0}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "attention":
        lens = _lengths(case, case["seqs"])
        t, h, kv, d, dt = sum(lens), case["heads"], case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
        # q and k come out of the rotary step; v is a part of the fused projection where there is one.
        q, k = (2.0 * normal(t, h, d)).to(dt), normal(t, kv, d).to(dt)
        v = normal(t, h + 2 * kv if case["fused"] else kv, d).to(dt)[:, -kv:]
        cu = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        return {"case": case, "q": q, "k": k, "v": v, "cu": cu, "longest": max(lens)}
    if case["op"] == "rotary":
        t, h, kv, d, dt = case["tokens"], case["heads"], case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
        qkv = normal(t, h + 2 * kv, d).to(dt)
        pos = torch.randint(0, case["far"], (case["axes"], t), generator=g, device=dev, dtype=torch.int32)
        p = case["pairs"]
        freq = 10000.0 ** (-torch.arange(p, device=dev, dtype=torch.float64) / p)
        state = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:], "pos": pos, "freq": freq}
        if case["cache"]:
            bs = case["block"]
            pages = -(-t // bs) + 3
            order = torch.randperm(pages, generator=g, device=dev)
            at = torch.arange(t, device=dev)
            state["slots"] = (order[at // bs] * bs + at % bs).to(torch.int32)
            state["kc"] = torch.zeros(pages, bs, kv, d, dtype=torch.float16, device=dev)
            state["vc"] = torch.zeros(pages, bs, kv, d, dtype=torch.float16, device=dev)
        return state
    b, bs, width = case["rows"], case["block"], case["width"]
    old, new = _old_lengths(case), _lengths(case, b)
    before, more = _pages_needed(case)
    total = before + more + more // 4 + 5
    ids = torch.randperm(total, generator=g, device=dev, dtype=torch.int32)
    owned = torch.tensor([-(-o // bs) for o in old], device=dev)
    at = torch.arange(width, device=dev)
    table_rows = b + 3  # a few rows that this batch does not touch
    inside = at[None, :] < owned[:, None]
    first = owned.cumsum(0) - owned
    picked = ids[(first[:, None] + at[None, :]).clamp(max=total - 1)]
    rows = torch.randperm(table_rows, generator=g, device=dev)[:b]
    tables = torch.full((table_rows, width), -1, dtype=torch.int32, device=dev)
    tables[rows] = torch.where(inside, picked, torch.full_like(picked, -1))
    lens = torch.zeros(table_rows, dtype=torch.int32, device=dev)
    lens[rows] = torch.tensor(old, dtype=torch.int32, device=dev)
    ring = torch.full((total,), -1, dtype=torch.int32, device=dev)
    head, count = total // 3, total - before
    ring[(head + torch.arange(count, device=dev)) % total] = ids[before:]
    return {"case": case, "tables": tables, "lens": lens, "ring": ring, "rows": rows.to(torch.int32),
            "pool": torch.tensor([head, count, 0, 0], dtype=torch.int32, device=dev),
            "new": torch.tensor(new, dtype=torch.int32, device=dev),
            "old": torch.tensor(old, dtype=torch.int32, device=dev), "tokens": sum(new) + case["pad"]}


def _plain_attention(s):
    """Every sequence padded to the longest; masked scores leave no weight."""
    c, q, k, v, cu = s["case"], s["q"], s["k"], s["v"], s["cu"].long()
    t, h, d = q.shape
    kv, longest = k.shape[1], s["longest"]
    n = cu[1:] - cu[:-1]
    at = torch.arange(longest, device=q.device)
    index = cu[:-1, None] + at[None, :]                      # [S, L] packed row of each padded place
    inside = at[None, :] < n[:, None]
    index = torch.where(inside, index, torch.zeros_like(index)).clamp(max=max(t - 1, 0))

    def padded(x):  # [S, KV, heads of the group, L, D] in 32 bits, zeros outside
        y = x[index].float() * inside[:, :, None, None]
        return y.permute(0, 2, 1, 3).reshape(y.shape[0], kv, -1, longest, d)

    score = padded(q) @ padded(k).transpose(-1, -2)
    score *= d ** -0.5
    end = at[:, None] + 1 if c["causal"] else n[:, None, None].expand(-1, longest, 1)
    first = (end - (c["window"] if c["window"] > 0 else longest + 1)).clamp(min=0)
    seen = (at < end) & (at >= first)                       # [L, L] or [S, L, L]
    seen = seen.expand(n.shape[0], longest, longest) & inside[:, None, :]
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    score -= top
    score.exp_()
    sums = score.sum(-1, keepdim=True)
    out = (score @ padded(v)) / torch.where(sums > 0, sums, torch.ones_like(sums))
    out = out.reshape(n.shape[0], h, longest, d).permute(0, 2, 1, 3)
    return out[inside].to(q.dtype)


def _angles(s):
    c = s["case"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=s["pos"].device),
                                   torch.tensor(_sections(c), device=s["pos"].device))
    return s["pos"].double()[axis].T * s["freq"][None, :]   # [T, pairs], 64 bits: positions go far


def _rotated(x, cos, sin, interleaved):
    p = cos.shape[-1]
    turned, rest = x[..., : 2 * p], x[..., 2 * p:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = turned[..., :p], turned[..., p:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    c = s["case"]
    angle = _angles(s)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotated(s["q"].float(), cos, sin, c["interleaved"]).to(s["q"].dtype)
    k32 = _rotated(s["k"].float(), cos, sin, c["interleaved"])
    k = k32.to(s["k"].dtype)
    if not c["cache"]:
        return {"q": q, "k": k}
    slots = s["slots"].long()
    s["kc"].view(-1, *s["kc"].shape[2:])[slots] = k32.half()
    s["vc"].view(-1, *s["vc"].shape[2:])[slots] = s["v"].half()
    return {"q": q, "k": k, "key_cache": s["kc"], "value_cache": s["vc"]}


def _plain_pages(s):
    c, bs = s["case"], s["case"]["block"]
    tables, lens, ring, pool, rows = s["tables"], s["lens"], s["ring"], s["pool"], s["rows"].long()
    size, dev = ring.shape[0], ring.device
    # reserve
    old, new = lens[rows].long(), s["new"].long()
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    had = (old + bs - 1) // bs
    need = (old + new + bs - 1) // bs - had
    base = need.cumsum(0) - need
    t = torch.arange(s["tokens"], device=dev)
    real = t < cu[-1]
    t = torch.minimum(t, cu[-1] - 1)
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = old[seq] + t - cu[seq]
    page_at = pos // bs
    fresh = page_at - had[seq]
    taken = ring[(pool[0] + base[seq] + fresh.clamp(min=0)) % size]
    page = torch.where(fresh >= 0, taken, tables[rows[seq], page_at])
    tables[rows[seq], page_at] = page
    slots = torch.where(real, page * bs + (pos % bs).int(), torch.full_like(page, -1))
    positions = torch.where(real, pos, torch.zeros_like(pos)).int()
    lens[rows] = (old + new).int()
    pool[0] = (pool[0] + need.sum()) % size
    pool[1] -= need.sum()
    batch_tables, batch_lens = tables[rows], lens[rows]
    # truncate to what the rows had
    length, keep = lens[rows].long(), s["old"].long()
    first = (keep + bs - 1) // bs
    freed = (length + bs - 1) // bs - first
    base = freed.cumsum(0) - freed
    at = torch.arange(tables.shape[1], device=dev)
    gone = (at >= first[:, None]) & (at < (first + freed)[:, None])
    rank = base[:, None] + at - first[:, None]
    mine = tables[rows]
    ring[(pool[0] + pool[1] + rank[gone]) % size] = mine[gone]
    tables[rows] = mine.masked_fill(gone, -1)
    lens[rows] = keep.int()
    pool[1] += freed.sum()
    return {"cu_seqlens": cu.int(), "slot_mapping": slots, "positions": positions, "batch_tables": batch_tables,
            "batch_lens": batch_lens, "tables": tables, "lens": lens, "ring": ring, "pool": pool}


def _own_pages(s):
    C, bs = _ops(), s["case"]["block"]
    cu, slots, positions, tables, lens = C.reserve_slots(s["tables"], s["lens"], s["ring"], s["pool"], s["rows"],
                                                         s["new"], bs, s["tokens"])
    C.truncate_rows(s["tables"], s["lens"], s["ring"], s["pool"], s["rows"], s["old"], bs)
    return {"cu_seqlens": cu, "slot_mapping": slots, "positions": positions, "batch_tables": tables,
            "batch_lens": lens, "tables": s["tables"], "lens": s["lens"], "ring": s["ring"], "pool": s["pool"]}


def run(state):
    c = state["case"]
    if c["op"] == "attention":
        if own:
            return _ops().packed_attention(state["q"], state["k"], state["v"], state["cu"], state["longest"],
                                           c["window"], c["causal"])
        return _plain_attention(state)
    if c["op"] == "rotary":
        if not own:
            return _plain_rotary(state)
        if not c["cache"]:
            q, k = _ops().apply_rotary(state["q"], state["k"], state["pos"], state["freq"], _sections(c),
                                       c["interleaved"])
            return {"q": q, "k": k}
        q, k = _ops().rotary_write_cache(state["q"], state["k"], state["v"], state["pos"], state["freq"],
                                         _sections(c), state["slots"], state["kc"], state["vc"], c["interleaved"])
        return {"q": q, "k": k, "key_cache": state["kc"], "value_cache": state["vc"]}
    return _own_pages(state) if own else _plain_pages(state)


def exact(case, seed):
    """The operators' definitions in 64 bits, one sequence or one axis at a time."""
    if case["op"] == "pages":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "attention":
        q, k, v, cu = s["q"], s["k"], s["v"], s["cu"].tolist()
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        group = case["heads"] // case["kv_heads"]
        for lo, hi in zip(cu[:-1], cu[1:]):
            n = hi - lo
            if n == 0:
                continue
            i = torch.arange(n, device=q.device)
            ends = i + 1 if case["causal"] else torch.full_like(i, n)
            starts = torch.clamp(ends - case["window"], min=0) if case["window"] > 0 else torch.zeros_like(i)
            hidden = (i[None, :] >= ends[:, None]) | (i[None, :] < starts[:, None])
            for head in range(case["heads"]):
                kk, vv = k[lo:hi, head // group].double(), v[lo:hi, head // group].double()
                logits = q[lo:hi, head].double() @ kk.t() / case["dim"] ** 0.5
                out[lo:hi, head] = torch.softmax(logits.masked_fill(hidden, float("-inf")), -1) @ vv
        return out
    p = case["pairs"]
    got = {}
    for name in ("q", "k"):
        x = s[name].double()
        y = x.clone()
        begin = 0
        for axis, count in enumerate(_sections(case)):
            for i in range(begin, begin + count):
                a = s["pos"][axis].double() * s["freq"][i]
                one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + p)
                cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None]
                y[:, :, one] = x[:, :, one] * cos - x[:, :, two] * sin
                y[:, :, two] = x[:, :, one] * sin + x[:, :, two] * cos
            begin += count
        got[name] = y
    if case["cache"]:
        for name, rows in (("key_cache", got["k"]), ("value_cache", s["v"].double())):
            pool = torch.zeros(s["kc"].shape, dtype=torch.float64, device=rows.device)
            pool.view(-1, *pool.shape[2:])[s["slots"].long()] = rows
            got[name] = pool
    return got
