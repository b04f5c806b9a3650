"""Measured cases of four operators of a serving step: attention with a
sliding window and first positions that stay visible (sinks) over the paged
8-bit cache, norms and rotation of query and key heads, the pages of the cache
(forked, reserved with copies of what is shared, released, compacted), and
routing of tokens to experts.

``run`` computes an operator in elementary torch operations where ``own`` is
false and through the framework's entry points where it is true; ``exact``
gives the same outputs from the definition, numbers in 64 bits.

The cache is held in 8-bit codes with one scale per block of 16 positions and
kv head, keys and values apart:

* key codes   ``[n_pages, n_kv_heads, page_tokens / 16, 16, d_head]``,
* value codes ``[n_pages, n_kv_heads, page_tokens / 16, d_head, 16]``,
* scales      ``[n_pages, n_kv_heads, page_tokens / 16]``.

A batch is ``n_seqs`` sequences: rows ``row_offsets[s] .. row_offsets[s + 1]``
are the newest positions of sequence ``s``, the last of them at
``seq_lens[s] - 1``; ``pages[s]`` holds its page ids in order, -1 where it has
no page.  ``refs[p]`` counts the table entries that name page p, 0 where it is
free.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -----------------------------------------------------------------

def listed():
    return [
        # the next token of one long chat: latency
        {"name": "sinks_1", "kind": "sinks", "seqs": 1, "new": 1, "ctx": 5000, "ragged": False, "q": 32, "kv": 4,
         "d": 64, "rope": 64, "dtype": "f32", "page": 64, "window": 1024, "sinks": 4},
        # a serving batch of long chats whose middles are freed
        {"name": "sinks_64", "kind": "sinks", "seqs": 64, "new": 1, "ctx": 30000, "ragged": True, "q": 32, "kv": 8,
         "d": 128, "rope": 128, "dtype": "f16", "page": 16, "window": 4096, "sinks": 4},
        # chunks of prompts against what is cached
        {"name": "sinks_chunk", "kind": "sinks", "seqs": 3, "new": 500, "ctx": 9000, "ragged": True, "q": 32, "kv": 8,
         "d": 128, "rope": 128, "dtype": "bf16", "page": 128, "window": 2048, "sinks": 64},
        # whole prompts
        {"name": "sinks_prompts", "kind": "sinks", "seqs": 2, "new": 6000, "ctx": 6000, "ragged": True, "q": 32,
         "kv": 8, "d": 128, "rope": 128, "dtype": "f16", "page": 64, "window": 1024, "sinks": 4},
        # one token's heads in front of the cache, f32 from the GEMV
        {"name": "rotate_1", "kind": "rotate", "seqs": 1, "new": 1, "ctx": 700, "ragged": False, "q": 32, "kv": 4,
         "d": 64, "rope": 64, "layout": "half", "dtype": "f32", "out": "f32", "norm": True},
        # a serving batch's single tokens, a quarter of each head rotated
        {"name": "rotate_64", "kind": "rotate", "seqs": 64, "new": 1, "ctx": 4000, "ragged": True, "q": 16, "kv": 2,
         "d": 256, "rope": 64, "layout": "half", "dtype": "f32", "out": "f16", "norm": True},
        # prompts, neighbouring values as pairs
        {"name": "rotate_prompts", "kind": "rotate", "seqs": 5, "new": 2500, "ctx": 2500, "ragged": True, "q": 32,
         "kv": 8, "d": 128, "rope": 128, "layout": "neighbours", "dtype": "f16", "out": "f16", "norm": True},
        # four beams of one prompt go on to their next token
        {"name": "fork_4", "kind": "fork", "prompts": 1, "beams": 4, "ctx": 300, "kv": 4, "d": 64, "page": 64},
        # eight answers to each of sixteen prompts
        {"name": "fork_128", "kind": "fork", "prompts": 16, "beams": 8, "ctx": 2040, "kv": 8, "d": 128, "page": 128},
        # half of a serving batch ends, the rest moves together, new prompts take the room
        {"name": "compact_64", "kind": "compact", "seqs": 64, "ctx": 4096, "kv": 8, "d": 128, "page": 16},
        # one decode step of a model of eight experts
        {"name": "route_64", "kind": "route", "rows": 64, "experts": 8, "top_k": 2, "dtype": "f32",
         "scoring": "softmax", "bias": False, "groups": 1, "kept": 1, "group_top": 1, "normalize": True},
        # prompts through a layer of many experts: groups first, a bias that balances them
        {"name": "route_prompts", "kind": "route", "rows": 12289, "experts": 256, "top_k": 8, "dtype": "bf16",
         "scoring": "sigmoid", "bias": True, "groups": 8, "kept": 4, "group_top": 2, "normalize": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["sinks", "sinks", "sinks", "rotate", "rotate", "fork", "compact", "route", "route"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 4, 512 // groups)
        kept = groups if groups < 4 else rng.randint(2, groups)
        return {"kind": kind, "rows": _log(rng, 1, min(16384, (1 << 22) // experts)), "experts": experts,
                "top_k": min(rng.choice([1, 2, 4, 6, 8]), kept * (experts // groups)),
                "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "scoring": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "kept": kept, "group_top": rng.choice([1, 2]),
                "normalize": rng.random() < 0.7}
    kv = rng.choice([1, 2, 4, 8, 8])
    if kind in ("fork", "compact"):
        c = {"kind": kind, "kv": kv, "d": rng.choice([64, 128, 128, 192, 256]), "page": rng.choice([16, 32, 64, 128, 256])}
        if kind == "fork":
            c["prompts"], c["beams"] = _log(rng, 1, 32), rng.randint(2, 8)
            c["ctx"] = _log(rng, 20, 4096)
        else:
            c["seqs"] = 2 * _log(rng, 1, 48)
            c["ctx"] = _log(rng, 20, 8192)
        while work(c)["bytes"] > 4e8:  # no more than the largest listed case
            c["ctx"] = max(20, c["ctx"] // 2)
        return c
    c = {"kind": kind, "kv": kv, "ragged": rng.random() < 0.8}
    mode = rng.choice(["token", "token", "draft", "chunk", "prompt"])
    if mode == "token":
        c["new"], c["seqs"] = 1, _log(rng, 1, 128)
        c["ctx"] = _log(rng, 16, 131072)
    elif mode == "draft":
        c["new"], c["seqs"] = rng.randint(2, 12), _log(rng, 1, 32)
        c["ctx"] = _log(rng, 64, 32768)
    elif mode == "chunk":
        c["new"], c["seqs"] = _log(rng, 16, 512), _log(rng, 1, 8)
        c["ctx"] = c["new"] + _log(rng, 1, 12000)
    else:
        c["seqs"] = _log(rng, 1, 6)
        c["new"] = c["ctx"] = _log(rng, 32, 12000 // c["seqs"] if kind == "rotate" else 6000)
    if kind == "rotate":
        c["q"] = kv * rng.choice([1, 2, 4, 8])
        c["d"] = rng.choice([64, 128, 128, 256, 80, 96, 112])
        c["rope"] = rng.choice([c["d"], c["d"], c["d"] // 2, c["d"] // 8 * 2, 0])
        c["layout"] = rng.choice(["half", "neighbours"])
        c["dtype"] = rng.choice(["f32", "f16", "bf16"])
        c["out"] = rng.choice([c["dtype"], c["dtype"], "f16", "f32"])
        c["norm"] = rng.random() < 0.7
    else:
        c["d"] = rng.choice([64, 128, 128, 192, 256])
        c["rope"] = rng.choice([0, c["d"] // 2, c["d"], c["d"]])
        c["dtype"] = rng.choice(["f32", "f16", "f16", "bf16"])
        c["page"] = rng.choice([16, 32, 64, 128, 256])
        c["q"] = kv * rng.choice([1, 2, 4, 4, 7, 8] if kv <= 4 else [1, 2, 3, 4])
        c["window"] = _log(rng, 1, 8192)
        c["sinks"] = rng.choice([0, 1, 4, 4, _log(rng, 1, 300)])
    while work(c)["flops"] > 1.9e11 or work(c)["bytes"] > 4e8:  # no more than the largest listed case
        if c["seqs"] > 1:
            c["seqs"] //= 2
        else:
            c["ctx"] = max(c["new"], c["ctx"] // 2)
            c["new"] = max(1, c["new"] // 2) if mode in ("chunk", "prompt") else c["new"]
    return c


# ---- what a program has in hand --------------------------------------------------

def _lengths(case):
    """(new, length) of every sequence."""
    rng = random.Random(case["seqs"] * 1000003 + case["ctx"] * 101 + case["new"])
    out = []
    for s in range(case["seqs"]):
        new, ctx = case["new"], case["ctx"]
        if case["ragged"] and s:  # the first one has the full size
            whole = new == ctx
            if new > 1:
                new = rng.randint(max(1, new // 4), new)
            ctx = new if whole else rng.randint(max(new, ctx // 4), ctx)
        out.append((new, max(new, ctx)))
    return out


def _pairs(case):
    """(query, key) pairs of one query head."""
    total, w, k = 0, case["window"], case["sinks"]
    for new, ctx in _lengths(case):
        for a, b, full in ((ctx - new, min(ctx, w), False), (max(ctx - new, w), ctx, True)):
            n = max(0, b - a)  # positions a .. b - 1: those before the window's length see all, the others it and sinks
            if not full:
                total += n * (a + b + 1) // 2
            else:
                hidden = [max(0, p + 1 - w) for p in (a, min(b, w + k))]  # the first of them see some of the sinks
                m = max(0, min(b, w + k) - a)
                total += n * w + (hidden[0] + hidden[1] - 1) * m // 2 + (n - m) * k
    return total


def _keys(case):
    """Cached positions that some query of the case sees."""
    return sum(min(ctx, new + case["window"] - 1 + min(case["sinks"], max(0, ctx - new - case["window"] + 1)))
               for new, ctx in _lengths(case))


def _rope_table(dim, n_pos):
    """[n_pos, dim / 2, 2] of (cos, sin), base 10000."""
    i = torch.arange(dim // 2, dtype=torch.float64, device=DEVICE)
    theta = torch.arange(n_pos, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (-2 * i / dim)
    return torch.stack([theta.cos(), theta.sin()], -1).float().contiguous()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _prefix(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _pool(case, n_pages, gen):
    """A pool of random codes and scales."""
    shape = (n_pages, case["kv"], case["page"] // BLOCK)
    n = n_pages * case["kv"] * case["page"] * case["d"]

    def codes():
        return (torch.randn(n, device=DEVICE, generator=gen) * 36).round_().clamp_(-127, 127).to(torch.int8)

    def scales(size):
        return (torch.rand(shape, device=DEVICE, generator=gen) * 0.7 + 0.65) * (size / 36)

    return {"n_pages": n_pages, "k": codes().view(*shape, BLOCK, case["d"]), "v": codes().view(*shape, case["d"], BLOCK),
            "k_scale": scales(1.2), "v_scale": scales(0.9)}


def _rows_of(case):
    lens = _lengths(case)
    offs = _prefix([new for new, _ in lens])
    return {"case": case, "kv": case["kv"], "d": case["d"], "n_rows": offs[-1], "n_seqs": len(lens),
            "max_new": max(n for n, _ in lens), "row_offsets": _i32(offs), "seq_lens": _i32([c for _, c in lens])}


def _prepare_sinks(case, gen):
    st, lens, page = _rows_of(case), _lengths(case), case["page"]
    # a program keeps the pages of the sinks and of the oldest query's window
    keep = []
    for new, ctx in lens:
        low = max(0, ctx - new - case["window"] + 1)
        keep.append([i for i in range(-(-ctx // page)) if i * page < case["sinks"] or (i + 1) * page > low])
    n_pages = sum(len(k) for k in keep) + 3
    ids = torch.randperm(n_pages, device=DEVICE, generator=gen).to(torch.int32).cpu()
    st["max_pages"] = max(-(-ctx // page) for _, ctx in lens)
    pages = torch.full((len(lens), st["max_pages"]), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(keep):
        pages[s, torch.tensor(k)] = ids[at:at + len(k)]
        at += len(k)
    st |= _pool(case, n_pages, gen)
    st["pages"] = pages.to(DEVICE)
    st["rope"] = _rope_table(case["rope"], st["max_pages"] * page) if case["rope"] else None
    q, kv, d, t = case["q"], case["kv"], case["d"], TYPES[case["dtype"]]
    st["qkv"] = torch.randn(st["n_rows"], (q + 2 * kv) * d, device=DEVICE, generator=gen).to(t)
    st["in"] = st["qkv"][:, :q * d]
    st["out"] = torch.zeros(st["n_rows"], q, d, dtype=t, device=DEVICE)
    return st


def _prepare_rotate(case, gen):
    st = _rows_of(case)
    rows, q, kv, d = st["n_rows"], case["q"], case["kv"], case["d"]
    # fused projections, tokens and channels of different size
    x = torch.randn(rows, (q + 2 * kv) * d, device=DEVICE, generator=gen)
    x *= (0.3 + 3 * torch.rand(rows, 1, device=DEVICE, generator=gen)) * (0.5 + torch.rand(x.shape[1], device=DEVICE, generator=gen))
    st["qkv"] = x.to(TYPES[case["dtype"]])
    st["in"] = (st["qkv"][:, :q * d], st["qkv"][:, q * d:(q + kv) * d])
    st["weight"] = [(1 + 0.3 * torch.randn(d, device=DEVICE, generator=gen)) if case["norm"] else None for _ in range(2)]
    st["eps"] = 1e-6
    st["n_pos"] = max(ctx for _, ctx in _lengths(case))
    st["rope"] = _rope_table(case["rope"], st["n_pos"]) if case["rope"] else None
    st["out"] = [torch.zeros(rows, n, d, dtype=TYPES[case["out"]], device=DEVICE) for n in (q, kv)]
    return st


def _prepare_fork(case, gen):
    n, page, beams = case["prompts"] * case["beams"], case["page"], case["beams"]
    rng = random.Random(case["ctx"] * 1009 + n * 31 + page)
    lens, counts, shared = [], [], []
    for p in range(case["prompts"]):
        ctx = case["ctx"] if p == 0 else rng.randint(max(2, case["ctx"] // 3), case["ctx"])
        lens += [ctx] * beams                  # the next token's position included
        counts.append(-(-(ctx - 1) // page))   # pages that hold something
        shared.append(int(0.7 * ctx) // page)  # the prompt's whole ones
    used = sum(s + beams * (c - s) for c, s in zip(counts, shared))
    n_pages = used + n + 3
    ids = torch.randperm(n_pages, device=DEVICE, generator=gen).to(torch.int32).cpu().tolist()
    max_pages = max(-(-ctx // page) for ctx in lens) + 1
    table, at = [], 0
    for c, s in zip(counts, shared):
        front, at = ids[at:at + s], at + s
        for _ in range(beams):
            table.append(front + ids[at:at + c - s] + [-1] * (max_pages - c))
            at += c - s
    refs = [0] * n_pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    pick = torch.randint(0, beams, (n,), device=DEVICE, generator=gen).cpu().tolist()
    parents = [i // beams * beams + pick[i] // 2 for i in range(n)]  # the better half of the beams goes on
    st = {"case": case, "page": page, "kv": case["kv"], "d": case["d"], "n_seqs": n, "n_rows": n, "max_pages": max_pages,
          "tables": [_i32(table), torch.full((n, max_pages), -1, dtype=torch.int32, device=DEVICE)], "refs": _i32(refs),
          "parents": _i32(parents), "row_offsets": _i32(list(range(n + 1))), "seq_lens": _i32(lens),
          "missing": torch.zeros(n, dtype=torch.int32, device=DEVICE)}
    return st | _pool(case, n_pages, gen)


def _compact_lens(case):
    """Lengths of the batch: sequences 2 i and 2 i + 1 of the same one."""
    rng = random.Random(case["ctx"] * 1013 + case["seqs"])
    out = []
    for s in range(case["seqs"] // 2):
        out += [case["ctx"] if s == 0 else rng.randint(max(1, case["ctx"] // 4), case["ctx"])] * 2
    return out


def _prepare_compact(case, gen):
    n, page, lens = case["seqs"], case["page"], _compact_lens(case)
    counts = [-(-x // page) for x in lens]
    half = sum(counts) // 2
    n_pages = 2 * half + 5
    low = torch.randperm(half, device=DEVICE, generator=gen).cpu().tolist()
    ids = [low, [half + i for i in torch.randperm(half, device=DEVICE, generator=gen).cpu().tolist()]]
    max_pages = max(counts)
    table, at = [], [0, 0]
    for s, c in enumerate(counts):  # the even ones, which end first, in the lower half
        g = s % 2
        table.append(ids[g][at[g]:at[g] + c] + [-1] * (max_pages - c))
        at[g] += c
    st = {"case": case, "page": page, "kv": case["kv"], "d": case["d"], "n_seqs": n, "max_pages": max_pages, "turn": 0,
          "tables": [_i32(table)], "refs": _i32([1] * (2 * half) + [0] * 5), "seq_lens": _i32(lens),
          "new_ids": torch.zeros(n_pages, dtype=torch.int32, device=DEVICE), "n_used": torch.zeros(1, dtype=torch.int32, device=DEVICE),
          "missing": torch.zeros(n, dtype=torch.int32, device=DEVICE)}
    st["ends"] = [_i32([max_pages * page if s % 2 == g else 0 for s in range(n)]) for g in range(2)]
    offs = [_prefix([x if s % 2 == g else 0 for s, x in enumerate(lens)]) for g in range(2)]
    st["offsets"], st["n_rows"] = [_i32(o) for o in offs], offs[0][-1]
    return st | _pool(case, n_pages, gen)


def _prepare_route(case, gen):
    n, e = case["rows"], case["experts"]
    stride = (e + 31) // 32 * 32 + 32  # rows of a fused projection's buffer
    lg = torch.randn(n, stride, device=DEVICE, generator=gen) * (0.5 + 1.5 * torch.rand(n, 1, device=DEVICE, generator=gen))
    lg += 0.5 * torch.randn(stride, device=DEVICE, generator=gen)  # experts that are liked more than others
    return {"case": case, "logits": lg.to(TYPES[case["dtype"]]), "stride": stride, "scale": 2.5 if case["scoring"] == "sigmoid" else 1.0,
            "bias": 0.2 * torch.randn(e, device=DEVICE, generator=gen) if case["bias"] else None,
            "ids": torch.zeros(n, case["top_k"], dtype=torch.int32, device=DEVICE),
            "weights": torch.zeros(n, case["top_k"], device=DEVICE)}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    make = {"sinks": _prepare_sinks, "rotate": _prepare_rotate, "fork": _prepare_fork, "compact": _prepare_compact,
            "route": _prepare_route}
    return make[case["kind"]](case, gen)


# ---- the framework's calls -------------------------------------------------------

_context = None


def _ctx():
    """The one context that a program keeps."""
    global _context
    if _context is None:
        import rce_amd
        _context = rce_amd.Context(0)
    return _context


def _own_cache(st):
    import rce_amd
    return rce_amd.KvCache(st["n_pages"], st["case"]["page"], st["kv"], st["d"], k=st["k"].data_ptr(), v=st["v"].data_ptr(),
                           k_scale=st["k_scale"].data_ptr(), v_scale=st["v_scale"].data_ptr())


def _own_batch(st, offsets, pages):
    import rce_amd
    return rce_amd.KvBatch(row_offsets=offsets.data_ptr(), seq_lens=st["seq_lens"].data_ptr(),
                           pages=0 if pages is None else pages.data_ptr(), n_seqs=st["n_seqs"], n_rows=st["n_rows"],
                           max_pages=0 if pages is None else st["max_pages"])


def _own_rope(st, n_pos):
    import rce_amd
    if st["rope"] is None:
        return None
    return rce_amd.Rope(st["rope"].data_ptr(), dim=st["case"]["rope"], n_pos=n_pos)


def _own_dtype(t):
    import rce_amd
    return {torch.float32: rce_amd.GgufDtype.F32, torch.float16: rce_amd.GgufDtype.F16,
            torch.bfloat16: rce_amd.GgufDtype.BF16}[t]


def _own_sinks(st):
    import rce_amd
    q, out, c = st["in"], st["out"], st["case"]
    rce_amd.kv_attention_sinks_dev(_ctx(), _own_cache(st), _own_batch(st, st["row_offsets"], st["pages"]), q.data_ptr(),
                                   _own_dtype(q.dtype), q.stride(0), c["q"], out.data_ptr(), _own_dtype(out.dtype),
                                   scale=1 / math.sqrt(st["d"]), window=c["window"], sinks=c["sinks"],
                                   rope=_own_rope(st, st["max_pages"] * c["page"]))
    return out


def _own_rotate(st):
    import rce_amd
    c, (q, k), (qo, ko), (qw, kw) = st["case"], st["in"], st["out"], st["weight"]
    heads = lambda x, o, w, n: rce_amd.Heads(x.data_ptr(), x.stride(0), n, o.data_ptr(), o.stride(0),  # noqa: E731
                                             weight=0 if w is None else w.data_ptr())
    rce_amd.qk_norm_rope_dev(_ctx(), _own_batch(st, st["row_offsets"], None), heads(q, qo, qw, c["q"]), heads(k, ko, kw, c["kv"]),
                             st["d"], _own_dtype(q.dtype), _own_dtype(qo.dtype), eps=st["eps"] if c["norm"] else None,
                             rope=_own_rope(st, st["n_pos"]), interleaved=c["layout"] == "neighbours")
    return {"q": qo, "k": ko}


def _own_table(st, t):
    import rce_amd
    return rce_amd.KvTable(t.data_ptr(), st["n_seqs"], st["max_pages"])


def _own_fork(st):
    import rce_amd
    ctx, cache, (a, b) = _ctx(), _own_cache(st), st["tables"]
    ta, tb, refs = _own_table(st, a), _own_table(st, b), st["refs"].data_ptr()
    rce_amd.kv_fork_dev(ctx, cache, ta, tb, st["parents"].data_ptr(), refs)
    rce_amd.kv_release_dev(ctx, cache, ta, refs)
    rce_amd.kv_reserve_dev(ctx, cache, _own_batch(st, st["row_offsets"], b), refs, st["missing"].data_ptr())
    st["tables"] = [b, a]
    return _pages_out(st)


def _own_compact(st):
    import rce_amd
    ctx, cache, table, g = _ctx(), _own_cache(st), st["tables"][0], st["turn"]
    t, refs = _own_table(st, table), st["refs"].data_ptr()
    rce_amd.kv_release_dev(ctx, cache, t, refs, to_dev=st["ends"][g].data_ptr())
    rce_amd.kv_compact_dev(ctx, cache, t, refs, st["new_ids"].data_ptr(), st["n_used"].data_ptr())
    rce_amd.kv_reserve_dev(ctx, cache, _own_batch(st, st["offsets"][g], table), refs, st["missing"].data_ptr())
    st["turn"] = 1 - g
    return _pages_out(st)


def _own_route(st):
    import rce_amd
    c = st["case"]
    how = rce_amd.MoeRouting(c["top_k"], sigmoid=c["scoring"] == "sigmoid", bias_dev=0 if st["bias"] is None else st["bias"].data_ptr(),
                             n_group=c["groups"], topk_group=c["kept"], group_top=c["group_top"], normalize=c["normalize"],
                             scale=st["scale"])
    rce_amd.moe_route_dev(_ctx(), st["logits"].data_ptr(), _own_dtype(st["logits"].dtype), c["rows"], c["experts"], st["stride"],
                          how, st["ids"].data_ptr(), st["weights"].data_ptr())
    return {"ids": st["ids"], "weights": st["weights"]}


# ---- the plain form --------------------------------------------------------------

def _rows(st):
    """Sequence and position of every row."""
    r, offsets = torch.arange(st["n_rows"], device=DEVICE), st["row_offsets"]
    s = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    return s, st["seq_lens"].long()[s] - (offsets.long()[s + 1] - r)


def _rotate(st, x, pos, neighbours=False):
    """[rows, heads, d] in f32, pairs (i, i + rope / 2), or (2 i, 2 i + 1), of each head's first `rope` values rotated."""
    if st["rope"] is None:
        return x
    h = st["rope"].shape[1]
    cs = st["rope"][pos][:, None]
    c, s = cs[..., 0], cs[..., 1]
    a, b = (x[..., :2 * h:2], x[..., 1:2 * h:2]) if neighbours else (x[..., :h], x[..., h:2 * h])
    a, b = a * c - b * s, a * s + b * c
    front = torch.stack([a, b], -1).flatten(-2) if neighbours else torch.cat([a, b], -1)
    return torch.cat([front, x[..., 2 * h:]], -1)


def _plain_sinks(st):
    c, d, kv = st["case"], st["d"], st["kv"]
    heads, per, w, page = c["q"], c["q"] // kv, c["window"], c["page"]
    s, pos = _rows(st)
    at = torch.arange(st["n_rows"], device=DEVICE) - st["row_offsets"].long()[s]
    q = torch.zeros(st["n_seqs"], st["max_new"], heads, d, device=DEVICE)
    q[s, at] = _rotate(st, st["in"].reshape(-1, heads, d).float(), pos)
    q = q.view(-1, st["max_new"], kv, per, d).permute(0, 2, 3, 1, 4).reshape(-1, kv, per * st["max_new"], d)
    # the positions that some row of the sequence sees: the sinks, and from the oldest row's window on
    first = st["seq_lens"].long() - (st["row_offsets"][1:] - st["row_offsets"][:-1]).long()
    low = (first - w + 1).clamp(min=0)
    n = min(c["ctx"], st["max_new"] + w - 1)
    sink = torch.arange(c["sinks"], device=DEVICE).expand(st["n_seqs"], -1)
    j = torch.cat([torch.where(sink < low[:, None], sink, -1), low[:, None] + torch.arange(n, device=DEVICE)], 1)
    ok = (j >= 0) & (j < st["seq_lens"][:, None])
    jc = torch.where(ok, j, low[:, None])
    pg, blk, slot = st["pages"].long().gather(1, jc // page), jc % page // BLOCK, jc % BLOCK
    k = (st["k"][pg, :, blk, slot].float() * st["k_scale"][pg, :, blk][..., None]).permute(0, 2, 3, 1).contiguous()
    v = (st["v"][pg, :, blk, :, slot].float() * st["v_scale"][pg, :, blk][..., None]).transpose(1, 2).contiguous()
    score = torch.matmul(q, k) * (1 / math.sqrt(d))
    p = torch.full((st["n_seqs"], st["max_new"]), -1, device=DEVICE)
    p[s, at] = pos
    jj = j[:, None]
    see = ok[:, None] & (jj <= p[..., None]) & ((jj > p[..., None] - w) | (jj < c["sinks"]))
    score = score.view(-1, kv, per, st["max_new"], j.shape[1])
    score = torch.where(see[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(-1, kv, per * st["max_new"], j.shape[1]), v).view(-1, kv, per, st["max_new"], d)
    o = torch.where(total > 0, o / torch.where(total > 0, total, 1.0), 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(st["n_seqs"], st["max_new"], heads, d)
    return o[s, at].to(st["out"].dtype)


def _plain_rotate(st):
    c, (q, k) = st["case"], st["in"]
    _, pos = _rows(st)

    def one(x, w, out):
        x = x.reshape(st["n_rows"], -1, st["d"]).float()
        if c["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + st["eps"]) * w
        return _rotate(st, x, pos, c["layout"] == "neighbours").to(out.dtype)

    return {"q": one(q, st["weight"][0], st["out"][0]), "k": one(k, st["weight"][1], st["out"][1])}


def _pages_out(st):
    out = {n: st[n] for n in ("refs", "k", "v", "k_scale", "v_scale", "missing") + (("new_ids", "n_used") if "turn" in st else ())}
    return out | {"table": st["tables"][0]}


def _count(st, entries, by):
    """refs plus `by` for each of the entries that names a page."""
    ok = (entries >= 0) & (entries < st["n_pages"])
    st["refs"].scatter_add_(0, torch.where(ok, entries, 0).long().flatten(), (ok * by).to(torch.int32).flatten())


def _plain_reserve(st, table, offsets):
    """Every page that the batch's rows touch becomes one of their sequence's own: a free one (the lowest first) where it
    has none or others name it too; what stands in front of the rows is copied.  Where all that name a page ask, the first keeps it."""
    page, refs, n_pages = st["page"], st["refs"], st["n_pages"]
    new = (offsets[1:] - offsets[:-1]).long()
    first, last = st["seq_lens"].long() - new, st["seq_lens"].long() - 1
    i = torch.arange(st["max_pages"], device=DEVICE)
    touched = (i >= first[:, None] // page) & (i <= last[:, None] // page) & (new > 0)[:, None]
    e = table.long()
    named = (e >= 0) & (e < n_pages)
    ec = torch.where(named, e, 0)
    ask = (touched & named & (refs[ec] > 1)).flatten()
    ec = ec.flatten()
    asked = torch.zeros(n_pages, dtype=torch.int32, device=DEVICE).scatter_add_(0, ec, ask.to(torch.int32))
    order = torch.arange(ec.numel(), device=DEVICE)
    first_ask = torch.full((n_pages,), ec.numel(), device=DEVICE).scatter_reduce_(0, ec, torch.where(ask, order, ec.numel()), "amin")
    leave = ask & ~((asked == refs)[ec] & (first_ask[ec] == order))
    need = leave | (touched & ~named).flatten()
    rank = need.long().cumsum(0) - 1
    free = torch.nonzero(refs == 0).flatten()
    got = torch.where(rank < free.numel(), torch.cat([free, free.new_zeros(1)])[rank.clamp(max=free.numel())], -1)
    refs.scatter_add_(0, ec, -leave.to(torch.int32))
    to = got[need]
    refs[to[to >= 0]] = 1
    st["missing"].copy_((need & (got < 0)).view(table.shape).sum(1))
    table.copy_(torch.where(need, got, e.flatten()).view(table.shape))
    # blocks in front of the first new position of its page
    at = order % st["max_pages"]
    f = first.repeat_interleave(st["max_pages"])
    blocks = torch.where(at == f // page, (f % page + BLOCK - 1) // BLOCK, 0)
    b = torch.arange(page // BLOCK, device=DEVICE)
    item, b = torch.nonzero((leave & (got >= 0))[:, None] & (b < blocks[:, None]), as_tuple=True)
    src, dst = ec[item], got[item]
    for n in ("k", "v", "k_scale", "v_scale"):
        st[n][dst, :, b] = st[n][src, :, b]


def _plain_fork(st):
    a, b = st["tables"]
    b.copy_(a[st["parents"].long()])
    _count(st, b, 1)
    _count(st, a, -1)
    a.fill_(-1)
    _plain_reserve(st, b, st["row_offsets"])
    st["tables"] = [b, a]
    return _pages_out(st)


def _plain_compact(st):
    table, g, n_pages, refs = st["tables"][0], st["turn"], st["n_pages"], st["refs"]
    i = torch.arange(st["max_pages"], device=DEVICE)
    gone = (i + 1) * st["page"] <= st["ends"][g][:, None]
    _count(st, torch.where(gone, table, -1), -1)
    table.masked_fill_(gone, -1)
    used = refs != 0
    n_used = used.sum()
    p = torch.arange(n_pages, device=DEVICE)
    src, dst = torch.nonzero(used & (p >= n_used)).flatten(), torch.nonzero(~used & (p < n_used)).flatten()
    new_ids = torch.where(used, p, -1)
    new_ids[src] = dst
    for n in ("k", "v", "k_scale", "v_scale"):
        st[n][dst] = st[n][src]
    refs[dst] = refs[src]
    refs[src] = 0
    ok = (table >= 0) & (table < n_pages)
    table.copy_(torch.where(ok, new_ids[torch.where(ok, table, 0).long()], table))
    st["new_ids"].copy_(new_ids)
    st["n_used"].copy_(n_used)
    _plain_reserve(st, table, st["offsets"][g])
    st["turn"] = 1 - g
    return _pages_out(st)


def _plain_route(st):
    c = st["case"]
    n, e, g = c["rows"], c["experts"], c["groups"]
    lg = st["logits"][:, :e].double()
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    if c["scoring"] == "sigmoid":
        score = 1 / (1 + torch.exp(-lg))
    else:
        top = lg.amax(-1, keepdim=True)
        w = torch.where(lg == top, 1.0, torch.exp(lg - top))
        score = w / w.sum(-1, keepdim=True)
    # without a bias the scores' order is the logits' own
    key = score + st["bias"].double() if c["bias"] else lg if c["group_top"] == 1 or g == 1 else score
    key = torch.where((lg == -math.inf) | torch.isnan(key), -math.inf, key)
    if g > 1:
        best = torch.sort(key.view(n, g, e // g), dim=-1, descending=True).values[..., :c["group_top"]]
        size = torch.where(best > -math.inf, best, 0.0).sum(-1)
        size = torch.where(best[..., 0] > -math.inf, size, -math.inf)
        kept = torch.sort(size, dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        see = torch.zeros(n, g, dtype=torch.bool, device=DEVICE).scatter_(1, kept, True).repeat_interleave(e // g, 1)
        key = key if c["bias"] else lg
        order = torch.sort(torch.where(see, key, -math.inf), dim=-1, descending=True, stable=True).indices
        # where what is left has no weight: the kept groups' first, by their ids
        order = order.gather(1, torch.sort((~see.gather(1, order)).to(torch.int8), dim=-1, stable=True).indices)
    else:
        order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    ids = order[:, :c["top_k"]]
    w = torch.where(key.gather(1, ids) > -math.inf, score.gather(1, ids), 0.0)
    if c["normalize"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / torch.where(total > 0, total, 1.0), 0.0)
    return {"ids": ids.to(torch.int32), "weights": (w * st["scale"]).float()}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"sinks": _own_sinks, "rotate": _own_rotate, "fork": _own_fork, "compact": _own_compact, "route": _own_route}[kind](state)
    return {"sinks": _plain_sinks, "rotate": _plain_rotate, "fork": _plain_fork, "compact": _plain_compact,
            "route": _plain_route}[kind](state)


# ---- work ------------------------------------------------------------------------

def _page_bytes(case, blocks):
    """Codes and scales of so many blocks of every head."""
    return 2 * case["kv"] * blocks * (BLOCK * case["d"] + 4)


def work(case):
    kind = case["kind"]
    if kind == "route":
        n = case["rows"] * case["experts"]
        return {"bytes": n * TYPES[case["dtype"]].itemsize + case["rows"] * case["top_k"] * 8, "flops": 10 * n}
    if kind == "fork":
        n, page = case["prompts"] * case["beams"], case["page"]
        entries = n * (-(-case["ctx"] // page) + 1)
        # half of the beams' last pages are copied, half full; three passes over the tables
        copied = n // 2 * _page_bytes(case, max(1, page // BLOCK // 2))
        return {"bytes": 2 * copied + 4 * 5 * entries, "flops": entries}
    if kind == "compact":
        lens, page = _compact_lens(case), case["page"]
        pages = sum(-(-x // page) for x in lens) // 2  # one half's, read and written
        return {"bytes": 2 * pages * _page_bytes(case, page // BLOCK) + 4 * 10 * pages, "flops": 4 * pages}
    d, kv, lens = case["d"], case["kv"], _lengths(case)
    rows, size = sum(n for n, _ in lens), TYPES[case["dtype"]].itemsize
    if kind == "rotate":
        values = rows * (case["q"] + kv) * d
        return {"bytes": values * (size + TYPES[case["out"]].itemsize) + 4 * min(rows, case["ctx"]) * case["rope"],
                "flops": 8 * values}
    keys = _keys(case)
    return {"bytes": 2 * kv * keys * d + kv * keys // 2 + 2 * rows * case["q"] * d * size,
            "flops": 4 * d * case["q"] * _pairs(case)}


# ---- the definition in 64 bits ----------------------------------------------------

def _exact_rope(st, x, pos, neighbours=False):
    """x [rows, heads, d] of the positions `pos` as complex pairs times the table's."""
    if st["rope"] is None:
        return x
    h = st["rope"].shape[1]
    if neighbours:
        z = torch.view_as_complex(x[..., :2 * h].reshape(*x.shape[:-1], h, 2).contiguous())
    else:
        z = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous())
    z = z * torch.view_as_complex(st["rope"].double())[pos][:, None]
    front = torch.view_as_real(z).flatten(-2) if neighbours else torch.cat([z.real, z.imag], -1)
    return torch.cat([front, x[..., 2 * h:]], -1)


def _exact_values(st, name, s, p):
    """[positions, heads, d] of one cache at the positions p of sequence s."""
    page = st["case"]["page"]
    pg, blk, slot = st["pages"][s].long()[p // page], p % page // BLOCK, p % BLOCK
    codes = st[name] if name == "k" else st[name].transpose(-1, -2)
    return codes[pg, :, blk, slot].double() * st[name + "_scale"][pg, :, blk].double()[..., None]


def _exact_sinks(st):
    c, offs = st["case"], st["row_offsets"].tolist()
    d, per, w, sinks = st["d"], c["q"] // st["kv"], c["window"], c["sinks"]
    out = torch.zeros(st["n_rows"], c["q"], d, dtype=torch.float64, device=DEVICE)
    for s, (new, ctx) in enumerate(_lengths(c)):
        for a in range(0, new, 1024):  # rows together
            b = min(new, a + 1024)
            pos = torch.arange(ctx - new + a, ctx - new + b, device=DEVICE)
            low = max(0, int(pos[0]) - w + 1)
            key = torch.cat([torch.arange(min(sinks, low), device=DEVICE), torch.arange(low, int(pos[-1]) + 1, device=DEVICE)])
            k, v = _exact_values(st, "k", s, key), _exact_values(st, "v", s, key)
            r = slice(offs[s] + a, offs[s] + b)
            q = _exact_rope(st, st["in"][r].double().reshape(b - a, c["q"], d), pos)
            back = pos[:, None] - key
            hide = (back < 0) | ((back >= w) & (key >= sinks))
            for h in range(c["q"]):
                p = q[:, h] @ k[:, h // per].T / math.sqrt(d)
                out[r, h] = torch.softmax(p.masked_fill_(hide, -math.inf), -1) @ v[:, h // per]
    return out


def _exact_rotate(st):
    c, out = st["case"], {}
    pos = torch.cat([torch.arange(ctx - new, ctx, device=DEVICE) for new, ctx in _lengths(c)])
    for name, x, w in zip("qk", st["in"], st["weight"]):
        x = x.double().reshape(st["n_rows"], -1, st["d"])
        if c["norm"]:
            x = x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / st["d"] + st["eps"]).sqrt() * w.double()
        out[name] = _exact_rope(st, x, pos, c["layout"] == "neighbours")
    return out


def _exact_reserve(table, refs, rows, page, copies):
    """rows: (sequence, first, last position); the pages of the table one after the other."""
    named = {}
    items = [(s, i, first) for s, first, last in rows for i in range(first // page, last // page + 1)]
    for s, i, _ in items:
        p = table[s][i]
        if p >= 0 and refs[p] > 1:
            named.setdefault(p, []).append((s, i))
    keep = {v[0] for p, v in named.items() if len(v) == refs[p]}
    free = (p for p, n in enumerate(list(refs)) if n == 0)
    missing = [0] * len(table)
    asks = {x for v in named.values() for x in v} - keep
    for s, i, first in items:
        old = table[s][i]
        if old >= 0 and (s, i) not in asks:
            continue
        new = next(free, -1)
        if old >= 0:
            refs[old] -= 1
        if new < 0:
            missing[s] += 1
        else:
            refs[new] = 1
            if old >= 0 and i == first // page:
                copies.append((old, new, -(-(first % page) // BLOCK)))
        table[s][i] = new
    return missing


def _exact_pages(st):
    c, page, lens = st["case"], st["case"]["page"], st["seq_lens"].tolist()
    refs, table, copies, moved = st["refs"].tolist(), st["tables"][0].tolist(), [], []
    out = {}
    if c["kind"] == "fork":
        parents = st["parents"].tolist()
        new = [list(table[p]) for p in parents]
        for rows, by in ((new, 1), (table, -1)):
            for row in rows:
                for p in row:
                    if p >= 0:
                        refs[p] += by
        table = new
        rows = [(s, n - 1, n - 1) for s, n in enumerate(lens)]
    else:
        for s in range(0, len(table), 2):
            for i, p in enumerate(table[s]):
                if p >= 0:
                    refs[p] -= 1
                table[s][i] = -1
        n_used = sum(n != 0 for n in refs)
        holes = [p for p in range(n_used) if refs[p] == 0]
        moved = list(zip([p for p in range(n_used, len(refs)) if refs[p]], holes))
        to = dict(moved)
        out["new_ids"] = _i32([to.get(p, p) if n else -1 for p, n in enumerate(refs)])
        out["n_used"] = _i32([n_used])
        for a, b in moved:
            refs[b], refs[a] = refs[a], 0
        table = [[to.get(p, p) for p in row] for row in table]
        rows = [(s, 0, n - 1) for s, n in enumerate(lens) if s % 2 == 0]
    out["missing"] = _i32(_exact_reserve(table, refs, rows, page, copies))
    for n in ("k", "v", "k_scale", "v_scale"):
        x = st[n].clone()
        for a, b in moved:
            x[b] = st[n][a]
        for a, b, blocks in copies:
            x[b, :, :blocks] = x[a, :, :blocks]
        out[n] = x.double() if "scale" in n else x
    return out | {"refs": _i32(refs), "table": _i32(table)}


def _exact_route(st):
    import numpy as np
    c = st["case"]
    e, g, k = c["experts"], c["groups"], c["top_k"]
    lg = st["logits"][:, :e].double().cpu().numpy()
    bias = st["bias"].double().cpu().numpy() if c["bias"] else np.zeros(e)
    ids, weights = [], []
    for x in lg:
        s = np.exp(-np.logaddexp(0, -x)) if c["scoring"] == "sigmoid" else np.exp(x - x.max() - np.log(np.exp(x - x.max()).sum()))
        key = s + bias
        best = np.sort(key.reshape(g, -1), 1)[:, ::-1][:, :c["group_top"]].sum(1)
        kept = set(np.argsort(-best, kind="stable")[:c["kept"]].tolist())
        order = [i for i in np.lexsort((np.arange(e), -x if not c["bias"] else -key)) if i // (e // g) in kept][:k]
        w = s[order]
        ids.append(order)
        weights.append(w / w.sum() * st["scale"] if c["normalize"] else w * st["scale"])
    return {"ids": torch.tensor(np.array(ids), dtype=torch.int32), "weights": torch.tensor(np.array(weights))}


def exact(case, seed):
    st = prepare(case, seed)
    return {"sinks": _exact_sinks, "rotate": _exact_rotate, "fork": _exact_pages, "compact": _exact_pages,
            "route": _exact_route}[case["kind"]](st)
