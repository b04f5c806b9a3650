"""Measured cases of the batched serving operators: appending keys and values
to the paged 8-bit cache, attention over it, and drawing the next tokens.

``run`` computes an operator in elementary torch operations where ``own`` is
false and through the framework's entry points where it is true; ``exact``
gives the same outputs from the definition in 64 bits.

The cache is held in 8-bit codes with one scale per block of 16 positions and
kv head, keys and values apart:

* key codes   ``[n_pages, n_kv_heads, page_tokens / 16, 16, d_head]``,
* value codes ``[n_pages, n_kv_heads, page_tokens / 16, d_head, 16]``,
* scales      ``[n_pages, n_kv_heads, page_tokens / 16]``.

A batch is ``n_seqs`` sequences: rows ``row_offsets[s] .. row_offsets[s + 1]``
are the newest positions of sequence ``s``, the last of them at
``seq_lens[s] - 1``; ``pages[s]`` holds its page ids in order.
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
        # the smallest step of a chat: one token of one sequence, a small model's heads, f32 from the GEMV
        {"name": "append_1", "kind": "append", "seqs": 1, "new": 1, "ctx": 300, "ragged": False, "kv": 4, "d": 64,
         "rope": 64, "dtype": "f32", "page": 64},
        # a serving batch: one token for each of 64 sequences of different ages
        {"name": "append_64", "kind": "append", "seqs": 64, "new": 1, "ctx": 2048, "ragged": True, "kv": 8, "d": 128,
         "rope": 128, "dtype": "f16", "page": 16},
        # prompts of different lengths written into the cache together, half of each head rotated
        {"name": "append_prompts", "kind": "append", "seqs": 5, "new": 2500, "ctx": 2500, "ragged": True, "kv": 8,
         "d": 128, "rope": 64, "dtype": "f32", "page": 64},
        # one token of one sequence in the middle of a chat: latency
        {"name": "attn_1", "kind": "attn", "seqs": 1, "new": 1, "ctx": 700, "ragged": False, "q": 32, "kv": 4, "d": 64,
         "rope": 64, "dtype": "f32", "page": 64, "window": 0},
        # the serving batch's attention: 64 sequences of up to 4096 positions
        {"name": "attn_64", "kind": "attn", "seqs": 64, "new": 1, "ctx": 4096, "ragged": True, "q": 32, "kv": 8,
         "d": 128, "rope": 128, "dtype": "f16", "page": 16, "window": 0},
        # two long documents being answered
        {"name": "attn_long", "kind": "attn", "seqs": 2, "new": 1, "ctx": 131072, "ragged": True, "q": 32, "kv": 8,
         "d": 128, "rope": 128, "dtype": "bf16", "page": 128, "window": 0},
        # drafts of five tokens checked at once for sixteen sequences
        {"name": "attn_drafts", "kind": "attn", "seqs": 16, "new": 5, "ctx": 2000, "ragged": True, "q": 32, "kv": 8,
         "d": 128, "rope": 128, "dtype": "f16", "page": 64, "window": 0},
        # chunks of prompts against what is cached, every head its own keys, a sliding window, f32 throughout
        {"name": "attn_chunk", "kind": "attn", "seqs": 3, "new": 201, "ctx": 1500, "ragged": True, "q": 16, "kv": 16,
         "d": 64, "rope": 32, "dtype": "f32", "page": 32, "window": 512},
        # whole prompts
        {"name": "attn_prompts", "kind": "attn", "seqs": 3, "new": 4096, "ctx": 4096, "ragged": True, "q": 32, "kv": 8,
         "d": 128, "rope": 128, "dtype": "f16", "page": 64, "window": 0},
        # the next token of one chat
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 32000, "dtype": "f32", "top_k": 40, "top_p": 0.95,
         "min_p": 0.0, "temp": 0.8, "mixed": False},
        # a serving batch over a large vocabulary, nucleus sampling
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": 128000, "dtype": "f32", "top_k": 0, "top_p": 0.9,
         "min_p": 0.0, "temp": 1.0, "mixed": False},
        # many short answers with settings of their own each, rows of a padded buffer in 16 bits
        {"name": "sample_500", "kind": "sample", "rows": 500, "vocab": 32003, "dtype": "bf16", "top_k": 100,
         "top_p": 0.97, "min_p": 0.05, "temp": 0.7, "mixed": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "attn", "sample", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 160000)
        return {"kind": kind, "rows": _log(rng, 1, max(2, min(500, 8_000_000 // vocab))), "vocab": vocab,
                "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "top_k": rng.choice([0, 0, 1, _log(rng, 2, vocab)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 3)]),
                "temp": rng.choice([0.0, 1.0, round(rng.uniform(0.2, 1.5), 2), round(rng.uniform(0.2, 1.5), 2)]),
                "mixed": rng.random() < 0.4}
    d = rng.choice([64, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8, 8])
    c = {"kind": kind, "kv": kv, "d": d, "rope": rng.choice([0, d // 2, d, d]),
         "dtype": rng.choice(["f32", "f16", "f16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256])}
    mode = rng.choice(["token", "token", "draft", "chunk", "prompt"])
    c["ragged"] = rng.random() < 0.8
    if mode == "token":
        c["new"], c["seqs"] = 1, _log(rng, 1, 128)
        c["ctx"] = _log(rng, 16, min(131072, 262144 // c["seqs"]))
    elif mode == "draft":
        c["new"], c["seqs"] = rng.randint(2, 12), _log(rng, 1, 32)
        c["ctx"] = _log(rng, 64, min(32768, 131072 // c["seqs"]))
    elif mode == "chunk":
        c["new"], c["seqs"] = _log(rng, 16, 512), _log(rng, 1, 8)
        c["ctx"] = c["new"] + _log(rng, 1, 6000)
    else:
        c["seqs"] = _log(rng, 1, 6)
        c["new"] = c["ctx"] = _log(rng, 32, 8192 // c["seqs"] if kind == "append" else 4096)
    if kind == "attn":
        c["q"] = kv * rng.choice([1, 2, 4, 4, 7, 8] if kv <= 4 else [1, 2, 3, 4])
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, max(2, c["ctx"]))])
    while work(c)["flops"] > 3e11 or work(c)["bytes"] > 4e8:  # no more than the largest listed case
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
    total, w = 0, case["window"] or case["ctx"] + 1
    for new, ctx in _lengths(case):
        full = max(0, min(new, ctx - w + 1))  # queries whose window is full
        rest = new - full                     # the earlier ones: ctx - new + 1, ... keys
        first = ctx - new + 1
        total += full * w + rest * first + rest * (rest - 1) // 2
    return total


def _keys(case):
    """Cached positions that some query of the case reads."""
    w = case["window"] or case["ctx"] + 1
    return sum(min(ctx, new + w - 1) for new, ctx in _lengths(case))


def _rope_table(gen, dim, n_pos):
    """[n_pos, dim / 2, 2] of (cos, sin), base 10000."""
    i = torch.arange(dim // 2, dtype=torch.float64, device=DEVICE)
    theta = torch.arange(n_pos, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (-2 * i / dim)
    return torch.stack([theta.cos(), theta.sin()], -1).float().contiguous()


def _prepare_cache(case, gen):
    lens = _lengths(case)
    page, kv, d = case["page"], case["kv"], case["d"]
    counts = [-(-ctx // page) for _, ctx in lens]
    max_pages = max(counts)
    n_pages = sum(counts) + 3
    ids = torch.randperm(n_pages, device=DEVICE, generator=gen).to(torch.int32).cpu()
    pages = torch.zeros(len(lens), max_pages, dtype=torch.int32)
    at = 0
    for s, n in enumerate(counts):
        pages[s, :n] = ids[at:at + n]
        at += n
    blocks = page // BLOCK
    shape = (n_pages, kv, blocks)

    def codes(n):
        return (torch.randn(n, device=DEVICE, generator=gen) * 36).round_().clamp_(-127, 127).to(torch.int8)

    def scales(size):
        return (torch.rand(shape, device=DEVICE, generator=gen) * 0.7 + 0.65) * (size / 36)

    n_codes = n_pages * kv * page * d
    offs = [0]
    for new, _ in lens:
        offs.append(offs[-1] + new)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    st = {"case": case, "page": page, "kv": kv, "d": d, "n_pages": n_pages, "max_pages": max_pages, "n_rows": offs[-1],
          "n_seqs": len(lens), "max_new": max(n for n, _ in lens),
          "row_offsets": i32(offs), "seq_lens": i32([c for _, c in lens]), "pages": pages.to(DEVICE),
          "k": codes(n_codes).view(*shape, BLOCK, d), "v": codes(n_codes).view(*shape, d, BLOCK),
          "k_scale": scales(1.2), "v_scale": scales(0.9),
          "rope": _rope_table(gen, case["rope"], max_pages * page) if case["rope"] else None}
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    if case["kind"] == "sample":
        return _prepare_sample(case, gen)
    st = _prepare_cache(case, gen)
    rows, kv, d = st["n_rows"], st["kv"], st["d"]
    t = TYPES[case["dtype"]]
    if case["kind"] == "append":
        # one buffer of fused projections: this operator's rows are slices of it
        qkv = torch.randn(rows, 4 * kv * d, device=DEVICE, generator=gen)
        qkv *= 0.5 + torch.rand(rows, 1, device=DEVICE, generator=gen)  # tokens of different size
        st["qkv"] = qkv.to(t)
        st["in"] = (st["qkv"][:, 2 * kv * d:3 * kv * d], st["qkv"][:, 3 * kv * d:])
        # the blocks that the append writes, read back: from their first position to each sequence's end
        cnt = [ctx - (ctx - new) // BLOCK * BLOCK for new, ctx in _lengths(case)]
        offs = [0]
        for n in cnt:
            offs.append(offs[-1] + n)
        st["read_offsets"] = torch.tensor(offs, dtype=torch.int32, device=DEVICE)
        st["read_rows"] = offs[-1]
        st["out"] = [torch.zeros(offs[-1], kv, d, dtype=torch.float16, device=DEVICE) for _ in range(2)]
    else:
        q = case["q"]
        st["qkv"] = torch.randn(rows, (q + 2 * kv) * d, device=DEVICE, generator=gen).to(t)
        st["in"] = st["qkv"][:, :q * d]
        st["out"] = torch.zeros(rows, q, d, dtype=t, device=DEVICE)
    return st


def _prepare_sample(case, gen):
    n, v = case["rows"], case["vocab"]
    stride = (v + 127) // 128 * 128  # rows of a padded buffer
    sharp = 0.5 + 2.5 * torch.rand(n, 1, device=DEVICE, generator=gen)
    lg = torch.randn(n, stride, device=DEVICE, generator=gen) * sharp
    # a few tokens that the model favours, by different amounts from row to row
    at = torch.randint(0, v, (n, 8), device=DEVICE, generator=gen)
    lg.scatter_add_(1, at, 12 * torch.rand(n, 8, device=DEVICE, generator=gen) * torch.rand(n, 1, device=DEVICE, generator=gen))
    lg = lg.to(TYPES[case["dtype"]])
    one = torch.ones(n, device=DEVICE)
    if case["mixed"]:  # every row its own settings, some rows greedy or with a filter off
        pick = torch.rand(n, 4, device=DEVICE, generator=gen)
        temp = one * case["temp"] * (0.5 + pick[:, 0]) * (pick[:, 0] > 0.1)
        top_k = (one * case["top_k"] * (0.5 + pick[:, 1]) * (pick[:, 1] > 0.2)).round().to(torch.int32)
        top_p = torch.where(pick[:, 2] > 0.2, (one * case["top_p"] * (0.7 + 0.5 * pick[:, 2])).clamp(max=1.0), one)
        min_p = one * case["min_p"] * pick[:, 3] * (pick[:, 3] > 0.2)
    else:
        temp, top_p, min_p = one * case["temp"], one * case["top_p"], one * case["min_p"]
        top_k = (one * case["top_k"]).to(torch.int32)
    return {"case": case, "logits": lg, "rows": n, "vocab": v, "stride": stride, "temp": temp, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "u": torch.rand(n, device=DEVICE, generator=gen),
            "ids": torch.zeros(n, dtype=torch.int32, device=DEVICE), "probs": torch.zeros(n, device=DEVICE)}


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
    return rce_amd.KvCache(st["n_pages"], st["page"], st["kv"], st["d"], k=st["k"].data_ptr(), v=st["v"].data_ptr(),
                           k_scale=st["k_scale"].data_ptr(), v_scale=st["v_scale"].data_ptr())


def _own_batch(st, offsets, rows):
    import rce_amd
    return rce_amd.KvBatch(row_offsets=offsets.data_ptr(), seq_lens=st["seq_lens"].data_ptr(),
                           pages=st["pages"].data_ptr(), n_seqs=st["n_seqs"], n_rows=rows, max_pages=st["max_pages"])


def _own_rope(st):
    import rce_amd
    if st["rope"] is None:
        return None
    return rce_amd.Rope(st["rope"].data_ptr(), dim=st["case"]["rope"], n_pos=st["max_pages"] * st["page"])


def _own_dtype(t):
    import rce_amd
    return {torch.float32: rce_amd.GgufDtype.F32, torch.float16: rce_amd.GgufDtype.F16,
            torch.bfloat16: rce_amd.GgufDtype.BF16}[t]


def _run_own(st):
    import rce_amd
    ctx, kind = _ctx(), st["case"]["kind"]
    if kind == "sample":
        rce_amd.sample_dev(ctx, st["logits"].data_ptr(), _own_dtype(st["logits"].dtype), st["rows"], st["vocab"],
                           st["stride"], st["u"].data_ptr(), st["ids"].data_ptr(), probs_dev=st["probs"].data_ptr(),
                           temperature_dev=st["temp"].data_ptr(), top_k_dev=st["top_k"].data_ptr(),
                           top_p_dev=st["top_p"].data_ptr(), min_p_dev=st["min_p"].data_ptr())
        return {"ids": st["ids"], "probs": st["probs"]}
    cache, batch = _own_cache(st), _own_batch(st, st["row_offsets"], st["n_rows"])
    if kind == "append":
        k, v = st["in"]
        rce_amd.kv_append_dev(ctx, cache, batch, k.data_ptr(), v.data_ptr(), _own_dtype(k.dtype), k.stride(0), v.stride(0),
                              rope=_own_rope(st))
        ko, vo = st["out"]
        rce_amd.kv_read_dev(ctx, cache, _own_batch(st, st["read_offsets"], st["read_rows"]), ko.data_ptr(), vo.data_ptr(),
                            rce_amd.GgufDtype.F16)
        return {"k": ko, "v": vo, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    q, out = st["in"], st["out"]
    rce_amd.kv_attention_dev(ctx, cache, batch, q.data_ptr(), _own_dtype(q.dtype), q.stride(0), st["case"]["q"],
                             out.data_ptr(), _own_dtype(out.dtype), scale=1 / math.sqrt(st["d"]), rope=_own_rope(st),
                             window=st["case"]["window"])
    return out


# ---- the plain form --------------------------------------------------------------

def _rows(st, offsets, n_rows):
    """Sequence and position of every row."""
    r = torch.arange(n_rows, device=DEVICE)
    s = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    return s, st["seq_lens"].long()[s] - (offsets.long()[s + 1] - r)


def _rotate(st, x, pos):
    """[rows, heads, d] in f32, the first `rope` values of each head rotated in pairs (i, i + rope / 2)."""
    if st["rope"] is None:
        return x
    h = st["rope"].shape[1]
    cs = st["rope"][pos][:, None]
    c, s = cs[..., 0], cs[..., 1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * h:]], -1)


def _quantized(x, slot, inv, first, scale, codes):
    """One cache's blocks after the append: x [rows, heads, d] into the blocks `inv` of scale [blocks, heads] and
    codes [blocks, heads, 16, d]; `first`: the first new slot of each block."""
    nb, heads, d = scale.shape[0], x.shape[1], x.shape[2]
    amax = torch.zeros(nb, heads, device=DEVICE).scatter_reduce_(
        0, inv[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    old = torch.where(first[:, None] > 0, scale, 0.0)
    new = (amax.double() / 127).float()
    new = torch.maximum(old, torch.where(new < 2.0 ** -126, 0.0, new))
    some = (new > 0) & (new < math.inf)
    inv_new = torch.where(some, (1 / new.double()).float(), 0.0)
    ratio = torch.where(some, (old.double() / new.double()).float(), 0.0)
    before = torch.arange(BLOCK, device=DEVICE) < first[:, None]
    moved = (codes.float() * ratio[..., None, None]).round().to(torch.int8)
    codes = torch.where(before[:, None, :, None], moved, codes)
    q = (x * inv_new[inv][..., None]).round().clamp(-127, 127).to(torch.int8)
    codes[inv, :, slot] = q
    return new, codes


def _plain_append(st):
    kv, d, page = st["kv"], st["d"], st["page"]
    s, pos = _rows(st, st["row_offsets"], st["n_rows"])
    pg = st["pages"].long()[s, pos // page]
    block = pg * (page // BLOCK) + pos % page // BLOCK
    slot = pos % BLOCK
    touched, inv = torch.unique(block, return_inverse=True)
    first = torch.full_like(touched, BLOCK).scatter_reduce_(0, inv, slot, "amin")
    pg, b = touched // (page // BLOCK), touched % (page // BLOCK)
    k, v = st["in"]
    k, v = _rotate(st, k.reshape(-1, kv, d).float(), pos), v.reshape(-1, kv, d).float()
    scale, codes = _quantized(k, slot, inv, first, st["k_scale"][pg, :, b], st["k"][pg, :, b])
    st["k_scale"][pg, :, b], st["k"][pg, :, b] = scale, codes
    scale, codes = _quantized(v, slot, inv, first, st["v_scale"][pg, :, b], st["v"][pg, :, b].transpose(-1, -2))
    st["v_scale"][pg, :, b], st["v"][pg, :, b] = scale, codes.transpose(-1, -2)
    s, pos = _rows(st, st["read_offsets"], st["read_rows"])
    pg, b, slot = st["pages"].long()[s, pos // page], pos % page // BLOCK, pos % BLOCK
    k = st["k"][pg, :, b, slot].float() * st["k_scale"][pg, :, b][..., None]
    v = st["v"][pg, :, b, :, slot].float() * st["v_scale"][pg, :, b][..., None]
    return {"k": k.half(), "v": v.half(), "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _cached(st):
    """Keys and values [n_seqs, heads, positions, d] of every sequence's table."""
    at = st["pages"].long()
    k = st["k"][at].float() * st["k_scale"][at][..., None, None]
    v = st["v"][at].float() * st["v_scale"][at][..., None, None]
    join = lambda x: x.transpose(1, 2).reshape(at.shape[0], st["kv"], -1, st["d"])  # noqa: E731
    return join(k), join(v.transpose(-1, -2))


def _plain_attention(st):
    c, d, kv = st["case"], st["d"], st["kv"]
    heads, per = c["q"], c["q"] // kv
    s, pos = _rows(st, st["row_offsets"], st["n_rows"])
    at = torch.arange(st["n_rows"], device=DEVICE) - st["row_offsets"].long()[s]
    x = _rotate(st, st["in"].reshape(-1, heads, d).float(), pos)
    q = torch.zeros(st["n_seqs"], st["max_new"], heads, d, device=DEVICE)
    q[s, at] = x
    q = q.view(-1, st["max_new"], kv, per, d).permute(0, 2, 3, 1, 4).reshape(-1, kv, per * st["max_new"], d)
    k, v = _cached(st)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1 / math.sqrt(d))
    j = torch.arange(k.shape[2], device=DEVICE)
    p = torch.full((st["n_seqs"], st["max_new"]), -1, device=DEVICE)
    p[s, at] = pos
    see = (j <= p[..., None]) & (j > p[..., None] - (c["window"] or c["ctx"] + 1))
    score = score.view(-1, kv, per, st["max_new"], k.shape[2])
    score = torch.where(see[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(-1, kv, per * st["max_new"], k.shape[2]), v).view(-1, kv, per, st["max_new"], d)
    o = torch.where(total > 0, o / torch.where(total > 0, total, 1.0), 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(st["n_seqs"], st["max_new"], heads, d)
    return o[s, at].to(st["out"].dtype)


def _plain_sample(st):
    n, v = st["rows"], st["vocab"]
    lg = st["logits"][:, :v].double()
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    top = lg.amax(-1, keepdim=True)
    temp = st["temp"].double()[:, None]
    w = torch.exp((lg - top) / torch.where(temp > 0, temp, 1.0))
    w = torch.where(lg == top, 1.0, torch.where(lg == -math.inf, 0.0, w))
    order = torch.sort(lg, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(v, device=DEVICE)
    k = st["top_k"].long()[:, None]
    ws = torch.where((k <= 0) | (rank < k), ws, 0.0)
    p = st["top_p"].double()[:, None]
    before = ws.cumsum(-1) - ws
    keep = (rank == 0) | ((ws >= st["min_p"].double()[:, None]) & ((p >= 1) | (before < p * ws.sum(-1, keepdim=True))))
    keep &= (temp > 0) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    total = kept.sum(-1, keepdim=True)
    ids = torch.searchsorted(kept.cumsum(-1), st["u"].double()[:, None] * total, right=True).clamp(max=v - 1)
    prob = kept.gather(1, ids) / total
    dead = top[:, 0] == -math.inf
    return {"ids": torch.where(dead, -1, ids[:, 0]).to(torch.int32),
            "probs": torch.where(dead, 0.0, prob[:, 0]).float()}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attn": _plain_attention, "sample": _plain_sample}[state["case"]["kind"]](state)


# ---- work ------------------------------------------------------------------------

def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * TYPES[case["dtype"]].itemsize + case["rows"] * 28, "flops": 3 * n}
    size = TYPES[case["dtype"]].itemsize
    d, kv, lens = case["d"], case["kv"], _lengths(case)
    rows = sum(n for n, _ in lens)
    if case["kind"] == "append":
        back = sum(ctx - (ctx - new) // BLOCK * BLOCK for new, ctx in lens)
        # the new rows in, their codes out; their blocks' codes in and values out
        return {"bytes": 2 * kv * (rows * d * (size + 1) + back * d * (1 + 2) + back // BLOCK * 12),
                "flops": 2 * kv * d * (6 * rows + back)}
    keys = _keys(case)
    return {"bytes": 2 * kv * keys * d + kv * keys // 2 + 2 * rows * case["q"] * d * size,
            "flops": 4 * d * case["q"] * _pairs(case)}


# ---- the definition in 64 bits ----------------------------------------------------

def _exact_rope(st, x, pos):
    """x [rows, heads, d] of the positions `pos` as complex pairs times the table's."""
    if st["rope"] is None:
        return x
    h = st["rope"].shape[1]
    z = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous())
    z = z * torch.view_as_complex(st["rope"].double())[pos][:, None]
    return torch.cat([z.real, z.imag, x[..., 2 * h:]], -1)


def _exact_rows(st, s, a, b):
    """Page and offset of the positions a .. b - 1 of sequence s."""
    p = torch.arange(a, b, device=DEVICE)
    return st["pages"][s].long()[p // st["page"]], p % st["page"]


def _exact_values(st, name, s, a, b):
    """[positions, heads, d] of one cache in 64 bits."""
    pg, at = _exact_rows(st, s, a, b)
    blk, slot = at // BLOCK, at % BLOCK
    codes = st[name] if name == "k" else st[name].transpose(-1, -2)
    return codes[pg, :, blk, slot].double() * st[name + "_scale"][pg, :, blk].double()[..., None]


def _exact_append(st):
    lens, offs = _lengths(st["case"]), st["row_offsets"].tolist()
    outs = {"k": [], "v": []}
    scales = {n: st[n + "_scale"].double() for n in "kv"}
    for s, (new, ctx) in enumerate(lens):
        start = ctx - new
        low = start // BLOCK * BLOCK
        n_blocks = -(-(ctx - low) // BLOCK)
        for name, x in zip("kv", st["in"]):
            x = x[offs[s]:offs[s + 1]].double().view(new, st["kv"], st["d"])
            if name == "k":
                x = _exact_rope(st, x, torch.arange(start, ctx, device=DEVICE))
            had = _exact_values(st, name, s, low, start)
            full = torch.zeros(n_blocks * BLOCK, st["kv"], st["d"], dtype=torch.float64, device=DEVICE)
            full[start - low:ctx - low] = x
            size = full.view(n_blocks, BLOCK, st["kv"], st["d"]).abs().amax((1, 3)) / 127
            pg, at = _exact_rows(st, s, low, ctx)
            pg, at = pg[::BLOCK], at[::BLOCK] // BLOCK
            if start > low:
                size[0] = torch.maximum(size[0], scales[name][pg[0], :, at[0]])
            scales[name][pg, :, at] = size
            full[:start - low] = had
            step = size.repeat_interleave(BLOCK, 0)[:ctx - low, :, None]
            outs[name].append((full[:ctx - low] / step).round().clamp(-127, 127) * step)
    return {"k": torch.cat(outs["k"]), "v": torch.cat(outs["v"]), "k_scale": scales["k"], "v_scale": scales["v"]}


def _exact_attention(st):
    c, offs = st["case"], st["row_offsets"].tolist()
    d, per = st["d"], c["q"] // st["kv"]
    out = torch.zeros(st["n_rows"], c["q"], d, dtype=torch.float64, device=DEVICE)
    for s, (new, ctx) in enumerate(_lengths(c)):
        pos = torch.arange(ctx - new, ctx, device=DEVICE)
        low = max(0, ctx - new - c["window"] + 1) if c["window"] else 0
        k, v = _exact_values(st, "k", s, low, ctx), _exact_values(st, "v", s, low, ctx)
        q = _exact_rope(st, st["in"][offs[s]:offs[s + 1]].double().reshape(new, c["q"], d), pos)
        key = torch.arange(low, ctx, device=DEVICE)
        hide = key > pos[:, None]
        if c["window"]:
            hide = hide | (key <= pos[:, None] - c["window"])
        for h in range(c["q"]):
            p = q[:, h] @ k[:, h // per].T / math.sqrt(d)
            p = torch.softmax(p.masked_fill_(hide, -math.inf), -1)
            out[offs[s]:offs[s + 1], h] = p @ v[:, h // per]
    return out


def _exact_sample(st):
    import numpy as np
    lg = st["logits"][:, :st["vocab"]].double().cpu().numpy()
    ids, probs = [], []
    for r in range(st["rows"]):
        t, k, p, m, u = (float(st[n][r]) for n in ("temp", "top_k", "top_p", "min_p", "u"))
        x = lg[r]
        best = int(np.argmax(x))
        if t <= 0:
            ids.append(best)
            probs.append(1.0)
            continue
        w = np.exp((x - x[best]) / t)
        order = np.argsort(-x, kind="stable")[:int(k) if k > 0 else None]
        ws = w[order]
        if p < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(ws), p * ws.sum(), side="left"))]
        order = order[(w[order] >= m) | (order == best)]
        order = np.sort(order)
        cum = np.cumsum(w[order])
        i = order[min(len(order) - 1, int(np.searchsorted(cum, u * cum[-1], side="right")))]
        ids.append(int(i))
        probs.append(w[i] / cum[-1])
    return {"ids": torch.tensor(ids, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attention, "sample": _exact_sample}[case["kind"]](st)
