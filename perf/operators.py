"""The batched serving operators, as a program that drives a model's layers itself runs them.

Such a program keeps the keys and values of many sequences in a paged cache of 4-bit codes. A step
plans the pages and slots of its new tokens from the sequences' lengths (`plan`), puts the new rows
into the cache (`append`, here with the reading back of what they stand for), attends over it
(`attend`: one token a sequence while decoding, a draft's rows while verifying, prompt chunks, or
a mix) and reports on its logits (`logprobs`: log probabilities of given tokens, entropy, the most
likely alternatives). Head counts, head sizes and vocabularies are those of this repository's model
configurations; the cache's layout in memory is stated at `_unpack`.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# (query heads, key / value heads, head size): Qwen3-30B-A3B, Qwen3-0.6B, Granite-1B-A400M, SmolLM2-135M
HEADS = [(32, 4, 128), (16, 8, 128), (16, 8, 64), (9, 3, 64)]


def listed():
    return [
        # a decode step's bookkeeping: 24 sequences, a token each
        {"name": "plan-decode", "kind": "plan", "seqs": 24, "page": 32, "context": 4000, "q": 1, "prompts": 0},
        # a step of a loaded server: 500 sequences, 40 of them with prompt chunks
        {"name": "plan-mixed", "kind": "plan", "seqs": 500, "page": 64, "context": 8000, "q": 511, "prompts": 40},
        # a decode step's new rows of one layer
        {"name": "append-decode", "kind": "append", "type": "f32", "kv": 4, "hd": 128, "page": 32, "rows": 24},
        # a batch of prompt chunks: 8191 rows of one layer
        {"name": "append-prompt", "kind": "append", "type": "bf16", "kv": 8, "hd": 128, "page": 64, "rows": 8191},
        # one sequence decoding at 4K: few rows, a long axis
        {"name": "attend-single", "kind": "attend", "type": "f32", "heads": 32, "kv": 4, "hd": 128, "page": 32, "seqs": 1, "context": 4097, "q": 1, "prompts": 0, "window": 0},
        # 64 sequences of up to 16K decoding together
        {"name": "attend-batch", "kind": "attend", "type": "f16", "heads": 32, "kv": 4, "hd": 128, "page": 64, "seqs": 64, "context": 16384, "q": 1, "prompts": 0, "window": 0},
        # a k = 8 verify over twelve sequences of a small model
        {"name": "attend-verify", "kind": "attend", "type": "f32", "heads": 16, "kv": 8, "hd": 64, "page": 16, "seqs": 12, "context": 2050, "q": 9, "prompts": 12, "window": 0},
        # the second chunk of a long prompt
        {"name": "attend-prompt", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4, "hd": 128, "page": 64, "seqs": 1, "context": 4096, "q": 2048, "prompts": 1, "window": 0},
        # two prompt chunks among decoding sequences, over a window
        {"name": "attend-mixed", "kind": "attend", "type": "f32", "heads": 16, "kv": 8, "hd": 128, "page": 32, "seqs": 26, "context": 3001, "q": 333, "prompts": 2, "window": 2000},
        # a sampled token's report: one row
        {"name": "logprobs-one", "kind": "logprobs", "type": "f32", "rows": 1, "vocab": 151936, "top": 5},
        # a verify batch's rows, an odd vocabulary in 16 bits
        {"name": "logprobs-verify", "kind": "logprobs", "type": "bf16", "rows": 72, "vocab": 49155, "top": 20},
        # the scoring of a prompt
        {"name": "logprobs-prompt", "kind": "logprobs", "type": "f32", "rows": 500, "vocab": 151936, "top": 1},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        seqs = _log(rng, 1, 800)
        prompts = rng.choice([0, rng.randint(0, min(seqs, 40))])
        return {"kind": kind, "seqs": seqs, "page": page, "context": _log(rng, 600, 16000), "q": _log(rng, 2, 500) if prompts else 1, "prompts": prompts}
    if kind == "append":
        _, kv, hd = rng.choice(HEADS)
        return {"kind": kind, "type": rng.choice(list(TYPES)), "kv": kv, "hd": hd, "page": page, "rows": _log(rng, 1, 4000)}
    if kind == "logprobs":
        rows = _log(rng, 1, 400)
        return {"kind": kind, "type": rng.choice(list(TYPES)), "rows": rows, "vocab": rng.choice([49152, 49155, 151936, _log(rng, 1000, 150000)]), "top": rng.choice([0, 1, 5, 20, rng.randint(1, 32)])}
    heads, kv, hd = rng.choice(HEADS)
    case = {"kind": kind, "type": rng.choice(list(TYPES)), "heads": heads, "kv": kv, "hd": hd, "page": page}
    form = rng.choice(["decode", "decode", "verify", "prompt", "mixed"])
    if form == "decode":
        seqs = _log(rng, 1, 64)
        more = {"seqs": seqs, "context": _log(rng, 20, 12000), "q": 1, "prompts": 0}
    elif form == "verify":
        seqs = _log(rng, 1, 24)
        more = {"seqs": seqs, "context": _log(rng, 30, 6000), "q": rng.randint(2, 16), "prompts": seqs}
    elif form == "prompt":
        q = _log(rng, 17, 1500)
        more = {"seqs": 1, "context": q + rng.choice([0, _log(rng, 1, 2000)]), "q": q, "prompts": 1}
    else:
        q = _log(rng, 17, 300)
        more = {"seqs": rng.randint(3, 24), "context": q + _log(rng, 20, 2500), "q": q, "prompts": rng.randint(1, 2)}
    return {**case, **more, "window": rng.choice([0, 0, 0, _log(rng, 16, 4000)])}


# ------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Each sequence's new rows and its length with them, by the case alone: lengths spread from a
    quarter of the context up to all of it, the prompts' sequences the longest."""
    n, ctx = case["seqs"], case["context"]
    q = [1] * (n - case["prompts"]) + [case["q"]] * case["prompts"]
    return q, [max(a, ctx - (n - 1 - i) * 3 * ctx // (4 * n)) for i, a in enumerate(q)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _order(case, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    q, kv = _lengths(case)
    at = torch.randperm(len(q), generator=g).tolist()
    return [q[i] for i in at], [kv[i] for i in at], g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prefix(v):
    return [sum(v[:i]) for i in range(len(v) + 1)]


def _keys(g, rows, kv, hd, dtype):
    """Rows as projections leave them: normal, a few channels larger than the rest."""
    wide = 1.0 + 4.0 * (torch.rand(kv, hd, generator=g, device="cuda") < 0.05)
    return (torch.randn(rows, kv, hd, generator=g, device="cuda") * wide / wide.square().mean().sqrt()).to(dtype)


def prepare(case, seed):
    kind, st, g = case["kind"], {"case": case}, _gen(seed)
    if kind == "plan":
        q, kv, h = _order(case, seed)
        page = case["page"]
        old = [a - b for a, b in zip(kv, q)]
        held = [-(-n // page) for n in old]
        # every sequence holds its pages; one in sixteen ends with this step; the pool has room for
        # all but the last few sequences' new pages
        ends = [i % 16 == 7 for i in range(len(q))]
        cols = -(-(case["context"] + 2 * page) // page)
        want = sum(-(-(n + a) // page) - b for n, a, b, e in zip(old, q, held, ends) if not e)
        spare = max(1, want - sum(b for b, e in zip(held, ends) if e) - 2)
        ids = torch.randperm(sum(held) + spare, generator=h).to(torch.int32)
        tables, at = torch.full((len(q), cols), -1, dtype=torch.int32), 0
        for i, b in enumerate(held):
            tables[i, :b] = ids[at:at + b]
            at += b
        free = torch.full((ids.numel(),), -1, dtype=torch.int32)
        free[:spare] = ids[at:]
        st.update(lens=_ints(old), add=_ints([-1 if e else a for a, e in zip(q, ends)]), tables=tables.cuda(), free=free.cuda(), n_free=_ints([spare]),
                  rows=sum(q))
        return st
    if kind == "logprobs":
        x = torch.randn(case["rows"], case["vocab"], generator=g, device="cuda") * 2.5
        at = torch.randint(case["vocab"], (case["rows"],), generator=g, device="cuda")
        x[torch.arange(case["rows"], device="cuda"), at] += 8.0
        # every second row is asked for its likely token, the others for any
        other = torch.randint(case["vocab"], (case["rows"],), generator=g, device="cuda")
        st.update(logits=x.to(TYPES[case["type"]]), targets=torch.where(torch.arange(case["rows"], device="cuda") % 2 == 0, at, other).to(torch.int32))
        return st
    kv, hd, page, dtype = case["kv"], case["hd"], case["page"], TYPES[case["type"]]
    if kind == "append":
        n = case["rows"]
        pages = -(-n // page) + 3
        # pages in any order, rows in order within them, the last page part filled
        order = torch.randperm(pages, generator=g, device="cuda")
        r = torch.arange(n, device="cuda")
        st.update(pages=pages, pool=torch.zeros(pages * kv * page * hd * 9 // 8, dtype=torch.uint8, device="cuda"),
                  k=_keys(g, n, kv, hd, dtype), v=torch.randn(n, kv, hd, generator=g, device="cuda").to(dtype),
                  slots=(order[r // page] * page + r % page).to(torch.int32))
        return st
    q, lens, h = _order(case, seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    ids = torch.randperm(pages, generator=h).to(torch.int32)
    tables, at = torch.full((len(q), max(need)), -1, dtype=torch.int32), 0
    for i, b in enumerate(need):
        tables[i, :b] = ids[at:at + b]
        at += b
    pool = torch.empty(pages * kv * page * hd * 9 // 8, dtype=torch.uint8, device="cuda")
    for a in range(0, pages, 64):  # every slot of every page holds a row, as in a pool that has been in use
        b = min(pages, a + 64)
        k, v = _keys(g, (b - a) * page, kv, hd, torch.float32), torch.randn((b - a) * page, kv, hd, generator=g, device="cuda")
        size = kv * page * hd * 9 // 8
        _pack(pool[a * size:b * size], k, v, torch.arange((b - a) * page, device="cuda"), kv, hd, page)
    rows = sum(q)
    st.update(pages=pages, pool=pool, tables=tables.cuda(), lens=_ints(lens), start=_ints(_prefix(q)), rows=rows, most_q=max(q),
              q=torch.randn(rows, case["heads"], hd, generator=g, device="cuda").to(dtype))
    return st


# --------------------------------------------------------------------------------- plain forms
# nibble j of a 32-bit word of key codes holds the word's channel SLOT[j]
SLOT = [0, 2, 4, 6, 1, 3, 5, 7]
# the nibble that holds a word's channel c
NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]


def _quantize(x):
    """[..., hd] as scales [..., hd / 32] (f16) and codes -8..7 [..., hd / 32, 32]."""
    x = x.float().unflatten(-1, (-1, 32))
    mag = x.abs()
    most = mag.amax(-1, keepdim=True)
    first = torch.where(mag == most, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = (torch.gather(x, -1, first.clamp(max=31)) / -8.0).to(torch.bfloat16).float().clamp(-8160.0, 8160.0).to(torch.float16)
    safe = torch.where(d == 0, torch.ones_like(d), d).double()
    code = torch.where(d == 0, torch.zeros_like(x).double(), torch.round(x.double() / safe)).clamp(-8, 7)
    return d.squeeze(-1), code.to(torch.int32)


def _views(pool, kv, hd, page):
    """The pool's parts: pages of kv heads of tiles of 16 tokens; a tile holds the key codes
    [4][16 tokens][hd / 32][4 bytes], the value codes [4][16][4 tokens][hd / 32 bytes], the key scales
    [16 tokens][hd / 32] and the value scales [hd / 32][16 tokens]."""
    t = pool.view(-1, kv, page // 16, 18 * hd)
    k, v, ks, vs = t.split([8 * hd, 8 * hd, hd, hd], -1)
    return (k.unflatten(-1, (4, 16, hd // 32, 4)), v.unflatten(-1, (4, 16, 4, hd // 32)),
            ks.unflatten(-1, (16, hd // 32, 2)), vs.unflatten(-1, (hd // 32, 16, 2)))


def _halves(d):
    return d.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))


def _pack(pool, k, v, slots, kv, hd, page):
    """Quantizes rows k, v [rows, kv, hd] into the pool's slots."""
    kc, vc, ks, vs = _views(pool, kv, hd, page)
    slots = slots.long()
    p, t, i = slots // page, slots % page // 16, slots % 16
    d, c = _quantize(k)
    c = (c + 8).unflatten(-1, (4, 8))[..., SLOT].transpose(-2, -3)  # [rows, kv, 4, hd / 32, 8 nibbles]
    kc[p, :, t, :, i] = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
    ks[p, :, t, i] = _halves(d)
    d, c = _quantize(v)
    c = (c + 8).flatten(-2).unflatten(-1, (16, hd // 16))
    vc[p, :, t, i // 4, :, i % 4] = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
    vs[p, :, t, :, i] = _halves(d)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _unpack(tiles, hd):
    """Tiles [..., 18 hd bytes] as keys and values [..., 16, hd] in 32 bits."""
    k, v, ks, vs = tiles.split([8 * hd, 8 * hd, hd, hd], -1)
    ks = ks.contiguous().view(torch.float16).float().unflatten(-1, (16, hd // 32, 1))
    vs = vs.contiguous().view(torch.float16).float().unflatten(-1, (hd // 32, 16)).transpose(-1, -2).unsqueeze(-1)
    k = _nibbles(k.unflatten(-1, (4, 16, hd // 32, 4)))[..., NIBBLE]      # [..., 4, 16, hd / 32, 8]
    k = k.movedim(-4, -2).flatten(-2).float() - 8.0                       # [..., 16, hd / 32, 32]
    v = _nibbles(v.unflatten(-1, (4, 16, 4, hd // 32)))                   # [..., 4, 16, 4 tokens, hd / 16]
    v = v.transpose(-2, -3).flatten(-2).flatten(-3, -2).unflatten(-1, (hd // 32, 32)).float() - 8.0
    return (k * ks).flatten(-2), (v * vs).flatten(-2)


def _plain_plan(st):
    page, lens, add, tables, free, rows = st["case"]["page"], st["lens"], st["add"], st["tables"], st["free"], st["rows"]
    ends, more = add < 0, add.clamp(min=0)
    held = (lens + page - 1) // page
    col = torch.arange(tables.shape[1], device="cuda", dtype=torch.int32).unsqueeze(0)
    # pages of ended sequences go onto the free list, in order
    back = ends.unsqueeze(1) & (col < held.unsqueeze(1))
    at = st["n_free"].long() + torch.cumsum(back.flatten(), 0) - 1
    room = torch.cat([free, free.new_empty(1)])
    room[torch.where(back.flatten(), at, free.numel())] = tables.flatten()
    free = room[:-1]
    n_free = st["n_free"] + back.sum(dtype=torch.int32)
    fits = ~ends & (lens + more <= tables.shape[1] * page)
    need = torch.where(fits, (lens + more + page - 1) // page - held, 0)
    upto = torch.cumsum(need, 0, dtype=torch.int32)
    granted = fits & ((need == 0) | (upto <= n_free))
    need = torch.where(granted, need, 0)
    idx = col - held.unsqueeze(1)
    new = (idx >= 0) & (idx < need.unsqueeze(1))
    rank = (upto - need).unsqueeze(1) + idx
    tables = torch.where(new, free[(n_free.unsqueeze(0) - 1 - rank).clamp(0, free.numel() - 1).long()], tables)
    start = torch.cat([more.new_zeros(1), torch.cumsum(more, 0, dtype=torch.int32)])
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    s = torch.searchsorted(start[1:].contiguous(), r, right=True).clamp(max=lens.numel() - 1)
    pos = lens[s] + r - start[s]
    fine = (r < start[-1]) & granted[s]
    slots = tables[s, (pos // page).clamp(max=tables.shape[1] - 1).long()] * page + pos % page
    return {"lens": torch.where(ends, 0, torch.where(granted, lens + more, lens)), "n_free": n_free - need.sum(dtype=torch.int32), "tables": tables, "free": free,
            "start": start, "slots": torch.where(fine, slots, -1), "positions": torch.where(fine, pos, -1), "status": (~ends & ~granted).to(torch.int32)}


def _plain_append(st):
    case = st["case"]
    kv, hd, page, dtype = case["kv"], case["hd"], case["page"], TYPES[case["type"]]
    _pack(st["pool"], st["k"], st["v"], st["slots"], kv, hd, page)
    s = st["slots"].long()
    k, v = _unpack(st["pool"].view(-1, kv, page // 16, 18 * hd)[s // page, :, s % page // 16], hd)  # [rows, kv, 16, hd]
    at = (s % 16).view(-1, 1, 1, 1).expand(-1, kv, 1, hd)
    return {"k": torch.gather(k, 2, at).squeeze(2).to(dtype), "v": torch.gather(v, 2, at).squeeze(2).to(dtype)}


def _plain_attend(st):
    case = st["case"]
    kv, hd, page, heads, window = case["kv"], case["hd"], case["page"], case["heads"], case["window"]
    start, lens, n, most = st["start"].long(), st["lens"].long(), st["lens"].numel(), st["most_q"]
    tiles = st["pool"].view(-1, kv, page // 16, 18 * hd)[st["tables"].clamp(min=0).long()]  # [seqs, pages, kv, tiles, bytes]
    k, v = (x.transpose(1, 2).reshape(n * kv, -1, hd) for x in _unpack(tiles, hd))
    count = start[1:] - start[:-1]
    i = torch.arange(most, device="cuda")
    rows = (start[:-1, None] + i).clamp(max=st["rows"] - 1)
    q = st["q"][rows].float().unflatten(2, (kv, -1)).permute(0, 2, 1, 3, 4).reshape(n * kv, -1, hd)  # [seqs * kv, most * group, hd]
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(hd)).view(n, kv, most, heads // kv, -1)
    pos = ((lens - count)[:, None] + i).view(n, 1, most, 1, 1)
    key = torch.arange(s.shape[-1], device="cuda")
    seen = key <= pos
    if window:
        seen = seen & (key > pos - window)
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = e.sum(-1)
    o = torch.bmm(e.view(n * kv, -1, e.shape[-1]), v.contiguous()).view(n, kv, most, heads // kv, hd) / total.clamp(min=1e-30).unsqueeze(-1)
    r = torch.arange(st["rows"], device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), r, right=True)
    return o.permute(0, 2, 1, 3, 4).reshape(n, most, heads, hd)[b, r - start[b]].to(TYPES[case["type"]])


def _plain_logprobs(st):
    x, top = st["logits"].float(), st["case"]["top"]
    m = x.amax(-1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    out = {"logp": (torch.gather(z, 1, st["targets"].long().unsqueeze(1)) - log_total).squeeze(1), "entropy": (log_total - (z * e).sum(-1, keepdim=True) / total).squeeze(1)}
    if top:
        # keys that order by value and then by the lower id
        bits = x.view(torch.int32).long()
        key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device="cuda"))
        ids = 0x7FFFFFFF - (torch.topk(key, top, 1).values & 0xFFFFFFFF)
        out.update(top_ids=ids.to(torch.int32), top_logp=torch.gather(z, 1, ids) - log_total)
    return out


# ------------------------------------------------------------------------- the framework's calls
_ctx = []


def _context():
    """The program's one context; torch's work goes to the context's stream too."""
    if not _ctx:
        from spindle_amd import ops
        _ctx.append(ops.Context(0))
        torch.cuda.synchronize()
        torch.cuda.set_stream(_ctx[0].torch_stream())
    return _ctx[0]


def _own(st):
    from spindle_amd import ops
    case, ctx = st["case"], _context()
    kind = case["kind"]
    if kind == "plan":
        p = ops.pages_plan(ctx, st["lens"], st["add"], st["tables"], st["free"], st["n_free"], case["page"], st["rows"])
        return {"lens": p.lens, "n_free": p.n_free, "tables": st["tables"], "free": st["free"], "start": p.q_start, "slots": p.slots, "positions": p.positions, "status": p.status}
    if kind == "logprobs":
        r = ops.logprobs(ctx, st["logits"], st["targets"], top=case["top"])
        out = {"logp": r.logp, "entropy": r.entropy}
        if case["top"]:
            out.update(top_ids=r.top_ids, top_logp=r.top_logp)
        return out
    shape = ops.Kv4Shape(case["kv"], case["hd"], case["page"], st["pages"])
    if kind == "append":
        ops.kv4_append(ctx, shape, st["pool"], st["k"], st["v"], st["slots"])
        k, v = ops.kv4_read(ctx, shape, st["pool"], st["slots"], TYPES[case["type"]])
        return {"k": k, "v": v}
    return ops.kv4_attention(ctx, shape, st["pool"], st["q"], st["start"], st["lens"], st["tables"], window=case["window"], max_kv=case["context"])


def run(st):
    if own:
        return _own(st)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[st["case"]["kind"]](st)


# ------------------------------------------------------------------- what a pass cannot do without
def _pairs(q, n, window):
    """Positions that the last q rows of a sequence of length n see, over all of them."""
    return sum(min(p + 1, window) if window else p + 1 for p in range(n - q, n))


def work(case):
    kind = case["kind"]
    if kind == "plan":
        q, lens = _lengths(case)
        new = sum(-(-n // case["page"]) - -(-(n - a) // case["page"]) for a, n in zip(q, lens))
        return {"bytes": 4.0 * (5 * len(q) + 2 * new + 2 * sum(q)), "flops": 0.0}
    if kind == "logprobs":
        return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["type"]] + 12.0 + 8.0 * case["top"]), "flops": 5.0 * case["rows"] * case["vocab"]}
    per = case["kv"] * case["hd"] * 9 / 8  # a token's bytes in the cache
    if kind == "append":
        n = case["rows"] * case["kv"] * case["hd"]
        return {"bytes": 4.0 * SIZE[case["type"]] * n + 2 * per * case["rows"] + 8.0 * case["rows"], "flops": 12.0 * n}
    q, lens = _lengths(case)
    w = case["window"]
    read = sum(min(n, w + a - 1) if w else n for a, n in zip(q, lens))
    rows = case["heads"] * case["hd"] * sum(q)
    return {"bytes": per * read + 2.0 * SIZE[case["type"]] * rows, "flops": 4.0 * case["heads"] * case["hd"] * sum(_pairs(a, n, w) for a, n in zip(q, lens))}


# ------------------------------------------------------------------------- the same in 64 bits
def _exact_group(x):
    """Groups of 32 [..., 32] as the values that their 4-bit codes stand for."""
    at = torch.argmax((x.abs() == x.abs().amax(-1, keepdim=True)).to(torch.int8), -1, keepdim=True)  # the first of the largest
    d = torch.gather(x, -1, at) / -8.0
    _, e = torch.frexp(d)
    step = torch.ldexp(torch.ones_like(d), e - 8)  # eight significant bits
    d = torch.round(d / step) * step
    d = (torch.round(d * 2.0 ** 24) / 2.0 ** 24).clamp(-8160.0, 8160.0)  # f16's smallest step
    return torch.where(d == 0, torch.zeros_like(x), torch.round(x / torch.where(d == 0, torch.ones_like(d), d)).clamp(-8, 7) * d)


def _exact_tokens(pool, page_ids, kv, hd, page, n):
    """Keys and values [kv, n, hd] of a sequence's first n tokens, by each value's place in the pool."""
    tok, ch = torch.arange(n, device="cuda"), torch.arange(hd, device="cuda")
    base = (((page_ids.long()[tok // page].view(1, -1) * kv + torch.arange(kv, device="cuda").view(-1, 1)) * (page // 16) + (tok % page // 16)) * (18 * hd)).unsqueeze(2)
    t, g, w, c = (tok % 16).view(1, -1, 1), ch // 32, ch % 32 // 8, ch % 8
    nib = c // 2 + 4 * (c % 2)
    code = pool[base + ((w * 16 + t) * (hd // 32) + g) * 4 + nib // 2] >> (4 * (nib % 2)).to(torch.uint8)

    def half(at):
        return torch.stack([pool[at], pool[at + 1]], -1).view(torch.float16).squeeze(-1).double()

    k = ((code & 15).double() - 8.0) * half(base + 16 * hd + (t * (hd // 32) + g) * 2)
    lane, c = ch // (hd // 16), ch % (hd // 16)
    code = pool[base + 8 * hd + (((t // 4) * 16 + lane) * 4 + t % 4) * (hd // 32) + c // 2] >> (4 * (c % 2)).to(torch.uint8)
    v = ((code & 15).double() - 8.0) * half(base + 17 * hd + (g * 16 + t) * 2)
    return k, v


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None
    st = prepare(case, seed)
    if kind == "append":
        return {x: _exact_group(st[x].double().unflatten(-1, (-1, 32))).flatten(-2) for x in ("k", "v")}
    if kind == "logprobs":
        logp, entropy, best = [], [], []
        for a in range(0, case["rows"], 64):
            x = st["logits"][a:a + 64].double()
            lse = torch.logsumexp(x, 1, keepdim=True)
            logp.append((torch.gather(x, 1, st["targets"][a:a + 64].long().unsqueeze(1)) - lse).squeeze(1))
            entropy.append(-(torch.exp(x - lse) * (x - lse)).sum(1))
            best.append(torch.topk(x, case["top"], 1).values - lse)
        out = {"logp": torch.cat(logp), "entropy": torch.cat(entropy)}
        if case["top"]:
            out.update(top_ids=None, top_logp=torch.cat(best))
        return out
    kv, hd, heads, page, window = case["kv"], case["hd"], case["heads"], case["page"], case["window"]
    out = torch.zeros(st["rows"], heads, hd, dtype=torch.float64, device="cuda")
    start, lens = st["start"].tolist(), st["lens"].tolist()
    for b, n in enumerate(lens):
        k, v = _exact_tokens(st["pool"], st["tables"][b], kv, hd, page, n)
        for a in range(start[b], start[b + 1], 512):
            z = min(start[b + 1], a + 512)
            pos = n - (start[b + 1] - torch.arange(a, z, device="cuda")).unsqueeze(1)
            key = torch.arange(n, device="cuda")
            hidden = (key > pos) | (key <= pos - window) if window else key > pos
            for h in range(heads):
                s = (st["q"][a:z, h].double() @ k[h // (heads // kv)].t().contiguous()) / math.sqrt(hd)
                out[a:z, h] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v[h // (heads // kv)]
    return out
