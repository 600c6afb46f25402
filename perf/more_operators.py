"""The operators of a mixture of experts over a batch, as a program that drives a model's layers itself runs them.

Such a program has router logits of the batch's rows. It picks each row's experts and their weights
(`route`, and while the router is tuned the way back to its logits), sorts the rows by expert
(`dispatch`: the order, and the rows in it), puts the rows through the experts' matrices, which it keeps
in microscaled 4-bit floats (`quantise` makes them, and activations in the same format; `product` is the
matrix product, dense or by expert), and joins the experts' results back into rows (`combine`, and
while the router is tuned its gradient). Sizes are those of this repository's model configurations.

A microscaled matrix of `rows` x `cols` values: with cols padded by zeros to a multiple of 128, first the
codes [rows][padded / 2], two a byte, low half first, then a scale byte for each 32 columns
[rows][padded / 32]. A code is a sign bit over 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale byte b is 2^(b - 127),
255 is NaN.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "mx4": 17 / 32}
# (experts, experts a row, row width, expert width): Qwen3-30B-A3B, Granite-1B-A400M
EXPERTS = [(128, 8, 2048, 768), (32, 8, 1024, 512)]


def listed():
    return [
        # a decode step's routing: 24 sequences, a token each
        {"name": "route-decode", "kind": "route", "type": "f32", "rows": 24, "experts": 128, "k": 8, "norm": True, "grad": False},
        # a tuning step of a router: 8191 rows there and back
        {"name": "route-tune", "kind": "route", "type": "f32", "rows": 8191, "experts": 128, "k": 8, "norm": True, "grad": True},
        # a decode step's rows by expert
        {"name": "dispatch-decode", "kind": "dispatch", "type": "f32", "rows": 24, "experts": 128, "local": 128, "k": 8, "width": 2048},
        # a batch of prompt chunks by expert
        {"name": "dispatch-prompt", "kind": "dispatch", "type": "bf16", "rows": 8191, "experts": 128, "local": 128, "k": 8, "width": 2048},
        # their results joined
        {"name": "combine-prompt", "kind": "combine", "type": "bf16", "rows": 8191, "experts": 128, "local": 128, "k": 8, "width": 2048, "grad": False},
        # the joining's gradient in a tuning step of a small model
        {"name": "combine-tune", "kind": "combine", "type": "f32", "rows": 4097, "experts": 32, "local": 32, "k": 8, "width": 1024, "grad": True},
        # a prompt's activations into 4 bits and what they then stand for
        {"name": "quantise-prompt", "kind": "quantise", "type": "bf16", "rows": 8191, "cols": 2048},
        # the up matrices of 32 experts into 4 bits
        {"name": "quantise-weights", "kind": "quantise", "type": "f32", "rows": 32 * 512, "cols": 1024},
        # one token's logits
        {"name": "product-head", "kind": "product", "type": "f32", "out": "f32", "rows": 1, "cols": 2048, "n": 151936, "experts": 0, "k": 1, "gated": False, "sorted": False},
        # the gated half of the experts over a k = 8 verify of 24 sequences
        {"name": "product-experts-verify", "kind": "product", "type": "bf16", "out": "bf16", "rows": 216, "cols": 2048, "n": 768, "experts": 128, "k": 8, "gated": True, "sorted": False},
        # an attention output's projection over a prompt, 16-bit activations
        {"name": "product-prompt", "kind": "product", "type": "bf16", "out": "bf16", "rows": 4095, "cols": 4096, "n": 2048, "experts": 0, "k": 1, "gated": False, "sorted": False},
        # the gated half of the experts over a prompt, 4-bit activations
        {"name": "product-experts-prompt", "kind": "product", "type": "mx4", "out": "bf16", "rows": 4095, "cols": 2048, "n": 768, "experts": 128, "k": 8, "gated": True, "sorted": False},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["route", "dispatch", "combine", "quantise", "product", "product", "product"])
    experts, k, width, inner = rng.choice(EXPERTS)
    kind_of = rng.choice(list(TYPES))
    if kind == "quantise":
        cols = rng.choice([width, inner, _log(rng, 33, 5000)])
        return {"kind": kind, "type": kind_of, "rows": min(_log(rng, 1, 12000), 16_000_000 // cols), "cols": cols}
    if rng.random() < 0.3:  # other mixtures
        experts = _log(rng, 4, 200)
        k = rng.randint(1, min(experts, 10))
    if kind == "route":
        return {"kind": kind, "type": kind_of, "rows": _log(rng, 1, 8000), "experts": experts, "k": k, "norm": rng.random() < 0.7, "grad": rng.random() < 0.5}
    if kind in ("dispatch", "combine"):
        width = rng.choice([width, _log(rng, 60, 2500)])
        case = {"kind": kind, "type": kind_of, "rows": min(_log(rng, 1, 8000), 60_000_000 // (width * k)), "experts": experts, "k": k, "width": width}
        # all experts are here, or the other half is another device's
        case["local"] = rng.choice([experts, experts, max(1, experts // 2)])
        return {**case, "grad": rng.random() < 0.5} if kind == "combine" else case
    form = rng.choice(["dense", "experts", "experts"])
    case = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16", "mx4", "mx4"])}
    case["out"] = rng.choice(["bf16", "f16", "f32"]) if case["type"] == "mx4" else case["type"]
    if form == "dense":
        cols, n = rng.choice([(2048, 4096), (4096, 2048), (1024, 2048), (576, 1536), (1536, 576), (_log(rng, 100, 3000), _log(rng, 50, 3000))])
        rows = rng.choice([rng.randint(1, 16), _log(rng, 1, 300), _log(rng, 100, 4000)])
        return {**case, "rows": rows, "cols": cols, "n": n, "experts": 0, "k": 1, "gated": rng.random() < 0.3, "sorted": False}
    rows = rng.choice([rng.randint(1, 16), _log(rng, 1, 300), _log(rng, 100, 2500)])
    if rng.random() < 0.5:
        return {**case, "rows": rows, "cols": width, "n": inner, "experts": experts, "k": k, "gated": True, "sorted": False}
    return {**case, "rows": rows, "cols": inner, "n": width, "experts": experts, "k": k, "gated": False, "sorted": True}


# ------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(g, rows, experts):
    """Router logits: some experts are likelier than others."""
    return 1.5 * torch.randn(rows, experts, generator=g, device="cuda") + 0.5 * torch.randn(experts, generator=g, device="cuda")


def _rows(g, rows, width):
    """Rows as a norm leaves them: normal, a few channels larger than the rest."""
    wide = 1.0 + 4.0 * (torch.rand(width, generator=g, device="cuda") < 0.05)
    return torch.randn(rows, width, generator=g, device="cuda") * wide / wide.square().mean().sqrt()


def _matrix(g, rows, cols):
    """A matrix of weights in 4 bits."""
    out = torch.empty(rows * _padded(cols) * 17 // 32, dtype=torch.uint8, device="cuda")
    codes, scales = _parts(out, rows, cols)
    step = max(1, (1 << 26) // cols)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        codes[a:b], scales[a:b] = _quantise(0.02 * torch.randn(b - a, cols, generator=g, device="cuda"))
    return out


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    st = {"case": case}
    if kind == "quantise":
        st["x"] = _rows(g, case["rows"], case["cols"]).to(TYPES[case["type"]])
        return st
    rows, experts, k = case["rows"], case["experts"], case["k"]
    if kind == "route":
        st["logits"] = _logits(g, rows, experts).to(TYPES[case["type"]])
        if case["grad"]:
            st["d_weights"] = torch.randn(rows, k, generator=g, device="cuda")
        return st
    if kind == "product":
        cols, n = case["cols"], case["n"]
        held = rows * k if case["sorted"] else rows
        x = _rows(g, held, cols)
        if case["type"] == "mx4":
            codes, scales = _quantise(x)
            st["x"] = torch.cat([codes.flatten(), scales.flatten()])
        else:
            st["x"] = x.to(TYPES[case["type"]])
        st["w"] = _matrix(g, max(1, experts) * n, cols)
        if case["gated"]:
            st["up"] = _matrix(g, max(1, experts) * n, cols)
        if experts:
            chosen, _ = _plain_route(_logits(g, rows, experts), k, True)
            st.update(_plain_sort(chosen, experts))
            st["most"] = int((st["starts"][1:] - st["starts"][:-1]).max())
        return st
    chosen, weights = _plain_route(_logits(g, rows, experts), k, True)
    chosen = torch.where(chosen < case["local"], chosen, -1)
    if kind == "dispatch":
        st.update(chosen=chosen, x=_rows(g, rows, case["width"]).to(TYPES[case["type"]]))
        return st
    st.update(_plain_sort(chosen, case["local"]), weights=weights, y=torch.randn(rows * k, case["width"], generator=g, device="cuda").to(TYPES[case["type"]]))
    if case["grad"]:
        st["d_out"] = torch.randn(rows, case["width"], generator=g, device="cuda").to(TYPES[case["type"]])
    return st


# --------------------------------------------------------------------------------- plain forms
def _padded(cols):
    return -(-cols // 128) * 128


def _parts(data, rows, cols):
    """The codes [rows, padded / 2] and scale bytes [rows, padded / 32] of a matrix's bytes."""
    p = _padded(cols)
    return data[:rows * p // 2].view(rows, p // 2), data[rows * p // 2:rows * p * 17 // 32].view(rows, p // 32)


def _quantise(x):
    """Rows as codes and scale bytes."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, _padded(cols) - cols)).view(rows, -1, 32)
    most = x.abs().amax(-1, keepdim=True)
    e = ((most.view(torch.int32) >> 23) - 129).clamp(min=-127)  # floor(log2) - 2 (what is below the normal numbers: the lowest)
    m = torch.ldexp(x.abs(), -e)
    code = (m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
    code = code + 8 * torch.signbit(x)
    fine = torch.isfinite(most)
    code, byte = torch.where(fine, code, 0).view(rows, -1), torch.where(fine, e + 127, 255).squeeze(-1)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8), byte.to(torch.uint8)


def _values(data, rows, cols):
    """What a matrix's bytes stand for, in 32 bits."""
    codes, scales = _parts(data, rows, cols)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    v = table[torch.stack([codes & 15, codes >> 4], -1).flatten(1).int()].view(rows, -1, 32)
    s = torch.ldexp(torch.ones((), device="cuda"), scales.int() - 127)
    return (v * torch.where(scales == 255, math.nan, s).unsqueeze(-1)).flatten(1)[:, :cols]


def _plain_route(logits, k, norm):
    x = logits.float()
    best, ids = (t[:, :k] for t in torch.sort(x, dim=1, descending=True, stable=True))
    w = torch.exp(best - best[:, :1])
    total = w.sum(1, keepdim=True) if norm else torch.exp(x - best[:, :1]).sum(1, keepdim=True)
    return ids.to(torch.int32).contiguous(), w / total


def _plain_route_grad(logits, chosen, weights, d_weights, norm):
    dot = (weights * d_weights).sum(1, keepdim=True)
    at = chosen.long()
    if norm:
        return torch.zeros_like(logits).scatter_(1, at, (weights * (d_weights - dot)).to(logits.dtype))
    x = logits.float()
    e = torch.exp(x - x.amax(1, keepdim=True))
    g = (e / e.sum(1, keepdim=True)) * -dot
    return g.scatter_add_(1, at, weights * d_weights).to(logits.dtype)


def _plain_sort(chosen, experts):
    """The stable order of chosen [rows, k] by expert, and its inverse; -1 stands for no expert."""
    flat = chosen.flatten().long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(key, stable=True)
    starts = torch.searchsorted(key[order], torch.arange(experts + 1, device="cuda"))
    there = torch.arange(n, device="cuda") < starts[-1]
    place = torch.empty_like(order)
    place[order] = torch.where(there, torch.arange(n, device="cuda"), -1)
    return {"starts": starts.to(torch.int32), "order": torch.where(there, order, -1).to(torch.int32), "place": place.to(torch.int32).view(chosen.shape)}


def _plain_dispatch(st):
    s = _plain_sort(st["chosen"], st["case"]["local"])
    there = (s["order"] >= 0).unsqueeze(1)
    return {**s, "x": torch.where(there, st["x"][s["order"].clamp(min=0).long() // st["case"]["k"]], 0)}


def _plain_combine(st):
    dtype = st["y"].dtype
    place, there = st["place"].clamp(min=0).long(), (st["place"] >= 0).unsqueeze(-1)
    y = torch.where(there, st["y"][place].float(), 0.0)  # [rows, k, width]
    w = st["weights"].unsqueeze(-1)
    if not st["case"]["grad"]:
        return (w * y).sum(1).to(dtype)
    d = st["d_out"].float().unsqueeze(1)
    entry = st["order"].clamp(min=0).long()
    d_y = torch.where((st["order"] >= 0).unsqueeze(1), st["weights"].flatten()[entry].unsqueeze(1) * st["d_out"].float()[entry // st["case"]["k"]], 0.0)
    return {"d_y": d_y.to(dtype), "d_weights": (d * y).sum(-1)}


def _plain_product(st):
    case = st["case"]
    cols, n, experts, k = case["cols"], case["n"], case["experts"], case["k"]
    held = case["rows"] * k if case["sorted"] else case["rows"]
    x = _values(st["x"], held, cols) if case["type"] == "mx4" else st["x"].float()
    if experts:  # each expert's rows beside each other, as many places as the largest has
        r = torch.arange(case["rows"] * k, device="cuda")
        e = torch.searchsorted(st["starts"][1:].contiguous().long(), r, right=True)
        at = r - st["starts"][e].long()
        places = x.new_zeros(experts, st["most"], cols)
        places[e, at] = x if case["sorted"] else x[st["order"].long() // k]
    else:
        places = x.unsqueeze(0)
    out = []
    for w in [st["w"], st["up"]] if case["gated"] else [st["w"]]:
        w = _values(w, max(1, experts) * n, cols).view(-1, n, cols).transpose(1, 2).contiguous()
        out.append(torch.bmm(places, w))
    out = out[0] / (1.0 + torch.exp(-out[0])) * out[1] if case["gated"] else out[0]
    return (out[e, at] if experts else out[0]).to(TYPES[case["out"]])


def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "route":
        chosen, weights = _plain_route(st["logits"], case["k"], case["norm"])
        out = {"chosen": chosen, "weights": weights}
        return {**out, "d_logits": _plain_route_grad(st["logits"], chosen, weights, st["d_weights"], case["norm"])} if case["grad"] else out
    if kind == "quantise":
        codes, scales = _quantise(st["x"])
        return _values(torch.cat([codes.flatten(), scales.flatten()]), case["rows"], case["cols"]).to(st["x"].dtype)
    return {"dispatch": _plain_dispatch, "combine": _plain_combine, "product": _plain_product}[kind](st)


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
    case, kind, ctx = st["case"], st["case"]["kind"], _context()
    if kind == "route":
        chosen, weights = ops.moe_route(ctx, st["logits"], case["k"], norm=case["norm"])
        out = {"chosen": chosen, "weights": weights}
        return {**out, "d_logits": ops.moe_route_grad(ctx, st["logits"], chosen, st["d_weights"], norm=case["norm"])} if case["grad"] else out
    if kind == "dispatch":
        s = ops.moe_sort(ctx, st["chosen"], case["local"])
        return {"starts": s.starts, "order": s.order, "place": s.place, "x": ops.moe_gather(ctx, st["x"], s.order, case["k"])}
    if kind == "combine":
        if not case["grad"]:
            return ops.moe_combine(ctx, st["y"], st["place"], st["weights"])
        d_y, d_weights = ops.moe_combine_grad(ctx, st["d_out"], st["y"], st["order"], st["place"], st["weights"])
        return {"d_y": d_y, "d_weights": d_weights}
    if kind == "quantise":
        return ops.mx4_read(ctx, ops.mx4_quantize(ctx, st["x"]), st["x"].dtype)
    cols, experts, k = case["cols"], case["experts"], case["k"]
    x = ops.Mx4(st["x"], case["rows"] * k if case["sorted"] else case["rows"], cols) if case["type"] == "mx4" else st["x"]
    w, up = (ops.Mx4(st[m], max(1, experts) * case["n"], cols) if m in st else None for m in ("w", "up"))
    if not experts:
        return ops.mx4_matmul(ctx, x, w, up=up, dtype=TYPES[case["out"]])
    return ops.mx4_matmul(ctx, x, w, up=up, starts=st["starts"], order=None if case["sorted"] else st["order"], k=k, dtype=TYPES[case["out"]])


def run(st):
    return _own(st) if own else _plain(st)


# ------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, rows, size = case["kind"], case["rows"], SIZE[case["type"]]
    if kind == "quantise":
        # read, written as 4 bits, read again, written as what they stand for
        return {"bytes": 2.0 * rows * (case["cols"] * size + _padded(case["cols"]) * 17 / 32), "flops": 8.0 * rows * case["cols"]}
    k, experts = case["k"], case["experts"]
    if kind == "route":
        # logits, ids and weights; back: the weights' gradient, the logits (read again) and theirs
        back = 2 * experts * size + 8.0 * k if case["grad"] else 0.0
        return {"bytes": rows * (experts * size + 8.0 * k + back), "flops": (8.0 if case["grad"] else 5.0) * rows * experts}
    if kind == "product":
        n, cols, held = case["n"], case["cols"], rows * k if case["sorted"] else rows
        # the experts that even chances leave some row
        used = experts * (1.0 - (1.0 - k / experts) ** rows) if experts else 1.0
        both = 2 if case["gated"] else 1
        return {"bytes": held * cols * size + both * used * n * cols * 17 / 32 + rows * k * n * SIZE[case["out"]] + (4.0 * rows * k if experts else 0.0),
                "flops": 2.0 * both * rows * k * n * cols}
    width, here = case["width"] * size, rows * k * case["local"] / experts
    if kind == "dispatch":
        return {"bytes": rows * width + rows * k * width + 12.0 * rows * k, "flops": float(rows * k)}
    if case["grad"]:
        return {"bytes": rows * width + (here + rows * k) * width + 16.0 * rows * k, "flops": 3.0 * here * case["width"]}
    return {"bytes": (here + rows) * width + 8.0 * rows * k, "flops": 2.0 * here * case["width"]}


# ------------------------------------------------------------------------- the same in 64 bits
def _exact_values(data, rows, cols):
    """A matrix's values, each by its place in the bytes."""
    p = _padded(cols)
    r, c = torch.arange(rows, device="cuda").unsqueeze(1), torch.arange(cols, device="cuda")
    code = (data[r * (p // 2) + c // 2] >> (4 * (c % 2)).to(torch.uint8)) & 15
    e, m = ((code >> 1) & 3).double(), (code & 1).double()
    mag = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * 2.0 ** (e - 1.0))
    scale = torch.exp2(data[rows * (p // 2) + r * (p // 32) + c // 32].double() - 127.0)
    return torch.where(code >= 8, -mag, mag) * scale


def _exact_quantise(x):
    cols = x.shape[1]
    x = torch.nn.functional.pad(x, (0, _padded(cols) - cols)).unflatten(1, (-1, 32))
    _, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # in [0.5, 1) * 2^e
    step = torch.exp2((e - 3).clamp(min=-127).double())
    q = x / step
    mag = q.abs()
    grid = torch.where(mag < 2.0, 0.5, torch.where(mag < 4.0, 1.0, 2.0))
    return (torch.round(q / grid) * grid).clamp(-6.0, 6.0).mul(step).flatten(1)[:, :cols]


def exact(case, seed):
    kind, st = case["kind"], prepare(case, seed)
    if kind == "quantise":
        return _exact_quantise(st["x"].double())
    k = case["k"]
    if kind == "route":
        x = st["logits"].double()
        best = torch.topk(x, k, 1)
        p = torch.softmax(x, 1)
        w = torch.softmax(best.values, 1) if case["norm"] else torch.exp(best.values - torch.logsumexp(x, 1, keepdim=True))
        if not case["grad"]:
            return {"chosen": None, "weights": w}
        # as a product with the softmax's derivatives: equal logits are interchangeable for the weights, not for their
        # gradients, so the ids are those of the stable order
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        picked = torch.zeros_like(x).scatter_(1, ids, st["d_weights"].double())
        if case["norm"]:
            p = torch.softmax(x.masked_fill(torch.zeros_like(x).scatter_(1, ids, 1.0) == 0, -math.inf), 1)
        return {"chosen": None, "weights": w, "d_logits": p * picked - p * (p * picked).sum(1, keepdim=True)}
    if kind == "product":
        cols, n, experts = case["cols"], case["n"], case["experts"]
        if case["rows"] * k * n * cols > 3e11:
            return None
        held = case["rows"] * k if case["sorted"] else case["rows"]
        x = _exact_values(st["x"], held, cols) if case["type"] == "mx4" else st["x"].double()
        bounds = st["starts"].tolist() if experts else [0, case["rows"]]
        out = torch.empty(bounds[-1], n, dtype=torch.float64, device="cuda")
        size = n * _padded(cols)
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            if a == b:
                continue
            rows = x[a:b] if not experts or case["sorted"] else x[st["order"][a:b].long() // k]
            both = []
            for m in ("w", "up") if case["gated"] else ("w",):
                half = max(1, experts) * size // 2
                one = torch.cat([st[m][e * size // 2:(e + 1) * size // 2], st[m][half + e * size // 32:half + (e + 1) * size // 32]])
                both.append(rows @ _exact_values(one, n, cols).t())
            out[a:b] = both[0] * torch.sigmoid(both[0]) * both[1] if case["gated"] else both[0]
        return out
    if kind == "dispatch":
        order = torch.sort(torch.where(st["chosen"] < 0, case["local"], st["chosen"]).flatten().long() * (case["rows"] * k) + torch.arange(case["rows"] * k, device="cuda")).values
        at, none = order % (case["rows"] * k), order // (case["rows"] * k) >= case["local"]
        return {"starts": None, "order": None, "place": None, "x": st["x"].double()[at // k].masked_fill_(none.unsqueeze(1), 0.0)}
    y, w, place = st["y"].double(), st["weights"].double(), st["place"].long()
    if case["grad"]:
        d, d_w = st["d_out"].double(), torch.zeros_like(w)
        d_y = torch.zeros_like(y)
    out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
    for j in range(k):
        r = (place[:, j] >= 0).nonzero().squeeze(1)
        at = place[r, j]
        if case["grad"]:
            d_y[at] = w[r, j].unsqueeze(1) * d[r]
            d_w[r, j] = (d[r] * y[at]).sum(1)
        else:
            out[r] += w[r, j].unsqueeze(1) * y[at]
    return {"d_y": d_y, "d_weights": d_w} if case["grad"] else out
