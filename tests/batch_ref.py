"""The operators for batches of sequences in plain 64-bit numpy, from their definitions in
include/spx.h: the 4-bit format and its pool layout value by value, attention row by row, the page
plan sequence by sequence, log probabilities. Bounds on rounding go with each."""
import numpy as np

NAN = float("nan")


def log2(p):
    return int(p).bit_length() - 1


# ------------------------------------------------------------------------------ the 4-bit cache
def scale_of(group):
    """A group's scale from its 32 values (float64)."""
    if not np.isfinite(group).all():
        return NAN
    m = group[int(np.argmax(np.abs(group)))]  # the first of the largest
    d = -m / 8.0
    if d == 0.0:
        return 0.0
    e = np.frexp(d)[1] - 8  # bf16: eight significant bits
    d = np.rint(np.ldexp(d, -e)) * 2.0 ** e
    d = min(max(d, -8160.0), 8160.0)
    return np.rint(d * 2.0 ** 24) / 2.0 ** 24 + 0.0 if abs(d) < 2.0 ** -14 else d  # f16's smallest step; zero is +0


def codes_of(group, d):
    if d == 0.0 or not np.isfinite(d):
        return np.zeros(32, np.int64)
    return np.clip(np.rint(group / d), -8, 7).astype(np.int64)  # (exact near halves: d has eight bits)


def quantize(x):
    """[..., hd] -> (scales [..., hd / 32], codes [..., hd])."""
    x = np.asarray(x, np.float64)
    flat = x.reshape(-1, 32)
    d = np.array([scale_of(g) for g in flat])
    c = np.stack([codes_of(g, s) for g, s in zip(flat, d)]) if len(flat) else np.zeros((0, 32), np.int64)
    return d.reshape(*x.shape[:-1], -1), c.reshape(x.shape)


def values(x):
    """What rows stand for once they are in the cache."""
    d, c = quantize(x)
    return c * np.repeat(d, 32, axis=-1)


def places(shape, slot, head):
    """Byte offsets in the pool of a token's parts: (key code byte, shift), (value code byte, shift) for
    each channel, key scale, value scale for each group."""
    kv, hd, page, _ = shape
    G = hd // 32
    pg, t = divmod(slot, page)
    base = ((pg * kv + head) * (page // 16) + t // 16) * 18 * hd
    t %= 16
    nibble = [0, 4, 1, 5, 2, 6, 3, 7]  # of channels 0..7 of a word
    key, val = [], []
    for c in range(hd):
        g, h, n = c // 32, c % 32 // 8, nibble[c % 8]
        key.append((base + ((h * 16 + t) * G + g) * 4 + n // 2, 4 * (n % 2)))
        l, n = c // (hd // 16), c % (hd // 16)
        val.append((base + 8 * hd + (((t // 4) * 16 + l) * 4 + t % 4) * G + n // 2, 4 * (n % 2)))
    ks = [base + 16 * hd + (t * G + g) * 2 for g in range(G)]
    vs = [base + 17 * hd + (g * 16 + t) * 2 for g in range(G)]
    return key, val, ks, vs


def pool_bytes(shape):
    kv, hd, page, pages = shape
    return pages * kv * (page // 16) * 18 * hd


def write(pool, shape, slot, k, v):
    """One token's heads k, v [kv, hd] into the pool (a uint8 array)."""
    kv, hd, page, pages = shape
    if slot < 0 or slot >= pages * page:
        return
    for head in range(kv):
        key, val, ks, vs = places(shape, slot, head)
        for x, at, scales in ((k[head], key, ks), (v[head], val, vs)):
            d, c = quantize(x)
            for (b, s), code in zip(at, c):
                pool[b] = (pool[b] & (0xF0 if s == 0 else 0x0F)) | ((int(code) + 8) << s)
            for b, dd in zip(scales, d):
                pool[b:b + 2] = np.frombuffer(np.float16(dd).tobytes(), np.uint8)


# --------------------------------------------------------------------------------------- the plan
def plan(lens, add, tables, free, n_free, page, rows):
    """spx_pages_plan, a sequence at a time."""
    lens, tables, free = [int(v) for v in lens], np.array(tables), [int(v) for v in free]
    cols, n_pages, n = tables.shape[1], len(free), len(lens)
    need, have = [], int(n_free)
    start = [0]
    for a in add:
        start.append(start[-1] + max(int(a), 0))
    for s in range(n):
        held = -(-lens[s] // page)
        if add[s] < 0:
            for p in tables[s, :held]:
                if have < n_pages:
                    free[have] = int(p)
                    have += 1
        fits = add[s] >= 0 and lens[s] + add[s] <= cols * page and start[s + 1] <= rows
        need.append(-(-(lens[s] + int(add[s])) // page) - held if fits else 0)
    out_lens, status, taken, upto = [], [], 0, 0
    slots, positions = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    for s in range(n):
        upto += need[s]
        ok = add[s] >= 0 and lens[s] + add[s] <= cols * page and start[s + 1] <= rows and (need[s] == 0 or upto <= have)
        status.append(int(add[s] >= 0 and not ok))
        out_lens.append(0 if add[s] < 0 else lens[s] + int(add[s]) if ok else lens[s])
        if not ok:
            continue
        held = -(-lens[s] // page)
        for j in range(need[s]):
            tables[s, held + j] = free[have - 1 - taken]
            taken += 1
        for i in range(int(add[s])):
            pos = lens[s] + i
            positions[start[s] + i] = pos
            slots[start[s] + i] = tables[s, pos // page] * page + pos % page
    return {"lens": np.array(out_lens, np.int32), "n_free": np.array([have - taken], np.int32), "tables": tables, "free": np.array(free, np.int32),
            "q_start": np.minimum(start, rows).astype(np.int32), "slots": slots, "positions": positions, "status": np.array(status, np.int32)}


# ---------------------------------------------------------------------------------- attention
def attention(q, keys, vals, pos, window, scale, parts_q, parts_p):
    """One row's heads q [heads, hd] over keys / vals [n, kv, hd] (float64; what a page id outside the
    pool hides is NaN-free and marked in `hidden`): (out [heads, hd], bound on its error before the
    output's own rounding).

    The bound counts roundings. A score is a sum of hd products in 32 bits, at most 2^-24 of the sum
    of magnitudes each time it is rounded (hd + 8 times), with the query off by 2^-22 of its largest
    value where it is split in two parts (parts_q = 2; exact in one); scaling and the exponential's
    argument round three times more. A probability's relative error is twice its score's absolute
    one (numerator and denominator) and 2^-22, or 2^-11 in one f16 part. Sums over n tokens in 32
    bits round at most n / 8 + 64 times at 2^-24 of the sum of magnitudes."""
    heads, hd = q.shape
    n, kv = keys.shape[:2]
    lo, hi = (max(0, pos - window + 1) if window else 0), min(pos + 1, n)
    out, tol = np.zeros((heads, hd)), np.zeros((heads, hd))
    for h in range(heads):
        if hi <= lo:
            continue
        k, v = keys[lo:hi, h // (heads // kv)], vals[lo:hi, h // (heads // kv)]
        with np.errstate(invalid="ignore"):
            s = k @ q[h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h] = p @ v
            mag = np.abs(k) @ np.abs(q[h]) * abs(scale)
            split = 2.0 ** -22 * np.abs(q[h]).max() * np.abs(k).sum(1) * abs(scale) if parts_q == 2 else 0.0
            ds = (mag * (hd + 8) * 2.0 ** -24 + split + np.abs(s) * 3 * 2.0 ** -24).max()
            rel = 2 * ds + (2.0 ** -22 if parts_p == 2 else 2.0 ** -11) * 2 + ((hi - lo) / 8 + 64) * 2.0 ** -24
            tol[h] = rel * (p @ np.abs(v)) + 2.0 ** -35 * np.abs(v).sum(0) + 1e-37
    return out, tol


# ------------------------------------------------------------------------------ log probabilities
def logprobs(x, targets, top):
    """Rows x [rows, vocab] (float64, already over the scale)."""
    logp, ent, ids, best = [], [], [], []
    for r, row in enumerate(x):
        bad, none = bool((np.isnan(row) | (row == np.inf)).any()), bool((row == -np.inf).all())
        if bad:
            logp.append(NAN), ent.append(NAN), ids.append([-1] * top), best.append([NAN] * top)
            continue
        if none:
            lp = np.full(row.shape, -np.inf)
            ent.append(0.0)
        else:
            m = row.max()
            z = row - m
            e = np.exp(z)
            lp = z - np.log(e.sum())
            p = e / e.sum()
            ent.append(float(-(p[p > 0] * lp[p > 0]).sum()))
        t = -1 if targets is None else int(targets[r])
        logp.append(float(lp[t]) if 0 <= t < len(row) else NAN)
        order = [int(i) for i in np.lexsort((np.arange(len(row)), -row))[:top] if row[i] > -np.inf]
        ids.append(order + [-1] * (top - len(order)))
        best.append([float(lp[i]) for i in order] + [-np.inf] * (top - len(order)))
    return np.array(logp), np.array(ent), np.array(ids, np.int64).reshape(len(x), top), np.array(best).reshape(len(x), top)
