"""The operators of a mixture of experts over a batch in plain 64-bit numpy, from their definitions in
include/spx.h: the router and its gradient, the sort entry by entry, rows joined, microscaled 4-bit floats
value by value and their products. Bounds on rounding go with each."""
import math

import numpy as np

EPS = {"float32": 2.0 ** -23, "float16": 2.0 ** -10, "bfloat16": 2.0 ** -7}  # twice a rounding, relative
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}
U = 2.0 ** -24  # a rounding in 32 bits


def name_of(dtype):
    return str(dtype).replace("torch.", "")


def rounding(v, dtype):
    """The most that rounding v to a type moves it."""
    return np.abs(v) * EPS[name_of(dtype)] / 2 + TINY[name_of(dtype)]


# ------------------------------------------------------------------------------------ the router
def route(x, k, norm):
    """Rows x [rows, E] (float64): chosen, weights, a bound on the weights' error. An exponential's argument is
    rounded once and its result off by two roundings at most; sums over E or k terms round E / 64 + 8 times."""
    chosen, weights, tol = [], [], []
    for row in x:
        key = [(-math.inf if math.isnan(v) else -v, i) for i, v in enumerate(row)]
        nan = [i for i, v in enumerate(row) if math.isnan(v)]
        ids = (nan + [i for _, i in sorted(t for t in key if t[1] not in nan)])[:k]
        chosen.append(ids)
        if np.isnan(row).any() or (row == np.inf).any():
            weights.append([math.nan] * k), tol.append([0.0] * k)
            continue
        if (row == -np.inf).all():
            weights.append([0.0] * k), tol.append([0.0] * k)
            continue
        e = np.exp(row - row.max())
        p = e / (e[ids].sum() if norm else e.sum())
        far = np.where(e > 1e-45, row.max() - row, 0.0)
        weights.append(list(p[ids]))
        rel = (far + 3) * U
        among = ids if norm else slice(None)
        total = (e[among] * rel[among]).sum() / e[among].sum() + (len(row) / 64 + 9) * U
        tol.append(list(p[ids] * (rel[ids] + total) + 1e-44))
    return np.array(chosen), np.array(weights), np.array(tol)


def route_grad(x, chosen, g, norm):
    """(d logits, bound)."""
    d, tol = np.zeros_like(x), np.zeros_like(x)
    for r, row in enumerate(x):
        ids = chosen[r]
        if np.isnan(row).any() or (row == np.inf).any() or (ids < 0).any() or (ids >= len(row)).any():
            d[r] = math.nan
            continue
        if (row == -np.inf).all():
            continue
        e = np.exp(row - (row[ids].max() if norm and row[ids].max() > -np.inf else row.max()))
        total = e[ids].sum() if norm else e.sum()
        if total == 0.0:
            continue
        p = e / total
        far = np.where(e > 1e-45, np.abs(row.max() - row), 0.0).max()
        rel = 2 * (far + 3) * U + (len(row) / 64 + 12) * U
        s = (p[ids] * g[r]).sum()
        mag = (p[ids] * np.abs(g[r])).sum()
        if not norm:
            d[r] = -p * s
            tol[r] = p * (mag * (2 * rel + 12 * U))
        for j, c in enumerate(ids):
            d[r, c] += p[c] * ((g[r, j] - s) if norm else g[r, j])
            tol[r, c] += p[c] * ((abs(g[r, j]) + mag) * (2 * rel + 12 * U))
        tol[r] += 1e-44
    return d, tol


# -------------------------------------------------------------------------------------- the sort
def sort(chosen, n_expert):
    flat = chosen.reshape(-1)
    order = [i for e in range(n_expert) for i in range(len(flat)) if flat[i] == e]
    starts = np.cumsum([0] + [int((flat == e).sum()) for e in range(n_expert)])
    place = np.full(len(flat), -1)
    place[order] = np.arange(len(order))
    return starts, np.array(order + [-1] * (len(flat) - len(order)), np.int64), place.reshape(chosen.shape)


# ------------------------------------------------------------------------------------- 4-bit rows
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def padded(cols):
    return -(-cols // 128) * 128


def quantize(x):
    """Rows x [rows, cols] (float64 of a type's values): codes [rows, P], scale bytes [rows, P / 32]."""
    rows, cols = x.shape
    x = np.concatenate([x, np.zeros((rows, padded(cols) - cols))], 1).reshape(rows, -1, 32)
    codes, scales = np.zeros(x.shape, np.int64), np.zeros(x.shape[:2], np.int64)
    for r in range(rows):
        for b in range(x.shape[1]):
            v = x[r, b]
            if not np.isfinite(v).all():
                scales[r, b] = 255
                continue
            m = np.abs(v).max()
            e = max((int(math.floor(math.log2(m))) if m > 0 else -1000) - 2, -127)
            if m > 0 and not 2.0 ** (e + 2) <= m < 2.0 ** (e + 3) and e > -127:  # (log2 rounds near powers of two)
                e = int(np.frexp(m)[1]) - 3
            scales[r, b] = e + 127
            q = np.abs(v) / 2.0 ** e
            for i, a in enumerate(q):
                off = np.abs(GRID - a)
                near = np.flatnonzero(off == off.min())
                c = int(near[0]) if len(near) == 1 else int([n for n in near if n % 2 == 0][0])
                codes[r, b, i] = (7 if a > 6 else c) + 8 * int(np.signbit(v[i]))
    return codes.reshape(rows, -1), scales


def pack(codes, scales):
    return np.concatenate([(codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8).reshape(-1), scales.astype(np.uint8).reshape(-1)])


def unpack(data, rows, cols):
    """The values [rows, cols] that a matrix's bytes stand for."""
    p = padded(cols)
    c = data[:rows * p // 2].reshape(rows, p // 2)
    s = data[rows * p // 2:rows * p // 32 * 17].reshape(rows, p // 32).astype(np.float64)
    codes = np.stack([c & 15, c >> 4], -1).reshape(rows, p)
    v = GRID[codes & 7] * np.where(codes >= 8, -1.0, 1.0)
    return (v * np.repeat(np.where(s == 255, np.nan, np.exp2(s - 127)), 32, axis=1))[:, :cols]


# --------------------------------------------------------------------------------------- products
def product(x, w, up, parts):
    """x [rows, cols], w, up [n, cols] (float64; up or None): (out, a bound on its error before the output's rounding).

    A matrix instruction takes 128 columns of 4-bit rows, or 32 of a part of others, and its sum is off by at most a
    unit in the last place of the magnitudes so far; what the waves hold is joined with a few additions. What a 16- or
    32-bit value loses below 2^-133 is times a weight."""
    cols = x.shape[1]
    count = padded(cols) // 128 * (1 if parts == 0 else 4 * parts) + 8

    def one(m):
        v = x @ m.T
        return v, np.abs(x) @ np.abs(m).T * count * 2 * U + (2.0 ** -133 * np.abs(m).sum(1) if parts > 1 else 0.0) + 2.0 ** -140

    g, dg = one(w)
    if up is None:
        return g, dg
    u, du = one(up)
    with np.errstate(over="ignore", invalid="ignore"):
        s = g / (1.0 + np.exp(-g))
        # silu's slope is at most 1.1; the exponential is off by its argument's rounding and two of its own, the division
        # and the sum by one each
        ds = 1.1 * dg + np.abs(s) * (np.minimum(np.abs(g), 100.0) + 6) * 2 * U
        return s * u, ds * np.abs(u) + np.abs(s) * du + ds * du + np.abs(s * u) * 2 * U
