"""The operators for batches of sequences at the ends of their ranges: launches of many workgroups, numbers
at their types' limits, lengths near 2^31. References in 64 bits."""
import numpy as np
import pytest

from test_gpu_batch import BF16, F16, F32, Batch, ctx, f64, ints, queries  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PARTS = {F32: (2, 2), F16: (1, 2), BF16: (1, 1)}


def reference(b, q, counts, dtype, window=0, scale=None, lens=None):
    """batch_ref.attention and its bound for every row at once, in 64 bits on the device, the output's own
    rounding included. (Products of two-dimensional matrices, the right one made dense.)"""
    parts_q, parts_p = PARTS[dtype]
    rows, heads, hd = q.shape
    scale = scale or hd ** -0.5
    out, tol = (torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda") for _ in range(2))
    at = 0
    for s, c in enumerate(counts):
        n = b.lens[s] if lens is None else lens[s]
        k, v = (torch.from_numpy(x[b.slots(s, n)]).cuda() for x in (b.k, b.v))
        tok = torch.arange(n, device="cuda")
        for a in range(0, c, 1024):
            z = min(c, a + 1024)
            pos = (n - c + torch.arange(a, z, device="cuda"))[:, None]
            seen = (tok <= pos) & (tok > pos - window) if window else tok <= pos
            some = seen.any(1, keepdim=True)
            for h in range(heads):
                kh, vh, qh = k[:, h // (heads // b.kv)].contiguous(), v[:, h // (heads // b.kv)].contiguous(), q[at + a:at + z, h].double()
                x = (qh @ kh.t().contiguous()) * scale
                mag = (qh.abs() @ kh.abs().t().contiguous()) * scale
                split = 2.0 ** -22 * qh.abs().amax(1, keepdim=True) * kh.abs().sum(1) * scale if parts_q == 2 else 0.0
                ds = torch.where(seen, mag * (hd + 8) * 2.0 ** -24 + split + x.abs() * 3 * 2.0 ** -24, 0.0).amax(1, keepdim=True)
                p = torch.where(some, torch.softmax(torch.where(seen, x, -torch.inf), 1), 0.0)
                rel = 2 * ds + (2.0 ** -22 if parts_p == 2 else 2.0 ** -11) * 2 + (seen.sum(1, keepdim=True) / 8 + 64) * 2.0 ** -24
                out[at + a:at + z, h] = p @ vh
                tol[at + a:at + z, h] = torch.where(some, rel * (p @ vh.abs()) + 2.0 ** -35 * (seen.double() @ vh.abs()) + 1e-37, 0.0)
        at += c
    half = torch.finfo(dtype).eps / 2
    return out, tol + half * (out.abs() + tol) + (2.0 ** -25 if dtype == F16 else 0.0)


def held(ctx, b, q, counts, dtype, window=0, scale=None, **kw):
    """Runs the operator into an output of NaN and holds every row to its bound."""
    from spindle_amd import ops
    start = np.concatenate([[0], np.cumsum(counts)])
    out = torch.full_like(q, float("nan"))
    ops.kv4_attention(ctx, b.shape, b.pool, q, ints(start), ints(b.lens), ints(b.tables), scale=scale or 0.0, window=window, out=out, **kw)
    want, tol = reference(b, q, counts, dtype, window, scale)
    n = int(start[-1])
    bad = ~((out[:n].double() - want[:n]).abs() <= tol[:n])
    assert not bad.any(), (int(bad.any(-1).sum()), bad.nonzero()[0].tolist())
    assert out[n:].isnan().all()
    return out


# -------------------------------------------------------------------- launches of many workgroups
@pytest.mark.parametrize("heads,kv,hd,lens,counts,dtype", [
    (9, 3, 64, [8192], [8192], BF16),                                        # 579 workgroups of the prompt kernel, one chunk
    (9, 3, 64, [100] * 64, [78] * 63 + [86], F32),                           # 5000 rows over 64 sequences
    (12, 6, 64, [4096], [4096], F16),
    (40, 10, 128, [2100, 2048], [2000, 2048], BF16),
    (40, 10, 128, [4096], [4096], F32),
    (5, 5, 64, [3000, 40, 2900], [2700, 0, 2500], BF16),
])
def test_prompts_of_many_workgroups(ctx, heads, kv, hd, lens, counts, dtype):  # noqa: F811
    """Row tiles times key heads past 512, numbers of key heads that are no power of two."""
    b = Batch(ctx, lens, kv, hd, 64, seed=kv)
    held(ctx, b, queries(kv, sum(counts), heads, hd, dtype), counts, dtype)


@pytest.mark.parametrize("heads,kv,hd", [(9, 3, 64), (12, 6, 64), (20, 5, 128)])
@pytest.mark.parametrize("window", [0, 700])
def test_many_workgroups_split(ctx, heads, kv, hd, window):  # noqa: F811
    """The same where sequences are split into chunks, whose outputs are joined: many short row tiles."""
    n = 220
    lens, counts = [[1500, 260, 90][i % 3] for i in range(n)], [[30, 1, 3][i % 3] for i in range(n)]
    b = Batch(ctx, lens, kv, hd, 16, seed=heads)
    held(ctx, b, queries(heads, sum(counts), heads, hd, F32), counts, F32, window=window)


# ----------------------------------------------------------------------- scores far from zero
def whole_keys(b, step, seed):
    """Keys of whole multiples of `step` (a power of two) in every slot: -7 .. 7 times it, the first channel of
    each group -8 times, so that the cache holds them exactly."""
    from spindle_amd import ops
    rng = np.random.default_rng(seed)
    k = rng.integers(-7, 8, (b.pages * b.page, b.kv, b.hd)).astype(np.float32)
    k[:, :, ::32] = -8.0
    v = torch.from_numpy(b.v).float().cuda()
    ops.kv4_append(b.ctx, b.shape, b.pool, torch.from_numpy(k * np.float32(step)).cuda(), v, ints(np.arange(b.pages * b.page)))
    b.refresh()
    assert np.array_equal(b.k, k.astype(np.float64) * step)


def run_into_nan(ctx, b, q, counts, **kw):  # noqa: F811
    from spindle_amd import ops
    out = torch.full_like(q, float("nan"))
    ops.kv4_attention(ctx, b.shape, b.pool, q, ints(np.concatenate([[0], np.cumsum(counts)])), ints(b.lens), ints(b.tables), out=out, **kw)
    return out


def check_largest_scores(ctx, dtype, hd, size, step, scale, lens, counts):  # noqa: F811
    """Queries with one channel of +-size: a row's scores are exact and further apart than any
    exponential's range, so that it is the mean of the values of its largest keys. Bound: n / 8 + 64
    roundings of a 32-bit sum; every probability is the same power of two."""
    b = Batch(ctx, lens, 2, hd, 16, seed=50)
    whole_keys(b, step, 51)
    rows, heads = sum(counts), 8
    rng = np.random.default_rng(52)
    ch = rng.integers(1, 32, (rows, heads)) + 32 * rng.integers(0, hd // 32, (rows, heads))
    sign = rng.choice([-1.0, 1.0], (rows, heads))
    q = torch.zeros(rows, heads, hd, dtype=dtype, device="cuda")
    q[torch.arange(rows)[:, None], torch.arange(heads)[None], torch.from_numpy(ch)] = torch.from_numpy(sign * size).to(dtype).cuda()
    got = f64(run_into_nan(ctx, b, q, counts, scale=scale))
    half, at = torch.finfo(dtype).eps / 2, 0
    for s, c in enumerate(counts):
        slots = b.slots(s)
        for i in range(c):
            n = lens[s] - c + i + 1
            for h in range(heads):
                k, v = b.k[slots[:n], h // 4, ch[at, h]] * sign[at, h], b.v[slots[:n], h // 4]
                best = v[k == k.max()]
                want = best.mean(0)
                tol = (n / 8 + 64) * 2.0 ** -24 * np.abs(best).mean(0)
                tol += half * (np.abs(want) + tol) + 2.0 ** -25
                assert (np.abs(got[at, h] - want) <= tol).all(), (s, i, h)
            at += 1


FAR = [(F32, 2.0 ** 30, 1.0, 0.0), (F32, 2.0 ** 100, 1.0, 0.0), (BF16, 2.0 ** 30, 1.0, 0.0), (BF16, 2.0 ** 100, 1.0, 0.0), (F16, 2.0 ** 15, 2.0 ** 12, 1.0)]


@pytest.mark.parametrize("dtype,size,step,scale", FAR)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts", [[2, 1], [60, 1]])
def test_scores_far_apart(ctx, dtype, size, step, scale, hd, counts):  # noqa: F811
    """Scores past 2^28, where the rounding of the largest one alone is more than f16's range."""
    check_largest_scores(ctx, dtype, hd, size, step, scale, [150, 70], counts)


@pytest.mark.parametrize("dtype,size,step,scale", FAR)
def test_scores_far_apart_split(ctx, dtype, size, step, scale):  # noqa: F811
    check_largest_scores(ctx, dtype, 128, size, step, scale, [3000, 700], [2, 1])
    check_largest_scores(ctx, dtype, 64, size, step, scale, [1500, 70], [70, 3])


@pytest.mark.parametrize("dtype,size,scale", [(F32, 1e10, 0.0), (F32, 1e30, 0.0), (BF16, 1e10, 0.0), (BF16, 1e30, 0.0), (F16, 3e3, 1e6)])
@pytest.mark.parametrize("counts", [[2, 1], [60, 1]])
def test_large_queries(ctx, dtype, size, scale, counts):  # noqa: F811
    """Ordinary rows times a large number: where the largest score is further from the next than what
    rounding can move them (and 50 more), the row is that token's value; elsewhere it lies among the values."""
    b = Batch(ctx, [300, 90], 2, 128, 16, seed=53)
    q = queries(53, sum(counts), 8, 128, dtype, size).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    got, sc = run_into_nan(ctx, b, q, counts, scale=scale).double(), scale or 128 ** -0.5
    parts_q, parts_p = PARTS[dtype]
    at, sure = 0, 0
    for s, c in enumerate(counts):
        k, v = (torch.from_numpy(x[b.slots(s)]).cuda() for x in (b.k, b.v))
        for i in range(c):
            n = b.lens[s] - c + i + 1
            for h in range(8):
                kh, vh, qh = k[:n, h // 4], v[:n, h // 4], q[at, h].double()
                x = kh @ qh * sc
                ds = ((kh.abs() @ qh.abs()) * 136 * 2.0 ** -24 + qh.abs().max() * kh.abs().sum(1) * (2.0 ** -22 if parts_q == 2 else 0.0) + x.abs() / sc * 3 * 2.0 ** -24).max() * sc
                top = x.topk(2)
                assert (got[at, h].abs() <= vh.abs().max() * (1 + 2.0 ** -7)).all()
                if float(top.values[0] - top.values[1]) > 2 * float(ds) + 50:
                    want = vh[top.indices[0]]
                    tol = (2.0 ** -21 if parts_p == 2 else 2.0 ** -11) * want.abs() + 2.0 ** -20
                    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
                    assert ((got[at, h] - want).abs() <= tol).all(), (s, i, h)
                    sure += 1
            at += 1
    assert sure > 0.9 * at * 8


@pytest.mark.parametrize("dtype,size,scale", [(t, 2.0 ** e, s) for t in (F32, BF16) for e, s in ((121, 0.0), (127, 0.0), (110, 1e9), (20, 3e38), (127, 3e38))] +
                         [(F16, 2.0 ** 15, 3e38)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts", [[2, 1], [60, 1]])
def test_queries_at_their_types_end(ctx, dtype, size, scale, hd, counts):  # noqa: F811
    """Queries and scales up to the largest numbers there are."""
    check_largest_scores(ctx, dtype, hd, size, 1.0, scale, [150, 70], counts)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e36, 1e38])
@pytest.mark.parametrize("counts", [[2, 1], [60, 1]])
def test_largest_queries(ctx, dtype, size, counts):  # noqa: F811
    test_large_queries(ctx, dtype, size, 0.0, counts)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("counts", [[2, 1], [60, 1]])
def test_vanishing_scores(ctx, dtype, counts):  # noqa: F811
    """Scores that are zero in 32 bits: a row is the mean of the values it sees, what it does not see counts
    for nothing."""
    b = Batch(ctx, [150, 70], 2, 64, 16, seed=54)
    for size, scale in ((1e-38 if dtype != F16 else 6e-8, 1e-38), (1.0, 1e-45)):
        for window in (0, 20):
            held(ctx, b, queries(54, sum(counts), 8, 64, dtype, size), counts, dtype, window=window, scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts", [[3, 2], [60, 2]])
def test_infinite_queries(ctx, dtype, hd, counts):  # noqa: F811
    """A row with an infinity or a NaN among its queries is NaN, also where all its scores are -inf (every key's
    first channel is negative), unless it sees nothing; its neighbours keep their bits."""
    b = Batch(ctx, [100, 1], 2, hd, 16, seed=55)
    whole_keys(b, 1.0, 56)
    b.lens[0] = counts[0] - 1  # the first row of either sequence sits before position 0
    q = queries(55, sum(counts), 8, hd, dtype)
    want = run_into_nan(ctx, b, q, counts)
    bad = torch.zeros(sum(counts), 8, dtype=torch.bool, device="cuda")
    for row, head, ch, x in ((0, 0, 0, np.inf), (1, 0, 0, np.inf), (1, 5, 32, np.inf), (1, 6, 7, -np.inf), (2, 3, 0, -np.inf), (2, 4, 9, np.nan),
                             (counts[0], 1, 0, np.inf), (counts[0] + 1, 2, 0, np.inf), (counts[0] + 1, 7, 0, np.nan)):
        q[row, head, ch], bad[row, head] = x, True
    got = run_into_nan(ctx, b, q, counts)
    nothing = torch.zeros_like(bad)
    nothing[0], nothing[counts[0]] = True, True
    assert (want[nothing] == 0).all() and (got[nothing] == 0).all()
    assert torch.equal(got[~bad & ~nothing], want[~bad & ~nothing])
    assert got[bad & ~nothing].isnan().all()


# ------------------------------------------------------------------------ lengths near 2^31
def test_plan_lengths_at_their_end(ctx):  # noqa: F811
    """Tables with room for more than 2^31 tokens: a sequence of the longest length there is gives back the
    pages that the list has room for, one that would pass it is refused and takes no pages from those after
    it."""
    from spindle_amd import ops
    top, cols, pages = 2 ** 31 - 1, 2 ** 23 + 1, 20
    tables = torch.arange(3 * cols, dtype=torch.int32, device="cuda").view(3, cols)
    tables[1, 0] = 5
    free = ints([90, 91, 92] + [-1] * (pages - 3))

    def plan(lens, add, rows):
        t, f = tables.clone(), free.clone()
        p = ops.pages_plan(ctx, ints(lens), ints(add), t, f, ints([3]), 256, rows)
        return p, t, f

    p, t, f = plan([top, 10, 300], [-1, 5, -1], 6)
    assert p.lens.tolist() == [0, 15, 0] and p.status.tolist() == [0, 0, 0] and p.n_free.tolist() == [pages]
    assert f.tolist() == [90, 91, 92] + list(range(17)) and torch.equal(t, tables)
    assert p.slots.tolist() == [5 * 256 + i for i in range(10, 15)] + [-1] and p.positions.tolist() == [10, 11, 12, 13, 14, -1]
    p, t, f = plan([top - 3, 250, top], [4, 10, 0], 14)
    assert p.lens.tolist() == [top - 3, 260, top] and p.status.tolist() == [1, 0, 0] and p.n_free.tolist() == [2]
    assert p.q_start.tolist() == [0, 4, 14, 14] and t[1, 1] == 92 and torch.equal(f, free)
    assert p.slots.tolist() == [-1] * 4 + [5 * 256 + i for i in range(250, 256)] + [92 * 256 + i for i in range(4)]
    p, t, f = plan([top - 3, 0, 0], [3, 0, 0], 3)
    assert p.lens.tolist() == [top, 0, 0] and p.status.tolist() == [0, 0, 0] and p.n_free.tolist() == [3]
    assert p.positions.tolist() == [top - 3, top - 2, top - 1] and torch.equal(t, tables)


@pytest.mark.parametrize("kv,counts", [(300, [150, 2]), (300, [3, 1]), (1024, [70, 1]), (1024, [1, 1])])
def test_many_key_heads(ctx, kv, counts):  # noqa: F811
    """As many key heads as there may be, more than a turn of the prompt kernel's order."""
    b = Batch(ctx, [160, 40], kv, 64, 16, seed=57)
    held(ctx, b, queries(57, sum(counts), kv, 64, BF16), counts, BF16)
