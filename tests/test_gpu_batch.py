"""The operators for batches of sequences (include/spx.h: spx_pages_plan, spx_kv4_append, spx_kv4_read,
spx_kv4_attention, spx_logprobs) against 64-bit evaluations of their definitions (batch_ref.py)."""
import numpy as np
import pytest

import batch_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    from spindle_amd import ops
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = ops.Context(0)
    yield c
    c.close()


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def f64(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------------ the 4-bit cache
def rows_for(rng, n, kv, hd, dtype):
    x = rng.standard_normal((n, kv, hd)) * np.exp(rng.uniform(-3, 3, (n, kv, 1)))
    g = x.reshape(-1, 32)
    for i, kind in enumerate(rng.integers(0, 16, len(g))):  # special groups among ordinary ones
        if kind == 0:
            g[i] = 0.0
        elif kind == 1:
            g[i, rng.integers(32)] = [np.nan, np.inf, -np.inf][i % 3]
        elif kind == 2:  # two of the largest magnitude, either sign first
            g[i, [5, 21]] = (9.0, -9.0) if i % 2 else (-9.0, 9.0)
        elif kind == 3:  # every quotient a half
            g[i] = (rng.integers(-8, 7, 32) + 0.5) * 0.25
            g[i, 11] = -2.0
        elif kind == 4:
            g[i] *= 1e-7  # scales among f16's subnormals
        elif kind == 5:
            g[i] *= 1e-30
        elif kind == 6:
            g[i] *= 1e5 if dtype != F16 else 1e2  # scales at their limit
    big = {F32: 3e38, F16: 65504.0, BF16: 3e38}[dtype]
    return torch.from_numpy(np.clip(x, -big, big)).to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kv,hd,page", [(1, 64, 16), (3, 64, 32), (2, 128, 64), (1, 128, 256)])
def test_append_and_read(ctx, dtype, kv, hd, page):
    from spindle_amd import ops
    rng = np.random.default_rng(page + hd + kv)
    pages = 1 + 200 // page
    sh = (kv, hd, page, pages)
    shape = ops.Kv4Shape(*sh)
    n = 23
    pool = torch.from_numpy(rng.integers(0, 256, R.pool_bytes(sh), dtype=np.uint8)).cuda()
    want = pool.cpu().numpy().copy()
    slots = rng.permutation(pages * page)[:n]
    slots[[3, 7, 8]] = -1, pages * page, 2 ** 31 - 1  # passed over
    wide = rows_for(rng, n, 1, kv * hd * 2 + 32, dtype).cuda().squeeze(1)
    k, v = wide[:, :kv * hd].view(n, kv, hd), wide[:, kv * hd + 32:].view(n, kv, hd)  # rows apart by more than their width
    ops.kv4_append(ctx, shape, pool, k, v, ints(slots))
    for i, s in enumerate(slots):
        R.write(want, sh, int(s), f64(k[i]), f64(v[i]))
    assert np.array_equal(pool.cpu().numpy(), want)
    gk, gv = ops.kv4_read(ctx, shape, pool, ints(slots), dtype)
    inside = (slots >= 0) & (slots < pages * page)
    for got, x in ((gk, k), (gv, v)):
        ref = torch.from_numpy(np.where(inside[:, None, None], R.values(f64(x)), 0.0)).to(dtype)
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=12345.0), torch.nan_to_num(ref, nan=12345.0))


def test_append_one_row_rewrites_it(ctx):
    """A slot written again holds the last row alone; its neighbours stay."""
    from spindle_amd import ops
    rng = np.random.default_rng(4)
    shape = ops.Kv4Shape(2, 64, 16, 2)
    pool = shape.pool()
    a, b, c = (torch.from_numpy(rng.standard_normal((2, 2, 64))).float().cuda() for _ in range(3))
    ops.kv4_append(ctx, shape, pool, a, b, ints([4, 5]))
    ops.kv4_append(ctx, shape, pool, c[:1], a[:1], ints([4]))
    k, v = ops.kv4_read(ctx, shape, pool, ints([4, 5]))
    assert np.array_equal(f64(k), R.values(np.stack([f64(c[0]), f64(a[1])])))
    assert np.array_equal(f64(v), R.values(np.stack([f64(a[0]), f64(b[1])])))
    k, v = ops.kv4_read(ctx, shape, pool, ints([]))
    assert k.shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kv,hd", [(8, 128), (13, 64)])
def test_append_and_read_many_rows(ctx, dtype, kv, hd):
    """A prompt's thousands of rows, more than a thread each, at odd counts and addresses, against the
    same in small calls."""
    from spindle_amd import ops
    n, page = 9001, 64
    shape = ops.Kv4Shape(kv, hd, page, n // page + 2)
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    slots = torch.randperm(shape.n_pages * page, generator=g, device="cuda")[:n].to(torch.int32)
    slots[[5, 8000]] = -1
    for off in (0, 1):
        k, v = (torch.randn(n * kv * hd + 1, generator=g, device="cuda").to(dtype)[off:off + n * kv * hd].view(n, kv, hd) for _ in range(2))
        many, few = shape.pool(), shape.pool()
        ops.kv4_append(ctx, shape, many, k, v, slots)
        for a in range(0, n, 500):
            ops.kv4_append(ctx, shape, few, k[a:a + 500], v[a:a + 500], slots[a:a + 500])
        assert torch.equal(many, few)
        got = ops.kv4_read(ctx, shape, many, slots, dtype)
        for a in range(0, n, 500):
            one = ops.kv4_read(ctx, shape, few, slots[a:a + 500], dtype)
            assert all(torch.equal(x[a:a + 500], y) for x, y in zip(got, one))


# --------------------------------------------------------------------------------------- the plan
def run_plan(ctx, lens, add, tables, free, n_free, page, rows):
    from spindle_amd import ops
    t, f = ints(tables), ints(free)
    p = ops.pages_plan(ctx, ints(lens), ints(add), t, f, ints([n_free]), page, rows)
    got = {k: getattr(p, k).cpu().numpy() for k in ("lens", "n_free", "q_start", "slots", "positions", "status")}
    return got | {"tables": t.cpu().numpy(), "free": f.cpu().numpy()}


def plan_case(rng, n, page, most, room, rows_short=0):
    lens = rng.integers(0, most, n) * (rng.random(n) < 0.9)
    add = np.where(rng.random(n) < 0.15, -1, rng.integers(0, [2, 2, most][rng.integers(3)], n))
    cols = -(-2 * most // page) + rng.integers(0, 2)
    held = -(-lens // page)
    total = int(held.sum()) + room
    ids = rng.permutation(total)
    tables, at = np.full((n, cols), -7), 0
    for s in range(n):
        tables[s, :held[s]] = ids[at:at + held[s]]
        at += held[s]
    free = np.full(max(total, 1), -9)
    free[:room] = ids[at:]
    rows = max(0, int(np.maximum(add, 0).sum()) + [0, 3][rng.integers(2)] - rows_short)
    return lens, add, tables, free, room, page, rows


@pytest.mark.parametrize("seed", range(24))
def test_plan(ctx, seed):
    rng = np.random.default_rng(seed)
    n = [1, 2, 5, 63, 64, 65, 200, 1023, 1024, 1025][seed % 10]
    page = [16, 32, 64, 256][seed % 4]
    case = plan_case(rng, n, page, [3, 40, 300][seed % 3], int(rng.integers(0, 4 * n)), rows_short=[0, 0, 5][seed // 8])
    got, want = run_plan(ctx, *case), R.plan(*case)
    for k in want:
        assert np.array_equal(got[k], want[k]), k


def test_plan_most_sequences(ctx):
    rng = np.random.default_rng(1)
    case = plan_case(rng, 4096, 16, 40, 6000)
    got, want = run_plan(ctx, *case), R.plan(*case)
    for k in want:
        assert np.array_equal(got[k], want[k]), k


def test_plan_many_rows(ctx):
    """Prompts of tens of thousands of rows, a short table and no rows at all."""
    lens, add = [0, 100, 31, 5], [50000, 0, 20000, 1]
    tables = np.full((4, 1600), -1)
    tables[1, :4], tables[2, 0], tables[3, 0] = [0, 1, 2, 3], 4, 5
    for cols, rows in ((1600, 70001), (1000, 70001), (1600, 0), (1600, 60000)):
        case = (lens, add, tables[:, :cols].copy(), np.arange(6, 2500), 2300, 32, rows)
        got, want = run_plan(ctx, *case), R.plan(*case)
        for k in want:
            assert np.array_equal(got[k], want[k]), (k, cols, rows)


def test_plan_steps_in_place(ctx):
    """Lengths and the free count written over themselves, step after step: no page has two owners,
    and pages of ended sequences come back."""
    from spindle_amd import ops
    from spindle_amd._lib import check, lib
    from spindle_amd.ops import _p
    rng = np.random.default_rng(7)
    n, page, cols, pages, rows = 9, 16, 12, 60, 400
    lens, tables, free, n_free = ints([0] * n), torch.full((n, cols), -1, dtype=torch.int32, device="cuda"), ints(np.arange(pages)), ints([pages])
    q_start, slots, pos, status = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (n + 1, rows, rows, n))
    h = [np.zeros(n, int), np.full((n, cols), -1), np.arange(pages), pages]
    for step in range(40):
        add = ints(np.where(rng.random(n) < 0.1, -1, rng.integers(0, 40, n) * (rng.random(n) < 0.5)))
        torch.cuda.synchronize()
        check(lib.spx_pages_plan(ctx.h, n, page, cols, pages, rows, _p(lens), _p(add), _p(n_free), _p(tables), _p(free), _p(lens), _p(n_free),
                                 _p(q_start), _p(slots), _p(pos), _p(status)))
        ctx.sync()
        w = R.plan(h[0], add.cpu().numpy(), h[1], h[2], h[3], page, rows)
        h = [w["lens"], w["tables"], w["free"], int(w["n_free"][0])]
        assert np.array_equal(lens.cpu(), h[0]) and np.array_equal(tables.cpu(), h[1]) and int(n_free) == h[3] and np.array_equal(slots.cpu(), w["slots"])
        held = [int(p) for s in range(n) for p in h[1][s, :-(-h[0][s] // page)]]
        assert sorted(held + [int(p) for p in h[2][:h[3]]]) == list(range(pages))
    assert isinstance(ops.PagesPlan(), ops.PagesPlan)


# ---------------------------------------------------------------------------------- attention
class Batch:
    """A pool with sequences in it: `lens` tokens each, pages in any order, every other slot of the
    pool filled with something else."""

    def __init__(self, ctx, lens, kv, hd, page, seed=0, spread=1.0, extra_cols=0):
        from spindle_amd import ops
        self.ctx, self.kv, self.hd, self.page = ctx, kv, hd, page
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + 2
        ids = rng.permutation(self.pages)
        self.tables = np.full((len(lens), max(max(need), 1) + extra_cols), -1)
        at = 0
        for s, b in enumerate(need):
            self.tables[s, :b] = ids[at:at + b]
            at += b
        self.lens = list(lens)
        self.shape = ops.Kv4Shape(kv, hd, page, self.pages)
        self.pool = self.shape.pool()
        total = self.pages * page
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        k, v = (torch.randn(total, kv, hd, generator=g, device="cuda") * spread for _ in range(2))
        ops.kv4_append(ctx, self.shape, self.pool, k, v, ints(np.arange(total)))
        self.refresh()

    def refresh(self):
        from spindle_amd import ops
        k, v = ops.kv4_read(self.ctx, self.shape, self.pool, ints(np.arange(self.pages * self.page)))
        self.k, self.v = f64(k), f64(v)

    def slots(self, s, n=None):
        t = np.arange(self.lens[s] if n is None else n)
        return self.tables[s, t // self.page] * self.page + t % self.page

    def put(self, s, t, k=None, v=None):
        """Other keys / values (float32 arrays [kv, hd]) for token t of sequence s."""
        from spindle_amd import ops
        slot = int(self.slots(s, t + 1)[t])
        row = [torch.from_numpy(np.asarray(x, np.float32)).cuda()[None] for x in (self.k[slot] if k is None else k, self.v[slot] if v is None else v)]
        ops.kv4_append(self.ctx, self.shape, self.pool, row[0], row[1], ints([slot]))
        self.refresh()

    def check(self, q, counts, dtype, window=0, scale=None, out=None, lens=None, **kw):
        """Runs the operator on q [rows, heads, hd] and holds every row to its bound."""
        from spindle_amd import ops
        lens = self.lens if lens is None else lens
        start = np.concatenate([[0], np.cumsum(counts)])
        got = ops.kv4_attention(self.ctx, self.shape, self.pool, q, ints(start), ints(lens), ints(self.tables), scale=scale or 0.0, window=window, out=out, **kw)
        g, qd, sc = f64(got), f64(q), scale or 1.0 / np.sqrt(self.hd)
        parts = {F32: (2, 2), F16: (1, 2), BF16: (1, 1)}[dtype]
        half = torch.finfo(dtype).eps / 2
        worst = 0.0
        for s, c in enumerate(counts):
            n = min(max(lens[s], 0), self.tables.shape[1] * self.page)
            at = self.slots(s, n)
            k, v = self.k[at], self.v[at]
            for i in range(c):
                want, tol = R.attention(qd[start[s] + i], k, v, n - c + i, window, sc, *parts)
                tol = tol + half * (np.abs(want) + tol) + (2.0 ** -25 if dtype == F16 else 0.0)
                err = np.abs(g[start[s] + i] - want)
                assert np.isfinite(g[start[s] + i]).all() and (err <= tol).all(), (s, i, float((err / tol).max()))
                worst = max(worst, float((err / tol).max()))
        return got, worst


def queries(seed, rows, heads, hd, dtype, spread=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 99)
    return (torch.randn(rows, heads, hd, generator=g, device="cuda") * spread).to(dtype)


HEADS = [(4, 4, 64), (9, 3, 64), (16, 1, 64), (8, 2, 128), (16, 2, 128), (5, 1, 128), (34, 2, 128)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,hd", HEADS)
def test_attention_one_token(ctx, dtype, heads, kv, hd):
    """A new token a sequence: lengths around the tiles' and pages' ends, an empty sequence among them."""
    lens = [1, 2, 15, 16, 17, 31, 0, 32, 33, 64, 65, 100, 257]
    counts = [1 if n else 0 for n in lens]
    for page in (16, 64):
        b = Batch(ctx, lens, kv, hd, page, seed=heads + page)
        b.check(queries(heads, sum(counts), heads, hd, dtype), counts, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,hd", [(9, 3, 64), (16, 2, 128)])
@pytest.mark.parametrize("window", [0, 1, 30])
def test_attention_verify_rows(ctx, dtype, heads, kv, hd, window):
    """Two to seventeen rows a sequence, whole sequences that are new among them, none for some."""
    lens, counts = [70, 17, 5, 200, 33, 9], [9, 17, 5, 2, 0, 3]
    b = Batch(ctx, lens, kv, hd, 32, seed=window)
    b.check(queries(window, sum(counts), heads, hd, dtype), counts, dtype, window=window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,hd,page", [(3, 3, 64, 16), (16, 2, 64, 64), (8, 1, 128, 16), (6, 2, 128, 128)])
@pytest.mark.parametrize("window", [0, 45])
def test_attention_prompts(ctx, dtype, heads, kv, hd, page, window):
    """Prompt chunks, from the start and behind earlier ones, next to sequences with one row."""
    lens, counts = [150, 300, 77, 129, 1], [150, 130, 1, 64, 1]
    b = Batch(ctx, lens, kv, hd, page, seed=page)
    b.check(queries(page, sum(counts), heads, hd, dtype), counts, dtype, window=window)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_long(ctx, dtype):
    """A few long sequences, whose tokens are split among workgroups."""
    lens = [9001, 4096, 511]
    b = Batch(ctx, lens, 2, 128, 64, seed=3)
    b.check(queries(3, 3, 16, 128, dtype), [1, 1, 1], dtype)
    b.check(queries(4, 11, 16, 128, dtype), [5, 1, 5], dtype, window=3000)
    b.check(queries(5, 1, 16, 128, dtype), [1, 0, 0], dtype, max_kv=32)  # an untrue max_kv
    b = Batch(ctx, [7001], 1, 64, 16, seed=4)
    b.check(queries(6, 1, 3, 64, dtype), [1], dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q_spread,kv_spread", [(1e-6, 1.0), (30.0, 1.0), (1.0, 1e-3), (1.0, 300.0), (0.01, 2000.0)])
def test_attention_scales(ctx, dtype, q_spread, kv_spread):
    """Small and large queries, keys and values: sharp and flat rows."""
    b = Batch(ctx, [200, 61], 2, 128, 32, seed=5, spread=kv_spread)
    b.check(queries(7, 5, 4, 128, dtype, q_spread), [4, 1], dtype)
    b.check(queries(8, 5, 4, 128, dtype, q_spread), [4, 1], dtype, scale=0.02)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_one_token_outweighs_the_rest(ctx, dtype, rows):
    """A token that takes nearly all of the weight, thousands of others with some 2^-24 of its: what they
    have together is kept (their probabilities lie among f16's subnormals)."""
    n, hd = 6000, 128
    b = Batch(ctx, [n], 1, hd, 64, seed=30, spread=0.05)
    u = np.zeros(hd)
    u[::2], u[1::2] = 1.0, -1.0
    for at, far in ((0, 17.0), (n - rows - 1, 16.0)):  # exp(-17) = 2^-24.5
        b = Batch(ctx, [n], 1, hd, 64, seed=31, spread=0.05)
        b.put(0, at, k=(u * far / np.sqrt(hd))[None], v=np.full((1, hd), 0.5))
        q = torch.from_numpy(np.tile(u, (rows, 2, 1))).to(dtype).cuda()
        b.check(q, [rows], dtype)


def test_attention_window_past_everything(ctx):
    """The largest window there is sees what no window sees, rows before position 0 among them."""
    b = Batch(ctx, [300, 40], 2, 64, 16, seed=32)
    for counts in ([3, 1], [100, 45]):
        q = queries(32, sum(counts), 4, 64, F32)
        want, _ = b.check(q, counts, F32)
        for window in (2 ** 31 - 1, 2 ** 30 + 1, 2 ** 30, 301):
            got, _ = b.check(q, counts, F32, window=window)
            assert np.allclose(f64(got), f64(want), rtol=0, atol=1e-5)


def test_attention_captured_prompt(ctx):
    """A prompt's call captured, in its first use of the type, and replayed over other lengths, tables
    and queries, with eager calls and waits between."""
    from spindle_amd import ops
    with torch.cuda.stream(ctx.torch_stream()):
        for dtype in (F32, F16, BF16):
            b = Batch(ctx, [400, 90], 2, 128, 16, seed=33)
            q, start, lens, tables = queries(33, 130, 8, 128, dtype), ints([0, 120, 123]), ints([400, 90]), ints(b.tables)
            out = torch.full_like(q, 7.0)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=ctx.torch_stream()):
                ops.kv4_attention(ctx, b.shape, b.pool, q, start, lens, tables, out=out)
            for i, (s, n) in enumerate([([0, 120, 123], [400, 90]), ([0, 1, 130], [300, 80]), ([0, 0, 50], [5, 90]), ([0, 130, 130], [255, 1])]):
                start.copy_(ints(s)), lens.copy_(ints(n)), q.copy_(queries(40 + i, 130, 8, 128, dtype)), out.fill_(7.0)
                want = torch.full_like(q, 7.0)
                ops.kv4_attention(ctx, b.shape, b.pool, q, start, lens, tables, out=want)
                g.replay()
                if i % 2:
                    torch.cuda.synchronize()
                assert torch.equal(out, want) and (out[s[2]:] == 7.0).all()


@pytest.mark.parametrize("start,n", [([0, 130], 700), ([0, 1], 333), ([4, 9], 9), ([0, 0], 50), ([100, 130], 64), ([0, 130], 100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_one_sequence_room_to_spare(ctx, dtype, start, n):
    """One sequence in a call with room for a prompt: a whole one, a row, some in the middle, none."""
    from spindle_amd import ops
    b = Batch(ctx, [n], 2, 64, 16, seed=34)
    q = queries(34, 130, 8, 64, dtype)
    out = torch.full_like(q, 7.0)
    ops.kv4_attention(ctx, b.shape, b.pool, q, ints(start), ints([n]), ints(b.tables), out=out)
    lo, hi = start
    assert (out[:lo] == 7.0).all() and (out[hi:] == 7.0).all()
    at, half, parts = b.slots(0), torch.finfo(dtype).eps / 2, (2, 2) if dtype == F32 else (1, 1)
    got, qd = f64(out), f64(q)
    for i in range(lo, hi):
        want, tol = R.attention(qd[i], b.k[at], b.v[at], n - (hi - i), 0, 64 ** -0.5, *parts)
        assert (np.abs(got[i] - want) <= tol + half * (np.abs(want) + tol)).all(), i


def test_attention_many_sequences(ctx):
    rng = np.random.default_rng(6)
    lens = [int(v) for v in rng.integers(1, 60, 300)]
    b = Batch(ctx, lens, 1, 64, 16, seed=6)
    b.check(queries(6, 300, 2, 64, F16), [1] * 300, F16)
    counts = [int(v) for v in rng.integers(0, 3, 300)]  # more rows than sequences, some of them idle
    b.check(queries(7, sum(counts), 2, 64, F16), counts, F16)
    lens = [int(v) for v in rng.integers(1, 20, 4096)]
    b = Batch(ctx, lens, 1, 64, 16, seed=7)
    b.check(queries(8, 4096, 1, 64, BF16), [1] * 4096, BF16)


def test_attention_rows_it_leaves(ctx):
    """Rows behind the last sequence and the space between rows stay; q and out are views."""
    b = Batch(ctx, [40, 3], 2, 64, 16, seed=8)
    q = torch.full((9, 2, 4, 64), 5.0, device="cuda")
    q[:, 0] = queries(8, 9, 4, 64, F32)
    out = torch.full((9, 3, 4, 64), -7.0, device="cuda")
    got, _ = b.check(q[:, 0], [3, 1], F32, out=out[:, 1])
    assert got.data_ptr() == out[:, 1].data_ptr()
    assert (out[4:] == -7.0).all() and (out[:, 0] == -7.0).all() and (out[:, 2] == -7.0).all() and not (out[:4, 1] == -7.0).any()


def test_attention_alignment(ctx):
    """Queries and outputs at addresses that are multiples of their elements' size and no more."""
    b = Batch(ctx, [40, 33, 150], 2, 64, 16, seed=9)
    for dtype in (F32, F16, BF16):
        for counts in ([1, 2, 1], [3, 1, 100]):
            n = sum(counts)
            flat, oflat = torch.zeros(n * 257 + 1, dtype=dtype, device="cuda"), torch.zeros(n * 259 + 3, dtype=dtype, device="cuda")
            q = torch.as_strided(flat, (n, 4, 64), (257, 64, 1), 1)
            q.copy_(queries(9, n, 4, 64, dtype))
            b.check(q, counts, dtype, out=torch.as_strided(oflat, (n, 4, 64), (259, 64, 1), 3))


@pytest.mark.parametrize("counts", [[3, 1], [40, 2]])
def test_attention_nothing_to_see(ctx, counts):
    """More new rows than tokens: the first rows sit before position 0 and get zeros; so does a row
    whose pages are all outside the pool."""
    from spindle_amd import ops
    b = Batch(ctx, [50, 20], 2, 64, 16, seed=10)
    q = queries(10, sum(counts), 4, 64, F32)
    out = torch.full((sum(counts), 4, 64), -7.0, device="cuda")
    b.check(q, counts, F32, lens=[2, 20], out=out)
    # (a row that sees one token is that token's value, whose channels may be 0)
    assert (out[:counts[0] - 2] == 0).all() and out[counts[0] - 2:].ne(0).any(-1).all()
    for bad in (-1, b.pages, 2 ** 31 - 1, -2 ** 31):
        t = b.tables.copy()
        t[0, :] = bad
        got = ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, counts[0], sum(counts)]), ints([50, 20]), ints(t))
        assert (got[:counts[0]] == 0).all() and got[counts[0]:].ne(0).any(-1).all()


@pytest.mark.parametrize("counts", [[2, 1], [60, 1]])
def test_attention_page_outside_the_pool(ctx, counts):
    """The tokens of such a page are unseen: the row is the one over the others."""
    from spindle_amd import ops
    b = Batch(ctx, [100, 20], 1, 128, 32, seed=11)
    q = queries(11, sum(counts), 2, 128, F32)
    t = b.tables.copy()
    t[0, 1] = b.pages + 3
    got = f64(ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, counts[0], sum(counts)]), ints([100, 20]), ints(t)))
    at = b.slots(0)
    for i in range(counts[0]):
        pos = 100 - counts[0] + i
        keep = np.array([p for p in range(pos + 1) if not 32 <= p < 64])
        want, tol = R.attention(f64(q)[i], b.k[at][keep], b.v[at][keep], len(keep) - 1, 0, 128 ** -0.5, 2, 2)
        assert (np.abs(got[i] - want) <= tol + 2.0 ** -24 * np.abs(want)).all(), i


def test_attention_lengths_cut(ctx):
    """Lengths behind the table's end and below zero, starts behind the rows."""
    from spindle_amd import ops
    b = Batch(ctx, [64, 20], 1, 64, 16, seed=12)
    q = queries(12, 2, 2, 64, F32)
    got = ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, 1, 2]), ints([2 ** 31 - 1, -5]), ints(b.tables))
    ref = ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, 1, 2]), ints([64, 0]), ints(b.tables))
    assert torch.equal(got, ref) and (got[1] == 0).all() and got[0].ne(0).any(-1).all()
    got = ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, 1, 2 ** 31 - 1]), ints([64, 20]), ints(b.tables))
    ref = ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, 1, 2]), ints([64, 20]), ints(b.tables))
    assert torch.equal(got, ref)
    for start in ([0, -4, 2], [2, 1, 0], [-2 ** 31, 2 ** 31 - 1, 0], [2, 2, 2]):
        ops.kv4_attention(ctx, b.shape, b.pool, q, ints(start), ints([64, 20]), ints(b.tables))
    ctx.sync()


@pytest.mark.parametrize("counts", [[1], [9], [90]])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_nan_in_masked_places(ctx, dtype, counts, hd):
    """NaN keys and values of tokens that a row does not see (behind the end, before the window, or
    newer than the row) do not reach it; a row that sees one has it."""
    from spindle_amd import ops
    n, window = 120, 50
    b = Batch(ctx, [n], 2, hd, 16, seed=13)
    c, nan = counts[0], np.full((2, hd), np.nan)
    t = np.arange(b.tables.shape[1] * 16)
    behind = (b.tables[0, t // 16] * 16 + t % 16)[n:]
    rest = np.setdiff1d(np.arange(b.pages * 16), b.slots(0))
    assert set(behind) <= set(rest)
    x = torch.full((len(rest), 2, hd), float("nan"), device="cuda")
    ops.kv4_append(ctx, b.shape, b.pool, x, x, ints(rest))
    b.refresh()
    q = queries(13, c, 4, hd, dtype)
    b.check(q, counts, dtype)
    for p in range(0, n - c - window + 1, 7):
        b.put(0, p, nan, nan)
    b.check(q, counts, dtype, window=window)
    # the last token's value and key, one after the other: the last row alone sees them
    for what in ("v", "k"):
        b2 = Batch(ctx, [n], 2, hd, 16, seed=13)
        one = b2.v[b2.slots(0)[n - 1]].copy()
        one[1, 40] = np.inf
        b2.put(0, n - 1, **{what: one})
        got = f64(ops.kv4_attention(ctx, b2.shape, b2.pool, q, ints([0, c]), ints([n]), ints(b2.tables)))
        assert np.isfinite(got[:-1]).all()
        assert np.isfinite(got[-1, :2]).all()  # the other key head's
        assert np.isnan(got[-1, 2:, 32:64]).all()
        assert np.isnan(got[-1, 2:]).all() if what == "k" else np.isfinite(np.delete(got[-1, 2:], np.s_[32:64], 1)).all()
        if c > 1:
            ref = f64(ops.kv4_attention(ctx, b2.shape, b2.pool, q[:-1].contiguous(), ints([0, c - 1]), ints([n - 1]), ints(b2.tables)))
            assert np.allclose(got[:-1], ref, rtol=0, atol=4 * torch.finfo(dtype).eps * np.abs(ref).max())


def test_attention_nan_query(ctx):
    """A NaN or an infinity in one query head stays in that head."""
    from spindle_amd import ops
    b = Batch(ctx, [90], 2, 128, 16, seed=14)
    for rows in (2, 40):
        q = queries(14, rows, 4, 128, F32)
        q[1, 2, 7], q[0, 1, 100] = float("nan"), float("inf")
        got = ops.kv4_attention(ctx, b.shape, b.pool, q, ints([0, rows]), ints([90]), ints(b.tables))
        assert got[1, 2].isnan().all() and got[0, 1].isnan().all()
        got[1, 2], got[0, 1] = 0, 0
        assert got.isfinite().all()


def test_attention_past_4_gib(ctx):
    """Pages whose bytes lie past 32-bit offsets."""
    from spindle_amd import ops
    shape = ops.Kv4Shape(8, 128, 256, 15200)
    assert shape.nbytes > 1.04 * 2 ** 32
    pool = torch.empty(shape.nbytes, dtype=torch.uint8, device="cuda")
    table = [15199, 3, 15100, 14600]
    n = 3 * 256 + 40
    slots = np.array([table[t // 256] * 256 + t % 256 for t in range(n)])
    g = torch.Generator(device="cuda")
    g.manual_seed(15)
    k, v = (torch.randn(n, 8, 128, generator=g, device="cuda") for _ in range(2))
    ops.kv4_append(ctx, shape, pool, k, v, ints(slots))
    kk, vv = (f64(x) for x in ops.kv4_read(ctx, shape, pool, ints(slots)))
    assert np.array_equal(kk[-1], R.values(f64(k[-1]))) and np.array_equal(vv[0], R.values(f64(v[0])))
    for c in (1, 30):
        q = queries(15, c, 8, 128, F32)
        got = f64(ops.kv4_attention(ctx, shape, pool, q, ints([0, c]), ints([n]), ints([table])))
        for i in (0, c - 1):
            want, tol = R.attention(f64(q)[i], kk, vv, n - c + i, 0, 128 ** -0.5, 2, 2)
            assert (np.abs(got[i] - want) <= tol + 2.0 ** -24 * np.abs(want)).all()


def test_attention_repeats_bit_for_bit(ctx):
    b = Batch(ctx, [3000, 100, 700], 2, 128, 32, seed=16)
    for counts in ([1, 1, 1], [9, 2, 120]):
        q = queries(16, sum(counts), 16, 128, F32)
        a = [b.check(q, counts, F32)[0].clone() for _ in range(2)] if sum(counts) < 20 else [b.check(q, counts, F32)[0], b.check(q, counts, F32)[0]]
        assert torch.equal(a[0], a[1])


# ------------------------------------------------------------------------------ log probabilities
def check_logprobs(ctx, x, targets, top, scale=1.0, **kw):
    """Bounds: x - m and its exponential round at 2^-24 and 2^-23 of themselves, the argument of the
    exponential (times log2 e) at 2^-23 of |x - m|, sums of n terms at most n / 512 + 32 times."""
    from spindle_amd import ops
    r = ops.logprobs(ctx, x, ints(targets) if targets is not None else None, top=top, logit_scale=scale, **kw)
    x32 = x.float().cpu().numpy()
    xs = (x32 / np.float32(scale)).astype(np.float64) if scale != 1.0 else x32.astype(np.float64)
    logp, ent, ids, best = R.logprobs(xs, targets, top)
    n = x.shape[1]
    with np.errstate(invalid="ignore"):
        span = np.nan_to_num(np.where(np.isfinite(xs), xs.max(1, keepdims=True) - xs, 0.0).max(1), nan=0.0, posinf=0.0)
    tol = (n / 512 + 32 + 4 * np.minimum(span, 100)) * 2.0 ** -24

    def near(got, want, extra):
        got, want = f64(got), np.asarray(want)
        same = (np.isnan(got) & np.isnan(want)) | (got == want)
        with np.errstate(invalid="ignore"):
            return (same | (np.abs(got - want) <= extra + 2.0 ** -22 * np.abs(want))).all()

    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    assert near(r.top_logp, best, tol[:, None])
    assert near(r.entropy, ent, tol * (2 + np.log(n)))
    if targets is not None:
        assert near(r.logp, logp, tol)
    else:
        assert r.logp is None
    return r


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (1, 1000), (5, 4097), (2, 49155), (1, 151936), (40, 5003), (300, 777)])
def test_logprobs(ctx, dtype, rows, vocab):
    rng = np.random.default_rng(rows + vocab)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)) * 3).to(dtype).cuda()  # 16 bits: many equal logits
    for top in (0, 1, 5, 32):
        check_logprobs(ctx, x, rng.integers(0, vocab, rows), top)
    check_logprobs(ctx, x, None, 3, scale=2.5)


def test_logprobs_edges(ctx):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((12, 3001)) * 2).astype(np.float32)
    x[0, ::2] = -np.inf
    x[1] = -np.inf
    x[2, 77] = np.nan
    x[3, 3000] = np.inf
    x[4] = 1.25                     # all equal
    x[5, 100] = 1e4                 # certain
    x[6] *= 1e30                    # logits past any exponential's range
    x[7, 5:] = -np.inf              # five alternatives
    x[8] = np.finfo(np.float32).min
    x[8, 9] = 0.0                   # the type's lowest value as a mask
    x[9] = -1e-3
    x[9, 40], x[9, 20] = 0.0, -0.0  # equal alternatives
    x[10, :] = np.linspace(-5, 5, 3001)   # ascending: every value a new largest
    x[11, :] = np.linspace(5, -5, 3001)
    t = rng.integers(0, 3001, 12)
    t[[0, 5, 7, 9]] = 2, 100, 2999, 40
    for top in (1, 8, 32):
        check_logprobs(ctx, torch.from_numpy(x).cuda(), t, top)
    for bad in (-1, 3001, 2 ** 31 - 1, -2 ** 31):
        r = check_logprobs(ctx, torch.from_numpy(x).cuda(), np.full(12, bad), 2)
        assert r.logp.isnan().all()


def test_logprobs_rows_apart(ctx):
    """Rows further apart than their width, at odd addresses; what lies between them is not read."""
    rng = np.random.default_rng(5)
    for dtype in (F32, F16, BF16):
        x = torch.from_numpy(rng.standard_normal((4, 5001))).to(dtype).cuda()
        flat = torch.full((4 * 5011 + 8,), float("nan"), dtype=dtype, device="cuda")
        for off in (1, 3, 6):
            v = torch.as_strided(flat, (4, 5001), (5011, 1), off)
            v.copy_(x)
            check_logprobs(ctx, v, [0, 5000, 17, 3], 4)
            flat.fill_(float("nan"))


def test_logprobs_agree_with_the_sampler(ctx):
    """The greedy sampler's pick is the first alternative where one logit is the largest."""
    from spindle_amd import ops
    x = torch.randn(151936, device="cuda")
    s = ops.Sampler(ctx, 151936, temperature=0.0, repeat_penalty=1.0)
    assert s.sample(x) == int(ops.logprobs(ctx, x[None], top=1).top_ids)
    s.close()


# ------------------------------------------------------------------------------------ together
class Step:
    """A decode step of one attention layer and the head, as a host drives it: plan, append, attend,
    the head's matrix (spx_matvec), the report; everything in buffers that live as long as it does."""

    def __init__(self, ctx, seqs=6, heads=4, kv=2, hd=64, page=16, pages=64, vocab=1000):
        from spindle_amd import model as M
        from spindle_amd import ops
        self.ctx, self.n, self.heads, self.kv, self.hd, self.page, self.vocab = ctx, seqs, heads, kv, hd, page, vocab
        self.shape = ops.Kv4Shape(kv, hd, page, pages)
        self.pool = self.shape.pool()
        self.tables = torch.full((seqs, 12), -1, dtype=torch.int32, device="cuda")
        self.free, self.n_free, self.lens = ints(np.arange(pages)), ints([pages]), ints([0] * seqs)
        self.w = ops.Tensor(ctx, M.F32, heads * hd, vocab, M.synth_tensor(M.TensorSpec("w", M.F32, heads * hd, vocab, kind=1), 3))
        self.rows = 16
        self.q, self.k, self.v = (torch.zeros(self.rows, h, hd, device="cuda") for h in (heads, kv, kv))
        self.add, self.targets = ints([0] * seqs), ints([0] * self.rows)
        self.out, self.logits = torch.zeros(self.rows, heads, hd, device="cuda"), torch.zeros(self.rows, vocab, device="cuda")

    def step(self):
        from spindle_amd import ops
        from spindle_amd._lib import check, lib
        p = ops.pages_plan(self.ctx, self.lens, self.add, self.tables, self.free, self.n_free, self.page, self.rows)
        ops.kv4_append(self.ctx, self.shape, self.pool, self.k, self.v, p.slots)
        ops.kv4_attention(self.ctx, self.shape, self.pool, self.q, p.q_start, p.lens, self.tables, out=self.out)
        x = self.out.view(self.rows, -1)
        check(lib.spx_matvec(self.ctx.h, self.w.h, 0, ops._p(x), x.shape[1], self.rows, ops._p(self.logits), self.vocab))
        r = ops.logprobs(self.ctx, self.logits, self.targets, top=4)
        self.lens.copy_(p.lens)
        self.n_free.copy_(p.n_free)
        return p, r


def inputs(rng, s):
    add = np.array([[7, 1, 0, 3, 1, 4], [1, 1, 1, 1, 1, 1], [-1, 1, 1, 2, 1, 1], [9, 1, 1, 1, 1, 1]][rng.integers(4)])
    f = lambda h: torch.from_numpy(rng.standard_normal((s.rows, h, s.hd)).astype(np.float32)).cuda()  # noqa: E731
    return add, f(s.heads), f(s.kv), f(s.kv), rng.integers(0, s.vocab, s.rows)


def fill(s, add, q, k, v, t):
    s.add.copy_(ints(add)), s.q.copy_(q), s.k.copy_(k), s.v.copy_(v), s.targets.copy_(ints(t))


def test_steps_of_a_batch(ctx):
    """Steps of a batch, sequences ending and starting among them, against the same in 64 bits."""
    rng = np.random.default_rng(20)
    with torch.cuda.stream(ctx.torch_stream()):
        s = Step(ctx)
        keys = [[] for _ in range(s.n)]
        w = f64(torch.from_numpy(s.w.download().view(np.float32).reshape(s.vocab, -1)))
        for _ in range(12):
            add, q, k, v, t = inputs(rng, s)
            fill(s, add, q, k, v, t)
            p, r = s.step()
            torch.cuda.current_stream().synchronize()
            at = 0
            assert not p.status.any()
            got, lp = f64(s.out), f64(r.logp)
            for i, a in enumerate(add):
                if a < 0:
                    keys[i] = []
                for j in range(max(a, 0)):
                    keys[i].append((R.values(f64(k[at + j])), R.values(f64(v[at + j]))))
                kk, vv = (np.array([x[z] for x in keys[i]]).reshape(-1, s.kv, s.hd) for z in (0, 1))
                for j in range(max(a, 0)):
                    want, tol = R.attention(f64(q[at + j]), kk, vv, len(kk) - a + j, 0, s.hd ** -0.5, 2, 2)
                    assert (np.abs(got[at + j] - want) <= tol + 2.0 ** -24 * np.abs(want)).all()
                    x = got[at + j].reshape(-1) @ w.T  # the head's matrix has its own tests: 1e-5 of the logits' size covers its sums
                    ref = R.logprobs(x[None], t[at + j:at + j + 1], 0)[0][0]
                    assert abs(lp[at + j] - ref) <= 1e-5 * max(1.0, np.abs(x).max())
                at += max(a, 0)
        s.w.close()


def test_steps_captured_and_replayed(ctx):
    """The step captured into a graph and replayed, eager work and waits between the replays: every
    replay gives the eager step's bits."""
    from spindle_amd import ops
    rng = np.random.default_rng(21)
    with torch.cuda.stream(ctx.torch_stream()):
        a, b = Step(ctx), Step(ctx)
        x = inputs(rng, a)
        for s in (a, b):  # a first step each, eager (workspaces of the matrix product)
            fill(s, *x)
            s.step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=ctx.torch_stream()):
            pb, rb = b.step()
        for i in range(6):
            x = inputs(rng, a)
            fill(a, *x), fill(b, *x)
            pa, ra = a.step()
            g.replay()
            if i % 2:
                torch.cuda.synchronize()
            for u, v in ((a.out, b.out), (a.lens, b.lens), (a.tables, b.tables), (a.free, b.free), (a.pool, b.pool), (pa.slots, pb.slots),
                         (ra.logp, rb.logp), (ra.entropy, rb.entropy), (ra.top_ids, rb.top_ids), (ra.top_logp, rb.top_logp)):
                assert torch.equal(u, v)
            ops.logprobs(ctx, a.logits, top=7)  # eager work of other sizes between
            torch.zeros(1 << 20, device="cuda").sum()
        for s in (a, b):
            s.w.close()


def test_two_streams_at_once(ctx):
    """Two contexts' calls with nothing between them, and torch's own stream as the source: calls are
    ordered after what torch's stream holds, and do not share scratch."""
    from spindle_amd import ops
    other = ops.Context(0)
    b = Batch(ctx, [5000, 4000], 2, 128, 64, seed=22)
    x = torch.randn(2, 151936, device="cuda")
    q = queries(22, 2, 16, 128, F32)
    args = (ints([0, 1, 2]), ints(b.lens), ints(b.tables))
    want = ops.kv4_attention(ctx, b.shape, b.pool, q, *args).clone()
    lp = ops.logprobs(ctx, x, ints([1, 2]), top=9)
    torch.cuda.synchronize()
    for _ in range(5):
        y = torch.zeros_like(q)
        for _ in range(20):
            y += 0.05 * q  # (torch's stream is busy with q's copy)
        y.copy_(q)
        z = x + 0.0
        got = [ops.kv4_attention(c, b.shape, b.pool, y, *args) for c in (ctx, other, ctx, other)]
        rep = [ops.logprobs(c, z, ints([1, 2]), top=9) for c in (ctx, other, ctx, other)]
        y.zero_(), z.zero_()  # after the calls, on torch's stream
        for g, r in zip(got, rep):
            assert torch.equal(g, want) and torch.equal(r.logp, lp.logp) and torch.equal(r.top_ids, lp.top_ids) and torch.equal(r.entropy, lp.entropy)
    other.close()


def test_python_refusals(ctx):
    from spindle_amd import ops
    shape = ops.Kv4Shape(2, 64, 16, 2)
    pool, k, q = shape.pool(), torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 4, 64, device="cuda")
    s3 = ints([0, 1, 2])
    att = dict(q=q, q_start=ints([0, 3]), kv_lens=ints([3]), tables=ints([[0, 1]]))
    bad = [lambda: ops.kv4_append(ctx, shape, pool[:-1], k, k, s3), lambda: ops.kv4_append(ctx, shape, pool, k.double(), k.double(), s3),
           lambda: ops.kv4_append(ctx, shape, pool, k, k.half(), s3), lambda: ops.kv4_append(ctx, shape, pool, k[:2], k, s3),
           lambda: ops.kv4_append(ctx, shape, pool, k.transpose(0, 1), k, s3), lambda: ops.kv4_append(ctx, shape, pool, k, k, s3.long()),
           lambda: ops.kv4_append(ctx, shape, pool, k.cpu(), k, s3), lambda: ops.kv4_read(ctx, shape, pool, s3, torch.int32),
           lambda: ops.kv4_attention(ctx, shape, pool, **(att | dict(q=q[:, :, :32]))), lambda: ops.kv4_attention(ctx, shape, pool, **(att | dict(kv_lens=s3))),
           lambda: ops.kv4_attention(ctx, shape, pool, **att, out=q.half()), lambda: ops.kv4_attention(ctx, shape, pool, **(att | dict(tables=ints([0, 1])))),
           lambda: ops.logprobs(ctx, q), lambda: ops.logprobs(ctx, q[0].t()), lambda: ops.logprobs(ctx, q[0], s3),
           lambda: ops.pages_plan(ctx, ints([1]), s3, ints([[0]]), ints([1]), ints([1]), 16, 1)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print(i)
    with pytest.raises(ops.SpxError if hasattr(ops, "SpxError") else RuntimeError, match="n_heads"):
        ops.kv4_attention(ctx, shape, pool, **(att | dict(q=torch.zeros(3, 3, 64, device="cuda"))))
