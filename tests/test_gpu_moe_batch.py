"""The router, the sort by expert and rows joined again (include/spx.h: spx_moe_route, spx_moe_route_grad,
spx_moe_sort, spx_moe_gather, spx_moe_combine, spx_moe_combine_grad) against 64-bit evaluations of their
definitions (moe_ref.py)."""
import numpy as np
import pytest

import moe_ref as R

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


def close(got, want, tol, what=""):
    got = f64(got) if isinstance(got, torch.Tensor) else got
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    with np.errstate(invalid="ignore"):
        off = np.where(np.isnan(want) | (got == want), 0.0, np.abs(got - want) - tol)
    assert (off <= 0).all(), (what, float(np.nanmax(off)))


# ------------------------------------------------------------------------------------ the router
def logits_for(rng, rows, n, dtype):
    x = rng.standard_normal((rows, n)) * 2
    for r in range(rows):
        kind = r % 9
        if kind == 1:
            x[r] = np.round(x[r])  # many equal ones
        elif kind == 2:
            x[r, rng.random(n) < 0.9] = -np.inf
        elif kind == 3:
            x[r] = -np.inf
        elif kind == 4:
            x[r, rng.integers(n)] = np.nan
        elif kind == 5:
            x[r, rng.integers(n)] = np.inf
        elif kind == 6:
            x[r] = rng.choice([0.0, -0.0], n)  # equal, whatever their signs
        elif kind == 7:
            x[r] *= 30
    x[-1, -1] = 9.0
    return torch.from_numpy(x).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,k", [(1, 1), (2, 2), (32, 8), (63, 5), (64, 32), (65, 1), (128, 8), (200, 7), (300, 3), (1024, 32)])
@pytest.mark.parametrize("norm", [True, False])
def test_route(ctx, dtype, n, k, norm):
    from spindle_amd import ops
    rng = np.random.default_rng(n + k)
    x = logits_for(rng, 29, n, dtype)
    chosen, weights = ops.moe_route(ctx, x, k, norm=norm)
    want, w, tol = R.route(f64(x), k, norm)
    assert np.array_equal(chosen.cpu().numpy(), want)
    close(weights, w, tol)
    wide = torch.cat([torch.full_like(x, 99.0), x], 1)[:, n:]  # rows apart by more than their width
    c2, w2 = ops.moe_route(ctx, wide, k, norm=norm)
    assert torch.equal(c2, chosen) and torch.equal(w2.nan_to_num(7.0), weights.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,k", [(1, 1), (32, 8), (64, 2), (65, 9), (128, 8), (300, 32), (1024, 3)])
@pytest.mark.parametrize("norm", [True, False])
def test_route_grad(ctx, dtype, n, k, norm):
    from spindle_amd import ops
    rng = np.random.default_rng(n * 3 + k)
    x = logits_for(rng, 19, n, dtype)
    chosen, _ = ops.moe_route(ctx, x, k, norm=norm)
    g = torch.from_numpy(rng.standard_normal((19, k))).float().cuda()
    ids = chosen.clone()
    ids[10, k - 1] = -1  # rows with such ids are NaN
    ids[13, 0] = n
    d = ops.moe_route_grad(ctx, x, ids, g, norm=norm)
    assert d.dtype == dtype
    want, tol = R.route_grad(f64(x), ids.cpu().numpy(), f64(g), norm)
    close(d, want, tol + R.rounding(want, dtype))


@pytest.mark.parametrize("norm", [True, False])
def test_route_grad_by_differences(ctx, norm):
    """Against differences of a loss in 64 bits: ids held fixed, an id given twice counts twice."""
    from spindle_amd import ops
    rng = np.random.default_rng(3)
    rows, n, k = 5, 12, 4
    x = torch.from_numpy(rng.standard_normal((rows, n))).float().cuda()
    ids = np.stack([rng.permutation(n)[:k] for _ in range(rows)])
    ids[2, 1] = ids[2, 3]
    g = rng.standard_normal((rows, k)).astype(np.float32).astype(np.float64)

    def loss(v):
        e = np.exp(v)
        at = np.take_along_axis(e, ids, 1)
        return (g * at / (at.sum(1, keepdims=True) if norm else e.sum(1, keepdims=True))).sum()

    base, h = f64(x), 1e-5
    want = np.zeros_like(base)
    for i in np.ndindex(*base.shape):
        up, down = base.copy(), base.copy()
        up[i] += h
        down[i] -= h
        want[i] = (loss(up) - loss(down)) / (2 * h)
    d = ops.moe_route_grad(ctx, x, ints(ids), torch.from_numpy(g).float().cuda(), norm=norm)
    # a difference is off by h^2 times a third derivative (below 10 here) and by 64 bits' rounding over h; the call by some
    # forty roundings of values below 8
    close(d, want, 1e-9 + 1e-9 + 40 * 8 * R.U)


def test_route_no_rows(ctx):
    from spindle_amd import ops
    c, w = ops.moe_route(ctx, torch.zeros(0, 8, device="cuda"), 2)
    assert c.shape == (0, 2) and w.shape == (0, 2)
    assert ops.moe_route_grad(ctx, torch.zeros(0, 8, device="cuda"), c, w).shape == (0, 8)


# -------------------------------------------------------------------------------------- the sort
def ids_for(rng, rows, k, n, drop):
    ids = rng.integers(0, n, (rows, k))
    if rows > 2:
        ids[: rows // 2] = ids[0, 0]  # a crowded expert
        ids[rows // 2] = n - 1        # the same one k times
    if drop:
        ids[rng.random((rows, k)) < 0.3] = -1
        ids.flat[-1] = n
        ids.flat[0] = 2 ** 31 - 1
        if rows > 5:
            ids[3] = -2 ** 31
    return ids


@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 8, 128), (24, 8, 128), (24, 8, 1024), (65, 3, 7), (511, 8, 32), (513, 8, 128), (700, 6, 129),
                                      (2047, 5, 1000), (9000, 1, 2)])
@pytest.mark.parametrize("drop", [False, True])
def test_sort(ctx, rows, k, n, drop):
    from spindle_amd import ops
    rng = np.random.default_rng(rows + n)
    ids = ids_for(rng, rows, k, n, drop)
    o = ops.moe_sort(ctx, ints(ids), n)
    starts, order, place = R.sort(ids, n)
    assert np.array_equal(o.starts.cpu().numpy(), starts)
    assert np.array_equal(o.order.cpu().numpy(), order)
    assert np.array_equal(o.place.cpu().numpy(), place)


def test_sort_many(ctx):
    """Millions of entries, runs of several thousand a workgroup, against torch's stable sort."""
    from spindle_amd import ops
    rows, k, n = 262144, 9, 77
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    ids = torch.randint(0, n, (rows, k), generator=g, device="cuda", dtype=torch.int32)
    o = ops.moe_sort(ctx, ids, n)
    values, order = torch.sort(ids.flatten(), stable=True)
    assert torch.equal(o.order.long(), order)
    assert torch.equal(o.starts.long(), torch.searchsorted(values, torch.arange(n + 1, device="cuda", dtype=torch.int32)))
    assert torch.equal(o.place.flatten()[order].long(), torch.arange(rows * k, device="cuda"))


def test_sort_nothing(ctx):
    from spindle_amd import ops
    o = ops.moe_sort(ctx, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), 6)
    assert o.starts.tolist() == [0] * 7
    o = ops.moe_sort(ctx, torch.full((5, 2), -1, dtype=torch.int32, device="cuda"), 3)
    assert o.starts.tolist() == [0] * 4 and (o.order == -1).all() and (o.place == -1).all()


# ----------------------------------------------------------------------------- rows there and back
WIDTHS = [1, 3, 8, 31, 64, 100, 256, 1000, 2048, 2056]


def sorted_rows(rng, ctx, rows, k, n, drop):
    from spindle_amd import ops
    ids = ids_for(rng, rows, k, n, drop)
    return ops.moe_sort(ctx, ints(ids), n)


def strided(rng, rows, width, dtype, pad, off=0):
    base = torch.from_numpy(rng.standard_normal((rows, width + pad + off))).to(dtype).cuda()
    return base[:, off:off + width]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("drop,pad,off", [(False, 0, 0), (True, 8, 0), (True, 5, 1)])
def test_gather(ctx, dtype, width, drop, pad, off):
    from spindle_amd import ops
    rng = np.random.default_rng(width)
    rows, k = 23, 3
    o = sorted_rows(rng, ctx, rows, k, 9, drop)
    x = strided(rng, rows, width, dtype, pad, off)
    order = o.order.cpu().numpy()
    want = np.where(order[:, None] >= 0, f64(x)[np.maximum(order, 0) // k], 0.0)
    assert np.array_equal(f64(ops.moe_gather(ctx, x, o.order, k)), want)
    w = torch.from_numpy(rng.standard_normal((rows, k))).float().cuda()
    into = strided(rng, rows * k, width, dtype, pad, off)
    assert ops.moe_gather(ctx, x, o.order, k, weights=w, out=into) is into
    want = want * np.where(order >= 0, f64(w).reshape(-1)[np.maximum(order, 0)], 0.0)[:, None]
    close(into, want, np.abs(want) * R.U + R.rounding(want * (1 + R.U), dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("drop,pad,off", [(False, 0, 0), (True, 8, 0), (True, 5, 1)])
def test_combine(ctx, dtype, width, drop, pad, off):
    from spindle_amd import ops
    rng = np.random.default_rng(width + 1)
    rows, k = 21, 5
    o = sorted_rows(rng, ctx, rows, k, 9, drop)
    y = strided(rng, rows * k, width, dtype, pad, off)
    if drop:
        y[int(o.starts[-1]):] = float("nan")  # no entry names these
    place, v = o.place.cpu().numpy(), f64(y)
    each = np.where(place[..., None] >= 0, v[np.maximum(place, 0)], 0.0)
    for w in (None, torch.from_numpy(rng.standard_normal((rows, k))).float().cuda()):
        got = ops.moe_combine(ctx, y, o.place, w, out=strided(rng, rows, width, dtype, pad, off) if off else None)
        terms = each if w is None else each * f64(w)[..., None]
        want, tol = terms.sum(1), np.abs(terms).sum(1) * k * R.U
        close(got, want, tol + R.rounding(np.abs(want) + tol, dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("drop,pad,off", [(False, 0, 0), (True, 8, 0), (True, 5, 1)])
def test_combine_grad(ctx, dtype, width, drop, pad, off):
    from spindle_amd import ops
    rng = np.random.default_rng(width + 2)
    rows, k = 21, 5
    o = sorted_rows(rng, ctx, rows, k, 9, drop)
    y, d = strided(rng, rows * k, width, dtype, pad, off), strided(rng, rows, width, dtype, pad, off)
    w = torch.from_numpy(rng.standard_normal((rows, k))).float().cuda()
    d_y, d_w = ops.moe_combine_grad(ctx, d, y, o.order, o.place, w)
    place, order = o.place.cpu().numpy(), o.order.cpu().numpy()
    terms = np.where(place[..., None] >= 0, f64(y)[np.maximum(place, 0)], 0.0) * f64(d)[:, None]
    close(d_w, terms.sum(-1), np.abs(terms).sum(-1) * (width / 64 + 24) * R.U)
    e = np.maximum(order, 0)
    want = np.where(order[:, None] >= 0, f64(w).reshape(-1)[e][:, None] * f64(d)[e // k], 0.0)
    close(d_y, want, np.abs(want) * R.U + R.rounding(want * (1 + R.U), dtype))


def test_gather_gradient_is_combine(ctx):
    """<gather(x), y> = <x, combine(y)>, with weights and without: whole numbers, so without rounding."""
    from spindle_amd import ops
    rng = np.random.default_rng(8)
    rows, k, width = 40, 4, 72
    o = sorted_rows(rng, ctx, rows, k, 11, True)
    whole = lambda *s: torch.from_numpy(rng.integers(-8, 9, s)).float().cuda()  # noqa: E731
    x, y, w = whole(rows, width), whole(rows * k, width), whole(rows, k)
    for v in (None, w):
        there, back = ops.moe_gather(ctx, x, o.order, k, weights=v), ops.moe_combine(ctx, y, o.place, v)
        assert float((f64(there) * f64(y)).sum()) == float((f64(x) * f64(back)).sum())


def test_combine_grad_by_differences(ctx):
    """d_weights and d_y against differences of the joined rows' loss; the loss is linear in each, so differences over
    whole numbers are exact."""
    from spindle_amd import ops
    rng = np.random.default_rng(9)
    rows, k, width = 6, 3, 16
    o = sorted_rows(rng, ctx, rows, k, 4, False)
    whole = lambda *s: torch.from_numpy(rng.integers(-5, 6, s)).float().cuda()  # noqa: E731
    y, w, d = whole(rows * k, width), whole(rows, k), whole(rows, width)
    d_y, d_w = ops.moe_combine_grad(ctx, d, y, o.order, o.place, w)
    loss = lambda y_, w_: float((f64(ops.moe_combine(ctx, y_, o.place, w_)) * f64(d)).sum())  # noqa: E731
    base = loss(y, w)
    for i in [(0, 0), (3, 2), (5, 1)]:
        w2 = w.clone()
        w2[i] += 1
        assert loss(y, w2) - base == float(d_w[i])
    for i in [(0, 0), (7, 15), (17, 3)]:
        y2 = y.clone()
        y2[i] += 1
        assert loss(y2, w) - base == float(d_y[i])


def test_places_out_of_range(ctx):
    """Orders and places that name nothing read and write nothing."""
    from spindle_amd import ops
    rows, k, width = 4, 2, 24
    x, y = torch.ones(rows, width, device="cuda"), torch.ones(rows * k, width, device="cuda")
    bad = ints([0, -1, 8, 2 ** 31 - 1, -2 ** 31, 7, 1, 100])
    got = ops.moe_gather(ctx, x, bad, k)
    assert got[:, 0].tolist() == [1, 0, 0, 0, 0, 1, 1, 0]
    assert ops.moe_combine(ctx, y, bad.view(rows, k))[:, 0].tolist() == [1, 0, 1, 1]
    order = ints([0, 5, -1, -1, -1, -1, -1, -1])
    place = ints([[0, -1], [8, -5], [-1, 1], [-1, -1]])
    d_y, d_w = ops.moe_combine_grad(ctx, x, y, order, place, torch.full((rows, k), 2.0, device="cuda"))
    assert d_y[:, 0].tolist() == [2, 2, 0, 0, 0, 0, 0, 0] and d_w.tolist() == [[24, 0], [0, 0], [0, 24], [0, 0]]


def test_no_rows(ctx):
    from spindle_amd import ops
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 16, device="cuda")
    assert ops.moe_gather(ctx, x, none.flatten(), 3).shape == (0, 16)
    assert ops.moe_combine(ctx, x, none).shape == (0, 16)
    d_y, d_w = ops.moe_combine_grad(ctx, x, x, none.flatten(), none, torch.zeros(0, 3, device="cuda"))
    assert d_y.shape == (0, 16) and d_w.shape == (0, 3)


def test_far_rows(ctx):
    """Sorted rows past 2^32 bytes: gathered, joined, and the gradient, looked at in some of them."""
    from spindle_amd import ops
    rows, k, width, experts = 150_000, 8, 2048, 40
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    ids = torch.randint(0, experts, (rows, k), generator=g, device="cuda", dtype=torch.int32)
    o = ops.moe_sort(ctx, ids, experts)
    x = torch.randn(rows, width, generator=g, device="cuda", dtype=BF16)
    y = ops.moe_gather(ctx, x, o.order, k)
    some = torch.cat([torch.arange(5, device="cuda"), torch.arange(rows * k - 5, rows * k, device="cuda"), torch.randint(0, rows * k, (50,), generator=g, device="cuda")])
    assert torch.equal(y[some], x[o.order[some].long() // k])
    w = torch.randint(-3, 4, (rows, k), generator=g, device="cuda").float()
    got = ops.moe_combine(ctx, y, o.place, w)
    want = f64(x[-50:]) * f64(w[-50:]).sum(1)[:, None]  # (every place of a row holds the row)
    close(got[-50:], want, np.abs(f64(x[-50:])) * f64(w[-50:].abs()).sum(1)[:, None] * k * R.U + R.rounding(want * (1 + 2.0 ** -20), BF16))
    d_y, d_w = ops.moe_combine_grad(ctx, x, y, o.order, o.place, w)
    e = o.order[some].long()
    want = f64(w).reshape(-1)[e.cpu().numpy()][:, None] * f64(x[e // k])
    close(d_y[some], want, np.abs(want) * R.U + R.rounding(want * (1 + R.U), BF16))
    sq = f64(x[-20:]) ** 2
    close(d_w[-20:], np.repeat(sq.sum(1)[:, None], k, 1), np.repeat(sq.sum(1)[:, None], k, 1) * (width / 64 + 24) * R.U)


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("rows,k,width,experts,drop", [(4097, 8, 1024, 32, 0.0), (6200, 2, 1040, 8, 0.3), (1025, 32, 8192, 128, 0.9), (12300, 1, 768, 3, 0.0), (3001, 5, 4104, 1, 1.0)])
def test_gather_of_many_rows(ctx, dtype, rows, k, width, experts, drop):
    """Rows past an L2's size, taken slice by slice: every place is written once, places of no expert with zeros."""
    from spindle_amd import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    ids = torch.randint(0, experts, (rows, k), generator=g, device="cuda", dtype=torch.int32)
    ids[torch.rand(rows, k, generator=g, device="cuda") < drop] = -1
    o = ops.moe_sort(ctx, ids, experts)
    big = torch.randn(rows, width + 16, generator=g, device="cuda").to(dtype)
    x = big[:, 8:8 + width]
    some = o.order >= 0
    e = torch.where(some, o.order, 0).long()
    want = torch.where(some[:, None], x[e // k], torch.zeros((), dtype=dtype, device="cuda"))
    out = torch.full((rows * k + 1, width + 8), 7.0, dtype=dtype, device="cuda")
    ops.moe_gather(ctx, x, o.order, k, out=out[:-1, :width])
    assert torch.equal(out[:-1, :width], want) and bool((out[:-1, width:] == 7).all()) and bool((out[-1] == 7).all())
    w = torch.randn(rows, k, generator=g, device="cuda")
    got = ops.moe_gather(ctx, x, o.order, k, weights=w)
    scaled = torch.where(some[:, None], (x[e // k].float() * w.reshape(-1)[e][:, None]).to(dtype), torch.zeros((), dtype=dtype, device="cuda"))
    assert torch.equal(got, scaled)
    # any order that the call may be given, the same entry twice and entries out of range among them
    other = torch.randint(-2, rows * k + 3, (rows * k,), generator=g, device="cuda", dtype=torch.int32)
    some = (other >= 0) & (other < rows * k)
    want = torch.where(some[:, None], x[torch.where(some, other, 0).long() // k], torch.zeros((), dtype=dtype, device="cuda"))
    assert torch.equal(ops.moe_gather(ctx, x, other, k), want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("norm", [True, False])
def test_route_grad_of_rows_of_padding(ctx, dtype, norm):
    """A row of nothing but -inf gets zeros whatever its weights' gradient is, infinities and NaN among it; an id out of range makes
    it NaN all the same."""
    from spindle_amd import ops
    rng = np.random.default_rng(4)
    rows, n, k = 12, 40, 5
    x = torch.from_numpy(rng.standard_normal((rows, n))).to(dtype).cuda()
    x[1::2] = float("-inf")
    chosen, weights = ops.moe_route(ctx, x, k, norm=norm)
    assert not weights[1::2].any()
    g = torch.from_numpy(rng.standard_normal((rows, k))).float().cuda()
    g[1], g[3, 2], g[5, 0], g[7, k - 1] = float("nan"), float("inf"), float("-inf"), float("nan")
    chosen[11, 3] = n
    d = ops.moe_route_grad(ctx, x, chosen, g, norm=norm)
    assert not d[1:11:2].any() and d[11].isnan().all()
    want, tol = R.route_grad(f64(x[::2]), chosen[::2].cpu().numpy(), f64(g[::2]), norm)
    close(d[::2], want, tol + R.rounding(want, dtype))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,k,width,experts,drop", [(40000, 1, 512, 16, 0.1), (33000, 2, 512, 16, 0.5), (33000, 3, 512, 40, 0.0), (9000, 4, 2056, 40, 0.1), (5003, 6, 2056, 64, 0.2)])
def test_gather_of_many_rows_by_each_rule(ctx, dtype, rows, k, width, experts, drop):
    """Sizes at which rows with weights and without go different ways, or the same one."""
    test_gather_of_many_rows(ctx, dtype, rows, k, width, experts, drop)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("drop", [False, True])
def test_weighted_gather_gradient(ctx, dtype, drop):
    """Both gradients of the weighted gather: of x the joining with the same weights, of the weights that of the joining's gradient with
    x for d_out and out's gradient for y. The loss is linear in each, so over whole numbers differences are exact."""
    from spindle_amd import ops
    rng = np.random.default_rng(12)
    rows, k, width = 9, 3, 24
    o = sorted_rows(rng, ctx, rows, k, 5, drop)
    whole = lambda *s: torch.from_numpy(rng.integers(-3, 4, s)).cuda()  # noqa: E731
    x, w, d = whole(rows, width).to(dtype), whole(rows, k).float(), whole(rows * k, width).to(dtype)
    loss = lambda x_, w_: float((f64(ops.moe_gather(ctx, x_, o.order, k, weights=w_)) * f64(d)).sum())  # noqa: E731
    d_x = ops.moe_combine(ctx, d, o.place, w)
    _, d_w = ops.moe_combine_grad(ctx, x, d, o.order, o.place, w)
    base = loss(x, w)
    for i in np.ndindex(rows, k):
        w2 = w.clone()
        w2[i] += 1
        assert loss(x, w2) - base == float(d_w[i])
    for i in [(0, 0), (3, 7), (4, 23), (8, 11)]:
        x2 = x.clone()
        x2[i] += 1
        assert loss(x2, w) - base == float(d_x[i])


def test_sort_and_route_at_their_limits(ctx):
    """As many rows, experts and choices as there may be: 2^18 rows, 1024 experts, 32 of them a row."""
    from spindle_amd import ops
    rows, n, k = 1 << 18, 1024, 32
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    # distinct logits in each row, so that the choice does not hang on ties: a permutation's values
    x = torch.rand(rows, n, generator=g, device="cuda").argsort(1).float() / 64
    chosen, weights = ops.moe_route(ctx, x, k)
    values, ids = x.topk(k, 1)
    assert torch.equal(chosen.long(), ids)
    # (64 bits; logits apart by less than 16 and exact, a few roundings each: 64 * 2^-24)
    assert (weights.double() - torch.softmax(values.double(), 1)).abs().max() <= 64 * R.U
    o = ops.moe_sort(ctx, chosen, n)
    sorted_ids, order = torch.sort(chosen.flatten(), stable=True)
    assert torch.equal(o.order.long(), order)
    assert torch.equal(o.starts.long(), torch.searchsorted(sorted_ids, torch.arange(n + 1, device="cuda", dtype=torch.int32)))
    assert torch.equal(o.place.flatten()[order].long(), torch.arange(rows * k, device="cuda"))
    one = torch.arange(rows, device="cuda", dtype=torch.float32).view(rows, 1)
    assert torch.equal(ops.moe_gather(ctx, one, o.order, k).view(-1).long(), order // k)
    assert torch.equal(ops.moe_combine(ctx, (order // k).float().view(-1, 1), o.place), one * k)  # (whole numbers below 2^24)


def test_two_contexts_at_once(ctx):
    """Layers' sorts and gathers on two contexts' streams at the same time keep to themselves."""
    from spindle_amd import ops
    other = ops.Context(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    rows, k, n = 9000, 4, 40
    ids = [torch.randint(0, n, (rows, k), generator=g, device="cuda", dtype=torch.int32) for _ in range(2)]
    x = [torch.randn(rows, 256, generator=g, device="cuda") for _ in range(2)]
    want = [x[i][torch.sort(ids[i].flatten(), stable=True).indices // k] for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, c in enumerate((ctx, other)):
            with torch.cuda.stream(c.torch_stream()):
                got[i].append(ops.moe_gather(c, x[i], ops.moe_sort(c, ids[i], n).order, k))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[i]) for i in range(2) for v in got[i])
    other.close()
