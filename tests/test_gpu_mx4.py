"""Matrices in microscaled 4-bit floats (include/spx.h: spx_mx4_quantize, spx_mx4_read, spx_mx4_matmul) against
64-bit evaluations of their definitions (moe_ref.py), and a layer of experts put together."""
import numpy as np
import pytest

import moe_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PARTS = {F32: 3, F16: 2, BF16: 1, "mx4": 0}


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


# ----------------------------------------------------------------------------------- the format
def rows_for(rng, rows, cols, dtype):
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, 1)))
    big = {F32: 3.4e38, F16: 65504.0, BF16: 3.38e38}[dtype]
    for r in range(rows):
        kind = r % 11
        if kind == 1:
            x[r] = 0.0
        elif kind == 2:
            x[r, rng.integers(cols)] = [np.nan, np.inf, -np.inf][r // 11 % 3]
        elif kind == 3:  # every quotient on the grid's halves, the largest 6 or 7.99
            x[r] = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], cols) * rng.choice([-1, 1], cols)
        elif kind == 4:
            x[r] *= 1e-7 if dtype == F16 else 1e-38  # around and below the smallest normal numbers
        elif kind == 5:
            x[r] = rng.choice([-big, big, 1.0], cols)
        elif kind == 6:
            x[r] = rng.choice([-0.0, 0.0], cols)
        elif kind == 7:
            x[r] = np.exp2(rng.integers(-10, 10, cols))
    return torch.from_numpy(np.clip(x, -big, big)).to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (22, 32), (23, 33), (5, 127), (12, 128), (34, 129), (11, 576), (3, 2050)])
@pytest.mark.parametrize("pad,off", [(0, 0), (16, 0), (3, 1)])
def test_quantize_and_read(ctx, dtype, rows, cols, pad, off):
    from spindle_amd import ops
    rng = np.random.default_rng(rows + cols)
    wide = torch.full((rows, cols + pad + off), float("nan"), dtype=dtype)
    wide[:, off:off + cols] = rows_for(rng, rows, cols, dtype)
    x = wide.cuda()[:, off:off + cols]
    m = ops.Mx4(torch.full((ops.Mx4.nbytes(rows, cols) + 8,), 0xA5, dtype=torch.uint8, device="cuda"), rows, cols)
    assert ops.mx4_quantize(ctx, x, out=m) is m
    want = R.pack(*R.quantize(f64(x)))
    got = m.data.cpu().numpy()
    assert np.array_equal(got[:-8], want) and (got[-8:] == 0xA5).all()
    values = torch.from_numpy(R.unpack(want, rows, cols))
    for t in (F32, F16, BF16):
        v = ops.mx4_read(ctx, m, t)
        ref = values.float().to(t)
        assert torch.equal(v.cpu().nan_to_num(nan=77.0), ref.nan_to_num(nan=77.0))
        into = torch.zeros(rows, cols + pad + off, dtype=t, device="cuda")
        ops.mx4_read(ctx, m, t, out=into[:, off:off + cols])
        assert torch.equal(into[:, off:off + cols].nan_to_num(nan=77.0), v.nan_to_num(nan=77.0)) and not into[:, :off].any() and not into[:, off + cols:].any()


def test_read_every_code_and_scale(ctx):
    from spindle_amd import ops
    data = np.concatenate([np.tile(np.arange(16, dtype=np.uint8) * 17, 256 * 4), np.repeat(np.arange(256, dtype=np.uint8), 4)])
    m = ops.Mx4(torch.from_numpy(data).cuda(), 256, 128)
    with np.errstate(over="ignore"):
        want = R.unpack(data, 256, 128).astype(np.float32)
    assert np.array_equal(ops.mx4_read(ctx, m).cpu().numpy(), want, equal_nan=True)


def test_quantize_many_rows(ctx):
    """As many rows as a prompt has, against the same in small calls."""
    from spindle_amd import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = torch.randn(9001, 700, generator=g, device="cuda", dtype=BF16)
    got = ops.mx4_read(ctx, ops.mx4_quantize(ctx, x), BF16)
    for a in range(0, 9001, 1000):
        assert torch.equal(ops.mx4_read(ctx, ops.mx4_quantize(ctx, x[a:a + 1000]), BF16), got[a:a + 1000])


# --------------------------------------------------------------------------------------- products
def matrix(rng, rows, cols, spread=6):
    """A random matrix's bytes (padding columns zeros)."""
    from spindle_amd import ops
    p = R.padded(cols)
    codes = rng.integers(0, 16, (rows, p))
    codes[:, cols:] = 0
    data = R.pack(codes, rng.integers(127 - spread, 128 + spread, (rows, p // 32)))
    return ops.Mx4(torch.from_numpy(data).cuda(), rows, cols), R.unpack(data, rows, cols)


def rows_of_x(rng, kind, rows, cols, pad=0, off=0):
    """x as the call takes it, its values in 64 bits."""
    if kind == "mx4":
        m, v = matrix(rng, max(rows, 1), cols)
        return m, v
    x = torch.from_numpy(rng.standard_normal((rows, cols + pad + off)) * np.exp2(rng.integers(-4, 4, (rows, 1)))).to(kind).cuda()[:, off:off + cols]
    return x, f64(x)


def check(got, x, w, up, kind, dtype):
    want, tol = R.product(x, w, up, PARTS[kind])
    got = f64(got)
    # What lies half a step or more above a type's largest number rounds to infinity: in f16 from 65504 + 32 / 2 on.
    # Where the exact value is that near to it, its infinity is as right as a finite result.
    limit = {F32: 2.0 ** 128, BF16: 2.0 ** 128, F16: 65520.0}[dtype]
    over = np.isinf(got) & (np.abs(want) + tol >= limit) & (np.sign(got) == np.sign(want))
    assert not (np.isfinite(got) & (np.abs(want) - tol >= limit)).any()
    close(np.where(over, want, got), want, tol + R.rounding(np.abs(want) + tol, dtype), (x.shape, w.shape))


SIZES = [(1, 1, 1), (1, 2048, 33), (2, 128, 16), (3, 100, 31), (16, 129, 64), (17, 576, 65), (33, 256, 129), (64, 1000, 40), (130, 384, 200), (257, 64, 300),
         (12, 640, 600), (40, 128, 600), (90, 260, 600), (200, 1100, 530)]


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,cols,n", SIZES)
@pytest.mark.parametrize("gated", [False, True])
def test_dense(ctx, kind, rows, cols, n, gated):
    from spindle_amd import ops
    rng = np.random.default_rng(rows * 7 + cols + n)
    x, xv = rows_of_x(rng, kind, rows, cols)
    w, wv = matrix(rng, n, cols)
    up, uv = matrix(rng, n, cols) if gated else (None, None)
    for dtype in (F32, F16, BF16) if kind == "mx4" else (kind,):
        scale = 2.0 ** -9 if dtype == F16 else 1.0  # (sums stay in f16's range)
        if scale != 1.0:
            w2, wv2 = lowered(w, wv, scale)
            check(ops.mx4_matmul(ctx, x, w2, up=up, dtype=dtype) if not gated else ops.mx4_matmul(ctx, x, w2, up=lowered(up, uv, scale)[0], dtype=dtype),
                  xv, wv2, uv * scale if gated else None, kind, dtype)
        else:
            check(ops.mx4_matmul(ctx, x, w, up=up, dtype=dtype), xv, wv, uv, kind, dtype)


def lowered(m, v, scale):
    """The matrix with its scales lowered by a power of two."""
    from spindle_amd import ops
    data = m.data.clone()
    codes = m.rows * R.padded(m.cols) // 2
    data[codes:] -= int(-np.log2(scale))
    return ops.Mx4(data, m.rows, m.cols), v * scale


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("pad,off", [(8, 0), (3, 1)])
def test_strides(ctx, kind, pad, off):
    """Rows of x and out apart by more than their width, at odd addresses; what lies between rows of out stays."""
    from spindle_amd import ops
    rng = np.random.default_rng(pad)
    rows, cols, n = 37, 200, 53
    x, xv = rows_of_x(rng, kind, rows, cols, pad, off)
    w, wv = lowered(*matrix(rng, n, cols), 2.0 ** -9)
    into = torch.full((rows, n + pad + off), 5.0, dtype=kind, device="cuda")
    ops.mx4_matmul(ctx, x, w, out=into[:, off:off + n])
    check(into[:, off:off + n], xv, wv, None, kind, kind)
    assert (into[:, :off] == 5.0).all() and (into[:, off + n:] == 5.0).all()


# Enough tiles for the kernels of many rows: of 32, 64 and 128 rows; odd columns, a part of a turn, of a step and of a block.
TILES = [(17, 192, 24700), (24, 320, 16500), (33, 130, 24700), (60, 576, 12600), (520, 200, 2900), (600, 64, 2700), (600, 300, 2625)]


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,cols,n", TILES)
@pytest.mark.parametrize("gated", [False, True])
def test_dense_tiles(ctx, kind, rows, cols, n, gated):
    from spindle_amd import ops
    rng = np.random.default_rng(rows * 7 + cols + n)
    x, xv = rows_of_x(rng, kind, rows, cols)
    w, wv = lowered(*matrix(rng, n, cols), 2.0 ** -9)
    up, uv = lowered(*matrix(rng, n, cols), 2.0 ** -9) if gated else (None, None)
    dtype = BF16 if kind == "mx4" else kind
    check(ops.mx4_matmul(ctx, x, w, up=up, dtype=dtype), xv, wv, uv, kind, dtype)


@pytest.mark.parametrize("kind,cols", [(F32, 131), (F16, 131), (BF16, 131), (F32, 200), (BF16, 200), (BF16, 192)])
@pytest.mark.parametrize("pad,off", [(8, 0), (3, 1), (0, 0)])
@pytest.mark.parametrize("rows,n", [(20, 25000), (530, 2900)])
def test_tile_strides(ctx, kind, cols, pad, off, rows, n):
    """Tiles over rows that are apart, at odd addresses, of odd lengths; what lies between rows of out stays."""
    from spindle_amd import ops
    rng = np.random.default_rng(pad + cols)
    x, xv = rows_of_x(rng, kind, rows, cols, pad, off)
    w, wv = lowered(*matrix(rng, n, cols), 2.0 ** -9)
    into = torch.full((rows, n + pad + off), 5.0, dtype=kind, device="cuda")
    ops.mx4_matmul(ctx, x, w, out=into[:, off:off + n])
    check(into[:, off:off + n], xv, wv, None, kind, kind)
    assert (into[:, :off] == 5.0).all() and (into[:, off + n:] == 5.0).all()


GROUPS = [(1, 8, 128, 128, 40), (5, 2, 4, 100, 33), (24, 8, 32, 256, 64), (100, 4, 6, 300, 100), (90, 8, 3, 64, 130), (300, 2, 5, 160, 72),
          (40, 2, 4, 700, 530), (100, 4, 9, 200, 300),
          # many tiles: 12, 40 and 600 rows a matrix, and more experts than a search keeps in registers
          (300, 4, 100, 128, 300), (700, 4, 70, 200, 260), (2400, 2, 8, 100, 300), (500, 2, 300, 64, 100)]


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,k,experts,cols,n", GROUPS)
@pytest.mark.parametrize("gated,sort_first,drop", [(True, False, False), (False, True, True), (False, False, True)])
def test_by_expert(ctx, kind, rows, k, experts, cols, n, gated, sort_first, drop):
    from spindle_amd import ops
    rng = np.random.default_rng(rows + cols)
    ids = rng.integers(0, experts, (rows, k))
    ids[: rows // 3] = ids[0, 0]  # a crowded expert, others with few rows or none
    if drop:
        ids[rng.random(ids.shape) < 0.4] = -1
    o = ops.moe_sort(ctx, ints(ids), experts)
    starts, order, _ = R.sort(ids, experts)
    x, xv = rows_of_x(rng, kind, rows * k if sort_first else rows, cols)
    w, wv = lowered(*matrix(rng, experts * n, cols), 2.0 ** -9)
    up, uv = lowered(*matrix(rng, experts * n, cols), 2.0 ** -9) if gated else (None, None)
    dtype = BF16 if kind == "mx4" else kind
    out = torch.full((rows * k, n), 123.0, dtype=dtype, device="cuda")
    ops.mx4_matmul(ctx, x, w, up=up, starts=o.starts, order=None if sort_first else o.order, k=k, dtype=dtype, out=out)
    assert (out[starts[-1]:] == 123.0).all()  # rows behind the last one stay
    for e in range(experts):
        a, b = starts[e], starts[e + 1]
        if a < b:
            rows_e = xv[a:b] if sort_first else xv[order[a:b] // k]
            at = slice(e * n, (e + 1) * n)
            check(out[a:b], rows_e, wv[at], uv[at] if gated else None, kind, dtype)


@pytest.mark.parametrize("kind", [F32, BF16, "mx4"])
@pytest.mark.parametrize("rows,n", [(6, 48), (150, 48), (40, 13000), (1200, 1600)])
def test_rows_without_an_entry(ctx, kind, rows, n):
    """A row whose order names no row of x stays as it was, among rows that have one; so do rows that starts leave out."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    cols = 128
    x, xv = rows_of_x(rng, kind, rows, cols)
    w, wv = matrix(rng, 2 * n, cols)
    dtype = F32
    order = rng.integers(0, rows * 2, rows)
    order[[1, 4]] = -1, rows * 2  # k = 2: that is a row behind x
    out = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
    cut = rows // 2
    ops.mx4_matmul(ctx, x, w, starts=ints([1, cut, rows - 1]), order=ints(order), k=2, dtype=dtype, out=out)
    none = [0, 1, 4, rows - 1]
    assert (out[none] == 7.0).all()
    for a, b, at in ((1, cut, slice(0, n)), (cut, rows - 1, slice(n, 2 * n))):
        some = [i for i in range(a, b) if i not in none]
        check(out[some], xv[order[some] // 2], wv[at], None, kind, dtype)
    # starts past the rows are cut there
    out.fill_(7.0)
    ops.mx4_matmul(ctx, x, w, starts=ints([-5, cut, 10 ** 6]), order=ints(order), k=2, dtype=dtype, out=out)
    check(out[rows - 1:], xv[order[rows - 1] // 2][None], wv[n:], None, kind, dtype)


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,n", [(3, 36), (70, 36), (200, 36), (20, 25000), (60, 12800), (530, 2900)])
def test_special_values(ctx, kind, rows, n):
    """NaN and infinities stay in their rows, NaN scales in their matrix's; scales to the ends of their range."""
    from spindle_amd import ops
    rng = np.random.default_rng(5)
    cols = 260
    w, wv = matrix(rng, n, cols)
    w.data[n * R.padded(cols) // 2 + 4 * R.padded(cols) // 32] = 255  # the first block of row 4
    if kind == "mx4":
        x, xv = matrix(rng, rows, cols)
        x.data[rows * R.padded(cols) // 2 + 2 * R.padded(cols) // 32 + 3] = 255
        xv = R.unpack(x.data.cpu().numpy(), rows, cols)
    else:
        x = torch.from_numpy(rng.standard_normal((rows, cols))).to(kind).cuda()
        x[2, 100] = float("nan")
        x[1, 7] = float("inf")
        xv = f64(x)
        if kind == F32:  # a NaN whose upper half is infinity's
            x.view(torch.int32)[2, 100] = 0x7F800001
    wv = R.unpack(w.data.cpu().numpy(), n, cols)
    got = f64(ops.mx4_matmul(ctx, x, w, dtype=F32))
    assert np.isnan(got[:, 4]).all() and np.isnan(got[2]).all()
    with np.errstate(invalid="ignore"):
        want = xv @ wv.T
    if kind != "mx4":
        rest = [j for j in range(n) if j != 4]
        inf = wv[rest, 7]
        assert np.array_equal(np.isnan(got[1, rest]), inf == 0) and np.array_equal(got[1, rest][inf != 0], np.sign(inf[inf != 0]) * np.inf)
    keep = [i for i in range(rows) if i not in (1, 2)]
    others = [j for j in range(n) if j != 4]
    if kind == "mx4":
        keep = [i for i in range(rows) if i != 2]
    ref, tol = R.product(xv[keep], wv[others], None, PARTS[kind])
    close(got[np.ix_(keep, others)], ref, tol + R.rounding(np.abs(ref) + tol, F32))
    assert not np.isnan(want[np.ix_(keep, others)]).any()


@pytest.mark.parametrize("rows,n", [(2, 24), (40, 24), (20, 6500), (80, 6500)])
def test_wide_scales(ctx, rows, n):
    """Products whose scales lie far apart, each way, keep their values: x times 2^40, the matrix times 2^-60."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    cols = 256
    w, wv = lowered(*matrix(rng, n, cols, 30), 2.0 ** -60)
    m, mv = matrix(rng, rows, cols, 30)
    m.data[rows * cols // 2:] += 40
    got = ops.mx4_matmul(ctx, m, w, dtype=F32)
    check(got, mv * 2.0 ** 40, wv, None, "mx4", F32)
    x = torch.from_numpy(mv * 2.0 ** 40).float().cuda()
    check(ops.mx4_matmul(ctx, x, w), f64(x), wv, None, F32, F32)


@pytest.mark.parametrize("x_rows", [3_300_000, 5_000_000])
@pytest.mark.parametrize("rows,n", [(5, 40), (80, 6500)])
def test_far_rows_of_x(ctx, x_rows, rows, n):
    """Rows of x whose codes lie past 2^31 and past 2^32 bytes."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    cols = 2048
    data = torch.zeros(ops.Mx4.nbytes(x_rows, cols), dtype=torch.uint8, device="cuda")
    some = np.concatenate([[0, x_rows - 1], rng.integers(x_rows - 100, x_rows, rows - 2)])
    codes, scales = rng.integers(0, 16, (100, cols)), rng.integers(121, 134, (100, cols // 32))
    packed = torch.from_numpy(R.pack(codes, scales)).cuda()
    end = x_rows * cols // 2
    data[end - 100 * cols // 2:end] = packed[:100 * cols // 2]
    data[end + (x_rows - 100) * cols // 32:] = packed[100 * cols // 2:]
    values = R.unpack(packed.cpu().numpy(), 100, cols)
    x = np.where((some >= x_rows - 100)[:, None], values[np.maximum(some - (x_rows - 100), 0)], 0.0)
    w, wv = matrix(rng, n, cols)
    got = ops.mx4_matmul(ctx, ops.Mx4(data, x_rows, cols), w, starts=ints([0, rows]), order=ints(some), dtype=F32)
    check(got, x, wv, None, "mx4", F32)


@pytest.mark.parametrize("kind", [BF16, "mx4"])
@pytest.mark.parametrize("rows,n", [(3, 40), (70, 9000)])
def test_far_matrix(ctx, kind, rows, n):
    """The matrix of an expert past 2^32 bytes."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    cols = 2048
    experts = min(1024, 4_400_000 // n)
    many = experts * n
    if many * 1088 < 2 ** 32:
        cols = 1 << 18 if n < 100 else cols
    p = R.padded(cols)
    data = torch.zeros(ops.Mx4.nbytes(many, cols), dtype=torch.uint8, device="cuda")
    assert data.numel() > 2 ** 32
    codes, scales = rng.integers(0, 16, (n, p)), rng.integers(112, 125, (n, p // 32))
    packed = torch.from_numpy(R.pack(codes, scales)).cuda()
    end = many * p // 2
    data[end - n * p // 2:end] = packed[:n * p // 2]
    data[end + (many - n) * p // 32:] = packed[n * p // 2:]
    x, xv = rows_of_x(rng, kind, rows, cols)
    starts = np.zeros(experts + 1, np.int64)
    starts[-1] = rows
    got = ops.mx4_matmul(ctx, x, ops.Mx4(data, many, cols), starts=ints(starts), dtype=F32)
    check(got, xv, R.unpack(packed.cpu().numpy(), n, cols), None, kind, F32)


def test_no_rows(ctx):
    from spindle_amd import ops
    w, _ = matrix(np.random.default_rng(1), 8, 64)
    assert ops.mx4_matmul(ctx, torch.zeros(0, 64, device="cuda"), w).shape == (0, 8)


def test_same_bits_every_time(ctx):
    from spindle_amd import ops
    rng = np.random.default_rng(11)
    w, _ = matrix(rng, 3 * 3000, 700)
    for kind in (F32, BF16, "mx4"):
        for rows in (5, 70, 90, 400, 1700):
            x, _ = rows_of_x(rng, kind, rows, 700)
            starts = ints([0, rows // 5, rows // 2, rows])
            a = ops.mx4_matmul(ctx, x, w, starts=starts, dtype=F32)
            for _ in range(3):
                assert torch.equal(ops.mx4_matmul(ctx, x, w, starts=starts, dtype=F32), a)


# ------------------------------------------------------------------------- a layer put together
def layer(ops, ctx, x, logits, k, gate, up, down, experts, four):
    """A mixture of experts over rows x: router, sort, gated products, down, joined."""
    chosen, weights = ops.moe_route(ctx, logits, k)
    o = ops.moe_sort(ctx, chosen, experts)
    h = ops.mx4_matmul(ctx, ops.mx4_quantize(ctx, x) if four else x, gate, up=up, starts=o.starts, order=o.order, k=k, dtype=x.dtype)
    y = ops.mx4_matmul(ctx, ops.mx4_quantize(ctx, h) if four else h, down, starts=o.starts, dtype=x.dtype)
    return ops.moe_combine(ctx, y, o.place, weights), (chosen, weights, o, h, y)


def layer_case(rng, rows, dtype):
    experts, k, dim, inner = 16, 4, 256, 96
    mats = []
    for r, c in ((inner, dim), (inner, dim), (dim, inner)):
        mats.append(lowered(*matrix(rng, experts * r, c, 2), 2.0 ** -5))
    x = torch.from_numpy(rng.standard_normal((rows, dim))).to(dtype).cuda()
    logits = torch.from_numpy(rng.standard_normal((rows, experts)) * 2).float().cuda()
    return experts, k, mats, x, logits


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 7, 150])
@pytest.mark.parametrize("four", [False, True])
def test_layer(ctx, dtype, rows, four):
    """Each step of the layer against its definition on the step's own inputs."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    experts, k, ((gate, gv), (up, uv), (down, dv)), x, logits = layer_case(rng, rows, dtype)
    got, (chosen, weights, o, h, y) = layer(ops, ctx, x, logits, k, gate, up, down, experts, four)
    ids, w, tol = R.route(f64(logits), k, True)
    assert np.array_equal(chosen.cpu().numpy(), ids)
    close(weights, w, tol)
    starts, order, place = R.sort(ids, experts)
    stand = lambda v: R.unpack(R.pack(*R.quantize(f64(v))), *v.shape) if four else f64(v)  # noqa: E731
    xv, hv, kind = stand(x), stand(h), "mx4" if four else dtype
    for e in range(experts):
        a, b = starts[e], starts[e + 1]
        if a < b:
            n, d = slice(e * 96, e * 96 + 96), slice(e * 256, e * 256 + 256)
            check(h[a:b], xv[order[a:b] // k], gv[n], uv[n], kind, dtype)
            check(y[a:b], hv[a:b], dv[d], None, kind, dtype)
    terms = f64(y)[place] * f64(weights)[..., None]
    want, tol = terms.sum(1), np.abs(terms).sum(1) * k * R.U
    close(got, want, tol + R.rounding(np.abs(want) + tol, dtype))


def test_layer_in_a_graph(ctx):
    """A captured layer, replayed over changing inputs with eager work between, gives the eager bits each time; on the
    context's stream and with another stream's work in order."""
    from spindle_amd import ops
    rng = np.random.default_rng(21)
    experts, k, ((gate, _), (up, _), (down, _)), x, logits = layer_case(rng, 200, BF16)
    inputs = [(torch.randn_like(x), torch.randn_like(logits)) for _ in range(4)]
    run = lambda: layer(ops, ctx, x, logits, k, gate, up, down, experts, True)[0]  # noqa: E731
    want = []
    side = torch.cuda.Stream()
    for i, (a, b) in enumerate(inputs):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            side.wait_stream(torch.cuda.default_stream())
            x.copy_(a)
            logits.copy_(b)
            want.append(run().clone())
            torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        out = run()
    for turn in range(3):
        for (a, b), w in zip(inputs, want):
            x.copy_(a)
            logits.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
            assert torch.equal(run(), w)  # eager work between replays


def test_tuning_step_in_a_graph(ctx):
    """A router's way back, captured and replayed: the eager bits each time."""
    from spindle_amd import ops
    rng = np.random.default_rng(22)
    rows, k, experts, width = 300, 4, 12, 64
    logits = torch.from_numpy(rng.standard_normal((rows, experts))).float().cuda()
    y = torch.from_numpy(rng.standard_normal((rows * k, width))).to(BF16).cuda()
    d = torch.from_numpy(rng.standard_normal((rows, width))).to(BF16).cuda()

    def step():
        chosen, weights = ops.moe_route(ctx, logits, k)
        o = ops.moe_sort(ctx, chosen, experts)
        out = ops.moe_combine(ctx, y, o.place, weights)
        d_y, d_w = ops.moe_combine_grad(ctx, d, y, o.order, o.place, weights)
        return out, d_y, ops.moe_route_grad(ctx, logits, chosen, d_w)

    first = [torch.randn_like(logits) for _ in range(3)]
    want = []
    for v in first:
        logits.copy_(v)
        want.append([t.clone() for t in step()])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for v, w in zip(first, want):
            logits.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, w))
            step()


# ------------------------------------------------------------------------ exactness of the gate
# few rows, and tiles of 32, 64 and 128 rows
GATES = [(250, 40), (20, 25000), (400, 6000), (600, 2700)]


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,n", GATES)
def test_gate_by_itself(ctx, kind, rows, n):
    """silu of sums that are exact, at every magnitude that it has a value at: out is silu(v) times 1, v one of x's values.

    Its error, with U = 2^-24 of a rounding: the exponential is off by a unit in the last place (2 U) and what its argument's
    rounding takes off it is put back by a multiplication and an addition of one rounding (U), 1 + e rounds (U), the reciprocal is
    off by a unit in the last place (2 U) and the product with v rounds (U): 7 U, and 1 U for all that is second order."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    cols = 64
    if kind == "mx4":  # 0.5 to 6 times 1 to 8, so up to 48
        codes, scales = np.zeros((rows, 128), np.int64), np.full((rows, 4), 127)
        codes[:, 0], codes[:, 32], scales[:, 0] = rng.integers(1, 8, rows) + 8 * rng.integers(0, 2, rows), 2, 127 + rng.integers(-1, 4, rows)
        data = R.pack(codes, scales)
        x, v = ops.Mx4(torch.from_numpy(data).cuda(), rows, cols), R.unpack(data, rows, cols)[:, 0]
    else:
        x = torch.zeros(rows, cols, device="cuda", dtype=kind)
        x[:, 0] = torch.from_numpy(rng.uniform(0.01, 86.0, rows) * np.where(np.arange(rows) % 4, -1, 1)).to(kind).cuda()
        x[:, 32] = 1.0
        v = f64(x[:, 0])
    one = lambda at: np.eye(1, 128, at, dtype=np.int64).repeat(n, 0) * 2  # noqa: E731 (code 2 is 1)
    gate, up = (ops.Mx4(torch.from_numpy(R.pack(one(at), np.full((n, 4), 127))).cuda(), n, cols) for at in (0, 32))
    got = f64(ops.mx4_matmul(ctx, x, gate, up=up, dtype=F32))
    want = v / (1.0 + np.exp(-v))
    close(got, np.repeat(want[:, None], n, 1), 8 * R.U * np.abs(want)[:, None])


# ----------------------------------------------------------------------------------- no rows at all
def test_no_four_bit_rows(ctx):
    """An empty batch in 4 bits, as in the other types: quantised, read, through a product, and a whole layer of none."""
    from spindle_amd import ops
    rng = np.random.default_rng(1)
    w, _ = matrix(rng, 8, 64)
    for dtype in (F32, BF16):
        m = ops.mx4_quantize(ctx, torch.zeros(0, 64, device="cuda", dtype=dtype))
        assert (m.rows, m.cols) == (0, 64)
        assert ops.mx4_quantize(ctx, torch.zeros(0, 64, device="cuda", dtype=dtype), out=m) is m
        v = ops.mx4_read(ctx, m, dtype)
        assert v.shape == (0, 64) and v.dtype == dtype
        out = ops.mx4_matmul(ctx, m, w, dtype=dtype)
        assert out.shape == (0, 8) and out.dtype == dtype
    into = torch.full((3, 8), 7.0, device="cuda")
    ops.mx4_matmul(ctx, m, w, starts=ints([0, 3]), order=ints([0, 1, 2]), out=into, dtype=F32)  # (rows of an x that has none)
    assert (into == 7.0).all()
    experts, k, ((gate, _), (up, _), (down, _)), x, logits = layer_case(rng, 3, BF16)
    for four in (False, True):
        got, _ = layer(ops, ctx, x[:0], logits[:0], k, gate, up, down, experts, four)
        assert got.shape == (0, 256) and got.dtype == BF16


# ---------------------------------------------------------------- many experts and far ones, in tiles
# rows a matrix past what the few rows' kernel takes: tiles of 32, 64 and (16-bit rows from 512 on) 128 rows
MANY = [(1500, 2, 300, 64, 100), (6000, 2, 300, 64, 100), (10200, 2, 257, 64, 72), (5700, 2, 1024, 64, 40)]


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,k,experts,cols,n", MANY)
@pytest.mark.parametrize("gated,drop", [(True, False), (False, True)])
def test_tiles_of_many_experts(ctx, kind, rows, k, experts, cols, n, gated, drop):
    """More experts than a workgroup's search for its tile keeps in registers."""
    from spindle_amd import ops
    assert rows * k // experts > 8 and (rows * k // 64 + experts) * -(-n // 128) > 192
    rng = np.random.default_rng(rows)
    ids = rng.integers(0, experts, (rows, k))
    ids[: rows // 6] = ids[0, 0]
    ids[(ids % 7 == 3) & (ids != ids[0, 0])] = experts - 1  # experts without a row
    if drop:
        ids[rng.random(ids.shape) < 0.2] = -1
    o = ops.moe_sort(ctx, ints(ids), experts)
    starts, order = o.starts.cpu().numpy(), o.order.cpu().numpy()
    x, xv = rows_of_x(rng, kind, rows, cols)
    w, wv = lowered(*matrix(rng, experts * n, cols), 2.0 ** -9)
    up, uv = lowered(*matrix(rng, experts * n, cols), 2.0 ** -9) if gated else (None, None)
    dtype = BF16 if kind == "mx4" else kind
    out = torch.full((rows * k, n), 123.0, dtype=dtype, device="cuda")
    ops.mx4_matmul(ctx, x, w, up=up, starts=o.starts, order=o.order, k=k, dtype=dtype, out=out)
    assert (out[starts[-1]:] == 123.0).all()
    for e in range(experts):
        a, b = starts[e], starts[e + 1]
        if a < b:
            at = slice(e * n, (e + 1) * n)
            check(out[a:b], xv[order[a:b] // k], wv[at], uv[at] if gated else None, kind, dtype)


@pytest.mark.parametrize("kind", [F32, BF16, "mx4"])
@pytest.mark.parametrize("rows", [80, 240, 560])
def test_far_matrix_in_tiles(ctx, kind, rows):
    """The last columns of the last of eight experts, past 2^32 bytes, in tiles of 32, 64 and (4-bit rows) 128 rows."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows)
    experts, n, cols, some = 8, 1 << 19, 2304, 200
    many = experts * n
    data = torch.zeros(ops.Mx4.nbytes(many, cols), dtype=torch.uint8, device="cuda")
    end = many * cols // 2
    assert end - some * cols // 2 > 2 ** 32 and rows // experts > 8
    codes, scales = rng.integers(0, 16, (some, cols)), rng.integers(112, 125, (some, cols // 32))
    packed = torch.from_numpy(R.pack(codes, scales)).cuda()
    data[end - some * cols // 2:end] = packed[:some * cols // 2]
    data[end + (many - some) * cols // 32:] = packed[some * cols // 2:]
    x, xv = rows_of_x(rng, kind, rows, cols)
    starts = np.zeros(experts + 1, np.int64)
    starts[-1] = rows
    out = ops.mx4_matmul(ctx, x, ops.Mx4(data, many, cols), starts=ints(starts), dtype=BF16 if kind == "mx4" else None)
    assert not out[:, :n - some].any()
    check(out[:, n - some:], xv, R.unpack(packed.cpu().numpy(), some, cols), None, kind, out.dtype)


# --------------------------------------------------------------------------- every bit of a value
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("rows,cols,n", [(1, 2048, 48), (5, 4096, 48), (40, 2048, 48), (20, 2048, 12500), (130, 4096, 9000), (600, 2048, 2700)])
def test_last_bits_of_long_rows(ctx, kind, rows, cols, n):
    """Long rows whose last bits make the whole sum: pairs of neighbours, a number plus some last bits and its negative, times
    equal weights. (fp32: 1 + 2^-8, whose parts are a bit each, so that the last bits are a third one's; fp16: 1.)

    A pair is in one instruction, whose sum is off by at most 2 U of what it adds up and of the sum so far. The latter is at
    most that of the last bits (the rest cancels in each), so the bound does not grow with the columns' square as it does
    for any order of any values; a part that was left out would be off by more (asserted)."""
    from spindle_amd import ops
    rng = np.random.default_rng(cols + n)
    first, low, step = (1.0 + 2.0 ** -8, 2.0 ** -15, 2.0 ** -23) if kind == F32 else (1.0, 2.0 ** -7, 2.0 ** -10)
    last = (np.floor(rng.uniform(0.5, 1.0, (rows, cols // 2)) * low / step)) * step
    v = np.stack([first + last, np.full_like(last, -first)], -1).reshape(rows, cols)
    x = torch.from_numpy(v).to(kind).cuda()
    assert np.array_equal(f64(x), v)
    codes = np.repeat(rng.integers(1, 8, (n, cols // 2)), 2, 1)
    data = R.pack(codes, rng.integers(124, 128, (n, cols // 32)))
    w, wv = ops.Mx4(torch.from_numpy(data).cuda(), n, cols), R.unpack(data, n, cols)
    got = f64(ops.mx4_matmul(ctx, x, w, dtype=F32))
    want, mag = v @ wv.T, np.abs(v) @ wv.T
    tol = 2 * R.U * (PARTS[kind] * (cols / 16 + 8) * want + mag) + np.abs(want) * R.U
    assert (tol < want / 4).all()
    close(got, want, tol)


# ------------------------------------------------------------------------------ ends of the scales
def ends_case(rng, kind, rows, cols, n, w_bytes, x_power):
    """A matrix with scales of these bytes, x of about 2^x_power."""
    from spindle_amd import ops
    p = R.padded(cols)
    codes = rng.integers(0, 16, (n, p))
    codes[:, cols:] = 0
    data = R.pack(codes, rng.choice(w_bytes, (n, p // 32)))
    w = ops.Mx4(torch.from_numpy(data).cuda(), n, cols)
    if kind == "mx4":
        codes = rng.integers(0, 16, (rows, p))
        codes[:, cols:] = 0
        xd = R.pack(codes, 127 + x_power + rng.integers(-2, 3, (rows, p // 32)))
        return w, R.unpack(data, n, cols), ops.Mx4(torch.from_numpy(xd).cuda(), rows, cols), R.unpack(xd, rows, cols)
    x = torch.from_numpy(rng.standard_normal((rows, cols)) * 2.0 ** x_power).to(kind).cuda()
    return w, R.unpack(data, n, cols), x, f64(x)


ENDS = [(3, 40), (70, 40), (20, 25000), (60, 12800), (530, 2900)]


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,n", ENDS)
@pytest.mark.parametrize("low", [True, False])
def test_smallest_and_largest_scales(ctx, kind, rows, n, low):
    """Matrices of the smallest scales (2^-127, whose values lie below the normal numbers, to 2^-124) against large x, and of the
    largest whose every value is a number (2^123 to 2^125) against small x."""
    rng = np.random.default_rng(rows)
    power = {F16: (12, -14)}.get(kind, (100, -110))[0 if low else 1]
    w, wv, x, xv = ends_case(rng, kind, rows, 260, n, [0, 1, 2, 3] if low else [250, 251, 252], power)
    from spindle_amd import ops
    check(ops.mx4_matmul(ctx, x, w, dtype=F32), xv, wv, None, kind, F32)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,n", ENDS)
def test_rows_below_the_normal_numbers(ctx, kind, rows, n):
    """x of 2^-133 to 2^-124 against large scales: what is at least 2^-133 counts."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows + 1)
    w, wv, x, xv = ends_case(rng, kind, rows, 260, n, [224, 225, 226, 227], -127)
    x = torch.where(torch.rand(x.shape, device="cuda") < 0.5, x, x / 16)
    xv = f64(x)
    assert (np.abs(xv) < 2.0 ** -126).mean() > 0.5
    check(ops.mx4_matmul(ctx, x, w, dtype=F32), xv, wv, None, kind, F32)


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
@pytest.mark.parametrize("rows,n", ENDS)
def test_scales_past_the_range(ctx, kind, rows, n):
    """Rows of the matrix with scales 2^126 and 2^127 may overflow, and do so in their own column of out; what does not is right."""
    from spindle_amd import ops
    rng = np.random.default_rng(rows + 2)
    w, wv, x, xv = ends_case(rng, kind, rows, 260, n, [125, 126, 127, 128], {F16: -10}.get(kind, -20))
    at, big = n * R.padded(260) // 2, [3, n // 2, n - 1]
    for i in big:
        w.data[at + i * 12 + 1] = 253 + (i & 1)
    wv = R.unpack(w.data.cpu().numpy(), n, 260)
    got = f64(ops.mx4_matmul(ctx, x, w, dtype=F32))
    want, tol = R.product(xv, wv, None, PARTS[kind])
    rest = np.setdiff1d(np.arange(n), big)
    close(got[:, rest], want[:, rest], (tol + R.rounding(np.abs(want) + tol, F32))[:, rest])
    fine = np.isfinite(got[:, big])
    close(np.where(fine, got[:, big], 0.0), np.where(fine, want[:, big], 0.0), (tol + R.rounding(np.abs(want) + tol, F32))[:, big])


@pytest.mark.parametrize("kind", [F32, F16, BF16, "mx4"])
def test_as_many_rows_as_there_may_be(ctx, kind):
    """2^23 rows, dense and by 1024 experts, looked at in some of them: whole numbers, so without rounding."""
    from spindle_amd import ops
    rows, cols, n = 1 << 23, 8, 5
    rng = np.random.default_rng(3)
    experts = 1024
    codes = np.zeros((experts * n, 128), np.int64)
    codes[:, :cols] = rng.choice([0, 2, 4, 5, 6, 7, 10, 12], (experts * n, cols))  # 0, 1, 2, 3, 4, 6, -1, -2
    data = R.pack(codes, np.full((experts * n, 4), 127))
    w, wv = ops.Mx4(torch.from_numpy(data).cuda(), experts * n, cols), R.unpack(data, experts * n, cols)
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    v = torch.randint(-4, 5, (rows, cols), generator=g, device="cuda", dtype=torch.float32)
    v[:, 0] = 4.0  # (the block's scale is 1: every value is a code)
    x = ops.mx4_quantize(ctx, v) if kind == "mx4" else v.to(kind)
    some = torch.cat([torch.arange(3, device="cuda"), torch.randint(0, rows, (200,), generator=g, device="cuda"), torch.arange(rows - 3, rows, device="cuda")])
    xv = f64(v[some])
    got = ops.mx4_matmul(ctx, x, ops.Mx4(torch.from_numpy(R.pack(codes[:n], np.full((n, 4), 127))).cuda(), n, cols), dtype=F32)
    assert np.array_equal(f64(got[some]), xv @ wv[:n].T)
    starts = torch.sort(torch.randint(0, rows, (experts + 1,), generator=g, device="cuda", dtype=torch.int32)).values
    starts[0], starts[-1] = 0, rows
    got = ops.mx4_matmul(ctx, x, w, starts=starts, dtype=F32)
    e = torch.searchsorted(starts[1:].contiguous(), some.int(), right=True).cpu().numpy()
    want = np.stack([xv[i] @ wv[e[i] * n:(e[i] + 1) * n].T for i in range(len(e))])
    assert np.array_equal(f64(got[some]), want)
