"""What the operators of a mixture of experts refuse, without a device: every check of arguments comes before
the context is looked at. And the 64-bit evaluations that the GPU tests hold them to, on known values."""
import ctypes as C

import numpy as np
import pytest

import moe_ref as R

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from spindle_amd import _lib
    return _lib.load()


BUF = np.zeros(1 << 16, np.uint8)
A = BUF.ctypes.data + (-BUF.ctypes.data) % 256  # an aligned address; nothing below reads it


def error(lib, rc):
    assert rc == -1
    return lib.spx_last_error().decode()


SIZES = [(dict(rows=-1), "rows"), (dict(rows=(1 << 18) + 1), "rows"), (dict(k=0), "k must"), (dict(k=33), "k must")]
EXPERTS = [(dict(n_expert=0), "n_expert"), (dict(n_expert=1025), "n_expert")]
TYPES = [(dict(type=8), "type"), (dict(type=39), "type"), (dict(type=-1), "type")]

ROUTE = dict(type=0, logits=A, ld=64, rows=4, n_expert=64, k=8, norm=1, chosen=A, weights=A)
GRAD = dict(type=0, logits=A, ld=64, rows=4, n_expert=64, k=8, norm=1, chosen=A, d_weights=A, d_logits=A, ld_d=64)


@pytest.mark.parametrize("kw,word", SIZES + EXPERTS + TYPES + [
    (dict(n_expert=4, k=5), "at most n_expert"), (dict(norm=2), "norm"), (dict(norm=-1), "norm"), (dict(ld=63), "leading"), ({}, "context")])
def test_route(lib, kw, word):
    assert word in error(lib, lib.spx_moe_route(None, *(ROUTE | kw).values()))
    assert word in error(lib, lib.spx_moe_route_grad(None, *(GRAD | kw).values()))


@pytest.mark.parametrize("name", ["logits", "chosen", "weights", "d_weights", "d_logits"])
def test_route_addresses(lib, name):
    for f, args in ((lib.spx_moe_route, ROUTE), (lib.spx_moe_route_grad, GRAD)):
        if name in args:
            assert "null" in error(lib, f(None, *(args | {name: None}).values()))
            assert "multiple" in error(lib, f(None, *(args | {name: A + 2}).values()))
    assert "multiple" in error(lib, lib.spx_moe_route(None, *(ROUTE | dict(type=1, logits=A + 1)).values()))
    assert "leading" in error(lib, lib.spx_moe_route_grad(None, *(GRAD | dict(ld_d=63)).values()))


SORT = dict(rows=1000, k=8, n_expert=64, chosen=A, starts=A, order=A, place=A, ws=A, ws_bytes=1 << 40)


@pytest.mark.parametrize("kw,word", SIZES + EXPERTS + [(dict([(n, None)]), "null") for n in ("chosen", "starts", "order", "place")] + [
    (dict([(n, A + 2)]), "multiples of 4") for n in ("chosen", "starts", "order", "place")] + [({}, "context")])
def test_sort(lib, kw, word):
    assert word in error(lib, lib.spx_moe_sort(None, *(SORT | kw).values()))


def test_sort_scratch(lib):
    need = lib.spx_moe_sort_ws(1000, 8, 64)
    assert need >= 4 * 65 * 2
    for kw in (dict(ws_bytes=need - 1), dict(ws=None), dict(ws=A + 8)):
        assert "ws must hold" in error(lib, lib.spx_moe_sort(None, *(SORT | kw).values()))
    assert "context" in error(lib, lib.spx_moe_sort(None, *(SORT | dict(ws_bytes=need)).values()))
    assert lib.spx_moe_sort_ws(24, 8, 128) == 0 and lib.spx_moe_sort_ws(-1, 8, 128) == 0 and lib.spx_moe_sort_ws(24, 8, 1025) == 0
    assert "context" in error(lib, lib.spx_moe_sort(None, *(SORT | dict(rows=24, ws=None, ws_bytes=0)).values()))
    assert 0 < lib.spx_moe_sort_ws(1 << 18, 32, 1024) < 1 << 21


GATHER = dict(type=0, x=A, ld_x=64, rows=4, k=2, width=64, order=A, weights=A, out=A, ld_out=64)
COMBINE = dict(type=0, y=A, ld_y=64, rows=4, k=2, width=64, place=A, weights=A, out=A, ld_out=64)
COMBINE_GRAD = dict(type=0, d_out=A, ld_d=64, y=A, ld_y=64, rows=4, k=2, width=64, order=A, place=A, weights=A, d_y=A, ld_dy=64, d_weights=A)


@pytest.mark.parametrize("kw,word", SIZES + TYPES + [(dict(width=0), "width"), (dict(width=(1 << 20) + 1), "width"), ({}, "context")])
def test_rows(lib, kw, word):
    assert word in error(lib, lib.spx_moe_gather(None, *(GATHER | kw).values()))
    assert word in error(lib, lib.spx_moe_combine(None, *(COMBINE | kw).values()))
    assert word in error(lib, lib.spx_moe_combine_grad(None, *(COMBINE_GRAD | kw).values()))


def test_rows_addresses(lib):
    for f, args, free in ((lib.spx_moe_gather, GATHER, ("weights",)), (lib.spx_moe_combine, COMBINE, ("weights",)), (lib.spx_moe_combine_grad, COMBINE_GRAD, ())):
        for name in args:
            if name.startswith("ld_"):
                assert "leading" in error(lib, f(None, *(args | {name: 63}).values()))
            elif args[name] == A:
                assert ("context" if name in free else "null") in error(lib, f(None, *(args | {name: None}).values()))
                assert "multiple" in error(lib, f(None, *(args | {name: A + 2}).values()))
        assert "context" in error(lib, f(None, *(args | dict(rows=0)).values()))


def matrix(lib_type=None, **kw):
    from spindle_amd import ops
    return ops._Mx4C(*(dict(data=A, rows=8, cols=100) | kw).values())


BAD = [(dict(data=None), "null"), (dict(data=A + 8), "multiple of 16"), (dict(rows=0), "rows"), (dict(rows=-4), "rows"), (dict(cols=0), "columns"),
       (dict(cols=(1 << 20) + 1), "columns")]


@pytest.mark.parametrize("kw,word", BAD)
def test_matrices(lib, kw, word):
    m = matrix(**kw)
    assert word in error(lib, lib.spx_mx4_quantize(None, 0, A, 100, C.byref(m)))
    assert word in error(lib, lib.spx_mx4_read(None, C.byref(m), 0, A, 100))
    assert word in error(lib, product(lib, w=m))
    assert word in error(lib, product(lib, up=m))


def test_quantize_and_read(lib):
    m = C.byref(matrix())
    for f in (lambda t=0, x=A, ld=100, m=m: lib.spx_mx4_quantize(None, t, x, ld, m), lambda t=0, x=A, ld=100, m=m: lib.spx_mx4_read(None, m, t, x, ld)):
        assert "type" in error(lib, f(t=39)) and "null" in error(lib, f(x=None)) and "leading" in error(lib, f(ld=99))
        assert "multiple" in error(lib, f(x=A + 2)) and "multiple" in error(lib, f(t=1, x=A + 1)) and "null" in error(lib, f(m=None)) and "context" in error(lib, f())


def test_bytes(lib):
    for rows, cols in [(1, 1), (3, 128), (5, 129), (1 << 20, 2048), (2 ** 31 - 1, 1 << 20)]:
        assert lib.spx_mx4_bytes(rows, cols) == rows * R.padded(cols) // 32 * 17
    assert lib.spx_mx4_bytes(0, 5) == 0 and lib.spx_mx4_bytes(5, 0) == 0 and lib.spx_mx4_bytes(5, (1 << 20) + 1) == 0


PRODUCT = dict(type=0, x=A, ld_x=100, x_rows=6, w=None, up=None, n_expert=2, starts=A, order=A, k=2, rows=12, out_type=0, out=A, ld_out=4)


def product(lib, **kw):
    a = PRODUCT | kw
    a["w"] = C.byref(a["w"] if a["w"] is not None else matrix())
    a["up"] = None if a["up"] is None else C.byref(a["up"])
    return lib.spx_mx4_matmul(None, *a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(type=8), "type"), (dict(out_type=39), "out_type"), (dict(n_expert=0), "n_expert"), (dict(n_expert=3), "n_expert"), (dict(n_expert=1025), "n_expert"),
    (dict(starts=None), "need starts"), (dict(starts=None, n_expert=1), "need starts"), (dict(k=0), "k must"), (dict(k=33), "k must"), (dict(rows=-1), "rows"),
    (dict(rows=(1 << 23) + 1), "rows"), (dict(x_rows=-1), "rows"), (dict(x_rows=(1 << 23) + 1), "rows"), (dict(order=None), "x_rows"), (dict(x=None), "null"),
    (dict(out=None), "null"), (dict(ld_x=99), "leading"), (dict(ld_out=3), "leading"), (dict(x=A + 2), "multiple"), (dict(type=39, x=A + 8), "multiple of 16"),
    (dict(out=A + 2), "multiple"), (dict(starts=A + 2), "multiple"), (dict(order=A + 2), "multiple"), (dict(up=matrix(rows=6)), "one shape"),
    (dict(up=matrix(cols=101)), "one shape"), (dict(w=matrix(rows=2 ** 22)), "2^20"), ({}, "context"), (dict(type=39, ld_x=0), "context"), (dict(up=matrix()), "context"),
    (dict(starts=None, order=None, n_expert=1, rows=6, ld_out=8), "context"), (dict(rows=0, x=None, out=None, x_rows=0), "context")])
def test_products(lib, kw, word):
    assert word in error(lib, product(lib, **kw))


# ----------------------------------------------------------------------------------- from Python
class Ctx:
    device, h, raw_stream = 0, None, 0


def test_python_refusals(lib):
    """Shapes, types and strides that the C entry cannot see, and numbers past its ints."""
    from spindle_amd import ops
    z, i32 = torch.zeros, lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    m = ops.Mx4(torch.zeros(ops.Mx4.nbytes(8, 100), dtype=torch.uint8), 8, 100)
    bad = [lambda: ops.moe_route(Ctx, z(4, 8).double(), 2), lambda: ops.moe_route(Ctx, z(8), 2), lambda: ops.moe_route(Ctx, z(8, 4).t(), 2),
           lambda: ops.moe_route(Ctx, z(4, 8), 2 ** 32 + 2), lambda: ops.moe_route(Ctx, z(4, 8), -1),
           lambda: ops.moe_route_grad(Ctx, z(4, 8), i32(3, 2), z(4, 2)), lambda: ops.moe_route_grad(Ctx, z(4, 8), i32(4, 2).long(), z(4, 2)),
           lambda: ops.moe_route_grad(Ctx, z(4, 8), i32(4, 2), z(4, 3)), lambda: ops.moe_route_grad(Ctx, z(4, 8), i32(4, 2), z(4, 2).half()),
           lambda: ops.moe_sort(Ctx, i32(4, 2).long(), 8), lambda: ops.moe_sort(Ctx, i32(8), 8), lambda: ops.moe_sort(Ctx, i32(4, 2), 2 ** 31),
           lambda: ops.moe_sort(Ctx, i32(4, 4)[:, ::2], 8), lambda: ops.moe_gather(Ctx, z(4, 8), i32(7), 2), lambda: ops.moe_gather(Ctx, z(4, 8), i32(8), 2, weights=z(4, 3)),
           lambda: ops.moe_gather(Ctx, z(4, 8), i32(8), 2, out=z(7, 8)), lambda: ops.moe_gather(Ctx, z(4, 8), i32(8), 2, out=z(8, 8).half()),
           lambda: ops.moe_gather(Ctx, z(4, 16)[:, ::2], i32(8), 2), lambda: ops.moe_combine(Ctx, z(7, 8), i32(4, 2)), lambda: ops.moe_combine(Ctx, z(8, 8), i32(4, 2), z(8)),
           lambda: ops.moe_combine(Ctx, z(8, 8), i32(4, 2), out=z(4, 9)), lambda: ops.moe_combine_grad(Ctx, z(4, 8), z(8, 9), i32(8), i32(4, 2), z(4, 2)),
           lambda: ops.moe_combine_grad(Ctx, z(4, 8).half(), z(8, 8), i32(8), i32(4, 2), z(4, 2)), lambda: ops.Mx4(torch.zeros(3, dtype=torch.uint8), 8, 100),
           lambda: ops.Mx4(torch.zeros(9999), 8, 100), lambda: ops.Mx4(torch.zeros(9999, dtype=torch.uint8), 2 ** 32 + 8, 100), lambda: ops.Mx4(torch.zeros(9999, dtype=torch.uint8), 0, 100),
           lambda: ops.mx4_quantize(Ctx, z(8, 99), out=m), lambda: ops.mx4_quantize(Ctx, z(8, 100).long(), out=m), lambda: ops.mx4_read(Ctx, m, torch.float64),
           lambda: ops.mx4_read(Ctx, m, out=z(8, 99)), lambda: ops.mx4_matmul(Ctx, z(4, 99), m), lambda: ops.mx4_matmul(Ctx, z(4, 100), m, starts=i32(4)),
           lambda: ops.mx4_matmul(Ctx, z(4, 100), m, starts=i32(1)), lambda: ops.mx4_matmul(Ctx, z(4, 100), m, out=z(4, 7)), lambda: ops.mx4_matmul(Ctx, z(4, 100), m, dtype=torch.int32),
           lambda: ops.mx4_matmul(Ctx, z(4, 100), m, starts=i32(3), order=i32(4), k=2 ** 32 + 1), lambda: ops.mx4_matmul(Ctx, z(4, 100), m, starts=i32(3), order=i32(2, 2))]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_python_other_devices(lib):
    """Tensors elsewhere than on the context's device are refused, each of a call's."""
    from spindle_amd import ops
    z, i32 = torch.zeros, lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    m = ops.Mx4(torch.zeros(ops.Mx4.nbytes(8, 100), dtype=torch.uint8), 8, 100)
    for f in (lambda: ops.moe_route(Ctx, z(4, 8), 2), lambda: ops.moe_route_grad(Ctx, z(4, 8), i32(4, 2), z(4, 2)), lambda: ops.moe_sort(Ctx, i32(4, 2), 8),
              lambda: ops.moe_gather(Ctx, z(4, 8), i32(8), 2), lambda: ops.moe_combine(Ctx, z(8, 8), i32(4, 2), z(4, 2)),
              lambda: ops.moe_combine_grad(Ctx, z(4, 8), z(8, 8), i32(8), i32(4, 2), z(4, 2)), lambda: ops.mx4_quantize(Ctx, z(8, 100)), lambda: ops.mx4_read(Ctx, m),
              lambda: ops.mx4_matmul(Ctx, z(4, 100), m, starts=i32(3), order=i32(4))):
        with pytest.raises(ValueError, match="cuda:0"):
            f()


def test_python_no_rows(lib):
    """A 4-bit matrix of no rows is made by empty alone, for columns that there may be, and takes no other shape's place."""
    from spindle_amd import ops
    m = ops.Mx4.empty(0, 100, device="cpu")
    assert (m.rows, m.cols, m.data.numel(), m.data.dtype) == (0, 100, 0, torch.uint8)
    z = torch.zeros
    for f in (lambda: ops.Mx4.empty(0, 0, device="cpu"), lambda: ops.Mx4.empty(0, (1 << 20) + 1, device="cpu"), lambda: ops.Mx4.empty(-1, 100, device="cpu"),
              lambda: ops.Mx4.empty(0, -(1 << 40), device="cpu"), lambda: ops.mx4_quantize(Ctx, z(1, 100), out=m), lambda: ops.mx4_quantize(Ctx, z(0, 99), out=m),
              lambda: ops.mx4_quantize(Ctx, z(0, 100).long()), lambda: ops.mx4_quantize(Ctx, z(0, 100)), lambda: ops.mx4_read(Ctx, m), lambda: ops.mx4_read(Ctx, m, torch.int32),
              lambda: ops.mx4_read(Ctx, m, out=z(1, 100))):
        with pytest.raises(ValueError):
            f()


def test_python_other_bytes(lib):
    """The calls take the bytes that a matrix has now, never those it was made with, and of the size that they were made for."""
    from spindle_amd import ops
    need = ops.Mx4.nbytes(8, 100)
    a, b = torch.zeros(need, dtype=torch.uint8), torch.zeros(need + 16, dtype=torch.uint8)
    m = ops.Mx4(a, 8, 100)
    assert (m._c.data, m._c.rows, m._c.cols) == (a.data_ptr(), 8, 100)
    m.data = b
    assert m.data is b and (m._c.data, m._c.rows, m._c.cols, m.rows, m.cols) == (b.data_ptr(), 8, 100, 8, 100)
    for bad in (torch.zeros(need - 1, dtype=torch.uint8), torch.zeros(need), b[::2]):
        with pytest.raises(ValueError):
            m.data = bad
    for name in ("rows", "cols"):
        with pytest.raises(AttributeError):
            setattr(m, name, 9)
    assert m.data is b and m._c.data == b.data_ptr()


# -------------------------------------------------------------------------- the references themselves
def test_reference_of_the_format():
    x = np.zeros((1, 33))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0]  # ties to the even code
    x[0, 32] = -9.0  # 8 <= 9 < 16: scale 2, 4.5 is nearest to 4
    codes, scales = R.quantize(x)
    assert list(codes[0, :8]) == [0, 2, 2, 4, 4, 6, 6, 15] and list(scales[0]) == [127, 128, 0, 0] and codes[0, 32] == 14
    v = R.unpack(R.pack(codes, scales), 1, 33)
    assert list(v[0, :8]) == [0, 1, 1, 2, 2, 4, 4, -6] and v[0, 32] == -8
    for m, byte in [(2.0 ** -149, 0), (2.0 ** -126, 0), (2.0 ** -125, 0), (2.0 ** -124, 1), (3.4e38, 252), (7.999999, 127), (8.0, 128), (np.nextafter(4.0, 0), 126), (np.inf, 255), (np.nan, 255)]:
        assert R.quantize(np.full((1, 32), m))[1][0, 0] == byte, m


def test_reference_of_the_router():
    x = np.array([[1.0, 3.0, 3.0, -np.inf], [-np.inf] * 4, [np.nan, 1, np.inf, 2]])
    ids, w, _ = R.route(x, 2, True)
    assert ids.tolist() == [[1, 2], [0, 1], [0, 2]] and w[0].tolist() == [0.5, 0.5] and w[1].tolist() == [0, 0] and np.isnan(w[2]).all()
    starts, order, place = R.sort(np.array([[1, 0], [5, 1]]), 2)
    assert starts.tolist() == [0, 1, 3] and order.tolist() == [1, 0, 3, -1] and place.tolist() == [[1, 0], [-1, 2]]
