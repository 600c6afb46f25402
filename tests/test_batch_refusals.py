"""What the operators for batches of sequences refuse, without a device: every check of arguments
comes before the context is looked at. And the pool's layout on the CPU: each slot's parts lie in the
pool and no two share a nibble."""
import ctypes as C

import numpy as np
import pytest

import batch_ref as R

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


def shape(**kw):
    from spindle_amd import ops
    return ops.Kv4Shape(*(dict(n_kv=2, head_dim=128, page_tokens=32, n_pages=4) | kw).values())


BAD_SHAPES = [(dict(head_dim=96), "head_dim"), (dict(n_kv=0), "n_kv"), (dict(n_kv=1025), "n_kv"), (dict(page_tokens=8), "page_tokens"),
              (dict(page_tokens=48), "page_tokens"), (dict(page_tokens=512), "page_tokens"), (dict(n_pages=0), "n_pages"),
              (dict(n_pages=1 << 27), "n_pages")]


@pytest.mark.parametrize("kw,word", BAD_SHAPES)
def test_shapes(lib, kw, word):
    s = shape(**kw)
    assert lib.spx_kv4_bytes(C.byref(s)) == 0
    with pytest.raises(ValueError):
        s.nbytes
    assert word in error(lib, lib.spx_kv4_append(None, C.byref(s), A, 0, A, 256, A, 256, 1, A))
    assert word in error(lib, lib.spx_kv4_read(None, C.byref(s), A, 0, 1, A, A, 256, A, 256))
    assert word in error(lib, attention(lib, s))


def test_bytes(lib):
    assert lib.spx_kv4_bytes(None) == 0
    for kv, hd, page, pages in [(1, 64, 16, 1), (3, 64, 256, 7), (8, 128, 64, 1000000)]:
        s = shape(n_kv=kv, head_dim=hd, page_tokens=page, n_pages=pages)
        assert lib.spx_kv4_bytes(C.byref(s)) == R.pool_bytes((kv, hd, page, pages)) == kv * pages * page * hd * 9 // 8


ROWS = dict(pool=A, type=0, k=A, ld_k=256, v=A, ld_v=256, rows=2, slots=A)


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(slots=None), "null"), (dict(type=8), "type"),
    (dict(type=-1), "type"), (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"), (dict(ld_k=255), "leading"),
    (dict(ld_v=0), "leading"), (dict(pool=A + 8), "multiple of 16"), (dict(k=A + 2), "multiple"), (dict(type=1, v=A + 1), "multiple"),
    (dict(slots=A + 2), "multiple"), ({}, "context")])
def test_rows(lib, kw, word):
    a, s = ROWS | kw, shape()
    assert word in error(lib, lib.spx_kv4_append(None, C.byref(s), a["pool"], a["type"], a["k"], a["ld_k"], a["v"], a["ld_v"], a["rows"], a["slots"]))
    assert word in error(lib, lib.spx_kv4_read(None, C.byref(s), a["pool"], a["type"], a["rows"], a["slots"], a["k"], a["ld_k"], a["v"], a["ld_v"]))


ATT = dict(pool=A, type=0, q=A, ld_q=512, heads=4, rows=2, n_seq=1, q_start=A, lens=A, tables=A, cols=3, scale=0.0, window=0, max_kv=90, out=A,
           ld_out=512, ws=None, ws_bytes=None)


def attention(lib, s, **kw):
    a = ATT | kw
    if a["ws"] is None:
        a["ws"] = A
    if a["ws_bytes"] is None:
        a["ws_bytes"] = 1 << 40
    return lib.spx_kv4_attention(None, C.byref(s), a["pool"], a["type"], a["q"], a["ld_q"], a["heads"], a["rows"], a["n_seq"], a["q_start"], a["lens"],
                                 a["tables"], a["cols"], a["scale"], a["window"], a["max_kv"], a["out"], a["ld_out"], a["ws"], a["ws_bytes"])


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(q_start=None), "null"), (dict(lens=None), "null"),
    (dict(tables=None), "null"), (dict(type=12), "type"), (dict(heads=3), "n_heads"), (dict(heads=0), "n_heads"), (dict(heads=1026), "n_heads"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 19), "rows"), (dict(n_seq=-1), "n_seq"), (dict(n_seq=4097), "n_seq"), (dict(window=-1), "window"), (dict(cols=0), "table_cols"),
    (dict(cols=1 << 26), "table_cols"), (dict(ld_q=511), "leading"), (dict(ld_out=511), "leading"), (dict(pool=A + 4), "multiple of 16"),
    (dict(q=A + 2), "multiple"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(max_kv=-1), "max_kv"), ({}, "context")])
def test_attention(lib, kw, word):
    assert word in error(lib, attention(lib, shape(), **kw))


def test_attention_scratch(lib):
    """Scratch that is missing, too small or not aligned is refused wherever the call needs some."""
    s = shape(n_pages=4096)
    need = lib.spx_kv4_attention_ws(C.byref(s), 4, 1, 1, 65536)
    assert need >= 0
    if need:
        big = dict(rows=1, cols=2048, max_kv=65536)
        assert "ws must hold" in error(lib, attention(lib, s, ws_bytes=need - 1, **big))
        assert "ws must hold" in error(lib, attention(lib, s, ws=A + 8, **big))
        assert "context" in error(lib, attention(lib, s, ws_bytes=need, **big))


PLAN = dict(n_seq=2, page=32, cols=4, n_pages=8, rows=3, lens=A, add=A, n_free=A, tables=A, free=A, lens_out=A, n_free_out=A, q_start=A, slots=A,
            positions=A, status=A)


@pytest.mark.parametrize("kw,word", [(dict([(k, None)]), "null") for k in list(PLAN)[5:]] + [
    (dict(n_seq=0), "n_seq"), (dict(n_seq=4097), "n_seq"), (dict(page=33), "page_tokens"), (dict(cols=0), "table_cols"), (dict(cols=1 << 30), "table_cols"),
    (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 26), "n_pages"), (dict(rows=-1), "rows"), (dict(rows=(1 << 18) + 1), "rows"), ({}, "context")])
def test_plan(lib, kw, word):
    assert word in error(lib, lib.spx_pages_plan(None, *(PLAN | kw).values()))


LP = dict(type=0, x=A, ld=1000, rows=2, vocab=1000, scale=1.0, targets=A, top=3, logp=A, entropy=A, ids=A, best=A, ws=A, ws_bytes=1 << 40)


@pytest.mark.parametrize("kw,word", [
    (dict(type=6), "type"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1), "vocab"), (dict(top=-1), "top_n"),
    (dict(top=33), "top_n"), (dict(scale=0.0), "logit_scale"), (dict(scale=-1.0), "logit_scale"), (dict(scale=float("nan")), "logit_scale"),
    (dict(scale=float("inf")), "logit_scale"), (dict(x=None), "null"), (dict(ids=None), "null"), (dict(best=None), "null"), (dict(targets=None), "together"),
    (dict(logp=None), "together"), (dict(ld=999), "leading"), (dict(x=A + 2), "multiple"), ({}, "context")])
def test_logprobs(lib, kw, word):
    assert word in error(lib, lib.spx_logprobs(None, *(LP | kw).values()))


def test_logprobs_scratch(lib):
    need = lib.spx_logprobs_ws(1, 151936, 5)
    assert need >= 0
    if need:
        big = dict(rows=1, vocab=151936, ld=151936, top=5)
        assert "ws must hold" in error(lib, lib.spx_logprobs(None, *(LP | big | dict(ws_bytes=need - 1)).values()))
        assert "ws must hold" in error(lib, lib.spx_logprobs(None, *(LP | big | dict(ws=None)).values()))
        assert "context" in error(lib, lib.spx_logprobs(None, *(LP | big | dict(ws_bytes=need)).values()))


@pytest.mark.parametrize("sh", [(2, 64, 16, 3), (1, 128, 32, 2)])
def test_layout_covers_the_pool(sh):
    """Every nibble and scale byte of the pool belongs to exactly one channel or scale."""
    kv, hd, page, pages = sh
    used = np.zeros((R.pool_bytes(sh), 2), np.int64)
    for slot in range(pages * page):
        for head in range(kv):
            key, val, ks, vs = R.places(sh, slot, head)
            for b, s in key + val:
                used[b, s // 4] += 1
            for b in ks + vs:
                used[b:b + 2] += 1
    assert (used == 1).all()


def test_reference_rounds_as_stated():
    x = np.zeros(32)
    x[5], x[9] = -3.0, 3.0  # the first of the largest gives the sign
    d, c = R.quantize(x)
    assert d[0] == 0.375 and c[5] == -8 and c[9] == 7
    x[:] = 0
    x[0], x[1], x[2] = -8.0, 0.5, 1.5  # halves to even
    assert list(R.codes_of(x, R.scale_of(x))[:3]) == [-8, 0, 2]
    assert np.isnan(R.values(np.where(np.arange(32) == 3, np.inf, 1.0))).all()
    assert R.scale_of(np.full(32, 1e9)) == -8160.0 and R.scale_of(np.zeros(32)) == 0.0


def test_python_numbers_past_the_c_ints():
    """Numbers that a C int would cut off are refused before anything else happens, negative ones too."""
    from spindle_amd import ops
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    sh, q = shape(), torch.zeros(2, 4, 128)
    pool = torch.zeros(4 * 2 * 2 * 18 * 128, dtype=torch.uint8)
    for bad in (2 ** 31, 2 ** 32, 2 ** 32 + 16, -1, -2 ** 31, -2 ** 32 + 16):
        calls = [lambda: ops.pages_plan(None, i32(2), i32(2), i32(2, 3), i32(5), i32(1), 16, bad),
                 lambda: ops.pages_plan(None, i32(2), i32(2), i32(2, 3), i32(5), i32(1), bad, 4),
                 lambda: ops.kv4_attention(None, sh, pool, q, i32(2), i32(1), i32(1, 4), window=bad),
                 lambda: ops.kv4_attention(None, sh, pool, q, i32(2), i32(1), i32(1, 4), max_kv=bad),
                 lambda: ops.logprobs(None, torch.zeros(2, 50), top=bad)]
        for f in calls:
            with pytest.raises(ValueError, match="2.31"):
                f()


def test_python_largest_numbers_reach_the_checks(lib):
    """2^31 - 1 goes through to the C entry's own checks (here as far as the tensors' device)."""
    from spindle_amd import ops

    class Ctx:
        device, h, raw_stream = 0, None, 0
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pool = torch.zeros(4 * 2 * 2 * 18 * 128, dtype=torch.uint8)
    for kw in (dict(window=2 ** 31 - 1), dict(max_kv=2 ** 31 - 1)):
        with pytest.raises(ValueError, match="cuda:0"):
            ops.kv4_attention(Ctx, shape(), pool, torch.zeros(2, 4, 128), i32(2), i32(1), i32(1, 4), ws=pool, **kw)
    with pytest.raises(ValueError, match="cuda:0"):
        ops.logprobs(Ctx, torch.zeros(2, 50), top=2 ** 31 - 1)


# ------------------------------------------------------------------ scratch that calls do need
def test_split_calls_need_scratch(lib):
    """What is split among workgroups needs scratch, and is refused without it; what is not needs none."""
    s = shape(n_pages=4096)
    need = lib.spx_kv4_attention_ws(C.byref(s), 4, 1, 1, 65536)
    assert need >= 4 * 2 * 16 * (128 + 2) * 2  # two parts of 16 rows of two key heads at the least
    big = dict(rows=1, cols=2048, max_kv=65536)
    for kw in (dict(ws_bytes=need - 1), dict(ws_bytes=0), dict(ws=A + 8)):
        assert "ws must hold" in error(lib, attention(lib, s, **kw, **big))
    none = lambda **kw: lib.spx_kv4_attention(None, C.byref(s), A, 0, A, 512, 4, kw["rows"], 1, A, A, A, kw["cols"], 0.0, 0, kw["max_kv"], A, 512, None, 0)  # noqa: E731
    assert "ws must hold" in error(lib, none(**big))
    assert lib.spx_kv4_attention_ws(C.byref(s), 4, 1, 1, 64) == 0
    assert "context" in error(lib, none(rows=1, cols=2, max_kv=64))
    need = lib.spx_logprobs_ws(1, 151936, 5)
    assert need >= 2 * (16 + 8 * 5)
    big = dict(rows=1, vocab=151936, ld=151936, top=5)
    for kw in (dict(ws_bytes=need - 1), dict(ws=None), dict(ws=A + 8)):
        assert "ws must hold" in error(lib, lib.spx_logprobs(None, *(LP | big | kw).values()))
    assert lib.spx_logprobs_ws(2, 1000, 3) == 0
    assert "context" in error(lib, lib.spx_logprobs(None, *(LP | dict(ws=None, ws_bytes=0)).values()))


# ------------------------------------------------------------------ addresses of 32-bit numbers
@pytest.mark.parametrize("name", list(PLAN)[5:])
def test_plan_addresses(lib, name):
    assert "multiples of 4" in error(lib, lib.spx_pages_plan(None, *(PLAN | {name: A + 2}).values()))


@pytest.mark.parametrize("name", ["q_start", "lens", "tables"])
def test_attention_addresses(lib, name):
    assert "multiple" in error(lib, attention(lib, shape(), **{name: A + 2}))


@pytest.mark.parametrize("name", ["targets", "logp", "entropy", "ids", "best"])
def test_logprobs_addresses(lib, name):
    assert "multiples" in error(lib, lib.spx_logprobs(None, *(LP | {name: A + 2}).values()))
