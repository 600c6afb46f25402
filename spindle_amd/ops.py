"""Operator-level mirror of the reference's kernel interface over the C ABI.

Names follow the reference: `matvec` / `matvec_multi` (smollm_chat.rs:309, 447),
`q8k_quantize` (Q8K::quantize, quant_q8k.rs:73), `matmul_rows_q8k` (quant_q8k::matmul_rows,
:255). Device memory comes from torch (cuda == HIP on ROCm); torch is plumbing only.
"""
import ctypes as C
import weakref

import numpy as np

from ._lib import P, check, lib

try:  # device buffers of the operator functions below are torch tensors; a context needs no torch
    import torch
except ImportError:  # pragma: no cover - torch is part of this image
    torch = None

F32, F16, Q5_0, Q8_0, Q4K, Q6K, BF16 = 0, 1, 6, 8, 12, 14, 30


class Context:
    """A device + HIP stream (replaces the reference's WorkerPool as the execution resource)."""

    def __init__(self, device=0):
        self.device = device
        if torch is not None and torch.cuda.is_available():
            torch.cuda.set_device(device)  # torch's buffers on the same device
        h = P()
        check(lib.spx_create(device, C.byref(h)))  # fails (SpxError) without a visible GPU
        self.h = h
        self._stream, self.raw_stream = None, lib.spx_get_stream(h)
        self._children = weakref.WeakSet()   # engines / tensors to release before the context

    def adopt(self, obj):
        self._children.add(obj)

    def sync(self):
        check(lib.spx_sync(self.h))

    def torch_stream(self):
        """The context's stream as a torch stream: a program that makes it torch's current one
        (torch.cuda.set_stream) orders its own work and the operators' on one stream."""
        if self._stream is None:
            self._stream = torch.cuda.ExternalStream(self.raw_stream, device=self.device)
        return self._stream

    def close(self):
        if self.h:
            for ch in list(self._children):
                ch.close()
            lib.spx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Tensor:
    """An uploaded weight tensor: n_expert slabs of rows x cols in GGUF block layout (Mat)."""

    def __init__(self, ctx, dtype, cols, rows, ggml_bytes, n_expert=1):
        self.ctx, self.dtype, self.cols, self.rows, self.n_expert = ctx, dtype, cols, rows, n_expert
        data = np.ascontiguousarray(ggml_bytes, dtype=np.uint8)
        rb = lib.spx_row_bytes(dtype, cols)
        if rb <= 0 or data.size != rb * rows * n_expert:
            raise ValueError(f"expected {rb * rows * n_expert} bytes for dtype {dtype} {rows}x{cols}x{n_expert}, got {data.size}")
        h = P()
        check(lib.spx_tensor_upload(ctx.h, dtype, cols, rows, n_expert, data.ctypes.data_as(P), C.byref(h)))
        self.h = h
        self.nbytes = data.size
        ctx.adopt(self)

    def download(self):
        out = np.empty(self.nbytes, np.uint8)
        check(lib.spx_tensor_download(self.ctx.h, self.h, out.ctypes.data_as(P)))
        return out

    def free(self):
        if self.h and self.ctx.h:
            lib.spx_tensor_free(self.ctx.h, self.h)
        self.h = None

    close = free

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _p(t):
    return C.c_void_p(t.data_ptr())


def q8k_quantize(ctx, x):
    """x: [m, n] float32 cuda tensor -> (d [m, n/256] f32, qs [m, n] i8, bsums [m, n/16] i16)."""
    x = x.contiguous()
    m, n = x.shape
    d = torch.empty((m, n // 256), dtype=torch.float32, device=x.device)
    qs = torch.empty((m, n), dtype=torch.int8, device=x.device)
    bs = torch.empty((m, n // 16), dtype=torch.int16, device=x.device)
    torch.cuda.synchronize()
    check(lib.spx_q8k_quantize(ctx.h, _p(x), n, n, m, _p(d), _p(qs), _p(bs)))
    ctx.sync()
    return d, qs, bs


def matmul_rows_q8k(ctx, w, q, expert=0, r0=0, r1=None, out=None):
    d, qs, bs = q
    m = qs.shape[0]
    r1 = w.rows if r1 is None else r1
    if out is None:
        out = torch.full((m, w.rows), float("nan"), dtype=torch.float32, device=qs.device)
    torch.cuda.synchronize()
    check(lib.spx_matmul_rows_q8k(ctx.h, w.h, expert, _p(d), _p(qs), _p(bs), m, _p(out), out.shape[1], r0, r1))
    ctx.sync()
    return out


def block_sums_q8k(ctx, w, row, q, expert=0):
    d, qs, bs = q
    nb = w.cols // 256
    out = torch.empty((nb, 2), dtype=torch.int32, device=qs.device)
    torch.cuda.synchronize()
    check(lib.spx_block_sums_q8k(ctx.h, w.h, expert, row, _p(qs), _p(bs), _p(out)))
    ctx.sync()
    return out


def matvec(ctx, w, x, expert=0):
    """x: [m, cols] float32 cuda (m <= 16) -> [m, rows] (matvec for m == 1, matvec_multi above)."""
    x = x.contiguous()
    m = x.shape[0]
    out = torch.empty((m, w.rows), dtype=torch.float32, device=x.device)
    torch.cuda.synchronize()
    check(lib.spx_matvec(ctx.h, w.h, expert, _p(x), x.shape[1], m, _p(out), w.rows))
    ctx.sync()
    return out


def matvec_noalloc(ctx, w, x, expert=0):
    """matvec through spx_matvec_noalloc: the K-quant activations' Q8_K staged in the library's
    fixed per-device scratch array instead of an allocated workspace (same results)."""
    x = x.contiguous()
    m = x.shape[0]
    out = torch.empty((m, w.rows), dtype=torch.float32, device=x.device)
    torch.cuda.synchronize()
    check(lib.spx_matvec_noalloc(ctx.h, w.h, expert, _p(x), x.shape[1], m, _p(out), w.rows))
    ctx.sync()
    return out


matvec_multi = matvec


def moe(ctx, gate, up, down, x, chosen, weights):
    """ffns_fused / moe_batch_fused with the combine: x [m, dim] float32 cuda; chosen, weights
    [m, k] host arrays (each row's experts distinct). Returns y [m, dim]."""
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2
    ch = np.ascontiguousarray(chosen, np.int32)
    wt = np.ascontiguousarray(weights, np.float32)
    m, k = ch.shape
    y = torch.empty((m, down.rows), dtype=torch.float32, device=x.device)
    torch.cuda.synchronize()  # x is written on torch's stream, the library runs on the context's
    check(lib.spx_moe(ctx.h, gate.h, up.h, down.h, _p(x), x.stride(0), m, k, ch.ctypes.data_as(P), wt.ctypes.data_as(P),
                      _p(y), y.stride(0)))
    ctx.sync()
    return y


def moe_dev(ctx, gate, up, down, x, chosen, weights):
    """moe with the routing in device memory (spx_moe_dev): chosen [m, k] int32 and weights
    [m, k] float32 cuda tensors, as a router on the GPU leaves them; K-quant experts. A row whose
    ids are out of range or repeated comes back NaN. Returns y [m, dim]."""
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2
    assert chosen.is_cuda and chosen.dtype == torch.int32 and weights.is_cuda and weights.dtype == torch.float32
    chosen, weights = chosen.contiguous(), weights.contiguous()
    m, k = chosen.shape
    y = torch.empty((m, down.rows), dtype=torch.float32, device=x.device)
    torch.cuda.synchronize()  # inputs written on torch's stream, the library runs on the context's
    check(lib.spx_moe_dev(ctx.h, gate.h, up.h, down.h, _p(x), x.stride(0), m, k, _p(chosen), _p(weights), _p(y), y.stride(0)))
    ctx.sync()
    return y


# ------------------------------------------------------------------ batches of sequences
# These wait for nothing on the host: a call's work is ordered after what torch's current stream
# holds, and that stream's later work after the call's (no cost where the two are one stream, see
# Context.torch_stream). Inside a captured graph they record their launches. Calls this small are
# bound by the host, so arguments are checked with as few steps as it takes.
_ROW_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16} if torch is not None else {}


def _run(ctx, tensors, call, *args):
    """call(ctx.h, *args) in order with torch's current stream."""
    for t in tensors:
        if t.get_device() != ctx.device:
            raise ValueError(f"expected tensors on cuda:{ctx.device}, got {t.device}")
    if torch._C._cuda_getCurrentRawStream(ctx.device) == ctx.raw_stream:  # (the stream's number, without an object around it)
        check(call(ctx.h, *args))
        return
    ours, theirs = ctx.torch_stream(), torch.cuda.current_stream(ctx.device)
    ours.wait_stream(theirs)
    try:
        check(call(ctx.h, *args))
    finally:
        theirs.wait_stream(ours)


def _row_type(dtype):
    t = _ROW_TYPES.get(dtype)
    if t is None:
        raise ValueError(f"expected float32, float16 or bfloat16, got {dtype}")
    return t


def _i32(t, *shape):
    """The address of a dense int32 tensor of this shape."""
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"expected a contiguous int32 tensor {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _not_c_ints(names):
    """Raised where one of a call's numbers (their bits together, past bit 31) does not fit the C entry's
    ints: ctypes would cut it off without a word."""
    return ValueError(f"{names} must be in 0..2^31 - 1")


def _rows3(t, heads, hd, name):
    """The distance between the rows of a [rows, heads, hd] tensor whose rows are dense."""
    n, w = t.shape[0], heads * hd
    if t.shape != (n, heads, hd) or not (t.is_contiguous() or (t.stride(2) == 1 and (heads == 1 or t.stride(1) == hd))):
        raise ValueError(f"{name}: expected [rows, {heads}, {hd}] with dense rows, got {tuple(t.shape)}, strides {t.stride()}")
    return t.stride(0) if n > 1 else w


class PagesPlan:
    """What pages_plan leaves: lens, n_free, q_start, slots, positions, status (int32 tensors)."""
    __slots__ = ("lens", "n_free", "q_start", "slots", "positions", "status")


def pages_plan(ctx, lens, add, tables, free_list, n_free, page_tokens, rows):
    """One step's pages, slots and positions (spx_pages_plan): lens, add [n_seq], tables [n_seq,
    table_cols], free_list [n_pages] and n_free [1] are int32 cuda tensors; tables and free_list are
    updated in place, the rest comes back new (pass the plan's lens and n_free to the next step).
    rows: how many rows the step has room for, at least the sum of the positive adds."""
    n, cols, pages = lens.numel(), tables.shape[1] if tables.dim() == 2 else 0, free_list.numel()
    if (n | cols | pages | page_tokens | rows) >> 31:
        raise _not_c_ints("page_tokens, rows and the tensors' sizes")
    ins = _i32(lens, n), _i32(add, n), _i32(n_free, 1), _i32(tables, n, cols), _i32(free_list, pages)
    p = PagesPlan()
    buf = torch.empty(3 * n + 2 + 2 * rows, dtype=torch.int32, device=lens.device)
    p.lens, p.status, p.q_start, p.n_free, p.slots, p.positions = buf.split_with_sizes((n, n, n + 1, 1, rows, rows))
    at = buf.data_ptr()  # (the parts in this order)
    _run(ctx, (lens, add, tables, free_list, n_free), lib.spx_pages_plan, n, page_tokens, cols, pages, rows, *ins, at, at + 4 * (3 * n + 1),
         at + 8 * n, at + 4 * (3 * n + 2), at + 4 * (3 * n + 2 + rows), at + 4 * n)
    return p


class Kv4Shape(C.Structure):
    """spx_kv4_shape: the shape of a layer's 4-bit key / value pool."""
    _fields_ = [("n_kv", C.c_int), ("head_dim", C.c_int), ("page_tokens", C.c_int), ("n_pages", C.c_int)]

    @property
    def nbytes(self):
        n = lib.spx_kv4_bytes(C.byref(self))
        if n <= 0:
            raise ValueError("not a shape of a 4-bit cache: head_dim 64 or 128, page_tokens a power of two in 16..256, n_kv and n_pages positive")
        return n

    def pool(self, device="cuda"):
        """A layer's pool for this shape (a uint8 tensor of zeros)."""
        return torch.zeros(self.nbytes, dtype=torch.uint8, device=device)


def _pool(shape, pool):
    if pool.dtype is not torch.uint8 or not pool.is_contiguous() or pool.numel() < shape.nbytes:
        raise ValueError(f"the pool must be a contiguous uint8 tensor of {shape.nbytes} bytes")
    return pool.data_ptr()


def kv4_append(ctx, shape, pool, k, v, slots):
    """Puts rows k, v [rows, n_kv, head_dim] into the pool's slots [rows] (spx_kv4_append)."""
    t, n, kv, hd = _row_type(k.dtype), slots.numel(), shape.n_kv, shape.head_dim
    if n >> 31:
        raise _not_c_ints("the rows")
    if v.dtype is not k.dtype or k.shape[0] != n or v.shape[0] != n:
        raise ValueError("k and v must have one type and a row for each slot")
    _run(ctx, (pool, k, v, slots), lib.spx_kv4_append, C.byref(shape), _pool(shape, pool), t, k.data_ptr(), _rows3(k, kv, hd, "k"), v.data_ptr(),
         _rows3(v, kv, hd, "v"), n, _i32(slots, n))


def kv4_read(ctx, shape, pool, slots, dtype=None):
    """(k, v) [rows, n_kv, head_dim]: the values that the pool's slots [rows] stand for (spx_kv4_read)."""
    dtype = dtype or torch.float32
    t, n, w = _row_type(dtype), slots.numel(), shape.n_kv * shape.head_dim
    if n >> 31:
        raise _not_c_ints("the rows")
    size = (n, shape.n_kv, shape.head_dim)
    k, v = pool.new_empty(size, dtype=dtype), pool.new_empty(size, dtype=dtype)
    _run(ctx, (pool, slots), lib.spx_kv4_read, C.byref(shape), _pool(shape, pool), t, n, _i32(slots, n), k.data_ptr(), w, v.data_ptr(), w)
    return k, v


def _scratch(need, ws, like):
    """(address, bytes) of a call's scratch, and the tensor that keeps it."""
    if ws is None:
        if need <= 0:
            return None, 0, like
        ws = like.new_empty(need, dtype=torch.uint8)
    return ws.data_ptr(), ws.numel() * ws.element_size(), ws


def kv4_attention(ctx, shape, pool, q, q_start, kv_lens, tables, scale=0.0, window=0, max_kv=None, out=None, ws=None):
    """Attention of q [rows, n_heads, head_dim] over the pool (spx_kv4_attention): q_start [n_seq + 1],
    kv_lens [n_seq] and tables [n_seq, table_cols] int32. out: [rows, n_heads, head_dim] of q's type
    (rows behind the last sequence stay as they are there). ws: scratch, a uint8 tensor; without one
    the call takes its own from torch's allocator."""
    t, n, hd = _row_type(q.dtype), kv_lens.numel(), shape.head_dim
    rows, heads = q.shape[0], q.shape[1] if q.dim() == 3 else 0
    ld_q = _rows3(q, heads, hd, "q")
    if out is None:
        out, ld_out = q.new_empty((rows, heads, hd)), heads * hd
    elif out.dtype is not q.dtype or out.shape != q.shape:
        raise ValueError("out must have q's type and shape")
    else:
        ld_out = _rows3(out, heads, hd, "out")
    cols = tables.shape[1] if tables.dim() == 2 else 0
    max_kv = cols * shape.page_tokens if max_kv is None else max_kv
    if (rows | heads | n | cols | window | max_kv) >> 31:
        raise _not_c_ints("window, max_kv and the tensors' sizes")
    sh = C.byref(shape)
    at, size, ws = _scratch(lib.spx_kv4_attention_ws(sh, heads, rows, n, max_kv), ws, pool)
    _run(ctx, (pool, q, q_start, kv_lens, tables, out, ws), lib.spx_kv4_attention, sh, _pool(shape, pool), t, q.data_ptr(), ld_q, heads, rows, n,
         _i32(q_start, n + 1), _i32(kv_lens, n), _i32(tables, n, cols), cols, scale, window, max_kv, out.data_ptr(), ld_out, at, size)
    return out


class Logprobs:
    """What logprobs leaves: logp [rows] (None without targets), entropy [rows], top_ids and
    top_logp [rows, top]."""
    __slots__ = ("logp", "entropy", "top_ids", "top_logp")


def logprobs(ctx, logits, targets=None, top=0, logit_scale=1.0, ws=None):
    """Log probabilities of targets [rows] (int32), the entropy and the `top` most likely tokens of
    each row of logits [rows, vocab] (spx_logprobs). ws as in kv4_attention."""
    t = _row_type(logits.dtype)
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be [rows, vocab] with dense rows")
    rows, vocab = logits.shape
    if (rows | vocab | top) >> 31:
        raise _not_c_ints("top and the logits' sizes")
    r, n = Logprobs(), min(top, 32)  # (more are refused)
    r.entropy = logits.new_empty(rows, dtype=torch.float32)
    r.top_ids, r.top_logp = logits.new_empty((rows, n), dtype=torch.int32), logits.new_empty((rows, n), dtype=torch.float32)
    if targets is None:
        r.logp, ids, logp, targets = None, None, None, logits
    else:
        r.logp, ids = logits.new_empty(rows, dtype=torch.float32), _i32(targets, rows)
        logp = r.logp.data_ptr()
    scratch, size, ws = _scratch(lib.spx_logprobs_ws(rows, vocab, top), ws, logits)
    _run(ctx, (logits, targets, ws), lib.spx_logprobs, t, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, logit_scale, ids,
         top, logp, r.entropy.data_ptr(), r.top_ids.data_ptr(), r.top_logp.data_ptr(), scratch, size)
    return r


class SamplerParams(C.Structure):
    """spx_sampler_params (SamplerConfig, smollm_chat.rs:1523-1555)."""
    _fields_ = [("temperature", C.c_float), ("top_k", C.c_int), ("top_p", C.c_float), ("min_p", C.c_float),
                ("repeat_penalty", C.c_float), ("seed", C.c_uint64), ("stop_ids", C.POINTER(C.c_int32)),
                ("n_stop", C.c_int), ("think_open", C.c_int)]


def sampler_params(temperature=0.6, top_k=40, top_p=0.9, min_p=0.05, repeat_penalty=1.1, seed=1, stop_ids=(),
                   think_open=-1):
    """The reference's defaults (a fixed seed instead of the clock); returns (params, keep-alive)."""
    stop = (C.c_int32 * max(1, len(stop_ids)))(*stop_ids)
    return SamplerParams(temperature, top_k, top_p, min_p, repeat_penalty, seed,
                         C.cast(stop, C.POINTER(C.c_int32)), len(stop_ids), think_open), stop


class Sampler:
    """sample_from_logits over device logits with its own SplitMix64 state (spx_sampler)."""

    def __init__(self, ctx, vocab, **kw):
        self.ctx, self.vocab = ctx, vocab
        params, keep = sampler_params(**kw)
        h = P()
        check(lib.spx_sampler_create(ctx.h, C.byref(params), vocab, C.byref(h)))
        self.h = h
        ctx.adopt(self)

    def reseed(self, seed):
        check(lib.spx_sampler_reseed(self.h, seed))

    def sample(self, logits, recent=(), forbid_stop=False, forbid_think=False, logit_scale=1.0):
        """One token from one row of device logits [vocab] (a float32 cuda tensor)."""
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.numel() == self.vocab and logits.is_contiguous()
        rc = np.ascontiguousarray(np.asarray(recent, np.int32).reshape(-1))
        tok = C.c_int32()
        torch.cuda.synchronize()
        check(lib.spx_sample(self.h, _p(logits), logit_scale, rc.ctypes.data_as(P) if rc.size else None, rc.size,
                             int(forbid_stop), int(forbid_think), C.byref(tok)))
        return tok.value

    def sample_verify(self, logits, recent, draft, generated, max_accept, forbid_think=False, logit_scale=1.0):
        """The verify loop's sampling over rows 0..len(draft) of logits [>= len(draft)+1, vocab]."""
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.shape[-1] == self.vocab
        rc = np.ascontiguousarray(np.asarray(recent, np.int32).reshape(-1))
        dr = np.ascontiguousarray(np.asarray(draft, np.int32).reshape(-1))
        toks = np.empty(dr.size + 1, np.int32)
        n = C.c_int()
        torch.cuda.synchronize()
        check(lib.spx_sample_verify(self.h, _p(logits), logits.stride(0), dr.size, logit_scale,
                                    rc.ctypes.data_as(P) if rc.size else None, rc.size,
                                    dr.ctypes.data_as(P) if dr.size else None, generated, max_accept,
                                    int(forbid_think), toks.ctypes.data_as(P), C.byref(n)))
        return toks[:n.value]

    def close(self):
        if self.h:
            lib.spx_sampler_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
