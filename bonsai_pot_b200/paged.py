"""Many requests at once over one paged KV cache held in 4 bits: rotary positions, append, read-back, attention.

`PagedContext` owns scratch memory only; cache, RoPE table and activations are the caller's CUDA tensors. Every method calls
straight into the C ABI of include/bonsai_paged.h, which says what each operator computes and how a pool's bytes are laid
out. Rows are tensors [tokens, heads, head_dim] of float16 or bfloat16 with any strides between tokens and heads; index
tensors are int32, slots int64. A call without a `stream` goes to torch's current stream of the context's device (the C entries' null
stream is CUDA's legacy default stream, for which torch's other streams do not wait).
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .attention import _stream
from .errors import ConfigError, raise_for_status

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {None: 0, "linear": 1, "ntk": 2, "yarn": 3}
_DTYPES, _I32, _I64 = {}, None, None
_U32 = 0xFFFFFFFF


def _types():
    """The torch types (the package itself does not import torch; whoever calls with tensors has)."""
    global _I32, _I64
    import torch
    _DTYPES.update({torch.float16: 0, torch.bfloat16: 1})
    _I32, _I64 = torch.int32, torch.int64


def _current(device):
    """The handle of torch's current stream; the first call puts torch's own function here."""
    global _current
    import torch
    _current = torch._C._cuda_getCurrentRawStream
    return _current(device)


def _bad(text):
    raise ConfigError("invalid config: " + text)


def _code(dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        _types()
        code = _DTYPES.get(dtype)
        if code is None:
            _bad(f"rows are float16 or bfloat16, not {dtype}")
    return code


# The checks below are on the path of every call (a decoded token makes three of them per layer), hence as few tensor methods as will do (each
# takes 50 to 130 ns, and a shape is made anew whenever it is asked for).
def _elsewhere(t, what, device):
    """An address of host memory or of another device must not reach a kernel."""
    _bad(f"{what} must be on cuda:{device}, not on {t.device}")


def _rows(to, t, what, device):
    """t's address and strides into a RowsStruct."""
    if t.get_device() != device:
        _elsewhere(t, what, device)
    strides = t.stride()
    if len(strides) != 3:
        _bad(f"{what} must be [tokens, heads, head_dim], not {tuple(t.shape)}")
    to.tok_stride, to.head_stride, dense = strides
    if dense != 1 and t.shape[2] > 1:
        _bad(f"a row of {what} must be dense")
    to.data = t.data_ptr()


def _like(t, dtype, shape, what):
    if t.dtype is not dtype or t.shape != shape:
        _bad(f"{what} must have the shape and type of the rows it goes with: {tuple(t.shape)} {t.dtype}, not {tuple(shape)} {dtype}")


def _index(t, what, n, device, slots=False):
    if t.get_device() != device:
        _elsewhere(t, what, device)
    if t.dtype is not (_I64 if slots else _I32) or t.shape != (n,) or not t.is_contiguous():
        _bad(f"{what} must be {n} dense values of {_I64 if slots else _I32}, not {tuple(t.shape)} {t.dtype}")
    return t.data_ptr()


def _weight(w, dtype, dim, what, device):
    if w.get_device() != device:
        _elsewhere(w, what, device)
    if w.dtype is not dtype or w.numel() != dim or not w.is_contiguous():
        _bad(f"{what} must be {dim} dense values of the rows' type")
    return w.data_ptr()


class RopeTable:
    """A float32 CUDA tensor [positions, rot_dim / 2, 2] of (cos, sin) and the layout of the pairs: "half" or "interleaved"."""

    def __init__(self, data, layout="half"):
        if layout not in _LAYOUTS:
            raise ConfigError(f"invalid config: layout must be one of {sorted(_LAYOUTS)}, not {layout!r}")
        if str(data.dtype) != "torch.float32" or data.dim() != 3 or data.shape[2] != 2 or not data.is_contiguous():
            raise ConfigError("invalid config: a RoPE table is a dense float32 tensor [positions, rot_dim / 2, 2]")
        if not data.is_cuda:
            _bad(f"a RoPE table must be on a CUDA device, not on {data.device}")
        self.data, self.device = data, data.get_device()
        self._c = _lib.RopeTableStruct(data.data_ptr(), data.shape[0], 2 * data.shape[1], _LAYOUTS[layout])
        self._p = C.addressof(self._c)


class KV4Pool:
    """The 4-bit pages of one layer in a uint8 CUDA tensor of at least KV4Pool.bytes(...) bytes."""

    def __init__(self, data, n_pages, page_tokens, n_kv_head, head_dim):
        need = KV4Pool.bytes(n_pages, page_tokens, n_kv_head, head_dim)
        if str(data.dtype) != "torch.uint8" or not data.is_contiguous() or data.numel() < need:
            raise ConfigError(f"invalid config: a pool of this shape is a dense uint8 tensor of at least {need} bytes")
        if not data.is_cuda:
            _bad(f"a pool must be on a CUDA device, not on {data.device}")
        self.data, self.device = data, data.get_device()
        self.page_tokens, self.n_kv_head, self.head_dim = page_tokens, n_kv_head, head_dim
        self._c = _lib.PoolStruct(data.data_ptr(), n_pages, page_tokens, n_kv_head, head_dim)
        self._p = C.addressof(self._c)

    @staticmethod
    def bytes(n_pages, page_tokens, n_kv_head, head_dim):
        n = _lib.load().bp_kv4_pool_bytes(C.byref(_lib.PoolStruct(None, n_pages, page_tokens, n_kv_head, head_dim))) if 0 < min(n_pages, page_tokens, n_kv_head, head_dim) and max(n_pages, page_tokens, n_kv_head, head_dim) <= _U32 else 0
        if n == 0:
            raise ConfigError("invalid config: a pool has n_pages >= 1, page_tokens 16, 32 or 64, n_kv_head >= 1 and head_dim 64 or 128")
        return n


class PagedContext:
    """Scratch memory and errors of the paged operators on one device, on which every tensor of a call must lie."""

    def __init__(self, device=0):
        self._lib = _lib.load()
        self._h = C.c_void_p()
        self._device = device
        self._setup()
        st = self._lib.bp_paged_create(device, C.byref(self._h))
        if st != 0:
            msg = self._message()
            self.close()
            raise_for_status(st, msg)

    def _setup(self):
        # arguments of a call, filled anew by every one (a context is not thread-safe)
        self._a, self._b, self._attn = _lib.RowsStruct(), _lib.RowsStruct(), _lib.AttnStruct()
        self._q, self._o = self._attn.q, self._attn.out
        self._pa, self._pb, self._pattn = C.addressof(self._a), C.addressof(self._b), C.addressof(self._attn)

    def _message(self):
        return (self._lib.bp_paged_last_error(self._h) or b"").decode() if self._h else ""

    def _check(self, st):
        if st != 0:
            raise_for_status(st, self._message() or self._lib.bp_strerror(st).decode())

    def close(self):
        if self._h:
            self._lib.bp_paged_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def status(self, stream=None):
        """Waits for `stream`; raises if a position, slot, page id or number of keys was out of range since the last call."""
        self._check(self._lib.bp_paged_status(self._h, _current(self._device) if stream is None else _stream(stream)))

    def fill_rope(self, out, freq_base=1e6, scaling=None, factor=1.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=0, stream=None):
        """Fills a float32 tensor [positions, rot_dim / 2, 2]; scaling: None, "linear", "ntk" or "yarn"."""
        if scaling not in _SCALINGS:
            raise ConfigError(f"invalid config: scaling must be one of None, 'linear', 'ntk', 'yarn', not {scaling!r}")
        if RopeTable(out).device != self._device:
            _elsewhere(out, "a RoPE table", self._device)
        cfg = _lib.RopeConfigStruct(out.shape[0], 2 * out.shape[1], _SCALINGS[scaling], freq_base, factor, beta_fast, beta_slow, orig_ctx)
        self._check(self._lib.bp_rope_fill(self._h, _current(self._device) if stream is None else _stream(stream), C.byref(cfg), out.data_ptr()))

    def rope(self, x, out, positions, table, w_norm=None, eps=1e-6, inverse=False, stream=None):
        """x [tokens, heads, head_dim] -> out (may be x): RMS norm over the head if w_norm is given, then the rotation by `positions`; inverse:
        its transpose, the gradient with respect to x."""
        dtype, shape, device = x.dtype, x.shape, self._device
        code = _code(dtype)
        _rows(self._a, x, "x", device)
        _like(out, dtype, shape, "out")
        _rows(self._b, out, "out", device)
        if table.device != device:
            _elsewhere(table.data, "the RoPE table", device)
        n, heads, dim = shape
        st = self._lib.bp_rope(self._h, _current(device) if stream is None else _stream(stream), code, self._pa, self._pb, n, heads, dim, _index(positions, "positions", n, device), table._p,
                               None if w_norm is None else _weight(w_norm, dtype, dim, "w_norm", device), eps, inverse)
        if st:
            self._check(st)

    def append(self, pool, k, v, positions, slots, table=None, w_k_norm=None, eps=1e-6, stream=None):
        """k, v [tokens, KV heads, head_dim] -> the pool at `slots`; K is normalised (w_k_norm) and rotated (table) on the way."""
        code, n, device = self._kv(pool, k, v)
        if table is not None and table.device != device:
            _elsewhere(table.data, "the RoPE table", device)
        st = self._lib.bp_kv4_append(self._h, _current(device) if stream is None else _stream(stream), code, pool._p, self._pa, self._pb, n,
                                     None if positions is None else _index(positions, "positions", n, device), _index(slots, "slots", n, device, True),
                                     None if table is None else table._p, None if w_k_norm is None else _weight(w_k_norm, k.dtype, pool.head_dim, "w_k_norm", device), eps)
        if st:
            self._check(st)

    def read(self, pool, slots, k, v, stream=None):
        """The pool's rows at `slots` -> k, v [tokens, KV heads, head_dim]; keys are as they were stored."""
        code, n, device = self._kv(pool, k, v)
        st = self._lib.bp_kv4_read(self._h, _current(device) if stream is None else _stream(stream), code, pool._p, _index(slots, "slots", n, device, True), n, self._pa, self._pb)
        if st:
            self._check(st)

    def attention(self, pool, q, out, q_start, kv_len, page_table, max_q, max_kv, scale=None, window=0, stream=None):
        """q [tokens of all requests, heads, head_dim] -> out. Request r has the rows q_start[r] .. q_start[r + 1] and sees kv_len[r] keys in
        the pages page_table[r]; max_q, max_kv: no request has more. scale: 1 / sqrt(head_dim) if None; window: 0 = none."""
        dtype, shape, a, device = q.dtype, q.shape, self._attn, self._device
        code = _code(dtype)
        _rows(self._q, q, "q", device)
        _like(out, dtype, shape, "out")
        _rows(self._o, out, "out", device)
        if pool.device != device:
            _elsewhere(pool.data, "the pool", device)
        if page_table.get_device() != device:
            _elsewhere(page_table, "page_table", device)
        n, heads, dim = shape
        if dim != pool.head_dim:
            _bad(f"q has head_dim {dim}, the pool {pool.head_dim}")
        if page_table.dtype is not _I32 or page_table.dim() != 2:
            _bad("page_table must be int32 [requests, pages]")
        (n_req, pages), (stride, dense) = page_table.shape, page_table.stride()
        if (dense != 1 and pages > 1) or (stride < pages and n_req > 1):
            _bad("the rows of page_table must be dense and not overlap")
        if max_q < 0 or max_kv < 0 or window < 0:
            _bad("max_q, max_kv and window must be >= 0")
        # (what a row of the table holds bounds the keys that are looked at, not the distance of two rows)
        cap = pages * pool.page_tokens
        if max_kv > cap:
            max_kv = cap
        pitch = stride if n_req > 1 else pages
        if max_kv > _U32 or pitch > _U32:  # (the C entry's numbers have 32 bits: what is longer would arrive as another number)
            _bad("max_kv and the distance of two rows of page_table must be below 2^32")
        a.q_start, a.kv_len, a.page_table = _index(q_start, "q_start", n_req + 1, device), _index(kv_len, "kv_len", n_req, device), page_table.data_ptr()
        a.n_req, a.n_head, a.total_q, a.max_q, a.max_kv = n_req, heads, n, max_q if max_q < n else n, max_kv
        a.window = window if window < max_kv else 0  # (a window over all keys is none)
        a.table_stride = pitch
        a.scale = dim ** -0.5 if scale is None else scale
        st = self._lib.bp_kv4_attention(self._h, _current(device) if stream is None else _stream(stream), code, pool._p, self._pattn)
        if st:
            self._check(st)

    def _kv(self, pool, k, v):
        dtype, shape, device = k.dtype, k.shape, self._device
        code = _code(dtype)
        _rows(self._a, k, "k", device)
        _like(v, dtype, shape, "v")
        _rows(self._b, v, "v", device)
        if pool.device != device:
            _elsewhere(pool.data, "the pool", device)
        n, heads, dim = shape
        if heads != pool.n_kv_head or dim != pool.head_dim:
            _bad(f"the pool holds {pool.n_kv_head} heads of {pool.head_dim}, the rows have {heads} of {dim}")
        return code, n, device
