"""Many requests at once over one paged KV cache held in 4 bits: rotary positions, append, read-back, attention.

`PagedContext` owns scratch memory only; cache, RoPE table and activations are the caller's CUDA tensors. Every method calls
straight into the C ABI of include/bonsai_paged.h, which says what each operator computes and how a pool's bytes are laid
out. Rows are tensors [tokens, heads, head_dim] of float16 or bfloat16 with any strides between tokens and heads; index
tensors are int32, slots int64.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .attention import _stream
from .errors import ConfigError, raise_for_status

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {None: 0, "linear": 1, "ntk": 2, "yarn": 3}
_DTYPES = {}


def _dtype(t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        code = {"torch.float16": 0, "torch.bfloat16": 1}.get(str(t.dtype))
        if code is None:
            raise ConfigError(f"invalid config: rows are float16 or bfloat16, not {t.dtype}")
        _DTYPES[t.dtype] = code
    return code


def _rows(t, what, like=None):
    shape = t.shape
    if len(shape) != 3:
        raise ConfigError(f"invalid config: {what} must be [tokens, heads, head_dim], not {tuple(shape)}")
    if like is not None and (shape != like.shape or t.dtype != like.dtype):
        raise ConfigError(f"invalid config: {what} must have the shape and type of the rows it goes with: {tuple(shape)} {t.dtype}, not {tuple(like.shape)} {like.dtype}")
    a, b, c = t.stride()
    if c != 1 and shape[2] > 1:
        raise ConfigError(f"invalid config: a row of {what} must be dense")
    return _lib.RowsStruct(t.data_ptr(), a, b)


def _index(t, what, n, dtype="torch.int32"):
    if str(t.dtype) != dtype or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ConfigError(f"invalid config: {what} must be {n} dense {dtype} values, not {tuple(t.shape)} {t.dtype}")
    return t.data_ptr()


def _weight(w, rows, what):
    if w is None:
        return None
    if w.dtype != rows.dtype or w.numel() != rows.shape[2] or not w.is_contiguous():
        raise ConfigError(f"invalid config: {what} must be {rows.shape[2]} dense values of the rows' type")
    return w.data_ptr()


class RopeTable:
    """A float32 CUDA tensor [positions, rot_dim / 2, 2] of (cos, sin) and the layout of the pairs: "half" or "interleaved"."""

    def __init__(self, data, layout="half"):
        if layout not in _LAYOUTS:
            raise ConfigError(f"invalid config: layout must be one of {sorted(_LAYOUTS)}, not {layout!r}")
        if str(data.dtype) != "torch.float32" or data.dim() != 3 or data.shape[2] != 2 or not data.is_contiguous():
            raise ConfigError("invalid config: a RoPE table is a dense float32 tensor [positions, rot_dim / 2, 2]")
        self.data = data
        self._c = _lib.RopeTableStruct(data.data_ptr(), data.shape[0], 2 * data.shape[1], _LAYOUTS[layout])


class KV4Pool:
    """The 4-bit pages of one layer in a uint8 CUDA tensor of at least KV4Pool.bytes(...) bytes."""

    def __init__(self, data, n_pages, page_tokens, n_kv_head, head_dim):
        need = KV4Pool.bytes(n_pages, page_tokens, n_kv_head, head_dim)
        if str(data.dtype) != "torch.uint8" or not data.is_contiguous() or data.numel() < need:
            raise ConfigError(f"invalid config: a pool of this shape is a dense uint8 tensor of at least {need} bytes")
        self.data, self.n_kv_head, self.head_dim = data, n_kv_head, head_dim
        self._c = _lib.PoolStruct(data.data_ptr(), n_pages, page_tokens, n_kv_head, head_dim)

    @staticmethod
    def bytes(n_pages, page_tokens, n_kv_head, head_dim):
        n = _lib.load().bp_kv4_pool_bytes(_lib.PoolStruct(None, n_pages, page_tokens, n_kv_head, head_dim)) if min(n_pages, page_tokens, n_kv_head, head_dim) > 0 else 0
        if n == 0:
            raise ConfigError("invalid config: a pool has n_pages >= 1, page_tokens 16, 32 or 64, n_kv_head >= 1 and head_dim 64 or 128")
        return n


class PagedContext:
    """Scratch memory and errors of the paged operators on one device."""

    def __init__(self, device=0):
        self._lib = _lib.load()
        self._h = C.c_void_p()
        st = self._lib.bp_paged_create(device, C.byref(self._h))
        if st != 0:
            msg = self._message()
            self.close()
            raise_for_status(st, msg)

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
        self._check(self._lib.bp_paged_status(self._h, _stream(stream)))

    def fill_rope(self, out, freq_base=1e6, scaling=None, factor=1.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=0, stream=None):
        """Fills a float32 tensor [positions, rot_dim / 2, 2]; scaling: None, "linear", "ntk" or "yarn"."""
        if scaling not in _SCALINGS:
            raise ConfigError(f"invalid config: scaling must be one of None, 'linear', 'ntk', 'yarn', not {scaling!r}")
        RopeTable(out)
        cfg = _lib.RopeConfigStruct(out.shape[0], 2 * out.shape[1], _SCALINGS[scaling], freq_base, factor, beta_fast, beta_slow, orig_ctx)
        self._check(self._lib.bp_rope_fill(self._h, _stream(stream), C.byref(cfg), out.data_ptr()))

    def rope(self, x, out, positions, table, w_norm=None, eps=1e-6, inverse=False, stream=None):
        """x [tokens, heads, head_dim] -> out (may be x): RMS norm over the head if w_norm is given, then the rotation by `positions`."""
        rx, ro = _rows(x, "x"), _rows(out, "out", x)
        n, heads, dim = x.shape
        self._check(self._lib.bp_rope(self._h, _stream(stream), _dtype(x), rx, ro, n, heads, dim, _index(positions, "positions", n), table._c,
                                      _weight(w_norm, x, "w_norm"), eps, inverse))

    def append(self, pool, k, v, positions, slots, table=None, w_k_norm=None, eps=1e-6, stream=None):
        """k, v [tokens, KV heads, head_dim] -> the pool at `slots`; K is normalised (w_k_norm) and rotated (table) on the way."""
        rk, rv = _rows(k, "k"), _rows(v, "v", k)
        n = self._fits(pool, k)
        self._check(self._lib.bp_kv4_append(self._h, _stream(stream), _dtype(k), pool._c, rk, rv, n,
                                            None if positions is None else _index(positions, "positions", n), _index(slots, "slots", n, "torch.int64"),
                                            None if table is None else table._c, _weight(w_k_norm, k, "w_k_norm"), eps))

    def read(self, pool, slots, k, v, stream=None):
        """The pool's rows at `slots` -> k, v [tokens, KV heads, head_dim]; keys are as they were stored."""
        rk, rv = _rows(k, "k"), _rows(v, "v", k)
        n = self._fits(pool, k)
        self._check(self._lib.bp_kv4_read(self._h, _stream(stream), _dtype(k), pool._c, _index(slots, "slots", n, "torch.int64"), n, rk, rv))

    def attention(self, pool, q, out, q_start, kv_len, page_table, max_q, max_kv, scale=None, window=0, stream=None):
        """q [tokens of all requests, heads, head_dim] -> out. Request r has the rows q_start[r] .. q_start[r + 1] and sees kv_len[r] keys in
        the pages page_table[r]; max_q, max_kv: no request has more. scale: 1 / sqrt(head_dim) if None; window: 0 = none."""
        rq, ro = _rows(q, "q"), _rows(out, "out", q)
        n, heads, dim = q.shape
        if dim != pool.head_dim:
            raise ConfigError(f"invalid config: q has head_dim {dim}, the pool {pool.head_dim}")
        n_req = kv_len.shape[0]
        if page_table.dim() != 2 or page_table.shape[0] != n_req or str(page_table.dtype) != "torch.int32" or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ConfigError(f"invalid config: page_table must be int32 [{n_req}, pages] with dense rows")
        if min(max_q, max_kv, window) < 0:
            raise ConfigError("invalid config: max_q, max_kv and window must be >= 0")
        if n_req > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ConfigError("invalid config: the rows of page_table must not overlap")
        # (what a row of the table holds bounds the keys that are looked at, not the distance of two rows)
        cap = page_table.shape[1] * pool._c.page_tokens
        a = _lib.AttnStruct(rq, ro, _index(q_start, "q_start", n_req + 1), _index(kv_len, "kv_len", n_req), page_table.data_ptr(),
                            n_req, heads, n, max_q, min(max_kv, cap), page_table.stride(0) if n_req > 1 else page_table.shape[1], window,
                            dim ** -0.5 if scale is None else scale)
        self._check(self._lib.bp_kv4_attention(self._h, _stream(stream), _dtype(q), pool._c, a))

    @staticmethod
    def _fits(pool, rows):
        if rows.shape[1] != pool.n_kv_head or rows.shape[2] != pool.head_dim:
            raise ConfigError(f"invalid config: the pool holds {pool.n_kv_head} heads of {pool.head_dim}, the rows have {tuple(rows.shape[1:])}")
        return rows.shape[0]
