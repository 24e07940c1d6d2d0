"""Many requests at once over one paged KV cache held in 4 bits: rotary positions, append, read-back, attention; page tables on the device,
prefixes that requests have in common, attention over chosen pages.

`PagedContext` owns scratch memory only; cache, RoPE table and activations are the caller's CUDA tensors. Every method calls
straight into the C ABI of include/bonsai_paged.h and include/bonsai_pages.h, which say what each operator computes and how a pool's bytes are laid
out. Rows are tensors [tokens, heads, head_dim] of float16 or bfloat16 with any strides between tokens and heads; index
tensors are int32, slots int64. A call without a `stream` goes to torch's current stream of the context's device (the C entries' null
stream is CUDA's legacy default stream, for which torch's other streams do not wait).
"""
from __future__ import annotations

import ctypes as C
import struct

from . import _lib
from .attention import _stream
from .errors import ConfigError, raise_for_status

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {None: 0, "linear": 1, "ntk": 2, "yarn": 3}
_DTYPES, _I32, _I64, _F32 = {}, None, None, None
_U32 = 0xFFFFFFFF
# the structs of include/bonsai_pages.h up to their scale, written at once (a field at a time costs 60 ns each)
_SHARED, _CHOICE, _CHOSEN = struct.Struct("PqqPqq7P9I").pack_into, struct.Struct("Pqq5P9I").pack_into, struct.Struct("PqqPqq2P3I").pack_into


def _types():
    """The torch types (the package itself does not import torch; whoever calls with tensors has)."""
    global _I32, _I64, _F32
    import torch
    _DTYPES.update({torch.float16: 0, torch.bfloat16: 1})
    _I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


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
    if _I32 is None:
        _types()
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


class KV4Pools:
    """The pools of a model's layers, of one shape, and their summaries: what copy_pages copies in one call."""

    def __init__(self, pools, summaries=()):
        self.pools, self.summaries = list(pools), list(summaries)
        if not self.pools:
            _bad("at least one pool")
        one = self.pools[0]
        self.device, self.n_pages = one.device, one._c.n_pages
        for p in self.pools:
            if p.device != self.device or (p._c.n_pages, p.page_tokens, p.n_kv_head, p.head_dim) != (self.n_pages, one.page_tokens, one.n_kv_head, one.head_dim):
                _bad("the pools must have one shape and lie on one device")
        arrays = [(p.data.data_ptr(), one.page_tokens * one.n_kv_head * one.head_dim * 5 // 4) for p in self.pools]
        for s in self.summaries:
            if s.device != self.device or s.codes.shape[0] != self.n_pages:
                _bad("the summaries must have the pools' number of pages and lie on their device")
            arrays += [(s.codes.data_ptr(), s.codes[0].numel()), (s.scales.data_ptr(), 4 * s.scales.shape[1])]
        self.n_arrays = len(arrays)
        self._c = (_lib.PageArrayStruct * self.n_arrays)(*[_lib.PageArrayStruct(*a) for a in arrays])
        self._p = C.addressof(self._c)


class PageTables:
    """int32 CUDA tensors: table [rows, pages of a row], kv_len [rows], refs [pages of the pool] (how often a page is held; 0 is free)."""

    def __init__(self, table, kv_len, refs, page_tokens):
        for t, what, n in ((table, "table", 2), (kv_len, "kv_len", 1), (refs, "refs", 1)):
            if str(t.dtype) != "torch.int32" or t.dim() != n:
                _bad(f"{what} must be an int32 tensor of {n} dimension{'s' * (n > 1)}, not {tuple(t.shape)} {t.dtype}")
            if not t.is_cuda or t.get_device() != table.get_device():
                _bad(f"{what} must be on the CUDA device of the others, not on {t.device}")
        n_rows, row_pages = table.shape
        if (table.stride(1) != 1 and row_pages > 1) or (n_rows > 1 and table.stride(0) < row_pages) or not kv_len.is_contiguous() or not refs.is_contiguous():
            _bad("the rows of table must be dense and not overlap, kv_len and refs dense")
        if kv_len.shape[0] != n_rows or page_tokens not in (16, 32, 64):
            _bad("kv_len must have an entry per row of table, page_tokens must be 16, 32 or 64")
        pitch = table.stride(0) if n_rows > 1 else row_pages
        if max(n_rows, row_pages, pitch, refs.shape[0]) > _U32:
            _bad("page tables have fewer than 2^32 rows, pages and elements between rows")
        self.table, self.kv_len, self.refs, self.page_tokens, self.device = table, kv_len, refs, page_tokens, table.get_device()
        self._c = _lib.PageTablesStruct(table.data_ptr(), kv_len.data_ptr(), refs.data_ptr(), n_rows, row_pages, pitch, refs.shape[0], page_tokens)
        self._p, self.n_rows = C.addressof(self._c), n_rows


class BlockSummary:
    """What select() goes by: int8 CUDA tensor codes [pages, KV heads, 2, head_dim] and float32 scales [pages, KV heads]."""

    def __init__(self, codes, scales):
        if str(codes.dtype) != "torch.int8" or codes.dim() != 4 or codes.shape[2] != 2 or not codes.is_contiguous():
            _bad("codes are a dense int8 tensor [pages, KV heads, 2, head_dim]")
        if str(scales.dtype) != "torch.float32" or scales.shape != codes.shape[:2] or not scales.is_contiguous():
            _bad("scales are a dense float32 tensor [pages, KV heads]")
        if not codes.is_cuda or codes.get_device() != scales.get_device():
            _bad("codes and scales must be on one CUDA device")
        self.codes, self.scales, self.device = codes, scales, codes.get_device()
        self.shape = (codes.shape[0], codes.shape[1], codes.shape[3])
        self._c = _lib.SummaryStruct(codes.data_ptr(), scales.data_ptr())
        self._p = C.addressof(self._c)


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
        self._shared, self._choice, self._chosen = _lib.SharedStruct(), _lib.ChoiceStruct(), _lib.ChosenStruct()
        self._pshared, self._pchoice, self._pchosen = C.addressof(self._shared), C.addressof(self._choice), C.addressof(self._chosen)

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

    # ---- page tables ----

    def _tables(self, tables):
        if tables.device != self._device:
            _elsewhere(tables.table, "the page tables", self._device)
        return tables._p

    def _pairs(self, a, b, what_a, what_b):
        """Two int32 tensors of one length; the length and the addresses."""
        n = a.shape[0] if a.dim() == 1 else -1
        return n, _index(a, what_a, n, self._device), _index(b, what_b, n, self._device)

    def grow(self, tables, n_new, q_start, positions, slots, stream=None):
        """Every row gets n_new[row] further tokens and the pages for them; q_start [rows + 1], positions and (int64) slots [at least the
        new tokens] are written for what is done with the tokens, -1 behind the last."""
        device, n = self._device, positions.shape[0] if positions.dim() == 1 else -1
        p, rows = self._tables(tables), tables.n_rows
        at = (_index(n_new, "n_new", rows, device), _index(q_start, "q_start", rows + 1, device), _index(positions, "positions", n, device), _index(slots, "slots", n, device, True))
        st = self._lib.bp_pages_grow(self._h, _current(device) if stream is None else _stream(stream), p, *at, n)
        if st:
            self._check(st)

    def release(self, tables, rows, stream=None):
        """The rows (int32; negative: none) give their pages back and are empty."""
        device, n, p = self._device, rows.shape[0] if rows.dim() == 1 else -1, self._tables(tables)
        rows = _index(rows, "rows", n, device)
        st = self._lib.bp_pages_release(self._h, _current(device) if stream is None else _stream(stream), p, rows, n)
        if st:
            self._check(st)

    def fork(self, tables, parents, children, src, dst, stream=None):
        """Empty rows `children` become what `parents` are: full pages are shared, src and dst say which pages are to be copied (copy_pages)."""
        p, device = self._tables(tables), self._device
        n, parents, children = self._pairs(parents, children, "parents", "children")
        src, dst = _index(src, "src", n, device), _index(dst, "dst", n, device)
        st = self._lib.bp_pages_fork(self._h, _current(device) if stream is None else _stream(stream), p, parents, children, n, src, dst)
        if st:
            self._check(st)

    def compact(self, tables, src, dst, stream=None):
        """The highest used pages move into the lowest free ones, as many as src and dst have places; these say which pages are to be copied (copy_pages)."""
        p = self._tables(tables)
        n, src, dst = self._pairs(src, dst, "src", "dst")
        st = self._lib.bp_pages_compact(self._h, _current(self._device) if stream is None else _stream(stream), p, src, dst, n)
        if st:
            self._check(st)

    def copy_pages(self, pools, src, dst, stream=None):
        """Page src[i] of every pool and summary of a KV4Pools goes to page dst[i] (int32; a negative one of either: nothing)."""
        if pools.device != self._device:
            _elsewhere(pools.pools[0].data, "the pools", self._device)
        n, src, dst = self._pairs(src, dst, "src", "dst")
        st = self._lib.bp_pages_copy(self._h, _current(self._device) if stream is None else _stream(stream), pools._p, pools.n_arrays, pools.n_pages, src, dst, n)
        if st:
            self._check(st)

    # ---- a prefix in common; chosen pages ----

    def _table(self, t, what, page_tokens, most):
        """A page table's requests, address and pitch, and `most` cut to the keys that a row has pages for."""
        if t.get_device() != self._device:
            _elsewhere(t, what, self._device)
        shape, stride = t.shape, t.stride()
        if t.dtype is not _I32 or len(shape) != 2:
            _bad(f"{what} must be int32 [rows, pages]")
        (n, pages), (pitch, dense) = shape, stride
        if (dense != 1 and pages > 1) or (pitch < pages and n > 1):
            _bad(f"the rows of {what} must be dense and not overlap")
        if most < 0:
            _bad("the largest numbers of queries and keys must be >= 0")
        if most > pages * page_tokens:
            most = pages * page_tokens
        if n <= 1:
            pitch = pages
        if most > _U32 or pitch > _U32:
            _bad(f"the keys and the distance of two rows of {what} must be below 2^32")
        return n, t.data_ptr(), pitch, most

    def _queries(self, pool, q, what="q"):
        """The shape of q (or out), its address and strides."""
        if q.get_device() != self._device:
            _elsewhere(q, what, self._device)
        shape, stride = q.shape, q.stride()
        if len(stride) != 3:
            _bad(f"{what} must be [tokens, heads, head_dim], not {tuple(shape)}")
        if stride[2] != 1 and shape[2] > 1:
            _bad(f"a row of {what} must be dense")
        if pool.device != self._device:
            _elsewhere(pool.data, "the pool", self._device)
        if shape[2] != pool.head_dim:
            _bad(f"{what} has head_dim {shape[2]}, the pool {pool.head_dim}")
        return shape, q.data_ptr(), stride[0], stride[1]

    def shared_work(self, total_q, n_head, head_dim):
        """float32 values of attention_shared's `work` for that many rows."""
        if not (0 <= total_q <= _U32 and 0 <= n_head <= _U32 and 0 <= head_dim <= _U32):
            _bad("total_q, n_head and head_dim must be >= 0 and below 2^32")
        return self._lib.bp_kv4_shared_work(total_q, n_head, head_dim)

    def attention_shared(self, pool, q, out, q_start, kv_len, page_table, prefix_start, prefix_len, prefix_table, work, max_q, max_kv, max_prefix, scale=None, stream=None):
        """attention() for requests behind prefixes in common: the requests prefix_start[g] .. prefix_start[g + 1] see the prefix_len[g] keys in the
        pages prefix_table[g], then their own. work: a float32 tensor of at least shared_work(...) values, for this call's partial results."""
        a, device, dtype = self._shared, self._device, q.dtype
        code = _code(dtype)
        shape, *rows = self._queries(pool, q)
        _like(out, dtype, shape, "out")
        n_req, table, pitch, max_kv = self._table(page_table, "page_table", pool.page_tokens, max_kv)
        n_prefix, prefix, prefix_pitch, max_prefix = self._table(prefix_table, "prefix_table", pool.page_tokens, max_prefix)
        total, heads, dim = shape
        if max_q < 0:
            _bad("max_q must be >= 0")
        if work.get_device() != device:
            _elsewhere(work, "work", device)
        if work.dtype is not _F32 or not work.is_contiguous() or work.numel() < self._lib.bp_kv4_shared_work(total, heads, dim):
            _bad("work must be dense float32 of at least shared_work(total_q, n_head, head_dim) values")
        _SHARED(a, 0, *rows, *self._queries(pool, out, "out")[1:], _index(q_start, "q_start", n_req + 1, device), _index(kv_len, "kv_len", n_req, device), table,
                _index(prefix_start, "prefix_start", n_prefix + 1, device), _index(prefix_len, "prefix_len", n_prefix, device), prefix, work.data_ptr(),
                n_req, heads, total, max_q if max_q < total else total, max_kv, pitch, n_prefix, max_prefix, prefix_pitch)
        a.scale = dim ** -0.5 if scale is None else scale
        st = self._lib.bp_kv4_attention_shared(self._h, _current(device) if stream is None else _stream(stream), code, pool._p, self._pshared)
        if st:
            self._check(st)

    def _summary(self, pool, summary):
        if summary.device != self._device:
            _elsewhere(summary.codes, "the summary", self._device)
        if pool.device != self._device:
            _elsewhere(pool.data, "the pool", self._device)
        if summary.shape != (pool._c.n_pages, pool.n_kv_head, pool.head_dim):
            _bad(f"the summary is of {summary.shape} pages, KV heads and dims, the pool of {(pool._c.n_pages, pool.n_kv_head, pool.head_dim)}")
        return summary._p

    def summarise(self, pool, summary, pages, n_tok=None, stream=None):
        """The summaries of `pages` (int32; negative: none), of all their tokens or the first n_tok (int32) of each."""
        p, n, device = self._summary(pool, summary), pages.shape[0] if pages.dim() == 1 else -1, self._device
        pages, n_tok = _index(pages, "pages", n, device), None if n_tok is None else _index(n_tok, "n_tok", n, device)
        st = self._lib.bp_kv4_summarise(self._h, _current(device) if stream is None else _stream(stream), pool._p, p, pages, n_tok, n)
        if st:
            self._check(st)

    def select(self, pool, summary, q, pages, keys, q_start, kv_len, page_table, max_q, max_kv, first=1, last=1, stream=None):
        """For every token and KV head the pages with the highest scores among those it sees, as many as pages [tokens, KV heads, pages] (int32) has
        places, the first `first` and last `last` always; keys [tokens] (int32): the keys in them."""
        p, device = self._summary(pool, summary), self._device
        code = _code(q.dtype)
        (total, heads, _), *rows = self._queries(pool, q)
        n_req, table, pitch, max_kv = self._table(page_table, "page_table", pool.page_tokens, max_kv)
        pages, chosen = self._lists(pool, pages, total)
        if max_q < 0 or not (0 <= first <= _U32 and 0 <= last <= _U32) or chosen > _U32:
            _bad("max_q, first, last and the places of pages must be >= 0 and below 2^32")
        _CHOICE(self._choice, 0, *rows, _index(q_start, "q_start", n_req + 1, device), _index(kv_len, "kv_len", n_req, device), table, pages, _index(keys, "keys", total, device),
                n_req, heads, total, max_q if max_q < total else total, max_kv, pitch, chosen, first, last)
        st = self._lib.bp_kv4_select(self._h, _current(device) if stream is None else _stream(stream), code, pool._p, p, self._pchoice)
        if st:
            self._check(st)

    def _lists(self, pool, pages, n):
        if pages.get_device() != self._device:
            _elsewhere(pages, "pages", self._device)
        shape = pages.shape
        if pages.dtype is not _I32 or len(shape) != 3 or shape[0] != n or shape[1] != pool.n_kv_head or not pages.is_contiguous():
            _bad(f"pages must be dense int32 [{n}, {pool.n_kv_head}, pages], not {tuple(shape)} {pages.dtype}")
        return pages.data_ptr(), shape[2]

    def attention_selected(self, pool, q, out, pages, keys, scale=None, stream=None):
        """Attention of every token of q [tokens, heads, head_dim] over the pages that select() has chosen for it."""
        a, device, dtype = self._chosen, self._device, q.dtype
        code = _code(dtype)
        shape, *rows = self._queries(pool, q)
        _like(out, dtype, shape, "out")
        total, heads, dim = shape
        pages, chosen = self._lists(pool, pages, total)
        if chosen > _U32:
            _bad("the places of pages must be below 2^32")
        _CHOSEN(a, 0, *rows, *self._queries(pool, out, "out")[1:], pages, _index(keys, "keys", total, device), heads, total, chosen)
        a.scale = dim ** -0.5 if scale is None else scale
        st = self._lib.bp_kv4_attention_selected(self._h, _current(device) if stream is None else _stream(stream), code, pool._p, self._pchosen)
        if st:
            self._check(st)
