"""Page tables, shared prefixes and chosen pages without a GPU: the header, its ctypes and Rust tables, what is refused before a kernel could run."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import bonsai_pot_b200 as bp
from bonsai_pot_b200 import _lib, paged
from tests import pages_ref as P
from tests.test_ffi_crate import header_functions, rust_functions
from tests.test_paged_wrapper import Owner, Recorder

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "bonsai_pages.h")
RS = os.path.join(ROOT, "ffi", "bonsai-attn-sys", "src", "pages.rs")
STRUCTS = {"bp_page_tables": _lib.PageTablesStruct, "bp_page_array": _lib.PageArrayStruct, "bp_kv4_shared": _lib.SharedStruct, "bp_block_summary": _lib.SummaryStruct,
           "bp_kv4_choice": _lib.ChoiceStruct, "bp_kv4_chosen": _lib.ChosenStruct}


def test_ctypes_and_rust_tables_cover_the_header():
    h = header_functions(HEADER)
    lib = _lib.load()
    assert sorted(h) == sorted(_lib.PAGES_SIGNATURES) and len(h) == 10
    for name, (n_args, is_void) in h.items():
        assert hasattr(lib, name)
        res, args = _lib.PAGES_SIGNATURES[name]
        assert len(args) == n_args and (res is None) == is_void, name
    assert h == rust_functions(RS)
    assert "pub mod pages;" in open(os.path.join(os.path.dirname(RS), "lib.rs")).read()


def test_structs_match_the_header():
    head, rust = (re.sub(r"/\*.*?\*/|//[^\n]*", "", open(p).read(), flags=re.S) for p in (HEADER, RS))
    size = {"uint32_t": 4, "uint64_t": 8, "float": 4, "bp_rows": C.sizeof(_lib.RowsStruct)}
    for name, cls in STRUCTS.items():
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, head, flags=re.S).group(1)
        want = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            kind, star, names = re.match(r"(?:const )?(\w+)(\*?) (.*)", decl, flags=re.S).groups()
            want += [(n.strip().lstrip("*"), 8 if star or "*" in n else size[kind]) for n in names.split(",")]
        assert [(f[0], C.sizeof(f[1])) for f in cls._fields_] == want, name
        fields = re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, flags=re.S).group(1)
        assert re.findall(r"pub (\w+):", fields) == [n for n, _ in want], name


def test_nothing_runs_without_a_context():
    lib = _lib.load()
    assert lib.bp_pages_grow(None, None, None, None, None, None, None, 0) == 7
    assert lib.bp_pages_release(None, None, None, None, 0) == 7
    assert lib.bp_pages_fork(None, None, None, None, None, 0, None, None) == 7
    assert lib.bp_pages_compact(None, None, None, None, None, 0) == 7
    assert lib.bp_pages_copy(None, None, None, 0, 0, None, None, 0) == 7
    assert lib.bp_kv4_attention_shared(None, None, 0, None, None) == 7
    assert lib.bp_kv4_summarise(None, None, None, None, None, None, 0) == 7
    assert lib.bp_kv4_select(None, None, 0, None, None, None) == 7
    assert lib.bp_kv4_attention_selected(None, None, 0, None, None) == 7
    assert lib.bp_kv4_shared_work(3, 4, 64) == 2 * 3 * 4 * 68 and lib.bp_kv4_shared_work(1 << 31, 64, 128) == (1 << 38) * 132


@pytest.fixture
def ctx():
    c = paged.PagedContext.__new__(paged.PagedContext)
    c._lib, c._h, c._device = Recorder(), C.c_void_p(), 0
    c._setup()
    return c


I32 = dict(dtype=torch.int32)


def calls(ctx, owner, n=3):
    x, i, table = torch.zeros(n, 2, 64, dtype=torch.float16), torch.zeros(n, **I32), torch.zeros(1, 2, **I32)
    return {
        "grow": lambda **kw: ctx.grow(owner, i[:1], i[:2], i, torch.arange(n), **kw),
        "release": lambda **kw: ctx.release(owner, i, **kw),
        "fork": lambda **kw: ctx.fork(owner, i, i, i, i, **kw),
        "compact": lambda **kw: ctx.compact(owner, i, i, **kw),
        "copy_pages": lambda **kw: ctx.copy_pages(owner, i, i, **kw),
        "attention_shared": lambda **kw: ctx.attention_shared(owner, x, x, i[:2], i[:1], table, i[:2], i[:1], table, torch.zeros(4096), max_q=1, max_kv=1, max_prefix=1, **kw),
        "summarise": lambda **kw: ctx.summarise(owner, owner, i, **kw),
        "select": lambda **kw: ctx.select(owner, owner, x, torch.zeros(n, 2, 4, **I32), i, i[:2], i[:1], table, max_q=1, max_kv=1, **kw),
        "attention_selected": lambda **kw: ctx.attention_selected(owner, x, x, torch.zeros(n, 2, 4, **I32), i, **kw),
    }


class Any(Owner):
    """A table, a pool, pools and a summary as the context sees them."""
    n_rows, n_arrays, n_pages, shape = 1, 1, 7, (7, 2, 64)
    _c = type("S", (), {"n_pages": 7})()

    def __init__(self, device):
        super().__init__(device)
        self.table = self.data = self.codes = torch.zeros(1)
        self.pools = [self]


def test_host_tensors_and_other_devices_do_not_reach_a_kernel(ctx):
    for owner in (Any(0), Any(1), Any(-1)):
        for name, call in calls(ctx, owner).items():
            with pytest.raises(bp.ConfigError, match="^invalid config: .* must be on cuda:0, not on "):
                call()
    # the context's own (noted as the host's), some of the call's tensors not on it
    assert ctx._lib.calls == []


def test_without_a_stream_a_call_goes_to_the_current_one(ctx, monkeypatch):
    ctx._device = -1
    monkeypatch.setattr(paged, "_current", lambda device: 4711, raising=False)
    monkeypatch.setattr(ctx._lib.__class__, "bp_kv4_shared_work", lambda self, *a: 1, raising=False)
    for stream, want in ((None, 4711), (99, 99), (0, 0)):
        for call in calls(ctx, Any(-1)).values():
            call(stream=stream)
        assert [args[1] for _, args in ctx._lib.calls] == [want] * 9
        ctx._lib.calls.clear()


def test_shapes_and_types_are_looked_at(ctx, monkeypatch):
    ctx._device = -1
    monkeypatch.setattr(paged, "_current", lambda device: 0, raising=False)
    monkeypatch.setattr(ctx._lib.__class__, "bp_kv4_shared_work", lambda self, *a: 100, raising=False)
    o, i, x = Any(-1), torch.zeros(3, **I32), torch.zeros(3, 2, 64, dtype=torch.float16)
    table, lists = torch.zeros(1, 2, **I32), torch.zeros(3, 2, 4, **I32)

    def shared(work=torch.zeros(100), prefix=table, start=i[:2], **kw):
        ctx.attention_shared(o, x, x, i[:2], i[:1], table, start, i[:1], prefix, work, **{**dict(max_q=1, max_kv=1, max_prefix=1), **kw})

    def select(pages=lists, keys=i, **kw):
        ctx.select(o, o, x, pages, keys, i[:2], i[:1], table, **{**dict(max_q=1, max_kv=1), **kw})

    shared(), select()
    n = len(ctx._lib.calls)
    odd = Any(-1)
    odd.shape = (7, 2, 128)
    bad = [
        lambda: ctx.grow(o, i, i[:2], i, torch.arange(3)),
        lambda: ctx.grow(o, i[:1], i[:1], i, torch.arange(3)),
        lambda: ctx.grow(o, i[:1], i[:2], i, torch.arange(2)),
        lambda: ctx.grow(o, i[:1], i[:2], i, i),
        lambda: ctx.release(o, i.long()),
        lambda: ctx.release(o, i.view(1, 3)),
        lambda: ctx.fork(o, i, i[:2], i, i),
        lambda: ctx.fork(o, i, i, i[:2], i),
        lambda: ctx.compact(o, i, i[:1]),
        lambda: ctx.copy_pages(o, i, i[:1]),
        lambda: ctx.copy_pages(o, i[::2], i[::2]),
        lambda: shared(work=torch.zeros(99)),
        lambda: shared(work=torch.zeros(100, dtype=torch.float64)),
        lambda: shared(prefix=table.long()),
        lambda: shared(start=i[:1]),
        lambda: shared(max_q=-1),
        lambda: shared(max_prefix=-1),
        lambda: shared(max_prefix=1 << 40, prefix=torch.empty(1, 1 << 28, **I32)),
        lambda: ctx.summarise(o, odd, i),
        lambda: ctx.summarise(o, o, i, i[:2]),
        lambda: ctx.summarise(o, o, i.long()),
        lambda: select(pages=lists[:2]),
        lambda: select(pages=lists[:, :1]),
        lambda: select(pages=lists.long()),
        lambda: select(keys=i[:2]),
        lambda: select(first=-1),
        lambda: select(last=1 << 32),
        lambda: ctx.attention_selected(o, x, x[:2], lists, i),
        lambda: ctx.attention_selected(o, x[..., :32], x[..., :32], lists, i),
        lambda: ctx.attention_selected(o, x.float(), x.float(), lists, i),
        lambda: bp.PageTables(table, i[:1], i, 16),  # not on a CUDA device
        lambda: bp.PageTables(table.long(), i[:1], i, 16),
        lambda: bp.BlockSummary(torch.zeros(7, 2, 2, 64, dtype=torch.int8), torch.zeros(7, 2)),
        lambda: bp.BlockSummary(torch.zeros(7, 2, 64, dtype=torch.int8), torch.zeros(7, 2)),
        lambda: bp.KV4Pools([]),
        lambda: ctx.shared_work(-1, 2, 64),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(bp.ConfigError, match="^invalid config: "):
            call()
        assert len(ctx._lib.calls) == n, k


def test_a_summary_bounds_the_scores_of_its_page():
    """Rounded up in 8 bits: score * the query's unit is no less than the sum of q . k over the group, but for the query's own rounding (half a unit of
    each of its codes, 127 steps of the summary at most)."""
    rng = np.random.default_rng(0)
    keys = rng.standard_normal((50, 16, 64)) * np.where(np.arange(64) % 9 == 0, 6, 1)
    codes, scale = P.summary(keys)
    assert (codes[:, 0] * scale[:, None].astype(np.float64) >= keys.max(1)).all() and (codes[:, 1] * scale[:, None].astype(np.float64) >= -keys.min(1)).all()
    assert (codes.max((1, 2)) > 63).all()  # (seven bits of them are used at least)
    q = rng.standard_normal((4, 64)).astype(np.float32)
    top = max(np.maximum(q, 0).sum(0).max(), np.maximum(-q, 0).sum(0).max())
    unit = 2.0 ** (np.frexp(top)[1] - 8)
    bound = P.scores(q, codes, scale) * unit
    most = (q.astype(np.float64)[None, None] * keys[:, :, None]).sum((2, 3)).max(1)
    assert (bound + 0.5 * unit * 128 * 127 * scale >= most).all()
