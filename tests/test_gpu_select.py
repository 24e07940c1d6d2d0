"""Summaries of pages, the choice among them and attention over the chosen ones, on the GPU against their definitions (tests/pages_ref.py).

Summaries and choices are whole numbers (and powers of two): equal. Attention over chosen pages: as bp_kv4_attention (tests/test_gpu_paged.py)."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests import pages_ref as P  # noqa: E402
from tests import paged_ref as R  # noqa: E402
from tests.test_gpu_paged import HALF_UNIT, HEADS, Requests, f64, normal, strided  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bp.PagedContext()
    yield c
    c.status()
    c.close()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def keys_of_pages(ref, pages, n_tok=None):
    """[pages, heads, tokens, dims]"""
    return np.stack([np.stack([ref.read(0, int(p) * ref.page + t) for t in range(ref.page)], 1) for p in pages])


# ---- summaries -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("hkv", [1, 3, 8])
@pytest.mark.parametrize("gain", [0.0, 1e-7, 1.0, 3e4])
def test_summaries(ctx, dim, page, hkv, gain):
    rng = np.random.default_rng(dim + page)
    n_pages = 7
    ref = R.Pool(n_pages, page, hkv, dim, fill=0xFF)
    x = (rng.standard_normal((n_pages * page, hkv, dim)) * gain).astype(np.float32)
    x[:page, :, 5] = 0.5 * gain  # the same in every token
    x[page:2 * page] = -np.abs(x[page:2 * page])
    ref.write(0, np.arange(n_pages * page), *R.quantise(x))
    pool = bp.KV4Pool(torch.from_numpy(ref.bytes).cuda(), n_pages, page, hkv, dim)
    codes, scales = torch.full((n_pages, hkv, 2, dim), 9, dtype=torch.int8, device="cuda"), torch.full((n_pages, hkv), 9.0, device="cuda")
    summary = bp.BlockSummary(codes, scales)
    pages, n_tok = [6, 0, -1, 1, 4], [page, 1, 5, page - 1, 3]
    ctx.summarise(pool, summary, i32(pages), i32(n_tok))
    want_c, want_s = codes.cpu().numpy() * 0 + 9, scales.cpu().numpy() * 0 + 9

    def put(p, n):
        want_c[p], want_s[p] = P.summary(keys_of_pages(ref, [p])[0][:, :n])

    for p, n in zip(pages, n_tok):
        if p >= 0:
            put(p, n)
    assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(scales.cpu().numpy(), want_s)
    ctx.summarise(pool, summary, i32(range(n_pages)))
    for p in range(n_pages):
        put(p, page)
    assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(scales.cpu().numpy(), want_s)
    ctx.status()
    for p, n in ((n_pages, 1), (1 << 30, 1), (2, 0), (2, page + 1), (2, -1)):
        ctx.summarise(pool, summary, i32([p]), i32([n]))
        with pytest.raises(bp.ContextOverflow):
            ctx.status()
    assert np.array_equal(codes.cpu().numpy(), want_c)
    ctx.summarise(pool, summary, i32([]))


def test_summaries_of_numbers_that_are_none(ctx):
    """A block of a token that is NaN is passed over; a dim that has nothing else counts as 0; infinities are the largest codes."""
    page, dim = 16, 64
    ref = R.Pool(3, page, 1, dim)
    x = np.random.default_rng(1).standard_normal((3 * page, 1, dim)).astype(np.float32)
    q, d, m = R.quantise(x)
    d[3, 0, 0] = np.nan
    m[16:32, 0, 1] = np.nan
    m[40, 0, 0], d[40, 0, 0] = np.inf, 0
    m[41, 0, 1], d[41, 0, 1] = -np.inf, 0
    ref.write(0, np.arange(3 * page), q, d, m)
    pool = bp.KV4Pool(torch.from_numpy(ref.bytes).cuda(), 3, page, 1, dim)
    codes, scales = torch.zeros(3, 1, 2, dim, dtype=torch.int8, device="cuda"), torch.zeros(3, 1, device="cuda")
    ctx.summarise(pool, bp.BlockSummary(codes, scales), i32([0, 1, 2]))
    with np.errstate(invalid="ignore"):
        want = P.summary(keys_of_pages(ref, [0, 1, 2]))
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


# ---- the choice, and attention over it -------------------------------------------------------------------------------

class Chosen(Requests):
    """Requests over a pool with summaries of their full pages (bits that are no numbers elsewhere); the choice by definition."""

    def __init__(self, seed, dtype, q_len, kv_len, heads, hkv, dim, page, chosen, first=1, last=1, how="dense", same=0):
        super().__init__(seed, dtype, q_len, kv_len, heads, hkv, dim, page, how=how)
        self.chosen, self.first, self.last = chosen, first, last
        n_pages = self.ref.bytes.shape[0]
        self.codes = torch.full((n_pages, hkv, 2, dim), -128, dtype=torch.int8, device="cuda")
        self.scales = torch.full((n_pages, hkv), float("nan"), device="cuda")
        full = [self.table[r, i] for r, k in enumerate(kv_len) for i in range(k // page)]
        if full:
            c, s = P.summary(keys_of_pages(self.ref, full))
            if same:  # many equal scores
                c[:], s[:] = c[:same].repeat(-(-len(full) // same), 0)[:len(full)], s[:1]
            self.codes[torch.tensor(full).long()], self.scales[torch.tensor(full).long()] = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
        self.summary = bp.BlockSummary(self.codes, self.scales)
        n = self.q.shape[0]
        self.pages, self.keys_n = i32(np.full((n, hkv, chosen), 5)), i32(np.full(n, 5))

    def select(self, ctx, **kw):
        ctx.select(self.pool, self.summary, self.q, self.pages, self.keys_n, *self.args, max_q=kw.pop("max_q", max(self.q_len)), max_kv=kw.pop("max_kv", max(self.kv_len)),
                   first=self.first, last=self.last, **kw)

    def want(self):
        n, hkv, group = self.q.shape[0], self.hkv, self.q.shape[1] // self.hkv
        pages, keys = np.full((n, hkv, self.chosen), -1), np.full(n, -1)
        codes, scales, q = self.codes.cpu().numpy(), self.scales.cpu().numpy(), f64(self.q)
        for r, (nq, nk) in enumerate(zip(self.q_len, self.kv_len)):
            for i in range(nq):
                t, sees = self.start[r] + i, max(nk - nq + i + 1, 0)
                nb = -(-sees // self.page)
                keys[t] = sees - max(nb - self.chosen, 0) * self.page
                for h in range(hkv):
                    at = np.arange(nb)
                    if nb > self.chosen:
                        p = self.table[r, :nb]
                        with np.errstate(invalid="ignore"):
                            s = P.scores(q[t, h * group:(h + 1) * group], codes[p, h], scales[p, h])
                        at = P.choose(s, self.first, self.last, self.chosen)
                    pages[t, h, :len(at)] = self.table[r, at]
        return pages, keys

    def check_choice(self):
        pages, keys = self.want()
        assert np.array_equal(self.keys_n.cpu().numpy(), keys)
        assert np.array_equal(self.pages.cpu().numpy(), pages)

    def attend(self, ctx, out=None, **kw):
        out = torch.full_like(self.q, float("nan")) if out is None else out
        ctx.attention_selected(self.pool, self.q, out, self.pages, self.keys_n, **kw)
        return out

    def check_out(self, out, scale=None):
        pages, keys, q, group = self.pages.cpu().numpy(), self.keys_n.cpu().numpy(), f64(self.q), self.q.shape[1] // self.hkv
        whole = {}
        for r, nk in enumerate(self.kv_len):
            for i in range(-(-nk // self.page)):
                whole[int(self.table[r, i])] = (r, i)
        for t in range(q.shape[0]):
            n = max(int(keys[t]), 0)
            for h in range(self.hkv):
                k, v = np.zeros((0, 1, self.dim)), np.zeros((0, 1, self.dim))
                for p in pages[t, h, :-(-n // self.page)]:
                    r, i = whole[int(p)]
                    part = slice(i * self.page, (i + 1) * self.page)
                    k, v = np.concatenate([k, self.keys[r][part, h:h + 1]]), np.concatenate([v, self.values[r][part, h:h + 1]])
                k, v = k[:n], v[:n]
                rows = q[t, h * group:(h + 1) * group][None]
                want, weight = P.softmax_over(rows, k, v, np.ones((1, n), bool), self.dim ** -0.5 if scale is None else scale)
                err = np.abs(f64(out[t, h * group:(h + 1) * group])[None] - want)
                tol = HALF_UNIT[self.dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -24
                assert (err <= tol).all(), (t, h, err.max(), (err / tol).max())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", HEADS)
@pytest.mark.parametrize("page,chosen", [(16, 3), (16, 9), (32, 4), (64, 2)])
def test_one_token_each(ctx, dtype, heads, hkv, dim, page, chosen):
    kv = [1, 0, 15, 16, 17, 127, 128, 129, 300, 500, 144]
    s = Chosen(1, dtype, [1] * len(kv), kv, heads, hkv, dim, page, chosen)
    s.select(ctx)
    s.check_choice()
    s.check_out(s.attend(ctx))
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", [(8, 2, 128), (5, 1, 64), (14, 2, 64)])
@pytest.mark.parametrize("first,last,chosen", [(0, 1, 1), (0, 1, 4), (1, 2, 5), (2, 3, 5), (3, 1, 30)])
def test_several_tokens_each(ctx, dtype, heads, hkv, dim, first, last, chosen):
    """Every token sees its own keys; more queries than keys; requests without queries or keys."""
    s = Chosen(2, dtype, [5, 2, 0, 1, 8, 7, 3, 40], [200, 2, 50, 64, 300, 3, 0, 333], heads, hkv, dim, 16, chosen, first, last)
    s.select(ctx)
    s.check_choice()
    s.check_out(s.attend(ctx, scale=0.3), scale=0.3)
    ctx.status()


@pytest.mark.parametrize("same", [1, 2, 7])
@pytest.mark.parametrize("chosen", [4, 64, 150])
def test_equal_scores_go_to_the_earlier_page(ctx, same, chosen):
    s = Chosen(3, "f16", [1, 3], [5000, 3211], 4, 2, 64, 16, chosen, same=same)
    s.select(ctx)
    s.check_choice()


@pytest.mark.parametrize("heads,hkv,dim,page,kv", [(4, 1, 64, 16, 70_003), (2, 2, 128, 16, 20_000), (4, 1, 128, 64, 40_000)])
def test_long_contexts(ctx, heads, hkv, dim, page, kv):
    """Thousands of pages, chosen by their summaries alone (made up: nobody reads the keys)."""
    rng = np.random.default_rng(5)
    n = -(-kv // page)
    s = Chosen(4, "bf16", [1, 2], [40, 50], heads, hkv, dim, page, 200, 2, 2)
    s.codes = torch.from_numpy(rng.integers(-127, 128, (n, hkv, 2, dim)).astype(np.int8)).cuda()
    s.scales = torch.from_numpy(2.0 ** rng.integers(-3, 3, (n, hkv))).float().cuda()
    s.summary = bp.BlockSummary(s.codes, s.scales)
    s.pool = bp.KV4Pool(torch.empty(bp.KV4Pool.bytes(n, page, hkv, dim), dtype=torch.uint8, device="cuda"), n, page, hkv, dim)
    s.kv_len = [kv, kv // 2]
    s.table = np.stack([rng.permutation(n) for _ in range(2)]).astype(np.int32)
    s.args[1], s.args[2] = i32(s.kv_len), i32(s.table)
    s.select(ctx)
    s.check_choice()
    ctx.status()


def test_many_requests(ctx):
    rng = np.random.default_rng(6)
    n = 700
    s = Chosen(5, "f16", [int(x) for x in rng.integers(0, 3, n)], [int(x) for x in rng.integers(0, 150, n)], 4, 2, 64, 16, 4, 1, 2)
    s.select(ctx)
    s.check_choice()
    s.check_out(s.attend(ctx))
    ctx.status()


@pytest.mark.parametrize("gain", [0.0, 1e-7, 1e-3, 60.0, 1e30])
def test_queries_of_any_size(ctx, gain):
    s = Chosen(6, "bf16", [1, 2], [500, 400], 6, 2, 64, 16, 8)
    s.q *= gain
    s.q[0, 1, 5] = -3 * gain
    s.select(ctx)
    s.check_choice()


def test_queries_that_are_no_numbers(ctx):
    """They count as 0 (infinities as the largest code): some pages of the request, each once, the forced ones among them."""
    s = Chosen(7, "f16", [1, 1, 1], [500, 400, 300], 6, 2, 64, 16, 8, 2, 2)
    s.q[0, 0, 3] = float("nan")
    s.q[1] = float("nan")
    s.q[2, 4, 9] = float("inf")
    s.select(ctx)
    got = s.pages.cpu().numpy()
    s.q = torch.where(s.q.isnan(), 0.0, s.q)
    want, keys = s.want()
    assert np.array_equal(got[:2], want[:2]) and np.array_equal(s.keys_n.cpu().numpy(), keys)
    for h in range(2):
        at = [list(s.table[2]).index(p) for p in got[2, h]]
        assert at == sorted(set(at)) and at[:2] == [0, 1] and at[-2:] == [17, 18]


@pytest.mark.parametrize("how", ["fused", "odd", "heads"])
def test_strided_rows_and_outputs_over_the_queries(ctx, how):
    s = Chosen(8, "f16", [3, 1], [300, 170], 8, 2, 128, 16, 6, how=how)
    s.select(ctx)
    s.check_choice()
    out = strided(torch.zeros(4, 8, 128, dtype=torch.float16, device="cuda"), how)
    s.check_out(s.attend(ctx, out))
    keep, s.q = s.q, s.q.clone()
    over = s.attend(ctx, s.q)
    s.q = keep
    s.check_out(over)


def test_rows_of_no_request(ctx):
    s = Chosen(9, "bf16", [2, 1], [300, 100], 8, 2, 128, 16, 6)
    rows = torch.cat([s.q, torch.full((3, 8, 128), float("nan"), dtype=s.q.dtype, device="cuda")])
    s.q, out = rows, torch.full_like(rows, 7.0)
    s.pages, s.keys_n = i32(np.full((6, 2, 6), 5)), i32(np.full(6, 5))
    s.select(ctx)
    assert (s.keys_n[3:] == -1).all() and (s.pages[3:] == -1).all()
    s.attend(ctx, out)
    assert (out[3:] == 7.0).all()
    s.q, s.pages, s.keys_n = rows[:3], s.pages[:3], s.keys_n[:3]
    s.check_choice()
    s.check_out(out[:3])
    # a start behind the first rows leaves those before it, too
    s.q, s.pages, s.keys_n = rows[:4], i32(np.full((4, 2, 6), 5)), i32(np.full(4, 5))
    s.args[0] = s.args[0] + 1
    s.select(ctx)
    assert s.keys_n[0].item() == -1 and (s.keys_n[1:] > 0).all()
    ctx.status()


def test_what_is_out_of_range_is_reported(ctx):
    s = Chosen(10, "f16", [1, 1], [500, 300], 8, 2, 64, 16, 6)

    def reported(call):
        out = call()
        with pytest.raises(bp.ContextOverflow):
            ctx.status()
        return out

    reported(lambda: s.select(ctx, max_kv=320))
    want, _ = s.want()
    assert np.array_equal(s.pages[1].cpu().numpy(), want[1]) and s.keys_n[0].item() == 96
    keep = s.args[2].clone()
    s.args[2][0, 9] = 1 << 28  # never chosen, unless it has to be
    reported(lambda: s.select(ctx))
    assert (s.pages[0] < s.ref.bytes.shape[0]).all()
    s.args[2].copy_(keep)
    s.select(ctx)
    s.check_choice()
    good = s.attend(ctx)
    ctx.status()
    s.pages[0, 1, 2] = s.ref.bytes.shape[0]
    out = reported(lambda: s.attend(ctx))
    assert torch.equal(out[1], good[1]) and torch.equal(out[0, :4], good[0, :4])
    s.keys_n[0] = 6 * 16 + 1
    reported(lambda: s.attend(ctx))
    s.keys_n[:] = 0
    assert (s.attend(ctx) == 0).all()
    ctx.status()


def test_other_streams_and_graphs(ctx):
    """Summaries, choice and attention captured together follow the lengths on the device."""
    s = Chosen(11, "bf16", [1, 2], [700, 400], 8, 2, 128, 16, 10)
    filled = i32([int(s.table[0, 3]), -1])
    out = torch.zeros_like(s.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.summarise(s.pool, s.summary, filled)
        s.select(ctx)
        s.attend(ctx, out)
    for kv in ([700, 400], [655, 377], [30, 2]):
        s.args[1].copy_(i32(kv))
        s.kv_len = kv
        s.codes[s.table[0, 3]] = 0
        graph.replay()
        torch.cuda.synchronize()
        assert (s.codes[s.table[0, 3]] != 0).any()
        s.check_choice()
        s.check_out(out)
    ctx.status()


def test_two_contexts_at_once(ctx):
    """Choice (in clusters) and attention on two streams at once."""
    s = Chosen(14, "f16", [1, 1], [3000, 2500], 4, 2, 64, 16, 20)
    s.select(ctx)
    s.check_choice()
    want = [s.pages.clone(), s.keys_n.clone(), s.attend(ctx)]
    other, streams = bp.PagedContext(), [torch.cuda.Stream() for _ in range(2)]
    got = [[(torch.zeros_like(want[0]), torch.zeros_like(want[1]), torch.zeros_like(want[2])) for _ in range(20)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for c, stream, g in zip((ctx, other), streams, got):
            with torch.cuda.stream(stream):
                s.pages, s.keys_n = g[i][:2]
                s.select(c)
                s.attend(c, g[i][2])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for x in g for a, b in zip(x, want))
    other.status()
    other.close()


def test_refusals(ctx):
    s = Chosen(12, "f16", [1, 1], [300, 200], 4, 2, 64, 16, 4)
    lib, at = bp.paged._lib, torch.zeros(64, device="cuda").data_ptr()

    def choice(dtype=0, summary=None, **kw):
        a = lib.ChoiceStruct(lib.RowsStruct(s.q.data_ptr(), 256, 64))
        for k, v in {**dict(zip(("q_start", "kv_len", "page_table"), (t.data_ptr() for t in s.args))), **dict(pages=s.pages.data_ptr(), keys=s.keys_n.data_ptr(), n_req=2, n_head=4, total_q=2, max_q=1,
                     max_kv=300, table_stride=s.args[2].shape[1], chosen=4, first=1, last=1), **kw}.items():
            setattr(a, k, v)
        return ctx._lib.bp_kv4_select(ctx._h, None, dtype, s.pool._p, s.summary._p if summary is None else C.byref(summary), C.byref(a))

    for kw in (dict(dtype=2), dict(n_head=3), dict(last=0), dict(first=4), dict(chosen=1), dict(first=0xFFFFFFFF), dict(n_req=65536), dict(total_q=1 << 30), dict(max_kv=16 * 49153, table_stride=50000),
               dict(chosen=1 << 31), dict(pages=at + 2), dict(keys=at + 1), dict(q_start=at + 2), dict(summary=lib.SummaryStruct(at + 4, at)), dict(summary=lib.SummaryStruct(at, at + 2))):
        assert choice(**kw) == 1, kw
    for kw in (dict(q_start=None), dict(kv_len=None), dict(page_table=None), dict(pages=None), dict(keys=None), dict(summary=lib.SummaryStruct(None, at)), dict(summary=lib.SummaryStruct(at, None))):
        assert choice(**kw) == 7, kw
    assert choice(total_q=0) == 0

    def attend(dtype=0, **kw):
        a = lib.ChosenStruct(lib.RowsStruct(s.q.data_ptr(), 256, 64), lib.RowsStruct(s.q.data_ptr(), 256, 64))
        for k, v in {**dict(pages=s.pages.data_ptr(), keys=s.keys_n.data_ptr(), n_head=4, total_q=2, chosen=4, scale=0.1), **kw}.items():
            setattr(a, k, v)
        return ctx._lib.bp_kv4_attention_selected(ctx._h, None, dtype, s.pool._p, C.byref(a))

    for kw in (dict(dtype=2), dict(n_head=3), dict(scale=float("nan")), dict(total_q=65536), dict(chosen=1 << 28), dict(pages=at + 2), dict(keys=at + 1)):
        assert attend(**kw) == 1, kw
    assert attend(pages=None) == 7 and attend(keys=None) == 7 and attend(total_q=0) == 0

    def summarise(summary=None, pages=at, n_tok=None, n=1):
        return ctx._lib.bp_kv4_summarise(ctx._h, None, s.pool._p, s.summary._p if summary is None else C.byref(summary), pages, n_tok, n)

    assert summarise(summary=lib.SummaryStruct(at + 8, at)) == 1 and summarise(pages=at + 2) == 1 and summarise(n_tok=at + 2) == 1 and summarise(n=1 << 31) == 1
    assert summarise(pages=None) == 7 and summarise(summary=lib.SummaryStruct(at, None)) == 7 and summarise(n=0) == 0
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        bp.BlockSummary(s.codes, s.scales[:2])
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        ctx.summarise(s.pool, bp.BlockSummary(s.codes[1:], s.scales[1:]), i32([0]))
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        bp.KV4Pools([s.pool], [bp.BlockSummary(s.codes[1:], s.scales[1:])])
    ctx.status()
