"""Page tables on the GPU against their definition (tests/pages_ref.py): whole numbers, equal all of them; copied bytes are equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests import pages_ref as P  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = bp.PagedContext()
    yield c
    c.status()
    c.close()


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a), dtype=dtype).cuda()


class Both:
    """The same tables as the definition has them and on the GPU, there as views into larger tensors (nothing 16-byte aligned, rows apart)."""

    def __init__(self, seed, rows, width, n_pages, page, kv, pad=3):
        rng = np.random.default_rng(seed)
        need = [-(-k // page) for k in kv]
        order = rng.permutation(n_pages)
        table, refs, at = np.full((rows, width), 1 << 30, np.int32), np.zeros(n_pages, np.int32), 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            refs[order[at:at + n]] = 1
            at += n
        self.ref, self.page = P.Tables(table, np.array(kv, np.int32), refs, page), page
        big = torch.full((rows, width + pad), -9, dtype=torch.int32, device="cuda")
        self.table = big[:, 1:1 + width] if pad else big
        self.table.copy_(dev(table))
        self.kv, self.refs = dev(np.concatenate([[7], kv]))[1:], dev(np.concatenate([[7], refs, [8]]))[1:-1]
        self.big = big
        self.gpu = bp.PageTables(self.table, self.kv, self.refs, page)

    def check(self):
        assert np.array_equal(self.kv.cpu().numpy(), self.ref.kv)
        assert np.array_equal(self.refs.cpu().numpy(), self.ref.refs)
        table = self.table.cpu().numpy()
        for r in range(len(self.ref.kv)):
            n = self.ref.pages(self.ref.kv[r])
            assert np.array_equal(table[r, :n], self.ref.entries(r)), r
        if self.big.shape[1] > table.shape[1]:
            assert (self.big[:, 0] == -9).all() and (self.big[:, 1 + table.shape[1]:] == -9).all()

    def grow(self, ctx, n_new, n_out, refused=False):
        start, pos, slots = dev(np.full(len(n_new) + 1, 5)), dev(np.full(n_out, 5)), dev(np.full(n_out, 5), torch.int64)
        ctx.grow(self.gpu, dev(n_new), start, pos, slots)
        bad, *want = self.ref.grow(np.array(n_new), n_out)
        assert bad == refused
        if refused:
            with pytest.raises(bp.ContextOverflow):
                ctx.status()
        for a, b in zip((start, pos, slots), want):
            assert np.array_equal(a.cpu().numpy(), b)
        self.check()

    def release(self, ctx, rows):
        ctx.release(self.gpu, dev(rows))
        self.ref.release(rows)
        self.check()

    def fork(self, ctx, parents, children, refused=False):
        src, dst = dev(np.full(len(parents), 5)), dev(np.full(len(parents), 5))
        ctx.fork(self.gpu, dev(parents), dev(children), src, dst)
        bad, *want = self.ref.fork(parents, children)
        assert bad == refused
        if refused:
            with pytest.raises(bp.ContextOverflow):
                ctx.status()
        assert np.array_equal(src.cpu().numpy(), want[0]) and np.array_equal(dst.cpu().numpy(), want[1])
        self.check()

    def compact(self, ctx, most):
        src, dst = dev(np.full(most, 5)), dev(np.full(most, 5))
        ctx.compact(self.gpu, src, dst)
        want = self.ref.compact(most)
        assert np.array_equal(src.cpu().numpy(), want[0]) and np.array_equal(dst.cpu().numpy(), want[1])
        self.check()
        return src, dst


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("rows,n_pages,pad", [(1, 9, 0), (1, 70, 3), (7, 300, 3), (65, 2000, 0), (300, 33000, 1)])
def test_a_life_of_tables(ctx, page, rows, n_pages, pad):
    """Rows grow, end, are forked and compacted, in random order; some pages are held by somebody else, too."""
    rng = np.random.default_rng(rows + page)
    width = max(2, n_pages // rows)
    kv = [int(rng.integers(0, width * page // 3)) for _ in range(rows)]
    b = Both(page, rows, width, n_pages, page, kv, pad)
    pinned = rng.permutation(n_pages)[:n_pages // 20]
    b.ref.refs[pinned] += 1
    b.refs.copy_(dev(b.ref.refs))
    for step in range(12):
        room = np.maximum(0, width * page - b.ref.kv)
        n_new = np.minimum(rng.integers(0, [1, 2, page + 3, 3 * page][step % 4] + 1, rows), room)
        free = int((b.ref.refs == 0).sum()) - rows
        n_new = np.where(np.cumsum((n_new + page - 1) // page + 1) < free, n_new, 0)
        b.grow(ctx, n_new, int(n_new.sum()) + int(rng.integers(0, 3)))
        if rows > 2:
            ends = rng.permutation(rows)[:rows // 3]
            b.release(ctx, [int(r) for r in ends] + [-1])
            alive = np.setdiff1d(np.arange(rows), ends)
            parents = rng.choice(alive, len(ends))
            parents[0] = -1
            b.fork(ctx, [int(x) for x in parents], [int(x) for x in ends])
        b.compact(ctx, [1, n_pages // 9 + 1, n_pages + 5][step % 3])
    ctx.status()


def test_many_rows_and_pages(ctx):
    """Several rows per thread, free pages far behind one another, more new pages than are found at a time."""
    rows, n_pages, page = 5000, 120_000, 16
    rng = np.random.default_rng(1)
    b = Both(1, rows, 40, n_pages, page, [int(x) for x in rng.integers(0, 160, rows)])
    b.grow(ctx, rng.integers(0, 200, rows), 1_000_000)
    b.release(ctx, [int(x) for x in rng.permutation(rows)[:2500]])
    ends = np.flatnonzero(b.ref.kv == 0)
    b.fork(ctx, [int(x) for x in rng.choice(np.flatnonzero(b.ref.kv), len(ends))], [int(x) for x in ends])
    b.compact(ctx, 100_000)
    b.grow(ctx, np.ones(rows, np.int64), rows)
    ctx.status()


@pytest.mark.parametrize("most", [30, 5000])
def test_compaction_of_large_tables(ctx, most):
    """More entries than one cluster takes care of."""
    rows, width, n_pages, page = 300, 1000, 20_000, 16
    rng = np.random.default_rng(most)
    b = Both(9, rows, width, n_pages, page, [int(x) for x in rng.integers(0, 900, rows)])
    b.compact(ctx, most)
    b.compact(ctx, most)
    ctx.status()


def test_rows_that_are_refused_stay_as_they_were(ctx):
    """No room in the row, no pages in the pool, no places in the output, a negative number: the others grow."""
    page = 16
    b = Both(2, 6, 4, 12, page, [60, 0, 10, 33, 5, 16])  # 4 + 0 + 1 + 3 + 1 + 1 pages held, two free
    b.grow(ctx, [5, 3, 2, 4, 1, 0], 15, refused=True)  # the first would need a fifth page
    b.grow(ctx, [0, 40, 6, 1, 1, 2], 50, refused=True)  # one page is left: row 1 would need two more, row 5 (behind it) one
    b.grow(ctx, [0, -3, 1, 0, 9, 0], 10, refused=True)
    b.grow(ctx, [1, 2, 3, 4, 5, 0], 9, refused=True)  # tokens of row 3 (its last) and row 4 have no places
    b.grow(ctx, [0] * 6, 0)
    ctx.status()


@pytest.mark.parametrize("pairs", [5, 700])
def test_forks_without_pages_stay_empty(ctx, pairs):
    page = 32
    rows = pairs + 1
    b = Both(3, rows, 12, 11 + pairs // 2, page, [10 * page + 3] + [0] * pairs)
    b.fork(ctx, [0] * pairs, list(range(1, rows)), refused=True)
    assert (b.kv[1 + pairs // 2:] == 0).all() and (b.kv[1:1 + pairs // 2] == 10 * page + 3).all()


def test_bad_rows_and_pages_are_reported_and_left(ctx):
    page = 16
    b = Both(4, 5, 6, 40, page, [50, 20, 0, 0, 96])

    def reported(call):
        call()
        with pytest.raises(bp.ContextOverflow):
            ctx.status()
        ctx.status()

    src, dst = dev([5]), dev([5])
    for parent, child in ((7, 2), (0, 9), (1, 1), (0, 1), (0, 4)):  # no such rows, a row of its own, a child that is not empty
        reported(lambda: ctx.fork(b.gpu, dev([parent]), dev([child]), src, dst))
        assert src.item() == dst.item() == -1
        b.check()
    reported(lambda: ctx.release(b.gpu, dev([5, 1 << 30])))
    b.check()
    # the same child twice: one of the pairs has it
    src, dst = dev([5, 5]), dev([5, 5])
    reported(lambda: ctx.fork(b.gpu, dev([1, 1]), dev([2, 2]), src, dst))
    assert sorted((src < 0).tolist()) == [False, True] and b.kv[2].item() == 20
    won = 0 if src[0].item() >= 0 else 1
    _, s, d = b.ref.fork([1], [2])
    assert src[won].item() == s[0] and dst[won].item() == d[0]
    b.check()
    # the same row twice: it ends once
    b.ref.release([4])
    ctx.release(b.gpu, dev([4, 4]))
    b.check()
    ctx.status()
    # a page that is none, held by a row: it is passed over
    b.table[0, 1] = 4000
    reported(lambda: ctx.compact(b.gpu, dev([0]), dev([0])))
    kept = b.table[0, 1].item()
    assert kept == 4000
    reported(lambda: ctx.release(b.gpu, dev([0])))
    assert b.kv[0].item() == 0
    # counts that are too low do not become negative
    b.kv[0] = 16
    b.table[0, 0] = int(torch.nonzero(b.refs == 0)[0])
    reported(lambda: ctx.release(b.gpu, dev([0])))
    assert (b.refs >= 0).all()
    # a row whose length says more than it has room for, and a negative one
    b.kv[3] = 6 * 16 + 1
    reported(lambda: ctx.fork(b.gpu, dev([3]), dev([0]), dev([0]), dev([0])))
    reported(lambda: ctx.grow(b.gpu, dev([0, 0, 0, 1, 0]), dev([0] * 6), dev([0]), dev([0], torch.int64)))
    b.kv[3] = -5
    reported(lambda: ctx.grow(b.gpu, dev([0, 0, 0, 1, 0]), dev([0] * 6), dev([0]), dev([0], torch.int64)))
    assert b.kv[3].item() == -5


SHAPES = [(1, 4, 64), (3, 2, 128), (5, 1, 64)]


@pytest.mark.parametrize("layers,hkv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("summaries", [False, True])
def test_copy_pages(ctx, layers, hkv, dim, page, summaries):
    """Pools and summaries together; scales of a page are 4 to 16 bytes. Padding, places nobody copies to and pages that are none stay."""
    n_pages, g = 50, torch.Generator(device="cuda").manual_seed(1)
    size = page * hkv * dim * 5 // 4
    pools = torch.randint(0, 256, (layers, n_pages, size), generator=g, device="cuda", dtype=torch.uint8)
    codes = torch.randint(-128, 128, (layers, n_pages, hkv, 2, dim), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.randn(layers, n_pages, hkv, generator=g, device="cuda")
    both = bp.KV4Pools([bp.KV4Pool(p, n_pages, page, hkv, dim) for p in pools], [bp.BlockSummary(c, s) for c, s in zip(codes, scales)] if summaries else ())
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int32)
    src, dst = order[:20].clone(), order[20:40].clone()
    src[3], dst[7] = -1, -1
    want = [t.clone() for t in (pools, codes, scales)]
    real = [i for i in range(20) if i not in (3, 7)]
    for t in want[:3 if summaries else 1]:
        t[:, dst[real].long()] = t[:, src[real].long()]
    ctx.copy_pages(both, src, dst)
    for a, b in zip((pools, codes, scales), want):
        assert torch.equal(a, b)
    ctx.status()
    for s, d in ((n_pages, 1), (1, n_pages), (1 << 30, 2)):
        ctx.copy_pages(both, dev([s, 4]), dev([d, 4]))
        with pytest.raises(bp.ContextOverflow):
            ctx.status()
        assert torch.equal(pools, want[0])
    ctx.copy_pages(both, dev([]), dev([]))


def test_copy_of_many_layers_and_odd_bases(ctx):
    """More arrays than one launch takes; arrays of the C entry whose pages are not 16-byte aligned."""
    pools = torch.randint(0, 256, (150, 4, 16 * 64 * 5 // 4), device="cuda", dtype=torch.uint8)
    want = pools.clone()
    want[:, 3] = want[:, 1]
    ctx.copy_pages(bp.KV4Pools([bp.KV4Pool(p, 4, 16, 1, 64) for p in pools]), dev([1]), dev([3]))
    assert torch.equal(pools, want)
    lib = bp.paged._lib
    words = torch.arange(7 * 9 + 1, dtype=torch.int32, device="cuda")
    a = (lib.PageArrayStruct * 1)(lib.PageArrayStruct(words.data_ptr() + 4, 36))
    assert ctx._lib.bp_pages_copy(ctx._h, None, a, 1, 7, dev([6]).data_ptr(), dev([0]).data_ptr(), 1) == 0
    torch.cuda.synchronize()
    assert torch.equal(words[1:10], torch.arange(55, 64, dtype=torch.int32, device="cuda")) and words[0] == 0 and words[10] == 10


def test_pages_behind_four_gigabytes(ctx):
    page, hkv, dim = 64, 2, 128
    size = page * hkv * dim * 5 // 4
    n_pages = (9 << 29) // size
    data = torch.empty(n_pages, size, dtype=torch.uint8, device="cuda")
    data[-1], data[5] = 17, 3
    ctx.copy_pages(bp.KV4Pools([bp.KV4Pool(data, n_pages, page, hkv, dim)]), dev([n_pages - 1, 5]), dev([0, n_pages - 2]))
    assert (data[0] == 17).all() and (data[-2] == 3).all() and (data[-1] == 17).all()


def test_a_captured_step(ctx):
    """Release, grow and a fork in one graph, replayed: it follows what is on the device; on another stream than the tensors' own."""
    page = 16
    a, b = (Both(6, 4, 20, 100, page, [30, 20, 0, 7]) for _ in range(2))
    n_new, ends, parents, children = dev([1, 0, 0, 1]), dev([1]), dev([0]), dev([1])
    start, pos, slots, src, dst = dev([0] * 5), dev([0] * 4), dev([0] * 4, torch.int64), dev([0]), dev([0])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ctx.release(a.gpu, ends)
        ctx.fork(a.gpu, parents, children, src, dst)
        ctx.grow(a.gpu, n_new, start, pos, slots)
    for i in range(20):
        graph.replay()
        torch.cuda.synchronize()
        b.ref.release([1])
        _, s, d = b.ref.fork([0], [1])
        _, *want = b.ref.grow(np.array([1, 0, 0, 1]), 4)
        a.ref = b.ref
        a.check()
        for x, y in zip((src, dst, start, pos, slots), (s, d, *want)):
            assert np.array_equal(x.cpu().numpy(), y)
    ctx.status()


def test_refusals(ctx):
    b = Both(7, 3, 4, 10, 16, [1, 2, 3])
    lib, S = ctx._lib, bp.paged._lib.PageTablesStruct
    i = dev([0] * 64)
    at = i.data_ptr()

    def tables(**kw):
        t = S(at, at, at, 3, 4, 4, 10, 16)
        for k, v in kw.items():
            setattr(t, k, v)
        return t

    import ctypes as C
    for kw in (dict(page_tokens=8), dict(n_rows=0), dict(n_rows=16385, table_stride=4), dict(row_pages=0), dict(row_pages=1 << 28, table_stride=1 << 28), dict(table_stride=3), dict(n_pages=0),
               dict(n_pages=1 << 31), dict(table=at + 1), dict(kv_len=at + 2), dict(refs=at + 3)):
        t = tables(**kw)
        assert lib.bp_pages_release(ctx._h, None, C.byref(t), at, 1) == 1, kw
        assert lib.bp_pages_grow(ctx._h, None, C.byref(t), at, at, at, at, 1) == 1
        assert lib.bp_pages_fork(ctx._h, None, C.byref(t), at, at, 1, at, at) == 1
        assert lib.bp_pages_compact(ctx._h, None, C.byref(t), at, at, 1) == 1
    t = C.byref(tables())
    assert lib.bp_pages_grow(ctx._h, None, t, at, at, at, at + 4, 1) == 1 and lib.bp_pages_grow(ctx._h, None, t, at, at, at, at, (1 << 24) + 1) == 1
    assert lib.bp_pages_fork(ctx._h, None, t, at, at, 16385, at, at) == 1
    for args in ((None, at, at, at, 1), (at, None, at, at, 1), (at, at, None, at, 1), (at, at, at, None, 1)):
        assert lib.bp_pages_grow(ctx._h, None, t, *args) == 7
    assert lib.bp_pages_release(ctx._h, None, t, None, 1) == 7 and lib.bp_pages_release(ctx._h, None, C.byref(tables(refs=None)), at, 1) == 7
    assert lib.bp_pages_compact(ctx._h, None, t, at, None, 1) == 7 and lib.bp_pages_fork(ctx._h, None, t, at, at, 1, None, at) == 7
    A = bp.paged._lib.PageArrayStruct
    for a, want in ((A(at, 6), 1), (A(at, 0), 1), (A(at + 2, 8), 1), (A(at, 1 << 31), 1), (A(None, 8), 7)):
        assert lib.bp_pages_copy(ctx._h, None, C.byref(a), 1, 4, at, at, 1) == want
    assert lib.bp_pages_copy(ctx._h, None, None, 1, 4, at, at, 1) == 7 and lib.bp_pages_copy(ctx._h, None, C.byref(A(at, 8)), 1, 0, at, at, 1) == 1
    assert lib.bp_pages_copy(ctx._h, None, C.byref(A(at, 8)), 1, 4, None, at, 1) == 7
    for bad in (lambda: bp.PageTables(b.table[:, ::2], b.kv, b.refs, 16), lambda: bp.PageTables(b.table, b.kv[:2], b.refs, 16), lambda: bp.PageTables(b.table, b.kv, b.refs, 8),
                lambda: bp.PageTables(b.table, b.kv, b.refs.cpu(), 16), lambda: bp.PageTables(b.table, b.kv.long(), b.refs, 16),
                lambda: bp.KV4Pools([bp.KV4Pool(torch.zeros(9999, dtype=torch.uint8, device="cuda"), 1, p, 1, 64) for p in (16, 32)])):
        with pytest.raises(bp.ConfigError, match="^invalid config: "):
            bad()
    ctx.status()
