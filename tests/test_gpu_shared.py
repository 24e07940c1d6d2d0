"""Attention behind prefixes in common, on the GPU against the softmax over prefix and own keys in 64 bits.

Tolerances as for bp_kv4_attention: every P is rounded once to f16 (2^-11 of it), the result once to its type; binary32 sums and scores up to about 30
move a P by less than 2^-13 of it. Joining the two parts is three binary32 operations per value: 2^-22 of sum p |v|, within the latter."""
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


class Shared(Requests):
    """Requests of which prefix_start[g] .. prefix_start[g + 1] have the prefix g in common: the prefixes lie in the same pool, as requests without queries."""

    def __init__(self, seed, dtype, q_len, kv_len, prefix_start, prefix_len, heads, hkv, dim, page, how="dense"):
        super().__init__(seed, dtype, q_len + [0] * len(prefix_len), kv_len + prefix_len, heads, hkv, dim, page, how=how)
        self.n, self.prefix_start, self.prefix_len = len(q_len), prefix_start, prefix_len
        start, kv, table = self.args
        self.args = [start[:self.n + 1].contiguous(), kv[:self.n].contiguous(), table[:self.n], torch.tensor(prefix_start, dtype=torch.int32, device="cuda"),
                     kv[self.n:].contiguous(), table[self.n:]]
        self.most = max(prefix_len + [0])

    def run(self, ctx, out=None, **kw):
        out = torch.full_like(self.q, float("nan")) if out is None else out
        work = kw.pop("work", None)
        if work is None:
            work = torch.full((ctx.shared_work(self.q.shape[0], self.q.shape[1], self.dim),), float("nan"), device="cuda")
        ctx.attention_shared(self.pool, self.q, out, *self.args, work, max_q=kw.pop("max_q", max(self.q_len)), max_kv=kw.pop("max_kv", max(self.kv_len[:self.n])),
                             max_prefix=kw.pop("max_prefix", self.most), **kw)
        return out

    def want(self, r, scale):
        g = [i for i in range(len(self.prefix_len)) if self.prefix_start[i] <= r < self.prefix_start[i + 1]]
        k, v = self.keys[r], self.values[r]
        before = 0
        if g:
            before = self.prefix_len[g[0]]
            k, v = np.concatenate([self.keys[self.n + g[0]][:before], k]), np.concatenate([self.values[self.n + g[0]][:before], v])
        nq = self.q_len[r]
        return P.softmax_over(f64(self.q[self.start[r]:self.start[r + 1]]), k, v, P.shared_seen(nq, before, k.shape[0] - before), scale)

    def check(self, out, scale=None, only=None):
        for r in range(self.n) if only is None else only:
            want, weight = self.want(r, self.dim ** -0.5 if scale is None else scale)
            err = np.abs(f64(out[self.start[r]:self.start[r + 1]]) - want)
            tol = HALF_UNIT[self.dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -24
            assert (err <= tol).all(), (r, err.max(), (err / tol).max())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_one_token_each(ctx, dtype, heads, hkv, dim, page):
    """Two prefixes, one of them not of whole pages or tiles; requests before and behind them have none; one has no keys of its own, two none at all."""
    s = Shared(1, dtype, [1] * 9, [20, 0, 1, 33, 64, 0, 65, 0, 17], [2, 6, 8], [130, 64], heads, hkv, dim, page)
    s.check(s.run(ctx))
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", HEADS)
@pytest.mark.parametrize("q", [5, 70, 300])
def test_several_tokens_each(ctx, dtype, heads, hkv, dim, q):
    """Drafts and chunks of odd lengths; a request with more queries than own keys (the first of them see the prefix alone), one without queries, a
    prefix of nobody, an empty prefix."""
    s = Shared(2, dtype, [q, 2, 0, q - 1, 3, 1], [q, 200, 40, 2, 77, 0], [0, 3, 3, 5, 6], [150, 30, 71, 0], heads, hkv, dim, 32)
    s.check(s.run(ctx))
    ctx.status()


@pytest.mark.parametrize("n_req,prefix,own", [(1, 5000, 3), (40, 3001, 200), (200, 64, 30), (600, 100, 20)])
@pytest.mark.parametrize("heads,hkv,dim", [(8, 2, 128), (5, 1, 64)])
def test_batches(ctx, n_req, prefix, own, heads, hkv, dim):
    """Few to many rows behind one prefix, split over the device in either part; results do not depend on who comes when."""
    rng = np.random.default_rng(n_req)
    s = Shared(3, "bf16", [1] * n_req, [int(x) for x in rng.integers(1, own + 1, n_req)], [0, n_req], [prefix], heads, hkv, dim, 16)
    a = s.run(ctx)
    s.check(a)
    for _ in range(3):
        assert torch.equal(a, s.run(ctx))
    ctx.status()


def test_many_prefixes(ctx):
    rng = np.random.default_rng(4)
    start = np.sort(rng.integers(0, 701, 601))
    s = Shared(4, "f16", [int(x) for x in rng.integers(0, 3, 700)], [int(x) for x in rng.integers(2, 40, 700)], [int(x) for x in start], [int(x) for x in rng.integers(0, 90, 600)], 4, 2, 64, 16)
    s.check(s.run(ctx))
    ctx.status()


@pytest.mark.parametrize("n_req", [3, 70])
def test_is_attention_over_both(ctx, n_req):
    """Where a prefix has whole pages, a row of its pages and the own ones is the same request to attention()."""
    page, n_prefix = 32, 128
    s = Shared(5, "f16", [2] * n_req, [5 + i for i in range(n_req)], [0, n_req], [n_prefix], 8, 2, 128, page)
    both = torch.cat([s.args[5][:, :n_prefix // page].expand(n_req, -1), s.args[2]], 1).contiguous()
    out = torch.empty_like(s.q)
    ctx.attention(s.pool, s.q, out, s.args[0], s.args[1] + n_prefix, both, max_q=2, max_kv=n_prefix + 5 + n_req)
    want, weight = zip(*[s.want(r, 128 ** -0.5) for r in range(n_req)])
    off = (f64(out) - f64(s.run(ctx)))
    # each is within its tolerance of the 64-bit result
    assert (np.abs(off) <= 2 * (2.0 ** -11 * np.abs(np.concatenate(want)) + (2.0 ** -11 + 2.0 ** -13) * np.concatenate(weight) + 2.0 ** -24)).all()


@pytest.mark.parametrize("how", ["fused", "odd", "heads"])
@pytest.mark.parametrize("q", [1, 60, 130])
def test_strided_rows_and_outputs_over_the_queries(ctx, how, q):
    s = Shared(6, "f16", [q, q, q], [300, 170, 60], [0, 3], [200], 8, 2, 128, 64, how=how)
    out = strided(torch.zeros(3 * q, 8, 128, dtype=torch.float16, device="cuda"), how)
    s.check(s.run(ctx, out, scale=0.2), scale=0.2)
    keep, s.q = s.q, s.q.clone()
    over = s.run(ctx, s.q, scale=0.2)
    s.q = keep
    s.check(over, scale=0.2)


@pytest.mark.parametrize("q", [1, 40, 450])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3e6, 1e30])
def test_scales(ctx, q, scale):
    """Scores that are turned or level, and ones of any size: then one key has all the weight, in the one part or the other."""
    s = Shared(7, "bf16", [q] * 4, [60, 41, 50, 99], [0, 4], [80], 4, 2, 64, 16)
    if scale > 1:
        # queries of few bits and keys on their grid: scores are far enough apart for the largest to be no matter of rounding
        out = f64(s.run(ctx, scale=scale))
        for r in range(s.n):
            want, weight = s.want(r, scale)
            q64, k = f64(s.q[s.start[r]:s.start[r + 1]]), np.concatenate([s.keys[s.n][:80], s.keys[r]])
            seen = P.shared_seen(q, 80, k.shape[0] - 80)
            for h in range(4):
                sc = np.where(seen, q64[:, h] @ k[:, h // 2].T, -np.inf)
                two = np.sort(sc, -1)[:, -2:]
                # a binary32 score is off by 2^-20 of sum |q| |k| at most here (some hundred terms); a gap of four times that, times scale, leaves the second nothing
                clear = (two[:, 1] - two[:, 0]) > 2.0 ** -18 * (np.abs(q64[:, h]) @ np.abs(k[:, h // 2]).T).max(-1)
                clear &= (two[:, 1] - two[:, 0]) * scale > 100
                err = np.abs(out[s.start[r]:s.start[r + 1], h] - want[:, h])
                assert clear.any() and (err <= 2.0 ** -8 * np.abs(want[:, h]) + 2.0 ** -24)[clear].all()
        return
    s.check(s.run(ctx, scale=scale), scale=scale)


@pytest.mark.parametrize("q", [1, 40, 240])
def test_values_that_are_no_numbers(ctx, q):
    """One in a prefix reaches all of its requests, one among own keys the queries that see it; in that block of dims alone. (Unused places hold bits that are no numbers in every test.)"""
    s = Shared(8, "f16", [q] * 4, [q + 70] * 4, [0, 2, 4], [100, 90], 8, 2, 64, 16)
    good = s.run(ctx)
    bad = s.ref.bytes.copy()

    def spoil(row, key, head, block):
        slot = int(s.table[row, key // 16]) * 16 + key % 16
        _, d, _ = s.ref.place(1, slot)
        view = bad[slot // 16, head]
        at = 16 * 64 * 5 // 8 + 16 * 32 + 4 * (slot % 16) + 2 * block
        view[at:at + 2] = (0xFF, 0x7F)

    spoil(s.n, 50, 0, 1)  # the first prefix, KV head 0, dims 32 ..
    last = q + 70 - 1
    spoil(3, last, 1, 0)  # the last own key of the last request
    s.pool = bp.KV4Pool(torch.from_numpy(bad).cuda(), s.ref.bytes.shape[0], 16, 2, 64)
    out = s.run(ctx)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[:2 * q, :4, 32:] = True
    want[4 * q - 1, 4:, :32] = True
    assert torch.equal(out.isnan(), want) and torch.equal(out[~want], good[~want])


def test_lengths_and_pages_out_of_range(ctx):
    for q in (1, 50, 240):
        s = Shared(9, "f16", [q] * 4, [200, 150, 60, 90], [0, 2, 4], [100, 300], 8, 2, 64, 16)
        want = s.run(ctx)

        def reported(fine, **kw):
            out = s.run(ctx, **kw)
            with pytest.raises(bp.ContextOverflow):
                ctx.status()
            s.check(out, only=fine)

        reported([0, 1], max_prefix=250)
        reported([1, 2, 3], max_kv=180)
        keep = s.args[5]
        s.args[5] = keep.clone()
        s.args[5][0, 2] = 1 << 29
        reported([2, 3])
        s.args[5] = keep
        starts = s.args[3]
        for wrong in ([0, 2, 9], [-3, 2, 4]):  # (cut to the requests that there are)
            s.args[3] = torch.tensor(wrong, dtype=torch.int32, device="cuda")
            out = s.run(ctx)
            with pytest.raises(bp.ContextOverflow):
                ctx.status()
            s.check(out)
        s.args[3] = starts
        assert torch.equal(s.run(ctx), want)
        ctx.status()


def test_rows_of_no_request_stay(ctx):
    s = Shared(10, "bf16", [3, 2], [30, 40], [0, 2], [50], 8, 2, 128, 16)
    rows = torch.cat([s.q, torch.full((4, 8, 128), float("nan"), dtype=s.q.dtype, device="cuda")])
    s.q, out = rows, torch.full_like(rows, 7.0)
    s.run(ctx, out)
    s.check(out)
    assert (out[5:] == 7.0).all()
    ctx.status()


def test_no_prefix_and_no_keys(ctx):
    s = Shared(11, "f16", [1, 3], [40, 9], [0], [], 4, 2, 64, 16)
    s.args[5] = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    s.check(s.run(ctx))
    s = Shared(12, "f16", [1, 40], [0, 0], [0, 2], [0], 4, 2, 64, 16)
    assert (s.run(ctx) == 0).all()
    empty = s.q[:0]
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    ctx.attention_shared(s.pool, empty, empty, i, i[:0], none, i, i[:0], none, torch.empty(0, device="cuda"), max_q=0, max_kv=0, max_prefix=0)
    ctx.status()


@pytest.mark.parametrize("n_req", [40, 90])
def test_a_call_sees_what_was_written_just_before(ctx, n_req):
    """New lengths, queries turned into place and appended keys (of the prefix and the requests' own), in changing order, then attention whose two launches begin early, again and
    again without waiting: as with a wait in between."""
    s = Shared(17, "bf16", [1] * n_req, [33] * n_req, [0, n_req], [700], 8, 2, 128, 16)
    rows = list(range(n_req)) + [s.n]
    at = [32] * n_req + [699]
    slots = torch.tensor([int(s.table[r, k // 16]) * 16 + k % 16 for r, k in zip(rows, at)], device="cuda")
    new = [normal(i, (n_req + 1, 2, 128), "bf16", 3.0) for i in range(40)]
    work = torch.empty(ctx.shared_work(n_req, 8, 128), device="cuda")
    table = bp.RopeTable(torch.from_numpy(R.table(64, 128)).cuda())
    asked = [normal(100 + i, (n_req, 8, 128), "bf16") for i in range(40)]
    positions = [torch.randint(0, 64, (n_req,), device="cuda", dtype=torch.int32) for _ in new]
    lengths = [torch.randint(1, 34, (n_req,), device="cuda", dtype=torch.int32) for _ in new]
    back = [k.flip(0).contiguous() for k in new]

    def go(wait):
        outs = [torch.empty_like(s.q) for _ in new]
        for i, (k, out) in enumerate(zip(new, outs)):
            steps = [lambda: s.args[1].copy_(lengths[i]), lambda: ctx.rope(asked[i], s.q, positions[i], table), lambda: ctx.append(s.pool, k, back[i], None, slots)]
            for at in range(3):
                steps[(i + at) % 3]()
                if wait:
                    torch.cuda.synchronize()
            s.run(ctx, out, work=work)
            if wait:
                torch.cuda.synchronize()
        return torch.stack(outs)

    assert torch.equal(go(False), go(True))
    ctx.status()


def test_two_contexts_at_once(ctx):
    """Two streams, a context and a work memory each, the same pool: neither changes the other's results."""
    s = Shared(18, "f16", [1] * 50, [60] * 50, [0, 50], [900], 8, 2, 64, 32)
    want = s.run(ctx)
    other, streams = bp.PagedContext(), [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros_like(s.q) for _ in range(20)] for _ in streams]
    works = [torch.empty(ctx.shared_work(50, 8, 64), device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for c, stream, out, work in zip((ctx, other), streams, outs, works):
            with torch.cuda.stream(stream):
                s.run(c, out[i], work=work)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for out in outs for o in out)
    other.status()
    other.close()


@pytest.mark.parametrize("how", ["dense", "odd", "heads"])
def test_two_launches_over_strided_rows_and_over_the_queries(ctx, how):
    """Many rows behind a prefix, few of each request; rows before the first request and behind the last one stay."""
    s = Shared(19, "f16", [2] * 30, [20 + 5 * i for i in range(30)], [3, 30], [333], 8, 2, 128, 32, how=how)
    rows = torch.cat([torch.full((2, 8, 128), 5.0, dtype=s.q.dtype, device="cuda"), s.q, torch.full((3, 8, 128), 6.0, dtype=s.q.dtype, device="cuda")])
    keep = s.q
    s.args[0] = s.args[0] + 2
    s.q = strided(rows, how)
    for out in (strided(torch.full_like(rows, 7.0), how), s.q):
        before = out.clone()
        s.run(ctx, out)
        assert torch.equal(out[:2], before[:2]) and torch.equal(out[-3:], before[-3:])
        mine, s.q = s.q, keep
        s.check(out[2:-3])
        s.q = mine
    ctx.status()


@pytest.mark.parametrize("q,n", [(1, 5), (30, 5), (1, 45), (130, 5)])
def test_other_streams_and_graphs(ctx, q, n):
    """Captured twice with one work memory, replayed one behind the other: either follows the lengths on the device."""
    s = Shared(13, "bf16", [q] * n, [40 + 12 * (i % 5) for i in range(n)], [1, n], [400], 8, 2, 128, 32)
    want = s.run(ctx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.zeros_like(s.q) for _ in range(2)]
    work = torch.empty(ctx.shared_work(n * q, 8, 128), device="cuda")
    s.run(ctx, outs[0], work=work, stream=side)
    side.synchronize()
    assert torch.equal(outs[0], want)
    graphs = [torch.cuda.CUDAGraph() for _ in outs]
    for g, o in zip(graphs, outs):
        with torch.cuda.graph(g, stream=side):
            s.run(ctx, o, work=work)
    for cut in (0, 9):
        s.args[4].copy_(torch.tensor([400 - cut], dtype=torch.int32))
        s.prefix_len = [400 - cut]
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        s.check(outs[0])
    ctx.status()


def test_refusals(ctx):
    s = Shared(14, "f16", [2, 1], [30, 40], [0, 2], [50], 4, 2, 64, 16)
    run = lambda **kw: s.run(ctx, **kw)  # noqa: E731
    one = torch.zeros(3, 1, 64, dtype=torch.float16, device="cuda")
    bad = [lambda: run(scale=float("nan")), lambda: run(max_q=-1), lambda: run(work=torch.zeros(10, device="cuda")), lambda: run(work=torch.zeros(ctx.shared_work(3, 4, 64)).double()),
           lambda: ctx.attention_shared(s.pool, one, one, *s.args, torch.zeros(999, device="cuda"), max_q=2, max_kv=40, max_prefix=50),  # 1 head over 2
           lambda: run(work=torch.zeros(ctx.shared_work(3, 4, 64) + 1, device="cuda")[1:])]  # 16-byte alignment
    for call in bad:
        with pytest.raises(bp.ConfigError, match="^invalid config: "):
            call()
    lib = bp.paged._lib
    ok = dict(zip(("q_start", "kv_len", "page_table", "prefix_start", "prefix_len", "prefix_table"), (t.data_ptr() for t in s.args)))
    work = torch.zeros(ctx.shared_work(3, 4, 64), device="cuda")

    def entry(dtype=0, **kw):
        a = lib.SharedStruct(lib.RowsStruct(s.q.data_ptr(), 256, 64), lib.RowsStruct(s.q.data_ptr(), 256, 64))
        for k, v in {**ok, **dict(work=work.data_ptr(), n_req=2, n_head=4, total_q=3, max_q=2, max_kv=40, table_stride=4, n_prefix=1, max_prefix=50, prefix_stride=4, scale=0.1), **kw}.items():
            setattr(a, k, v)
        return ctx._lib.bp_kv4_attention_shared(ctx._h, None, dtype, s.pool._p, C.byref(a))

    for name in (*ok, "work"):
        assert entry(**{name: None}) == 7 and entry(**{name: (ok.get(name) or work.data_ptr()) + 2}) == 1, name
    # without prefixes there need be no tables of them, without own keys none of these
    none = dict(prefix_start=None, prefix_len=None, prefix_table=None, n_prefix=0)
    assert entry(**none) == 0 and entry(**none, max_prefix=0) == 0 and entry(page_table=None, max_kv=0) == 0
    with pytest.raises(bp.ContextOverflow):  # (which is reported: the requests say that they have some)
        ctx.status()
    assert entry(dtype=2) == 1 and entry(n_head=3) == 1 and entry(n_req=65536) == 1 and entry(n_prefix=65536) == 1 and entry(max_kv=1 << 31) == 1 and entry(max_prefix=1 << 31) == 1
    assert entry(total_q=1 << 30) == 1
    ctx.status()
