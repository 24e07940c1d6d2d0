"""The paged 4-bit operators on the GPU against their definitions (tests/paged_ref.py).

Tolerances. rope: one rounding to the 16-bit type (half a unit: 2^-11 or 2^-8 of the value, and 2^-25 below its smallest normal
number), and six binary32 operations on values of the size of the pair. append, read: none. attention: every P is rounded once to f16
(2^-11 of it at most, so 2^-11 of sum p |v|), the result once to its type; binary32 sums, of up to some thousand terms of either sign
and with scores up to about 30, move a P by less than 2^-13 of it."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    c = bp.PagedContext()
    yield c
    c.status()
    c.close()


def f64(t):
    return t.detach().cpu().double().numpy()


def normal(seed, shape, dtype, gain=1.0):
    x = np.random.default_rng(seed).standard_normal(shape) * gain
    return torch.from_numpy(x).to(TYPES[dtype]).cuda()


def strided(x, how):
    """The rows of x [n, heads, dim], laid out otherwise."""
    n, heads, dim = x.shape
    if how == "dense":
        return x.clone()
    if how == "fused":  # beside other heads
        big = torch.zeros(n, heads + 3, dim, dtype=x.dtype, device=x.device)
        view = big[:, 1:1 + heads]
    elif how == "odd":  # rows that are 2-byte aligned only
        big = torch.zeros(n * (heads * dim + 5) + 1, dtype=x.dtype, device=x.device)
        view = big[1:].as_strided((n, heads, dim), (heads * dim + 5, dim, 1), 1)
    else:  # heads outermost
        view = torch.zeros(heads, n, dim, dtype=x.dtype, device=x.device).transpose(0, 1)
    view.copy_(x)
    return view


# ---- rope ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rot", [2, 64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=2.0), dict(scaling="yarn", factor=8.0, orig_ctx=256),
                                dict(scaling="yarn", factor=1.0, orig_ctx=64)])
def test_rope_table(ctx, rot, kw):
    if kw.get("scaling") == "ntk" and rot == 2:
        pytest.skip("refused")
    out = torch.empty(1000, rot // 2, 2, device="cuda")
    ctx.fill_rope(out, freq_base=5e5, **kw)
    want = R.table(1000, rot, base=5e5, **kw)
    # cos and sin of an angle below 1000 in binary64, rounded once: half a unit of binary32, and what 64 bits lose
    assert np.abs(f64(out) - want.astype(np.float64)).max() <= 2 ** -23


ROPE = [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 128, 64), (2, 4, 64, 64), (7, 3, 256, 256), (5, 2, 80, 80), (4, 3, 96, 48), (3, 2, 80, 20), (2, 3, 64, 2), (33, 9, 128, 32), (2, 2, 6, 4)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("how", ["dense", "fused", "odd", "heads"])
@pytest.mark.parametrize("n,heads,dim,rot", ROPE)
def test_rope(ctx, dtype, layout, norm, how, n, heads, dim, rot):
    x = normal(n + dim, (n, heads, dim), dtype, 2.0)
    tab = R.table(300, rot)
    pos = np.random.default_rng(5).integers(0, 300, n).astype(np.int32)
    pos[0] = 299
    w = normal(7, (dim,), dtype) if norm else None
    want = f64(x)
    if norm:
        want = R.norm64(want, f64(w), 1e-5)
    size = np.abs(want)
    for inverse in (False, True):
        full = R.rotate(want, tab, pos, layout, inverse)
        p1, p2 = R.pairs(rot, layout)
        near = size.copy()
        near[..., p1] = near[..., p2] = size[..., p1] + size[..., p2]
        out = strided(torch.zeros_like(x), how)
        ctx.rope(strided(x, how), out, torch.from_numpy(pos).cuda(), bp.RopeTable(torch.from_numpy(tab).cuda(), layout), w_norm=w, eps=1e-5, inverse=inverse)
        err = np.abs(f64(out) - full)
        assert (err <= HALF_UNIT[dtype] * np.abs(full) + 2.0 ** -25 + 2.0 ** -20 * near).all(), err.max()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (80, 80), (64, 62)])
def test_rope_in_place_and_padding(ctx, layout, dim, rot):
    x = normal(1, (9, 4, dim), "bf16")
    tab = bp.RopeTable(torch.from_numpy(R.table(64, rot)).cuda(), layout)
    pos = torch.tensor([5, -1, 0, 63, 7, -2, 8, 9, 10], dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 3.0)
    ctx.rope(x, out, pos, tab)
    assert (out[[1, 5]] == 3.0).all()
    y = x.clone()
    ctx.rope(y, y, pos, tab)
    out[[1, 5]] = x[[1, 5]]
    assert torch.equal(y, out)
    ctx.status()
    ctx.rope(x, out, torch.full((9,), 64, dtype=torch.int32, device="cuda"), tab)
    with pytest.raises(bp.ContextOverflow):
        ctx.status()
    ctx.status()  # reported once


def test_rope_inverse_is_the_gradient(ctx):
    """d/dx of sum(g * rope(x)): by the inverse, and by central differences of the definition."""
    n, heads, dim, rot = 3, 2, 64, 32
    x, g = (f64(normal(s, (n, heads, dim), "f16")) for s in (1, 2))
    tab, pos = R.table(128, rot), np.array([3, 77, 127], np.int32)
    got = torch.empty(n, heads, dim, dtype=torch.float16, device="cuda")
    ctx.rope(torch.from_numpy(g).half().cuda(), got, torch.from_numpy(pos).cuda(), bp.RopeTable(torch.from_numpy(tab).cuda(), "interleaved"), inverse=True)
    h, want = 1e-3, np.empty_like(x)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += h
        down[i] -= h
        want[i] = ((R.rotate(up, tab, pos, "interleaved") - R.rotate(down, tab, pos, "interleaved")) * g).sum() / (2 * h)
    # the function is linear: differences are exact but for rounding, 64-bit noise over 2 h
    assert np.abs(f64(got) - want).max() <= 2.0 ** -11 * np.abs(want).max() + 1e-8


# ---- append and read -------------------------------------------------------------------------------------------------

def appended(pool, k, v, slots, pos, tab, layout, w, eps):
    x = k.float().cpu().numpy()
    if w is not None:
        x = R.norm32(x, w.float().cpu().numpy(), eps)
    if tab is not None:
        x = R.rotate(x, tab, pos, layout)
    for kind, rows in ((0, x), (1, v.float().cpu().numpy())):
        take = (slots >= 0) & (tab is None or pos >= 0)
        q, d, m = R.quantise(rows)
        pool.write(kind, slots[take], q[take], d[take], m[take])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("how", ["dense", "fused", "odd", "heads"])
@pytest.mark.parametrize("norm,layout,rot", [(True, "half", 1.0), (False, "half", 1.0), (True, "half", 0.5), (False, "half", 0.25), (True, "interleaved", 1.0),
                                             (False, "interleaved", 0.5), (True, None, 0), (False, None, 0), (True, "half", 0.1), (False, "interleaved", 0.1)])
@pytest.mark.parametrize("n,heads,dim,page", [(1, 8, 128, 16), (37, 3, 128, 64), (5, 1, 64, 32), (19, 8, 64, 16)])
def test_append_writes_the_defined_bytes(ctx, dtype, how, norm, layout, rot, n, heads, dim, page):
    rng = np.random.default_rng(n * dim)
    k, v = normal(1, (n, heads, dim), dtype, 1.7), normal(2, (n, heads, dim), dtype, 0.3)
    k[:, :, 5] *= 20
    v[0, 0, :32] = 0.75  # a constant block
    v[0, -1, 32:64] = 0.0
    k[-1, 0] = 3e-7 if dtype == "f16" else 1e-30  # below f16's normal numbers
    pages = -(-n // page) + 2
    slots = rng.permutation(pages * page)[:n].astype(np.int64)
    pos = rng.integers(0, 200, n).astype(np.int32)
    if n > 3:
        slots[2] = -1
        pos[3] = -7
    rot = int(dim * rot) // 2 * 2
    tab = R.table(200, rot) if layout else None
    w = (1 + 0.1 * normal(3, (dim,), dtype)).to(TYPES[dtype]) if norm else None
    want = R.Pool(pages, page, heads, dim, fill=0xA5)
    data = torch.from_numpy(want.bytes.copy()).cuda()
    appended(want, k, v, slots, pos, tab, layout, w, 1e-6)
    pool = bp.KV4Pool(data, pages, page, heads, dim)
    ctx.append(pool, strided(k, how), strided(v, how), torch.from_numpy(pos).cuda() if layout else None, torch.from_numpy(slots).cuda(),
               bp.RopeTable(torch.from_numpy(tab).cuda(), layout) if layout else None, w_k_norm=w)
    assert np.array_equal(data.cpu().numpy(), want.bytes)  # the places of padding and of nobody included
    # read back
    ko, vo = (strided(torch.full_like(k, 9.0), how) for _ in range(2))
    ctx.read(pool, torch.from_numpy(slots).cuda(), ko, vo)
    for kind, got in ((0, ko), (1, vo)):
        for i, s in enumerate(slots):
            if s < 0:
                assert (got[i] == 9.0).all()
            elif n <= 3 or i != 3:
                ref = torch.from_numpy(want.read(kind, int(s))).to(TYPES[dtype])
                assert torch.equal(got[i].cpu(), ref)
    ctx.status()


def test_append_of_numbers_that_are_none(ctx):
    n, heads, dim, page = 4, 2, 64, 16
    k, v = normal(1, (n, heads, dim), "bf16"), normal(2, (n, heads, dim), "bf16")
    k[0, 0, 3] = float("nan")
    v[1, 1, 40] = float("inf")
    v[2, 0, 7] = -1e30
    data = torch.zeros(bp.KV4Pool.bytes(1, page, heads, dim), dtype=torch.uint8, device="cuda")
    pool = bp.KV4Pool(data, 1, page, heads, dim)
    slots = torch.arange(n, device="cuda")
    ctx.append(pool, k, v, None, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ctx.read(pool, slots, ko, vo)
    assert ko[0, 0, :32].isnan().all() and not ko[0, 0, 32:].isnan().any() and not ko[1:].isnan().any()
    assert not vo.isinf().any() and not vo.isnan().any()
    # the largest value of a block lies within half a step of itself, a step is 129024 / 15 at most
    assert vo[1, 1, 40] >= 64512 - 4400 and vo[2, 0, 7] <= -64512 + 4400


def test_slots_out_of_range_are_reported(ctx):
    data = torch.zeros(bp.KV4Pool.bytes(2, 16, 1, 64), dtype=torch.uint8, device="cuda")
    pool = bp.KV4Pool(data, 2, 16, 1, 64)
    k = normal(1, (1, 1, 64), "f16")
    for call in (lambda s: ctx.append(pool, k, k, None, s), lambda s: ctx.read(pool, s, k.clone(), k.clone())):
        call(torch.tensor([31], device="cuda"))
        ctx.status()
        for slot in (32, 1 << 40):
            call(torch.tensor([slot], device="cuda"))
            with pytest.raises(bp.ContextOverflow):
                ctx.status()
    tab = bp.RopeTable(torch.from_numpy(R.table(8, 64)).cuda())
    before = data.clone()
    ctx.append(pool, 2 * k, k, torch.tensor([8], dtype=torch.int32, device="cuda"), torch.tensor([0], device="cuda"), tab)
    with pytest.raises(bp.ContextOverflow):
        ctx.status()
    assert torch.equal(before, data)


# ---- attention -------------------------------------------------------------------------------------------------------

class Requests:
    """Requests over a pool whose unused places and pages hold bits that are no numbers."""

    def __init__(self, seed, dtype, q_len, kv_len, heads, hkv, dim, page, spare=3, how="dense"):
        rng = np.random.default_rng(seed)
        self.q_len, self.kv_len, self.dtype, self.dim, self.page, self.hkv = q_len, kv_len, dtype, dim, page, hkv
        need = [-(-k // page) for k in kv_len]
        pages = sum(need) + spare
        self.ref = R.Pool(pages, page, hkv, dim, fill=0xFF)  # d, m = NaN
        order = rng.permutation(pages)
        self.table = np.full((len(kv_len), max(need + [1]) + 1), -1, np.int32)
        self.keys, self.values, at = [], [], 0
        for r, k in enumerate(kv_len):
            self.table[r, :need[r]] = order[at:at + need[r]]
            at += need[r]
            x = rng.standard_normal((2, k, hkv, dim)).astype(np.float32)
            x[0, :, :, 3] *= 6
            x[0] += 0.4
            got = []
            for kind in range(2):
                q, d, m = R.quantise(x[kind])
                i = np.arange(k)
                self.ref.write(kind, self.table[r, i // page].astype(np.int64) * page + i % page, q, d, m)
                got.append(R.dequantise(q, d, m))
            self.keys.append(got[0])
            self.values.append(got[1])
        self.pool = bp.KV4Pool(torch.from_numpy(self.ref.bytes).cuda(), pages, page, hkv, dim)
        self.q = strided(normal(seed + 1, (sum(q_len), heads, dim), dtype, 1.5), how)
        self.start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.args = [torch.from_numpy(a).cuda() for a in (self.start, np.array(kv_len, np.int32), self.table)]

    def run(self, ctx, out=None, **kw):
        out = torch.full_like(self.q, float("nan")) if out is None else out
        ctx.attention(self.pool, self.q, out, *self.args, max_q=kw.pop("max_q", max(self.q_len)), max_kv=kw.pop("max_kv", max(self.kv_len)), **kw)
        return out

    def check(self, out, scale=None, window=0, only=None):
        for r in range(len(self.q_len)) if only is None else only:
            rows = slice(self.start[r], self.start[r + 1])
            want, weight = R.attention(f64(self.q[rows]), self.keys[r], self.values[r], self.dim ** -0.5 if scale is None else scale, window)
            err = np.abs(f64(out[rows]) - want)
            tol = HALF_UNIT[self.dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -24
            assert (err <= tol).all(), (r, err.max(), (err / tol).max())


HEADS = [(4, 1, 128), (8, 8, 64), (6, 2, 128), (8, 1, 64), (32, 8, 128), (14, 2, 64), (16, 1, 128), (20, 1, 128), (40, 1, 64)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_one_token_each(ctx, dtype, heads, hkv, dim, page):
    kv = [1, 0, 15, 16, 17, 63, 64, 65, 127, 130, 300]
    r = Requests(1, dtype, [1] * len(kv), kv, heads, hkv, dim, page)
    r.check(r.run(ctx))
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", HEADS)
@pytest.mark.parametrize("window", [0, 1, 33, 100])
def test_several_tokens_each(ctx, dtype, heads, hkv, dim, window):
    r = Requests(2, dtype, [5, 2, 0, 1, 8, 7, 3], [200, 2, 50, 64, 8, 3, 0], heads, hkv, dim, 16)  # 7 queries over 3 keys: four rows see none
    r.check(r.run(ctx, window=window), window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", HEADS)
@pytest.mark.parametrize("window", [0, 70])
def test_chunks_of_prompts(ctx, dtype, heads, hkv, dim, window):
    r = Requests(3, dtype, [129, 64, 1, 77], [129, 500, 260, 90], heads, hkv, dim, 32)
    r.check(r.run(ctx, window=window), window=window)


@pytest.mark.parametrize("how", ["fused", "odd", "heads"])
@pytest.mark.parametrize("q", [1, 4, 150])
def test_strided_rows(ctx, how, q):
    r = Requests(4, "f16", [q, q], [300, 170], 8, 2, 128, 64, how=how)
    out = strided(torch.zeros(2 * q, 8, 128, dtype=torch.float16, device="cuda"), how)
    r.check(r.run(ctx, out, scale=0.2), scale=0.2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gain", [1e-4, 1.0, 40.0])
@pytest.mark.parametrize("q", [1, 130])
def test_small_and_large_queries(ctx, dtype, gain, q):
    """Queries far below f16's normal numbers once scaled, and scores of hundreds (one key has all the weight)."""
    r = Requests(5, dtype, [q], [260], 8, 2, 128, 16)
    r.q *= gain
    scale = 1.0 if gain < 1 else None
    out = r.run(ctx, scale=scale)
    if gain > 1:  # scores up to about 1000: a binary32 score is off by 2^-24 of it per sum, a P by some 2^-12 more
        want, weight = R.attention(f64(r.q), r.keys[0], r.values[0], 128 ** -0.5)
        assert (np.abs(f64(out) - want) <= HALF_UNIT[dtype] * np.abs(want) + 2.0 ** -9 * weight + 2.0 ** -24).all()
    else:
        r.check(out, scale=scale)


@pytest.mark.parametrize("q", [1, 130])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("window", [0, 50])
def test_scales_that_turn_or_level_the_scores(ctx, q, scale, window):
    r = Requests(13, "bf16", [q, q], [300, 140], 8, 2, 64, 16)
    r.check(r.run(ctx, scale=scale, window=window), scale=scale, window=window)


@pytest.mark.parametrize("heads,hkv,dim,kv", [(32, 8, 128, 9000), (4, 1, 128, 20011), (8, 8, 64, 5000)])
def test_long_contexts_are_split(ctx, heads, hkv, dim, kv):
    r = Requests(6, "f16", [1, 1, 2], [kv, 10, 3000], heads, hkv, dim, 64)
    a = r.run(ctx)
    r.check(a)
    for _ in range(3):  # the order in which parts of a row arrive does not show
        assert torch.equal(a, r.run(ctx))
    r.check(r.run(ctx, window=2500), window=2500)


def test_many_requests(ctx):
    rng = np.random.default_rng(3)
    kv = [int(x) for x in rng.integers(0, 200, 331)]
    r = Requests(7, "bf16", [1] * 331, kv, 4, 2, 64, 16)
    r.check(r.run(ctx))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q", [1, 6])
def test_more_requests_than_threads(ctx, dim, q):
    """A thread then counts the work of several requests; some have no queries, some no keys."""
    rng = np.random.default_rng(dim + q)
    kv = [int(x) for x in rng.integers(0, 90, 1100)]
    r = Requests(12, "f16", [int(x) for x in rng.integers(0, q + 1, 1100)], kv, 4, 1, dim, 16)
    r.check(r.run(ctx))
    ctx.status()


def test_pages_behind_four_gigabytes(ctx):
    heads, hkv, dim, page = 4, 2, 128, 64
    record = hkv * page * dim * 5 // 4
    pages = (9 << 29) // record + 200  # 4.8 GB
    r = Requests(8, "f16", [1, 130], [500, 300], heads, hkv, dim, page)
    big = torch.empty(pages * record, dtype=torch.uint8, device="cuda")
    shift = pages - r.ref.bytes.shape[0]
    big[shift * record:] = r.pool.data.flatten()
    r.pool = bp.KV4Pool(big, pages, page, hkv, dim)
    r.args[2] = torch.where(r.args[2] >= 0, r.args[2] + shift, r.args[2]).int()
    r.check(r.run(ctx))
    k, v = normal(1, (1, hkv, dim), "f16"), normal(2, (1, hkv, dim), "f16")
    last = torch.tensor([pages * page - 1], device="cuda")
    ctx.append(r.pool, k, v, None, last)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ctx.read(r.pool, last, ko, vo)
    assert torch.equal(ko.cpu().double(), torch.from_numpy(R.dequantise(*R.quantise(k.float().cpu().numpy()))))


@pytest.mark.parametrize("q", [1, 100])
def test_lengths_and_pages_out_of_range(ctx, q):
    r = Requests(9, "f16", [q, q], [200, 150], 8, 2, 64, 16)
    # a request with more keys than the caller said: the others are right, nothing faults, and it is reported
    out = r.run(ctx, max_kv=150)
    with pytest.raises(bp.ContextOverflow):
        ctx.status()
    r.check(out, only=[1])
    if q > 1:  # and with more queries
        out = r.run(ctx, out=torch.full_like(r.q, 7.0), max_q=q - 1)
        with pytest.raises(bp.ContextOverflow):
            ctx.status()
    wrong = r.args[2].clone()
    wrong[0, 3] = 1 << 30
    keep, r.args[2] = r.args[2], wrong
    out = r.run(ctx)
    with pytest.raises(bp.ContextOverflow):
        ctx.status()
    r.check(out, only=[1])
    r.args[2] = keep
    # pages before a window may be anybody's
    want = r.run(ctx, window=20)
    wrong = keep.clone()
    wrong[0, : (200 - q - 20 + 1) // 16 if q < 180 else 0] = -1
    r.args[2] = wrong
    assert torch.equal(r.run(ctx, window=20), want)
    ctx.status()


def test_a_key_that_is_no_number_stays_with_its_request(ctx):
    r = Requests(10, "f16", [1, 1], [100, 100], 4, 1, 128, 16)
    good = r.run(ctx)
    slot = int(r.table[0, 2]) * 16 + 5
    k = torch.full((1, 1, 128), float("nan"), dtype=torch.float16, device="cuda")
    ctx.append(r.pool, k, k, None, torch.tensor([slot], device="cuda"))
    out = r.run(ctx)
    assert out[0].isnan().all() and torch.equal(out[1], good[1])


@pytest.mark.parametrize("q,kv", [(1, 4000), (1, 60), (96, 500)])
def test_other_streams_and_graphs(ctx, q, kv):
    """A captured call follows the lengths on the device: the same graph serves the next token."""
    r = Requests(11, "bf16", [q, q], [kv, kv // 2], 8, 2, 128, 32)
    want = r.run(ctx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(r.q)
    with torch.cuda.stream(side):
        r.run(ctx, out, stream=side)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(graph, stream=side):
        r.run(ctx, out, stream=torch.cuda.current_stream())
    for cut in (0, 7, kv // 2 - q):
        r.args[1].copy_(torch.tensor([kv - cut, kv // 2 - min(cut, 3)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, r.run(ctx, max_kv=kv))
        r2 = r
        r2.keys = [x[:n] for x, n in zip(r.keys, (kv - cut, kv // 2 - min(cut, 3)))]
        r2.values = [x[:n] for x, n in zip(r.values, (kv - cut, kv // 2 - min(cut, 3)))]
        r2.check(got)
    ctx.status()


@pytest.mark.parametrize("q", [1, 200])
def test_no_keys_at_all(ctx, q):
    """Zeros for every query, without a look at a pool or a page table (the C entry takes neither)."""
    rows = normal(1, (2 * q, 4, 64), "f16")
    out = torch.full_like(rows, float("nan"))
    start, kv = torch.tensor([0, q, 2 * q], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    lib = bp.paged._lib
    r = [lib.RowsStruct(t.data_ptr(), 256, 64) for t in (rows, out)]
    a = lib.AttnStruct(*r, start.data_ptr(), kv.data_ptr(), None, 2, 4, 2 * q, q, 0, 0, 0, 0.125)
    assert ctx._lib.bp_kv4_attention(ctx._h, None, 0, C.byref(lib.PoolStruct(None, 1, 16, 2, 64)), C.byref(a)) == 0
    assert (out == 0).all()
    ctx.status()


def test_nothing_to_do(ctx):
    pool = bp.KV4Pool(torch.zeros(bp.KV4Pool.bytes(1, 16, 2, 64), dtype=torch.uint8, device="cuda"), 1, 16, 2, 64)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    i32 = torch.zeros(0, dtype=torch.int32, device="cuda")
    ctx.attention(pool, q, q, torch.zeros(1, dtype=torch.int32, device="cuda"), i32, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), max_q=0, max_kv=0)
    ctx.append(pool, k, k, None, torch.zeros(0, dtype=torch.int64, device="cuda"))
    ctx.read(pool, torch.zeros(0, dtype=torch.int64, device="cuda"), k, k)
    ctx.rope(q, q, i32, bp.RopeTable(torch.zeros(4, 32, 2, device="cuda")))
    ctx.status()


# ---- refusals --------------------------------------------------------------------------------------------------------

def test_refusals(ctx):
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    slots = torch.arange(3, device="cuda")
    tab = bp.RopeTable(torch.zeros(4, 32, 2, device="cuda"))
    data = torch.zeros(bp.KV4Pool.bytes(2, 16, 2, 64), dtype=torch.uint8, device="cuda")
    pool = bp.KV4Pool(data, 2, 16, 2, 64)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    start, kv = torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    bad = [
        lambda: ctx.rope(x.float(), x.float(), pos, tab),
        lambda: ctx.rope(x, x[:2], pos, tab),
        lambda: ctx.rope(x, x, pos[:2], tab),
        lambda: ctx.rope(x, x, pos.long(), tab),
        lambda: ctx.rope(x[..., :32], x[..., :32], pos, tab),  # rot_dim > head_dim
        lambda: ctx.rope(x[..., ::2], x[..., ::2], pos, tab),
        lambda: ctx.rope(x, x, pos, tab, w_norm=x[0, 0, :32]),
        lambda: ctx.rope(x, x, pos, tab, w_norm=x[0, 0], eps=-1.0),
        lambda: ctx.rope(x[..., :0], x[..., :0], pos, tab),
        lambda: bp.RopeTable(torch.zeros(4, 32, 2, device="cuda"), layout="other"),
        lambda: bp.RopeTable(torch.zeros(4, 64, device="cuda")),
        lambda: ctx.fill_rope(torch.zeros(4, 1, 2, device="cuda"), scaling="ntk", factor=2.0),
        lambda: ctx.fill_rope(torch.zeros(4, 8, 2, device="cuda"), scaling="yarn", factor=2.0),
        lambda: ctx.fill_rope(torch.zeros(4, 8, 2, device="cuda"), scaling="linear", factor=0.5),
        lambda: ctx.fill_rope(torch.zeros(4, 8, 2, device="cuda"), scaling="none"),
        lambda: ctx.fill_rope(torch.zeros(4, 8, 2, device="cuda"), freq_base=0.0),
        lambda: bp.KV4Pool(data, 3, 16, 2, 64),
        lambda: bp.KV4Pool(data, 1, 16, 2, 96),
        lambda: bp.KV4Pool(data, 1, 8, 2, 64),
        lambda: bp.KV4Pool(data[1:], 1, 16, 2, 64) and ctx.append(bp.KV4Pool(data[1:], 1, 16, 2, 64), x, x, None, slots),  # 16-byte alignment
        lambda: ctx.append(pool, x[:, :1], x[:, :1], None, slots),
        lambda: ctx.append(pool, x, x.bfloat16(), None, slots),
        lambda: ctx.append(pool, x, x, None, slots.int()),
        lambda: ctx.append(pool, x, x, pos[:1], slots, tab),
        lambda: ctx.read(pool, slots, x, x[:, :1]),
        lambda: ctx.attention(pool, x[:, :1], x[:, :1], start, kv, table, max_q=3, max_kv=3),  # 1 head over 2
        lambda: ctx.attention(pool, x, x, start, kv, table.long(), max_q=3, max_kv=3),
        lambda: ctx.attention(pool, x, x, start[:1], kv, table, max_q=3, max_kv=3),
        lambda: ctx.attention(pool, x, x, start, kv, table, max_q=-1, max_kv=3),
        lambda: ctx.attention(pool, x, x, start, kv, table, max_q=3, max_kv=3, scale=float("nan")),
        lambda: ctx.attention(pool, x[..., :32], x[..., :32], start, kv, table, max_q=3, max_kv=3),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(bp.ConfigError) as e:
            call()
        assert str(e.value).startswith("invalid config: "), i
    lib, rows = ctx._lib, C.byref(bp.paged._lib.RowsStruct(x.data_ptr(), 128, 64))
    assert lib.bp_rope(ctx._h, None, 0, rows, rows, 3, 2, 64, None, tab._p, None, 0.0, 0) == 7
    assert lib.bp_kv4_append(ctx._h, None, 0, pool._p, rows, rows, 3, pos.data_ptr(), None, tab._p, None, 0.0) == 7
    assert lib.bp_kv4_append(ctx._h, None, 0, pool._p, rows, rows, 3, None, slots.data_ptr(), tab._p, None, 0.0) == 7
    assert lib.bp_kv4_read(ctx._h, None, 0, None, slots.data_ptr(), 3, rows, rows) == 7
    assert lib.bp_kv4_attention(ctx._h, None, 0, pool._p, None) == 7
    assert lib.bp_kv4_attention(ctx._h, None, 2, pool._p, C.byref(bp.paged._lib.AttnStruct())) == 1
    with pytest.raises(bp.ConfigError):
        bp.PagedContext(device=99)
    empty = C.c_void_p()
    assert lib.bp_paged_create(-1, C.byref(empty)) == 1
    assert lib.bp_paged_status(empty, None) == 5
    lib.bp_paged_destroy(empty)
    ctx.status()


def test_the_serving_example(ctx):
    """Prompts in chunks, decoded tokens, pages that change owners: the outputs are the plain softmax's over what the cache holds. bf16 outputs below 4
    in magnitude: half a unit is 2^-7 at most, and P's rounding 2^-11 of at most 4."""
    from examples import paged_serving
    assert paged_serving.run(steps=20) <= 2.0 ** -7 + 2.0 ** -8
