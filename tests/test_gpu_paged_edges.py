"""The paged 4-bit operators where numbers, sizes and masks lie at an edge; the tolerances are those of tests/test_gpu_paged.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests import paged_ref as R  # noqa: E402
from tests.test_gpu_paged import HALF_UNIT, TYPES, Requests, ctx, f64, normal  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pitch", [40, (1 << 25) + 24])
@pytest.mark.parametrize("q", [1, 130])
def test_page_tables_whose_rows_lie_apart(ctx, q, pitch):
    """A view into a larger table: beyond 2^25 entries of 64 tokens a row could hold more keys than 31 bits count."""
    r = Requests(14, "f16", [q, q, q], [300, 170, 500], 8, 2, 64, 64)
    n, pages = r.args[2].shape
    big = torch.zeros((n - 1) * pitch + pages, dtype=torch.int32, device="cuda")
    view = big.as_strided((n, pages), (pitch, 1))
    view.copy_(r.args[2])
    r.args[2] = view
    r.check(r.run(ctx))
    ctx.status()


@pytest.mark.parametrize("heads", [1, 40])
def test_windows_beyond_a_billion_keys(ctx, heads):
    """All pages are the same one but the first, whose keys have so large a score that one of them outweighs all the others together: a window
    that reaches it must not be cut shorter, one that does not reach it must not see it."""
    kv, page, dim = (1 << 30) + 5000, 64, 64
    rng = np.random.default_rng(15)
    k, v = (rng.standard_normal((2 * page, 1, dim)).astype(np.float32) for _ in range(2))
    k[:, :, 0] = 0.0
    k[:page, :, 0] = 64.0
    ref = R.Pool(2, page, 1, dim)
    for kind, x in ((0, k), (1, v)):
        ref.write(kind, np.arange(2 * page), *R.quantise(x))
    pool = bp.KV4Pool(torch.from_numpy(ref.bytes).cuda(), 2, page, 1, dim)
    table = torch.ones(1, -(-kv // page), dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    q = torch.zeros(1, heads, dim, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 10.0  # a score of 80 (natural logarithm) against 0 for a billion others
    out = torch.empty_like(q)
    start, length = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([kv], dtype=torch.int32, device="cuda")
    keys, values = (R.dequantise(*R.quantise(x))[:, 0] for x in (k, v))
    score = keys @ f64(q[0, 0]) * dim ** -0.5
    place = np.arange(page)
    for window, first in ((kv - 3, 3), (kv - 63, 63), (0, 0), (kv, 0), (kv - 64, page)):
        ctx.attention(pool, q, out, start, length, table, max_q=1, max_kv=kv, window=window)
        # how often each place of the two pages is seen
        times = np.concatenate([place >= first, (kv - page - 1 - place) // page + 1]).astype(np.float64)
        p = times * np.exp(score - score[times > 0].max())
        p /= p.sum()
        want, weight = p @ values, p @ np.abs(values)
        if first < page:  # (binary32 sums of the rest do not count)
            assert (np.abs(f64(out[0]) - want) <= HALF_UNIT["f16"] * np.abs(want) + (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -24).all(), window
        else:
            # a tensor core's binary32 sum may be cut, not rounded, at each of its steps of 16 keys: 2^-23 of it per step, and a CTA has
            # 2^26 / SMs steps in a row
            steps = (1 << 26) / torch.cuda.get_device_properties(0).multi_processor_count
            assert (np.abs(f64(out[0]) - want) <= (2.0 ** -10 + steps * 2.0 ** -23) * weight).all(), window
    ctx.status()


@pytest.mark.parametrize("dim,n", [(128, 1 << 23), (128, (1 << 23) + 3), (64, 1 << 24)])
def test_zeros_for_more_rows_than_32_bits_of_values(ctx, dim, n):
    """16 heads of n queries without any key. The queries are one row, the outputs lie four values apart (all are zeros), so that 2^27 rows fit."""
    q = torch.zeros(1, 1, dim, dtype=torch.float16, device="cuda").expand(n, 16, dim)
    store = torch.ones(n * 64 + dim - 4, dtype=torch.float16, device="cuda")
    out = store.as_strided((n, 16, dim), (64, 4, 1))
    pool = bp.KV4Pool(torch.zeros(bp.KV4Pool.bytes(1, 16, 4, dim), dtype=torch.uint8, device="cuda"), 1, 16, 4, dim)
    i32 = dict(dtype=torch.int32, device="cuda")
    ctx.attention(pool, q, out, torch.tensor([0, n], **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32), max_q=n, max_kv=0)
    assert not store.any()
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [1e4, 3e7, -2e9, 1e33])
@pytest.mark.parametrize("q,heads,hkv,dim,kv", [(1, 8, 2, 128, 700), (3, 10, 2, 64, 90), (1, 4, 1, 128, 9000), (70, 8, 2, 128, 300), (130, 4, 1, 64, 200)])
def test_scores_of_any_size(ctx, dtype, scale, q, heads, hkv, dim, kv):
    """With such scales one key has all the weight of a row; rows whose two largest scores lie nearer than 32 bits can tell are left out."""
    r = Requests(16, dtype, [q, q], [kv, kv // 2], heads, hkv, dim, 32)
    out = f64(r.run(ctx, scale=scale))
    told = asked = 0
    for i in range(2):
        keys, values, rows = r.keys[i], r.values[i], f64(r.q[r.start[i]:r.start[i + 1]])
        for j in range(q):
            n = len(keys) - q + j + 1
            if n <= 0:
                assert (out[r.start[i] + j] == 0).all()
                continue
            asked += heads
            for h in range(heads):
                s = keys[:n, h // (heads // hkv)] @ rows[j, h] * scale
                best = int(s.argmax())
                second = np.partition(s, -2)[-2] if n > 1 else -np.inf
                # binary32 sums of some 130 terms: 2^-22 of the sum of magnitudes; what the second has is exp(-gap) of the weight, below 2^-24
                noise = 2.0 ** -22 * (np.abs(keys[:n, h // (heads // hkv)]) @ np.abs(rows[j, h])).max() * abs(scale)
                if s[best] - second < 2 * noise + 17:
                    continue
                told += 1
                want = values[best, h // (heads // hkv)]
                got = out[r.start[i] + j, h]
                assert (np.abs(got - want) <= (HALF_UNIT[dtype] + 2.0 ** -11) * np.abs(want) + 2.0 ** -24 + 2.0 ** -22).all(), (i, j, h)
    assert told >= 0.8 * asked
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", [(4, 1, 128), (10, 2, 64), (16, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("q,kv,window,at", [(2, 70, 0, [69]), (4, 200, 0, [199, 198, 3]), (3, 129, 0, [127, 128]), (4, 300, 100, [198, 199, 200, 299, 100, 150]),
                                            (3, 64, 64, [63, 1]), (130, 500, 0, [499, 450, 401, 370, 20]), (130, 130, 0, [0, 64, 129]), (200, 700, 90, [499, 411, 412, 640, 699]),
                                            (520, 1400, 0, [1399, 1100]), (300, 2000, 65, [1700, 1900, 1635])])
def test_values_that_are_no_numbers_reach_who_sees_them(ctx, dtype, heads, hkv, dim, q, kv, window, at):
    """NaN in one block of a value at some keys: only queries that see such a key have it in their outputs, and only in the block's dims."""
    r = Requests(17, dtype, [q, 1], [kv, 90], heads, hkv, dim, 16)
    for i, key in enumerate(at):  # by append, as a layer would
        k = torch.from_numpy(r.keys[0][key]).half().cuda()[None]
        v = torch.from_numpy(r.values[0][key]).half().cuda()[None]
        block = i % (dim // 32)
        v[0, i % hkv, 32 * block + 5] = float("nan")
        ctx.append(r.pool, k, v, None, torch.tensor([int(r.table[0, key // 16]) * 16 + key % 16], device="cuda"))
        ks, vs = torch.empty_like(k), torch.empty_like(v)  # quantised anew: what the cache now holds
        ctx.read(r.pool, torch.tensor([int(r.table[0, key // 16]) * 16 + key % 16], device="cuda"), ks, vs)
        r.keys[0][key], r.values[0][key] = f64(ks[0]), f64(vs[0])
    out = r.run(ctx, window=window)
    none = np.isnan(r.values[0])
    r.values[0] = np.where(none, 0.0, r.values[0])
    place = np.arange(kv - q, kv)[:, None]
    seen = (np.arange(kv) <= place) & ((np.arange(kv) > place - window) if window else True)
    spoiled = np.repeat(np.einsum("qk,khd->qhd", seen.astype(np.int64), none.astype(np.int64)) > 0, heads // hkv, axis=1)
    got = f64(out)
    assert np.array_equal(np.isnan(got[:q]), spoiled) and spoiled.any() and not spoiled.all()
    want, weight = R.attention(f64(r.q[:q]), r.keys[0], r.values[0], dim ** -0.5, window)
    tol = HALF_UNIT[dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -24
    assert (np.abs(got[:q] - want) <= tol)[~spoiled].all()
    r.check(out, window=window, only=[1])
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim", [(4, 1, 128), (10, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("q", [1, 5, 130])
def test_queries_with_a_wide_range_within_a_row(ctx, dtype, heads, hkv, dim, q):
    """The first 32 dims of all keys are zeros, and those of the queries larger than the others by 2^17: what counts are the small ones, whose bits
    must have been kept. (The sums that the zeros are in have no share in an error.)"""
    r = Requests(18, dtype, [q, q], [300, 170], heads, hkv, dim, 32)
    for i in range(2):
        k, v = (torch.from_numpy(x).half().cuda() for x in (r.keys[i], r.values[i]))
        k[:, :, :32] = 0
        at = np.arange(len(k))
        slots = torch.from_numpy(r.table[i, at // 32].astype(np.int64) * 32 + at % 32).cuda()
        ctx.append(r.pool, k, v, None, slots)
        ks, vs = torch.empty_like(k), torch.empty_like(v)
        ctx.read(r.pool, slots, ks, vs)
        r.keys[i], r.values[i] = f64(ks), f64(vs)
        assert (r.keys[i][:, :, :32] == 0).all()
    small = 1.0 if dtype == "bf16" else 0.125
    r.q *= small
    r.q[:, :, :32] = 2.0 ** 17 * small
    out = r.run(ctx, scale=dim ** -0.5 / small)
    r.check(out, scale=dim ** -0.5 / small)


def test_a_new_context_is_ready_for_every_stream():
    """Its counters are zeroed behind what the legacy stream still has to do: creation waits for that."""
    bp.PagedContext().close()  # (what is loaded once has been)
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)  # some 100 ms
    before = torch.cuda.Event()
    before.record()
    c = bp.PagedContext()
    assert before.query()
    c.close()


# ---- long stretches: every warp or CTA works on many units of several items ------------------------------------------

class Shared(Requests):
    """Requests whose pages are drawn from a few hundred, many of them several times: long contexts that cost little to make. rising: a request's pages
    lie in the order of the size of their keys, so that a running maximum grows again and again on the way."""

    def __init__(self, seed, dtype, q_len, kv_len, heads, hkv, dim, page, rising=False, pages=150):
        rng = np.random.default_rng(seed)
        self.q_len, self.kv_len, self.dtype, self.dim, self.page, self.hkv = q_len, kv_len, dtype, dim, page, hkv
        self.ref = R.Pool(pages, page, hkv, dim)
        x = rng.standard_normal((2, pages * page, hkv, dim)).astype(np.float32)
        if rising:
            x[0] *= np.linspace(0.2, 3.0, pages, dtype=np.float32).repeat(page)[:, None, None]
        self.rows = []
        for kind in range(2):
            parts = R.quantise(x[kind])
            self.ref.write(kind, np.arange(pages * page), *parts)
            self.rows.append(R.dequantise(*parts).reshape(pages, page, hkv, dim))
        self.table = rng.integers(0, pages, (len(kv_len), max(-(-max(kv_len) // page), 1))).astype(np.int32)
        if rising:
            for row, k in zip(self.table, kv_len):
                row[:-(-k // page)].sort()
        self.pool = bp.KV4Pool(torch.from_numpy(self.ref.bytes).cuda(), pages, page, hkv, dim)
        self.q = normal(seed + 1, (sum(q_len), heads, dim), dtype, 1.5)
        self.start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.args = [torch.from_numpy(a).cuda() for a in (self.start, np.array(kv_len, np.int32), self.table)]

    def gathered(self, kind):
        class Rows:
            def __getitem__(_, r):
                k = self.kv_len[r]
                return self.rows[kind][self.table[r, :-(-k // self.page)]].reshape(-1, self.hkv, self.dim)[:k]
        return Rows()

    keys = property(lambda self: self.gathered(0))
    values = property(lambda self: self.gathered(1))


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# (heads, KV heads, head_dim, tokens, page, warps of a CTA): one and two tiles of eight rows, both dims; pages of 16: more than 32 of them per warp
@pytest.mark.parametrize("heads,hkv,dim,q,page,warps", [(32, 8, 128, 1, 16, 12), (32, 8, 128, 1, 64, 12), (16, 8, 64, 1, 16, 16), (16, 8, 64, 4, 32, 16), (32, 8, 128, 4, 32, 8),
                                                        (32, 4, 128, 2, 16, 8), (14, 2, 64, 2, 16, 12), (40, 8, 64, 5, 64, 12)])
@pytest.mark.parametrize("window", [0, 1500])
@pytest.mark.parametrize("rising", [False, True])
def test_many_units_per_warp(ctx, heads, hkv, dim, q, page, warps, window, rising):
    """Some 12 (pages of 16) or 6 units of 64 keys for every warp of the device, of ragged requests: rings are filled again and again, items change within
    a warp's stretch and end in the middle of it, page ids are read anew."""
    rng = np.random.default_rng(heads + q)
    rows = q * heads // hkv
    tiles = -(-rows // 8) if rows <= 8 else -(-rows // 16)
    units = (12 if page == 16 else 6) * warps * sms()
    kv = []
    while sum(min(k, window or k) for k in kv) * hkv * tiles < units * 64:
        kv.append(int(rng.integers(1, 4300)))
    kv[3] = 0
    r = Shared(19, "bf16", [q] * len(kv), kv, heads, hkv, dim, page, rising)
    out = r.run(ctx, window=window)
    r.check(out, window=window, only=sorted({0, 3, len(kv) - 1, int(np.argmax(kv)), *(int(x) for x in rng.integers(0, len(kv), 12))}))
    assert torch.equal(out, r.run(ctx, window=window))
    ctx.status()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,hkv,dim,q,kv", [(16, 8, 128, [100], [12100]), (16, 8, 64, [110], [12100]), (32, 8, 128, [20], [12100]), (24, 8, 64, [33], [12500]),
                                                (8, 4, 128, [150, 7, 60, 1, 129], [9000, 7000, 4100, 8000, 6000])])
@pytest.mark.parametrize("rising", [False, True])
def test_many_key_tiles_per_cta(ctx, dtype, heads, hkv, dim, q, kv, rising):
    """Ten tiles of 64 keys and more of one item per CTA (all slots several times), one and two query tiles; rising: O is rescaled on the way."""
    r = Shared(20, dtype, q, kv, heads, hkv, dim, 32, rising)
    out = r.run(ctx)
    r.check(out)
    assert torch.equal(out, r.run(ctx))
    ctx.status()


@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_and_chunks_in_one_call(ctx, dim):
    """What a server with chunked prompts issues: hundreds of requests with one token beside a few with a chunk."""
    rng = np.random.default_rng(dim)
    q = [1] * 300 + [200, 77, 1, 300]
    kv = [int(x) for x in rng.integers(1, 1500, 300)] + [900, 77, 0, 1300]
    order = rng.permutation(len(q))
    q, kv = [q[i] for i in order], [kv[i] for i in order]
    r = Shared(21, "bf16", q, kv, 8, 2, dim, 16)
    out = r.run(ctx)
    r.check(out, only=[i for i in range(len(q)) if q[i] > 1 or kv[i] == 0 or i % 9 == 0])
    r.check(r.run(ctx, window=333), window=333, only=[i for i in range(len(q)) if q[i] > 1 or i % 9 == 0])
    ctx.status()


def test_two_contexts_at_once(ctx):
    """Each has its own scratch memory: calls on two streams do not meet."""
    a, b = Shared(22, "f16", [1] * 3, [30000, 5000, 20000], 32, 8, 128, 32), Shared(23, "f16", [70, 3], [9000, 4000], 16, 4, 128, 32)
    want = [x.run(ctx) for x in (a, b)]
    a.check(want[0])
    b.check(want[1])
    torch.cuda.synchronize()
    with bp.PagedContext() as other:
        streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
        for _ in range(10):
            for i, (c, x) in enumerate(((ctx, a), (other, b))):
                with torch.cuda.stream(streams[i]):
                    outs[i].append(x.run(c, out=torch.zeros_like(x.q)))
        for i, c in enumerate((ctx, other)):
            c.status(stream=streams[i])
            assert all(torch.equal(o, want[i]) for o in outs[i])


# ---- rope: several heads per thread ----------------------------------------------------------------------------------

@pytest.mark.parametrize("n,heads,dim,rot,layout,norm,dtype", [(30500, 5, 80, 80, "half", True, "bf16"), (30500, 5, 128, 64, "interleaved", False, "f16"), (17000, 9, 128, 128, "half", False, "bf16"),
                                                              (17000, 9, 80, 32, "interleaved", True, "f16"), (6400, 24, 128, 128, "half", True, "f16"), (13000, 24, 64, 64, "interleaved", True, "bf16"),
                                                              (20000, 2, 256, 256, "half", False, "f16")])
def test_rope_of_long_prompts(ctx, n, heads, dim, rot, layout, norm, dtype):
    """So many rows that a thread has four heads of a token (or as many as are left); out of place, in place, tokens that are padding."""
    lanes = 1 << (dim // 16 - 1).bit_length()
    assert n * heads * lanes // 4 >= 2048 * sms() or heads < 3
    x = normal(n, (n, heads + 1, dim), dtype, 2.0)[:, 1:]
    tab = R.table(500, rot)
    pos = np.random.default_rng(6).integers(0, 500, n).astype(np.int32)
    pos[[0, 7, n - 1]] = -1
    w = normal(8, (dim,), dtype) if norm else None
    want = f64(x)
    if norm:
        want = R.norm64(want, f64(w), 1e-6)
    full = R.rotate(want, tab, np.maximum(pos, 0), layout)
    near = np.abs(want)
    p1, p2 = R.pairs(rot, layout)
    near[..., p1] = near[..., p2] = near[..., p1] + near[..., p2]
    table, at = bp.RopeTable(torch.from_numpy(tab).cuda(), layout), torch.from_numpy(pos).cuda()
    out = torch.full((n, heads, dim), 3.0, dtype=TYPES[dtype], device="cuda")
    ctx.rope(x, out, at, table, w_norm=w)
    there = pos >= 0
    assert (out[torch.from_numpy(~there).cuda()] == 3.0).all()
    err = np.abs(f64(out) - full)[there]
    assert (err <= (HALF_UNIT[dtype] * np.abs(full) + 2.0 ** -25 + 2.0 ** -20 * near)[there]).all(), err.max()
    before = x.clone()
    ctx.rope(x, x, at, table, w_norm=w)
    keep = torch.from_numpy(~there).cuda()
    assert torch.equal(x[keep], before[keep]) and torch.equal(x[~keep], out[~keep])
    ctx.status()


def test_the_prompts_of_the_serving_example(ctx):
    """bf16 outputs: half a unit is 2^-8 of the value at most, which is no larger than sum p |v|; P's rounding and the binary32 sums as everywhere."""
    from examples import paged_serving
    decoded, of_prompts = paged_serving.serve(1, (700, 37, 1, 1300), seed=1)
    assert decoded <= 2.0 ** -7 + 2.0 ** -8
    assert of_prompts <= 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -13


@pytest.mark.parametrize("q", [1, 70])
def test_queries_behind_the_rows_are_reported(ctx, q):
    r = Requests(24, "f16", [q, q, q], [200, 150, 90], 8, 2, 64, 16)
    want = r.run(ctx)
    r.check(want)
    for at, value, right in ((3, 3 * q + 2, [0, 1]), (3, (1 << 31) - 1, [0, 1]), (0, -3, [1, 2]), (0, -(1 << 31), [1, 2])):
        starts = r.args[0].clone()
        starts[at] = value
        keep, r.args[0] = r.args[0], starts
        out = r.run(ctx, max_q=q + 5)
        with pytest.raises(bp.ContextOverflow):
            ctx.status()
        r.check(out, only=right)
        r.args[0] = keep
    # entries for nobody: as many as there are, all behind the last request
    more = torch.cat([r.args[0], r.args[0][-1:].repeat(5)])
    lengths = torch.cat([r.args[1], torch.tensor([0, -1, 3, 0, -9], dtype=torch.int32, device="cuda")])
    r.args = [more, lengths, torch.cat([r.args[2], r.args[2][:1].repeat(5, 1)])]
    assert torch.equal(r.run(ctx), want)
    ctx.status()


@pytest.mark.parametrize("q,kv", [(1, 9000), (5, 700), (64, 3000), (300, 2000)])
def test_outputs_over_the_queries(ctx, q, kv):
    """out may be q: whoever writes a row has read it, and so have the others."""
    r = Shared(25, "bf16", [q, 1, q], [kv, 300, kv // 2], 32, 8, 128, 16)
    want = r.run(ctx)
    r.q = r.q.clone()
    r.run(ctx, out=r.q)
    assert torch.equal(r.q, want)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 32), (20, 8)])
def test_rope_inverse_of_a_table_with_a_factor(ctx, layout, dim, rot):
    """A YaRN table's cos and sin have a factor: the inverse is the transpose still, <rope(x), y> = <x, inverse(y)>, and undoes the rotation but for
    the factor's square."""
    factor = 8.0
    tab = torch.empty(300, rot // 2, 2, device="cuda")
    ctx.fill_rope(tab, scaling="yarn", factor=factor, orig_ctx=64)
    table, pos = bp.RopeTable(tab, layout), torch.tensor([0, 17, 299], dtype=torch.int32, device="cuda")
    x, y = normal(1, (3, 2, dim), "f16"), normal(2, (3, 2, dim), "f16")
    rx, iy, back = (torch.empty_like(x) for _ in range(3))
    ctx.rope(x, rx, pos, table)
    ctx.rope(y, iy, pos, table, inverse=True)
    ctx.rope(rx, back, pos, table, inverse=True)
    left, right = (f64(rx) * f64(y)).sum(-1), (f64(x) * f64(iy)).sum(-1)
    size = (np.abs(f64(rx) * f64(y)) + np.abs(f64(x) * f64(iy))).sum(-1)
    assert (np.abs(left - right) <= 2.0 ** -10 * size).all()  # both sides are sums of terms with one rounding to f16 each
    want = f64(x)
    p1, p2 = R.pairs(rot, layout)
    for p in (p1, p2):
        want[..., p] *= (0.1 * np.log(factor) + 1) ** 2
    near = np.abs(f64(rx)).max(-1, keepdims=True)
    assert (np.abs(f64(back) - want) <= 2.0 ** -9 * near * 1.3).all()  # rx and back are rounded to f16 once each, next to values of that size
