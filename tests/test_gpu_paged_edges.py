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
