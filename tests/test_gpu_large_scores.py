"""Scores so large that neighbouring binary32 numbers are whole powers of two of a weight apart: what pieces of a row's keys are joined by.

Keys and queries are such that every q . k is a binary32 number that each of its partial sums is one for, too; a score is that times the scale in log2 units, which is a power of two
where a kernel rounds the product. So nothing rounds before the weights, and the tolerances are those of tests/test_gpu_paged.py: 2^-11 of a weight, half a unit of the output."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests.test_gpu_paged import HALF_UNIT, Requests, ctx, f64  # noqa: E402, F401
from tests.test_gpu_shared import Shared  # noqa: E402

pytestmark = pytest.mark.gpu

LARGE = 16 * 15 * 2.0 ** 15  # q . k but for its last step: between 2^22 and 2^23, where binary32 numbers are 0.5 apart


def scale_of(log2_units):
    """A binary32 scale whose product with binary32's log2(e) is exactly log2_units."""
    near = np.float32(log2_units * np.log(2.0))
    for step in range(-4, 5):
        s = (near.view(np.int32) + np.int32(step)).view(np.float32)
        if s * np.float32(1.4426950408889634) == np.float32(log2_units):
            return float(s)
    raise AssertionError("no such scale")


def exact(r, sign, order):
    """Keys of q . k = sign * (LARGE + c / 2) for whole c of 0 .. 15 in some order; whole values that go with c, so that a wrong weight shows."""
    rng = np.random.default_rng(5)
    dim, hkv = r.dim, r.hkv
    for row, n in enumerate(r.kv_len):
        at = np.arange(n)
        c = {"rising": 16 * at // max(n, 1), "falling": 15 - 16 * at // max(n, 1), "mixed": rng.integers(0, 16, n), "level": np.full(n, 6)}[order]
        k, v = np.zeros((n, hkv, dim), np.uint8), rng.integers(0, 8, (n, hkv, dim)).astype(np.uint8)
        k[:, :, :16] = 15
        k[:, :, 40] = c[:, None]
        v += (c[:, None, None] % 2 * 8).astype(np.uint8)
        if order == "level":
            v += (row % 2 * 8)
        one, none = np.ones((n, hkv, dim // 32), np.float16), np.zeros((n, hkv, dim // 32), np.float16)
        slots = r.table[row, at // r.page].astype(np.int64) * r.page + at % r.page
        for kind, codes in ((0, k), (1, v)):
            r.ref.write(kind, slots, codes, one, none)
        r.keys[row], r.values[row] = k.astype(np.float64), v.astype(np.float64)
    r.pool = bp.KV4Pool(torch.from_numpy(r.ref.bytes).cuda(), r.ref.bytes.shape[0], r.page, hkv, dim)
    r.q.zero_()
    r.q[:, :, :16] = sign * 2.0 ** 15
    r.q[:, :, 40] = sign * 0.5
    return r


# log2 units of a step of q . k are 2^(power - 1), largest scores 2^(22.9 + power)
POWERS = [-4, 0, 1, 2, 3, 4, 5, 6, 8, 30]


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("q,heads,hkv,dim,kv", [(1, 4, 1, 128, 3000), (3, 8, 2, 64, 700), (1, 2, 1, 64, 20000)])
def test_few_rows(ctx, power, sign, order, q, heads, hkv, dim, kv):
    """Maxima that grow or shrink along a warp's stretch, from warp to warp and from CTA to CTA."""
    r = exact(Requests(1, "f16", [q, q], [kv, kv // 3], heads, hkv, dim, 32), sign, order)
    scale = scale_of(2.0 ** power)
    r.check(r.run(ctx, scale=scale), scale=scale)
    ctx.status()


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("q,heads,hkv,dim,kv", [(40, 2, 2, 128, 3000), (130, 4, 1, 64, 900)])
def test_many_rows(ctx, power, order, q, heads, hkv, dim, kv):
    r = exact(Requests(2, "bf16", [q, q], [kv, kv // 3], heads, hkv, dim, 64), 1, order)
    scale = scale_of(2.0 ** power)
    r.check(r.run(ctx, scale=scale), scale=scale)
    ctx.status()


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("q,heads,hkv,dim,kv", [(40, 2, 2, 128, 3000), (130, 4, 1, 64, 900), (300, 1, 1, 64, 1500)])
def test_many_rows_of_any_scale(ctx, power, order, q, heads, hkv, dim, kv):
    """This kernel takes the maximum off before the scale comes in: no product is rounded before its difference is taken, in the joins neither."""
    r = exact(Requests(6, "f16", [q, q], [kv, kv // 3], heads, hkv, dim, 32), 1, order)
    for scale in (0.7 * 2.0 ** power, 1.13 * 2.0 ** power):
        r.check(r.run(ctx, scale=scale), scale=scale)
    ctx.status()


FORMS = [(1, 64, 4), (1, 5, 4), (3, 30, 4), (40, 5, 4), (450, 2, 4)]  # two launches side by side, one for few rows, two, one for many rows in parts, prefix and own keys in one item


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("order", ["rising", "mixed", "level"])
@pytest.mark.parametrize("q,n,heads", FORMS)
def test_behind_a_prefix(ctx, power, order, q, n, heads):
    """Prefix and own keys whose largest scores are equal, or steps apart, either way round."""
    prefix, own = 700, 90
    s = exact(Shared(3, "f16", [q] * n, [own if i % 3 else max(own, q) + 500 for i in range(n)], [0, n - 1], [prefix], heads, 2, 128 if q == 3 else 64, 32), 1, order)
    scale = scale_of(2.0 ** power)
    s.check(s.run(ctx, scale=scale), scale=scale)
    ctx.status()


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("order", ["rising", "mixed", "level"])
@pytest.mark.parametrize("q,n,heads", FORMS[3:])
def test_behind_a_prefix_with_any_scale(ctx, power, order, q, n, heads):
    """The same of the kernel for many rows alone; in parts its records hold what their maxima's products lose, up to 2^31."""
    s = exact(Shared(7, "f16", [q] * n, [590 if i % 3 else q + 500 for i in range(n)], [0, n - 1], [700], heads, 2, 64, 32), 1, order)
    for scale in (0.7 * 2.0 ** power, 1.13 * 2.0 ** power):
        if power < 9 or q > 40:
            s.check(s.run(ctx, scale=scale), scale=scale)
    ctx.status()


@pytest.mark.parametrize("power", [2, 3, 4, 5, 6])
@pytest.mark.parametrize("n_prefix,n_own", [(64, 64), (700, 100), (100, 700)])
def test_equal_keys_count_alike(ctx, power, n_prefix, n_own):
    """64 tokens: n_prefix keys with values of 1 behind n_own with values of 3, scores all the same."""
    s = exact(Shared(4, "f16", [1] * 64, [n_own] * 64, [0, 64], [n_prefix], 4, 2, 64, 32), 1, "level")
    for row, n in enumerate(s.kv_len):
        at = np.arange(n)
        slots = s.table[row, at // 32].astype(np.int64) * 32 + at % 32
        codes = np.full((n, 2, 64), 1 if row == s.n else 3, np.uint8)
        s.ref.write(1, slots, codes, np.ones((n, 2, 2), np.float16), np.zeros((n, 2, 2), np.float16))
    s.pool = bp.KV4Pool(torch.from_numpy(s.ref.bytes).cuda(), s.ref.bytes.shape[0], 32, 2, 64)
    out = s.run(ctx, scale=scale_of(2.0 ** power))
    want = (n_prefix + 3 * n_own) / (n_prefix + n_own)
    assert (np.abs(f64(out) - want) <= HALF_UNIT["f16"] * want + 2.0 ** -20).all()
    ctx.status()


@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("order", ["rising", "mixed"])
def test_chosen_pages(ctx, power, order):
    """A list of all pages."""
    kv, page = 1500, 32
    r = exact(Requests(5, "f16", [1] * 3, [kv, 700, 64], 8, 2, 128, page), 1, order)
    n = -(-kv // page)
    pages = torch.full((3, 2, n), -1, dtype=torch.int32, device="cuda")
    for i, k in enumerate(r.kv_len):
        pages[i, :, :-(-k // page)] = torch.from_numpy(r.table[i, :-(-k // page)]).cuda()
    out = torch.full_like(r.q, float("nan"))
    scale = scale_of(2.0 ** power)
    ctx.attention_selected(r.pool, r.q, out, pages, r.args[1], scale=scale)
    r.check(out, scale=scale)
    ctx.status()
