"""Page tables whose numbers are not what a server keeps in them: what a call refuses it reports and leaves."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests.test_gpu_pages import Both, ctx, dev  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def reported(ctx, call):
    call()
    with pytest.raises(bp.ContextOverflow):
        ctx.status()
    ctx.status()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("length", [-1, -(1 << 31), "one more", (1 << 31) - 1])
def test_a_row_of_no_possible_length_is_not_given_back(ctx, page, length):
    """Its length, its entries and every count stay; the other rows of the call end, one that is there twice once."""
    b = Both(1, 4, 5, 40, page, [3 * page + 1, 5 * page, 7, 2 * page])
    length = 5 * page + 1 if length == "one more" else length
    b.kv[1] = length
    table = b.table.clone()
    reported(ctx, lambda: ctx.release(b.gpu, dev([0, 1, 1, 3, 3])))
    assert b.kv.tolist() == [0, length, 7, 0] and torch.equal(b.table, table)
    b.kv[1] = 5 * page
    b.ref.release([0, 3])
    b.check()
    ctx.release(b.gpu, dev([1]))  # put right it ends like any other
    b.ref.release([1])
    b.check()
    ctx.status()


@pytest.mark.parametrize("rows,width", [(4, 30), (300, 1000)])
@pytest.mark.parametrize("count", [-1, -2, -6, -(1 << 31)])
def test_compaction_tells_counts_below_zero_from_moves(ctx, rows, width, count):
    """A page of such a count neither moves nor sends a row's entry elsewhere; it is reported. The others move."""
    page, n_pages = 16, 30000
    b = Both(2, rows, width, n_pages, page, [page * 20] + [page * 3] * (rows - 1))
    held = int(b.ref.table[0, 7])
    b.ref.refs[held] = count
    b.refs.copy_(dev(b.ref.refs))
    src, dst = dev([5] * 50), dev([5] * 50)
    reported(ctx, lambda: ctx.compact(b.gpu, src, dst))
    want = b.ref.compact(50)  # (which leaves alone what is neither free nor held)
    assert np.array_equal(src.cpu().numpy(), want[0]) and np.array_equal(dst.cpu().numpy(), want[1])
    assert (want[0] >= 0).sum() == min(50, 20 + 3 * (rows - 1) - 1) and b.ref.table[0, 7] == held
    b.check()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("pair", [0, 1, 2])
def test_forks_tell_a_length_below_zero_from_a_claimed_child(ctx, page, pair):
    """A child of any such length is not empty: its pair is reported, its row and every count stay. The other pairs are made."""
    b = Both(3, 8, 6, 60, page, [3 * page + 5, 2 * page, 0, 0, 0, 0, 4 * page + 1, 0])
    parents, children = [0, 1, 6, 0], [2, 3, 4, 5]
    b.ref.kv[children[pair]] = -1 - pair
    b.kv.copy_(dev(b.ref.kv))
    src, dst = dev([5] * 4), dev([5] * 4)
    reported(ctx, lambda: ctx.fork(b.gpu, dev(parents), dev(children), src, dst))
    parents[pair] = -1
    _, s, d = b.ref.fork(parents, children)
    assert np.array_equal(src.cpu().numpy(), s) and np.array_equal(dst.cpu().numpy(), d)
    b.check()
