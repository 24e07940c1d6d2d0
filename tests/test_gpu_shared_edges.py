"""Attention behind prefixes in common where a call's sizes lie at an edge."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from tests.test_gpu_shared import ctx  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,want", [(2600, 64, 0), (2980, 64, 1), (3600, 64, 1), (3600, 128, 1)])
def test_places_of_both_parts_fit_32_bits(ctx, heads, dim, want):
    """65535 requests and as many prefixes of up to 64 keys: an item takes 2 tiles and 10 places at most, so 2 * 65535 * heads * 12 of them have to be below 2^32, which is so up to 2730
    heads. Requests and prefixes are empty here; what is accepted writes nothing."""
    n, lib = 65535, bp.paged._lib
    size = bp.KV4Pool.bytes(1, 16, heads, dim)
    pool = bp.KV4Pool(torch.zeros(size, dtype=torch.uint8, device="cuda"), 1, 16, heads, dim)
    q = torch.ones(1, heads, dim, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    zeros, table = torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    work = torch.zeros(ctx.shared_work(1, heads, dim), device="cuda")
    a = lib.SharedStruct(lib.RowsStruct(q.data_ptr(), heads * dim, dim), lib.RowsStruct(out.data_ptr(), heads * dim, dim))
    for k in ("q_start", "kv_len", "prefix_start", "prefix_len"):
        setattr(a, k, zeros.data_ptr())
    a.page_table = a.prefix_table = table.data_ptr()
    a.work, a.n_req, a.n_prefix, a.n_head, a.total_q, a.max_q, a.max_kv, a.max_prefix, a.table_stride, a.prefix_stride, a.scale = work.data_ptr(), n, n, heads, 1, 1, 64, 64, 4, 4, 1.0
    assert ctx._lib.bp_kv4_attention_shared(ctx._h, None, 0, pool._p, C.byref(a)) == want
    assert (out == 7.0).all()
    ctx.status()
