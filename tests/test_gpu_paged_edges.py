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
