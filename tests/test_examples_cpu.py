"""The serving examples' own comparison: outputs that are no numbers, or that nobody wrote, are no small deviation."""
import pytest

torch = pytest.importorskip("torch")

import bonsai_pot_b200 as bp  # noqa: E402
from examples import paged_serving, shared_serving  # noqa: E402


class Cache:
    """Keys and values of one row."""

    def __init__(self, module, device="cpu"):
        g = torch.Generator().manual_seed(1)
        self.k, self.v = (torch.randn(9, module.N_KV_HEAD, module.HEAD_DIM, generator=g).to(device) for _ in range(2))

    def keys(self, *row):
        return self.k, self.v


DEVIATIONS = {"paged": lambda c, q, out: max(paged_serving.deviation(c, 0, q, out)), "shared": lambda c, q, out: shared_serving.deviation(c, 0, 1, q, out, alone=True)}


@pytest.mark.parametrize("name", DEVIATIONS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_outputs_that_are_no_numbers_deviate(name, bad):
    module = paged_serving if name == "paged" else shared_serving
    c = Cache(module)
    q = torch.randn(3, module.N_HEAD, module.HEAD_DIM)
    k, v = (t.repeat_interleave(module.N_HEAD // module.N_KV_HEAD, 1) for t in (c.k, c.v))
    scores = torch.einsum("qhd,thd->qht", q, k) / module.HEAD_DIM ** 0.5
    p = torch.softmax(scores.masked_fill((torch.arange(9) > torch.arange(6, 9)[:, None])[:, None], float("-inf")), -1)
    out = torch.einsum("qht,thd->qhd", p, v)
    assert DEVIATIONS[name](c, q, out) < 1e-4
    out[1, 5, 17] = bad
    assert max(0.0, DEVIATIONS[name](c, q, out)) == float("inf")


@pytest.mark.parametrize("name", DEVIATIONS)
def test_a_weight_of_zero_is_no_deviation(name):
    module = paged_serving if name == "paged" else shared_serving
    c = Cache(module)
    c.k, c.v = c.k[:1], c.v[:1]
    c.v[0, 2, 40] = 0.0
    out = c.v.repeat_interleave(module.N_HEAD // module.N_KV_HEAD, 1)
    q = torch.randn(out.shape)
    assert DEVIATIONS[name](c, q, out) == 0
    out[0, 2 * module.N_HEAD // module.N_KV_HEAD, 40] = 1e-3
    assert DEVIATIONS[name](c, q, out) == float("inf")


@pytest.mark.gpu
def test_outputs_that_nobody_writes_show(monkeypatch):
    for name in ("attention", "attention_shared"):
        monkeypatch.setattr(bp.PagedContext, name, lambda self, *a, **kw: None)
    assert paged_serving.serve(2, (40, 3)) == (float("inf"), float("inf"))
    assert shared_serving.run(2, 1000, (7,), 2)[0] == float("inf")


@pytest.mark.gpu
def test_a_decoded_step_says_that_rows_get_one_token(monkeypatch):
    """By max_q a call goes to the kernel for single tokens or to the one for prompts."""
    asked, call = [], bp.PagedContext.attention_shared
    monkeypatch.setattr(bp.PagedContext, "attention_shared", lambda self, *a, **kw: (asked.append((a[1].shape[0], kw["max_q"])), call(self, *a, **kw))[1])
    shared_serving.run(2, 1000, (7, 30), 5)
    layers = shared_serving.LAYERS
    assert asked == [(1000, 1000)] * layers + [(37, 30)] * layers + [(10, 1)] * layers
