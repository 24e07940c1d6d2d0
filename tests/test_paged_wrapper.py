"""What PagedContext refuses, and what it hands to the C entry, without a GPU: the library is a stand-in that records its calls."""
import ctypes as C

import pytest

import bonsai_pot_b200 as bp
from bonsai_pot_b200 import paged

torch = pytest.importorskip("torch")


class Recorder:
    """Every entry of the library: notes its arguments and says that all went well."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0
        return entry


class Owner:
    """A table or pool as the context sees it."""
    _p, n_kv_head, head_dim, page_tokens = 0, 2, 64, 16

    def __init__(self, device=0):
        self.device = device


@pytest.fixture
def ctx():
    c = paged.PagedContext.__new__(paged.PagedContext)
    c._lib, c._h, c._device = Recorder(), C.c_void_p(), 0
    c._setup()
    return c


@pytest.mark.parametrize("name", ["rope", "append", "read", "attention"])
def test_host_tensors_do_not_reach_a_kernel(ctx, name):
    x, i32, slots = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32), torch.arange(3)
    owner = Owner()
    call = {
        "rope": lambda: ctx.rope(x, x, i32, owner),
        "append": lambda: ctx.append(owner, x, x, i32, slots, owner),
        "read": lambda: ctx.read(owner, slots, x, x),
        "attention": lambda: ctx.attention(owner, x, x, i32[:2], i32[:1], i32[:2].view(1, 2), max_q=3, max_kv=3),
    }[name]
    with pytest.raises(bp.ConfigError, match="^invalid config: .* must be on cuda:0, not on cpu"):
        call()
    assert ctx._lib.calls == []


def test_tables_and_pools_are_device_memory(ctx):
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        bp.RopeTable(torch.zeros(4, 32, 2))
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        bp.KV4Pool(torch.zeros(bp.KV4Pool.bytes(1, 16, 2, 64), dtype=torch.uint8), 1, 16, 2, 64)
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        ctx.fill_rope(torch.zeros(4, 32, 2))
    assert ctx._lib.calls == []


@pytest.mark.gpu
def test_every_tensor_of_a_call_is_looked_at():
    """One tensor at a time is on the host; nothing is launched."""
    cuda = {"x": torch.zeros(3, 2, 64, dtype=torch.float16), "out": torch.zeros(3, 2, 64, dtype=torch.float16), "pos": torch.zeros(3, dtype=torch.int32),
            "slots": torch.arange(3), "w": torch.ones(64, dtype=torch.float16), "table": torch.zeros(1, 2, dtype=torch.int32),
            "start": torch.tensor([0, 3], dtype=torch.int32), "kv": torch.tensor([3], dtype=torch.int32)}
    cuda = {k: v.cuda() for k, v in cuda.items()}
    tab = bp.RopeTable(torch.zeros(4, 32, 2, device="cuda"))
    pool = bp.KV4Pool(torch.zeros(bp.KV4Pool.bytes(1, 16, 2, 64), dtype=torch.uint8, device="cuda"), 1, 16, 2, 64)
    c = bp.PagedContext()
    calls = {
        ("x", "out", "pos", "w"): lambda t: c.rope(t["x"], t["out"], t["pos"], tab, w_norm=t["w"]),
        ("x", "out", "pos", "slots", "w"): lambda t: c.append(pool, t["x"], t["out"], t["pos"], t["slots"], tab, w_k_norm=t["w"]),
        ("x", "out", "slots"): lambda t: c.read(pool, t["slots"], t["x"], t["out"]),
        ("x", "out", "start", "kv", "table"): lambda t: c.attention(pool, t["x"], t["out"], t["start"], t["kv"], t["table"], max_q=3, max_kv=3),
    }
    real, c._lib = c._lib, Recorder()
    for names, call in calls.items():
        for name in names:
            with pytest.raises(bp.ConfigError, match="must be on cuda:0, not on cpu"):
                call({**cuda, name: cuda[name].cpu()})
        assert c._lib.calls == []
        call(cuda)
        assert len(c._lib.calls) == 1
        c._lib.calls.clear()
    other = bp.PagedContext.__new__(bp.PagedContext)  # a context of the next device: tables and pools of this one are refused too
    other._lib, other._h, other._device = Recorder(), C.c_void_p(), 1
    other._setup()
    with pytest.raises(bp.ConfigError, match="must be on cuda:1, not on cuda:0"):
        other.fill_rope(tab.data)
    with pytest.raises(bp.ConfigError, match="must be on cuda:1, not on cuda:0"):
        other.rope(cuda["x"], cuda["out"], cuda["pos"], tab)
    assert other._lib.calls == []
    c._lib = real
    c.close()


def test_without_a_stream_a_call_goes_to_the_current_one(ctx, monkeypatch):
    ctx._device = -1  # where host tensors lie: nothing here is refused
    x, i32, slots, owner = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32), torch.arange(3), Owner(-1)
    asked = []
    monkeypatch.setattr(paged, "_current", lambda device: asked.append(device) or 4711, raising=False)
    monkeypatch.setattr(bp.RopeTable, "__init__", lambda self, data, layout="half": setattr(self, "device", -1))
    for stream, want in ((None, 4711), (99, 99), (0, 0)):
        ctx.rope(x, x, i32, owner, stream=stream)
        ctx.append(owner, x, x, i32, slots, owner, stream=stream)
        ctx.read(owner, slots, x, x, stream=stream)
        ctx.attention(owner, x, x, i32[:2], i32[:1], i32[:2].view(1, 2), max_q=3, max_kv=3, stream=stream)
        ctx.fill_rope(torch.zeros(4, 32, 2), stream=stream)
        ctx.status(stream=stream)
        assert [args[1] for _, args in ctx._lib.calls] == [want] * 6
        ctx._lib.calls.clear()
    assert asked == [-1] * 6


def test_sizes_beyond_32_bits_are_not_cut_to_other_ones(ctx, monkeypatch):
    ctx._device = -1
    monkeypatch.setattr(paged, "_current", lambda device: 0)
    x, i32, owner = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32), Owner(-1)
    taken = []
    monkeypatch.setattr(ctx, "_lib", type("L", (), {"bp_kv4_attention": lambda self, *a: taken.append((ctx._attn.max_q, ctx._attn.max_kv, ctx._attn.window)) and 0})())

    def call(max_q=3, max_kv=3, window=0, page_table=i32[:2].view(1, 2)):
        ctx.attention(owner, x, x, i32[:2], i32[:1], page_table, max_q=max_q, max_kv=max_kv, window=window)
        return taken[-1]

    assert call() == (3, 3, 0) and call(window=2) == (3, 3, 2)
    assert call(max_q=1 << 32) == (3, 3, 0)  # no more queries than rows
    assert call(max_kv=1 << 32) == (3, 32, 0)  # no more keys than the table's pages hold
    assert call(window=(1 << 32) + 1) == (3, 3, 0) and call(window=3) == (3, 3, 0)  # a window over all keys is none
    n = len(taken)
    with pytest.raises(bp.ConfigError, match="^invalid config: "):
        call(max_kv=1 << 40, page_table=torch.empty(1, 1 << 28, dtype=torch.int32))  # pages of 2^32 tokens (nobody touches them)
    assert len(taken) == n
    for bad in ((1 << 32) + 1, 1 << 40):
        with pytest.raises(bp.ConfigError, match="^invalid config: "):
            bp.KV4Pool.bytes(bad, 16, 1, 64)
        with pytest.raises(bp.ConfigError, match="^invalid config: "):
            bp.KV4Pool.bytes(1, 16, bad, 64)


@pytest.mark.gpu
def test_calls_follow_the_current_stream():
    """On a stream of torch's own the rows are made late: a call that did not wait for them would take what was there before. And a call
    without a stream is captured like any other."""
    c = bp.PagedContext()
    tab = torch.empty(64, 32, 2, device="cuda")
    side = torch.cuda.Stream()
    x, out, pos = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda"), torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    ones = torch.ones_like(x)
    c.fill_rope(tab)
    table = bp.RopeTable(tab)
    want = torch.empty_like(x)
    c.rope(ones, want, pos, table)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # some 25 ms
        x.copy_(ones)
        c.rope(x, out, pos, table)
        c.status()  # waits for the same stream
        assert side.query()
    assert torch.equal(out, want)
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.rope(x, out, pos, table)
    assert (out == 0).all()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    c.close()
