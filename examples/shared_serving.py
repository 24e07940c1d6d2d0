"""One long instruction, several questions about it, several answers to each, over one paged 4-bit cache whose page tables live on the device.

Row 0 of the tables is the instruction, the other rows are conversations behind it. The instruction's pages are held once, and attention
reads them once per step for all conversations. Every question is forked into answers, which share its full pages; answers that
end give their pages back, the pool is compacted, the others go on. A step (pages, norm and rotary positions, append, attention) is captured once per layout and
replayed: nothing of it asks the host. In the end one conversation reads on over chosen pages alone. Two attention layers of the 8B shape (32 query / 8 KV
heads of 128) on made-up activations stand for a model's; the outputs are compared with a plain softmax over what the cache says it holds.

    python examples/shared_serving.py [--steps 32]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import bonsai_pot_b200 as bp  # noqa: E402

N_HEAD, N_KV_HEAD, HEAD_DIM, PAGE, N_PAGES, LAYERS, ROW_PAGES, MAX_POS = 32, 8, 128, 32, 300, 2, 64, 8192
I32 = dict(dtype=torch.int32, device="cuda")


class Server:
    def __init__(self, rows):
        self.ctx, self.rows = bp.PagedContext(device=0), rows
        self.table, self.kv, self.refs = (torch.zeros(*shape, **I32) for shape in ((rows, ROW_PAGES), (rows,), (N_PAGES,)))
        self.tables = bp.PageTables(self.table, self.kv, self.refs, PAGE)
        data = torch.zeros(LAYERS, bp.KV4Pool.bytes(N_PAGES, PAGE, N_KV_HEAD, HEAD_DIM), dtype=torch.uint8, device="cuda")
        self.pools = [bp.KV4Pool(d, N_PAGES, PAGE, N_KV_HEAD, HEAD_DIM) for d in data]
        self.summaries = [bp.BlockSummary(torch.zeros(N_PAGES, N_KV_HEAD, 2, HEAD_DIM, dtype=torch.int8, device="cuda"), torch.zeros(N_PAGES, N_KV_HEAD, device="cuda")) for _ in range(LAYERS)]
        self.all = bp.KV4Pools(self.pools, self.summaries)
        angles = torch.empty(MAX_POS, HEAD_DIM // 2, 2, device="cuda")
        self.ctx.fill_rope(angles, freq_base=1e6)
        self.rope = bp.RopeTable(angles)
        self.prefix_start = torch.tensor([1, rows], **I32)  # the rows from 1 on go on where row 0 ends

    def step(self, n_new, qkv, turned, out, each, most, prefix):
        """n_new[r] further tokens for every row, packed in qkv [layers, tokens, heads + 2 KV heads, head_dim]; `each`, `most`, `prefix`: new tokens of a row, tokens of a row, of the
        instruction, at most (by `each` and by the rows behind the instruction attention goes to its kernels for single tokens or for prompts: say 1 where it is 1).
        Rows behind the instruction see it, too."""
        n = qkv.shape[1]
        start, positions, slots = torch.empty(self.rows + 1, **I32), torch.empty(n, **I32), torch.empty(n, dtype=torch.int64, device="cuda")
        self.ctx.grow(self.tables, n_new, start, positions, slots)
        first = torch.arange(n, **I32) < start[1]  # tokens of the instruction itself
        where = torch.where(first | (positions < 0), positions, positions + self.kv[:1])
        work = torch.empty(self.ctx.shared_work(n, N_HEAD, HEAD_DIM), device="cuda")
        for layer, pool in enumerate(self.pools):
            q, k, v = qkv[layer].split([N_HEAD, N_KV_HEAD, N_KV_HEAD], 1)
            self.ctx.rope(q, turned[layer], where, self.rope)
            self.ctx.append(pool, k, v, where, slots, self.rope)
            self.ctx.attention_shared(pool, turned[layer], out[layer], start, self.kv, self.table, self.prefix_start, self.kv[:1], self.table[:1], work, max_q=each, max_kv=most, max_prefix=prefix)

    def fork(self, parents, children):
        parents, children = torch.tensor(parents, **I32), torch.tensor(children, **I32)
        src, dst = torch.empty_like(parents), torch.empty_like(parents)
        self.ctx.fork(self.tables, parents, children, src, dst)
        self.ctx.copy_pages(self.all, src, dst)

    def drop(self, rows):
        self.ctx.release(self.tables, torch.tensor(rows, **I32))
        src, dst = torch.empty(N_PAGES, **I32), torch.empty(N_PAGES, **I32)
        self.ctx.compact(self.tables, src, dst)
        self.ctx.copy_pages(self.all, src, dst)

    def keys(self, layer, row):
        """What the cache holds of a row, as float32 [tokens, KV heads, head_dim]."""
        n = int(self.kv[row])
        at = torch.arange(n, device="cuda")
        k, v = (torch.empty(n, N_KV_HEAD, HEAD_DIM, dtype=torch.float16, device="cuda") for _ in range(2))
        self.ctx.read(self.pools[layer], self.table[row, at // PAGE].long() * PAGE + at % PAGE, k, v)
        return k.float(), v.float()


def projections(n):
    return torch.randn(LAYERS, n, N_HEAD + 2 * N_KV_HEAD, HEAD_DIM, device="cuda").bfloat16()


def deviation(server, layer, row, q, out, alone=False):
    """The largest deviation of `out`, the outputs of the row's last tokens q, from the plain softmax, in parts of sum p |v|; infinite where an output is no number."""
    k, v = server.keys(layer, row)
    own = k.shape[0]
    if row and not alone:
        k, v = (torch.cat(pair) for pair in zip(server.keys(layer, 0), (k, v)))
    k, v = (t.repeat_interleave(N_HEAD // N_KV_HEAD, 1) for t in (k, v))
    n, total = q.shape[0], k.shape[0]
    scores = torch.einsum("qhd,thd->qht", q.float(), k) / HEAD_DIM ** 0.5
    hidden = torch.arange(total, device=q.device) > torch.arange(total - n, total, device=q.device)[:, None]
    p = torch.softmax(scores.masked_fill(hidden[:, None], float("-inf")), -1)
    off = (torch.einsum("qht,thd->qhd", p, v) - out.float()).abs()
    assert own >= n
    weight = torch.einsum("qht,thd->qhd", p, v.abs())
    largest = torch.where(off == 0, 0.0, off / weight).max().item()  # (a token that sees one key may have a value of 0, and a weight of 0 with it)
    return largest if largest == largest else float("inf")  # (max() would pass over what is no number)


def run(steps=32, instruction=1000, questions=(37, 160, 5), answers=3, seed=0):
    """Serves it all; returns the largest deviation of any output looked at from the plain softmax, in parts of sum p |v|, and how many pages are held in the end."""
    torch.manual_seed(seed)
    n_q, rows = len(questions), 1 + len(questions) * (1 + answers)
    server, worst = Server(rows), 0.0

    def feed(n_new, rows_to_check):
        nonlocal worst
        n = sum(n_new)
        qkv = projections(n)
        turned, out = (torch.full((LAYERS, n, N_HEAD, HEAD_DIM), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))  # (so that a row nobody writes shows)
        server.step(torch.tensor(n_new, **I32), qkv, turned, out, max(n_new), ROW_PAGES * PAGE, instruction)
        at = 0
        for r, k in enumerate(n_new):
            if k and r in rows_to_check:
                worst = max(worst, *(deviation(server, layer, r, turned[layer, at:at + k], out[layer, at:at + k]) for layer in range(LAYERS)))
            at += k

    feed([instruction] + [0] * (rows - 1), [0])
    feed([0, *questions] + [0] * (rows - 1 - n_q), range(1, 1 + n_q))
    parents = [1 + i // answers for i in range(n_q * answers)]
    children = list(range(1 + n_q, rows))
    server.fork(parents, children)
    live = children
    # one captured step serves all that follow; rows that get nothing cost nothing, padding is skipped
    n_new = torch.zeros(rows, **I32)
    qkv = projections(len(children))
    turned, out = (torch.zeros(LAYERS, len(children), N_HEAD, HEAD_DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        server.step(n_new, qkv, turned, out, 1, ROW_PAGES * PAGE, instruction)
    for step in range(steps):
        if step == steps // 2 and len(live) > 1:
            server.drop([1, live[0], live[-1]])  # a question, whose answers go on, and two answers
            live = live[1:-1]
        n_new.zero_()
        n_new[live] = 1
        qkv.copy_(projections(len(children)))
        out.fill_(float("nan"))
        graph.replay()
        if step in (0, steps // 2, steps - 1):
            for i, r in enumerate(live):
                worst = max(worst, *(deviation(server, layer, r, turned[layer, i:i + 1], out[layer, i:i + 1]) for layer in range(LAYERS)))
    # the instruction itself is asked, over chosen pages: with places for all of them the outputs are those over all keys
    full = server.table[0, :instruction // PAGE].contiguous()
    q = torch.randn(1, N_HEAD, HEAD_DIM, device="cuda").bfloat16()
    for layer in range(LAYERS):
        server.ctx.summarise(server.pools[layer], server.summaries[layer], full)
        for places in (ROW_PAGES, 6):
            pages, keys, got = torch.empty(1, N_KV_HEAD, places, **I32), torch.empty(1, **I32), torch.full_like(q, float("nan"))
            server.ctx.select(server.pools[layer], server.summaries[layer], q, pages, keys, torch.tensor([0, 1], **I32), server.kv[:1], server.table[:1], max_q=1, max_kv=instruction, first=1, last=2)
            server.ctx.attention_selected(server.pools[layer], q, got, pages, keys)
            if places == ROW_PAGES:
                worst = max(worst, deviation(server, layer, 0, q, got, alone=True))
            elif int(keys) != 5 * PAGE + instruction % PAGE or not got.isfinite().all():
                raise RuntimeError("six pages hold five full ones' keys and the last one's, and outputs are numbers")
    server.ctx.status()
    return worst, int((server.refs > 0).sum())


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=32)
    print("largest deviation from a plain softmax: %.2g of sum p |v|; %d pages held" % run(ap.parse_args().steps))
