"""Several requests at once over one paged 4-bit KV cache: prompts in chunks, then one token per request and step.

One attention layer of the 8B shape (32 query / 8 KV heads of 128) on made-up activations stands for a model's layers: what a layer
does with its cache is complete (norm, rotary positions, append, attention), the projections around it are not there. A request
gets pages as it grows and gives them back when it ends. The outputs of every prompt chunk and of the last step are compared with a
plain softmax over the keys and values that the cache says it holds.

    python examples/paged_serving.py [--steps 64]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import bonsai_pot_b200 as bp  # noqa: E402

N_HEAD, N_KV_HEAD, HEAD_DIM, PAGE, N_PAGES, CHUNK, MAX_POS = 32, 8, 128, 32, 512, 512, 8192


class Server:
    """Pages and lengths of the requests (host side), the cache of one layer and what its calls need (device side)."""

    def __init__(self):
        self.ctx = bp.PagedContext(device=0)
        self.pool = bp.KV4Pool(torch.empty(bp.KV4Pool.bytes(N_PAGES, PAGE, N_KV_HEAD, HEAD_DIM), dtype=torch.uint8, device="cuda"), N_PAGES, PAGE, N_KV_HEAD, HEAD_DIM)
        table = torch.empty(MAX_POS, HEAD_DIM // 2, 2, device="cuda")
        self.ctx.fill_rope(table, freq_base=1e6, scaling="yarn", factor=4.0, orig_ctx=MAX_POS // 4)
        self.rope = bp.RopeTable(table, layout="half")
        self.w_q, self.w_k = (1 + 0.1 * torch.randn(2, HEAD_DIM, device="cuda")).bfloat16()
        self.free, self.pages, self.length = list(range(N_PAGES)), {}, {}

    def add(self, request):
        self.pages[request], self.length[request] = [], 0

    def drop(self, request):
        self.free += self.pages.pop(request)
        del self.length[request]

    def layer(self, requests, new, qkv):
        """`new[i]` further tokens of requests[i], all of them packed in qkv [tokens, heads + 2 KV heads, head_dim]: their attention outputs."""
        positions, slots, starts = [], [], [0]
        for r, n in zip(requests, new):
            at = self.length[r]
            while len(self.pages[r]) * PAGE < at + n:
                self.pages[r].append(self.free.pop())
            positions += range(at, at + n)
            slots += [self.pages[r][p // PAGE] * PAGE + p % PAGE for p in range(at, at + n)]
            self.length[r] = at + n
            starts.append(starts[-1] + n)
        lengths = [self.length[r] for r in requests]
        most = max(len(self.pages[r]) for r in requests)
        i32 = dict(dtype=torch.int32, device="cuda")
        positions, slots = torch.tensor(positions, **i32), torch.tensor(slots, device="cuda")
        q, k, v = qkv[:, :N_HEAD], qkv[:, N_HEAD:N_HEAD + N_KV_HEAD], qkv[:, N_HEAD + N_KV_HEAD:]
        turned, out = torch.empty_like(q), torch.empty(q.shape, dtype=q.dtype, device="cuda")
        self.ctx.rope(q, turned, positions, self.rope, w_norm=self.w_q)
        self.ctx.append(self.pool, k, v, positions, slots, self.rope, w_k_norm=self.w_k)
        self.ctx.attention(self.pool, turned, out, torch.tensor(starts, **i32), torch.tensor(lengths, **i32),
                           torch.tensor([self.pages[r] + [0] * (most - len(self.pages[r])) for r in requests], **i32), max_q=max(new), max_kv=max(lengths))
        return turned, out

    def keys(self, request):
        """What the cache holds of a request, as float32 [tokens, KV heads, head_dim]."""
        n = self.length[request]
        slots = torch.tensor([self.pages[request][p // PAGE] * PAGE + p % PAGE for p in range(n)], device="cuda")
        k, v = (torch.empty(n, N_KV_HEAD, HEAD_DIM, dtype=torch.float16, device="cuda") for _ in range(2))
        self.ctx.read(self.pool, slots, k, v)
        return k.float(), v.float()


def projections(n):
    return torch.randn(n, N_HEAD + 2 * N_KV_HEAD, HEAD_DIM, device="cuda").bfloat16()


def deviation(server, request, q, out):
    """Of `out`, the outputs of the request's last tokens q, from the plain softmax: the largest, and the largest in parts of sum p |v|."""
    k, v = (t.repeat_interleave(N_HEAD // N_KV_HEAD, 1) for t in server.keys(request))
    n, total = q.shape[0], k.shape[0]
    scores = torch.einsum("qhd,thd->qht", q.float(), k) / HEAD_DIM ** 0.5
    hidden = torch.arange(total, device="cuda") > torch.arange(total - n, total, device="cuda")[:, None]
    p = torch.softmax(scores.masked_fill(hidden[:, None], float("-inf")), -1)
    off = (torch.einsum("qht,thd->qhd", p, v) - out.float()).abs()
    return off.max().item(), (off / torch.einsum("qht,thd->qhd", p, v.abs())).max().item()


def run(steps=64, prompts=(700, 37, 1, 1300), seed=0):
    """Serves the prompts for `steps` tokens each; returns the largest deviation of the last step's outputs from the plain softmax."""
    return serve(steps, prompts, seed)[0]


def serve(steps, prompts, seed=0):
    """The same; returns that deviation, and the largest of the prompts' outputs in parts of sum p |v|."""
    torch.manual_seed(seed)
    of_prompts = 0.0
    server = Server()
    for r, n in enumerate(prompts):
        server.add(r)
        for at in range(0, n, CHUNK):
            q, out = server.layer([r], [min(CHUNK, n - at)], projections(min(CHUNK, n - at)))
            of_prompts = max(of_prompts, deviation(server, r, q, out)[1])
    live, worst = list(range(len(prompts))), 0.0
    for step in range(steps):
        q, out = server.layer(live, [1] * len(live), projections(len(live)))
        rows = list(live)
        if step == steps // 2 and len(live) > 1:  # a request ends, its pages serve the others
            server.drop(live.pop(1))
    for row, r in enumerate(rows if steps else []):
        if r not in live:
            continue
        worst = max(worst, deviation(server, r, q[row:row + 1], out[row:row + 1])[0])
    server.ctx.status()
    return worst, of_prompts


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=64)
    decoded, of_prompts = serve(ap.parse_args().steps, (700, 37, 1, 1300))
    print("largest deviation from a plain softmax: %.2g decoded, %.2g of sum p |v| in prompts" % (decoded, of_prompts))
