"""The operators of paged serving with a 4-bit KV cache: rotary positions, append, attention.

  rope    rows [tokens, heads, head_dim] (a view into a fused projection's output) are rotated by their positions: half or
          interleaved layout, all or the first part of a head, with or without RMS norm first, forwards or inverse (the gradient)
  append  new keys (normalised, rotated) and values are quantised to 4 bits into the pages of a cache, and read back
  attend  queries of several requests, packed one behind the other, over each request's pages: one token, a few drafted
          tokens or a chunk of a prompt per request, causal up to the request's last key, optionally within a window

A cache page holds `page` tokens; a block is 32 consecutive dims of one head, a value is m + d * q with 16-bit d and m per
block and a whole q of 0 .. 15 (`_quantise` says which). `_unpack` says where a pool's bytes hold them.
"""
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one token of one request, the query heads of a layer: latency
        dict(name="rope_token", op="rope", n=1, n_head=32, head_dim=128, rot=128, layout="half", norm=True, inverse=False, dtype="f16"),
        # a prompt of the benchmark's length; half of every head rotated, interleaved
        dict(name="rope_prompt_2048", op="rope", n=2048, n_head=32, head_dim=128, rot=64, layout="interleaved", norm=False, inverse=False, dtype="bf16"),
        # the gradient of a long batch's queries, an odd number of tokens and narrow heads
        dict(name="rope_inverse_16383", op="rope", n=16383, n_head=24, head_dim=64, rot=64, layout="half", norm=False, inverse=True, dtype="bf16"),
        # one decoded token goes into its page
        dict(name="append_token", op="append", n=1, n_kv_head=8, head_dim=128, rot=128, layout="half", norm=True, page=16, dtype="f16"),
        # one token each of an odd number of requests
        dict(name="append_batch_47", op="append", n=47, n_kv_head=8, head_dim=128, rot=128, layout="half", norm=True, page=32, dtype="bf16"),
        # long prompts of several requests at once
        dict(name="append_prompt_16383", op="append", n=16383, n_kv_head=8, head_dim=128, rot=64, layout="interleaved", norm=False, page=64, dtype="bf16"),
        # a short conversation, one token
        dict(name="attend_token_300", op="attend", n_req=1, q=1, ragged=False, kv_min=300, kv=300, n_head=32, n_kv_head=8, head_dim=128, page=16, window=0, dtype="f16"),
        # a batch of conversations of all lengths, one of them not begun
        dict(name="attend_batch_64", op="attend", n_req=64, q=1, ragged=False, kv_min=0, kv=8191, n_head=32, n_kv_head=8, head_dim=128, page=32, window=0, dtype="bf16"),
        # the benchmark's long context, one token
        dict(name="attend_token_32768", op="attend", n_req=1, q=1, ragged=False, kv_min=32768, kv=32768, n_head=32, n_kv_head=8, head_dim=128, page=64, window=0, dtype="f16"),
        # drafted tokens are checked: up to five per request, narrow heads, a window
        dict(name="attend_draft_16x5", op="attend", n_req=16, q=5, ragged=True, kv_min=40, kv=4096, n_head=40, n_kv_head=8, head_dim=64, page=16, window=1024, dtype="bf16"),
        # chunks of the prompts of a few requests, of odd lengths, behind what is cached
        dict(name="attend_chunks_4x512", op="attend", n_req=4, q=512, ragged=True, kv_min=512, kv=4099, n_head=32, n_kv_head=8, head_dim=128, page=32, window=0, dtype="bf16"),
        # the last chunk of a long prompt
        dict(name="attend_chunk_2048_of_32768", op="attend", n_req=1, q=2048, ragged=False, kv_min=32768, kv=32768, n_head=32, n_kv_head=8, head_dim=128, page=64, window=0, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "rope":
        n_head, head_dim = rng.choice([(32, 128), (8, 128), (24, 64), (16, 256), (32, 80), (5, 96), (64, 128)])
        rot = rng.choice([head_dim, head_dim, head_dim // 2])
        return dict(op=op, n=_log(rng, 1, 8192), n_head=n_head, head_dim=head_dim, rot=rot, layout=rng.choice(["half", "interleaved"]),
                    norm=rng.random() < 0.4, inverse=rng.random() < 0.3, dtype=dtype)
    if op == "append":
        head_dim = rng.choice([64, 128, 128])
        return dict(op=op, n=_log(rng, 1, 16000), n_kv_head=rng.choice([1, 2, 4, 8, 8, 10]), head_dim=head_dim,
                    rot=rng.choice([head_dim, head_dim, head_dim // 2]), layout=rng.choice(["half", "interleaved"]), norm=rng.random() < 0.5,
                    page=rng.choice([16, 32, 64]), dtype=dtype)
    kind = rng.choice(["token", "token", "draft", "chunk", "chunk"])
    n_req = 1 if rng.random() < 0.3 else _log(rng, 2, 96 if kind == "token" else 24 if kind == "draft" else 4)
    kv = _log(rng, 20, min(32768, 400000 // n_req if kind != "chunk" else 32768 // n_req))
    q = 1 if kind == "token" else rng.randint(2, 8) if kind == "draft" else min(kv, _log(rng, 16, 2000 // n_req))
    n_head, n_kv_head, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (16, 16, 64), (24, 8, 128), (40, 8, 64), (32, 4, 128), (16, 1, 128), (14, 2, 64)])
    return dict(op=op, n_req=n_req, q=q, ragged=rng.random() < 0.6, kv_min=rng.choice([0, 1, max(1, kv // 8), kv]), kv=kv, n_head=n_head, n_kv_head=n_kv_head,
                head_dim=head_dim, page=rng.choice([16, 32, 64]), window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0, dtype=dtype)


def _lengths(case):
    """(queries, keys) of each request: the first has kv keys, the second kv_min, the others lie between a sixteenth of kv and kv.
    There are no more queries than keys unless there is no key at all."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, lo, hi = case["n_req"], max(1, case["kv_min"], case["kv"] // 16), case["kv"]
    kv = [hi] + [case["kv_min"] if i == 1 else _log(rng, lo, hi) for i in range(1, n)]
    q = [rng.randint(1, case["q"]) if case["ragged"] and i else case["q"] for i in range(n)]
    return [min(a, b) if b else a for a, b in zip(q, kv)], kv


# ---- what a user's program has in hand ------------------------------------------------------------------------------

def _rope_table(n_pos, rot, scale):
    """f32 (cos, sin) [n_pos][rot / 2][2], computed in 64 bits; `scale` > 1: positions stretched over a longer context."""
    inv = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot) / scale
    a = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _swapped(token, dim):
    """Whether a row of values has its two halves changed over: tokens with bit 1 set, where a row has 64 bytes."""
    return (token & 2).bool() if dim == 128 else torch.zeros_like(token, dtype=torch.bool)


def _k_codes(q):
    """q [.., dims] of 0 .. 15 (uint8) -> a row's bytes [.., dims / 2]: [chunk, block, half, byte, nibble]."""
    q = q.unflatten(-1, (-1, 4, 2, 2, 2)).movedim(-5, -4).movedim(-1, -3)
    return (q[..., 0] | (q[..., 1] << 4)).flatten(-4)


def _v_codes(q, swapped):
    """The same of values: [chunk, block, byte, nibble], then the halves; `swapped` goes with q without its last axis."""
    dim = q.shape[-1]
    q = q.unflatten(-1, (-1, 8, 2, 2)).movedim(-4, -3)
    q = (q[..., 0] | (q[..., 1] << 4)).flatten(-3).unflatten(-1, (2, dim // 4))
    return torch.where(swapped[..., None, None], q.flip(-2), q).flatten(-2)


def _pack(kq, kd, km, vq, vd, vm):
    """Codes [pages, heads, page, dims] (uint8) and scales [.., dims / 32] (f16) -> a pool [pages, heads, bytes]."""
    token = torch.arange(kq.shape[2], device="cuda")
    scales = [s.contiguous().view(torch.uint8) for s in (kd, km, vd, vm)]
    return torch.cat([t.flatten(2) for t in (_k_codes(kq), *scales[:2], _v_codes(vq, _swapped(token, kq.shape[3])), *scales[2:])], -1)


def _quantise(x):
    """x [.., dims] -> codes, d, m. With u = the distance of neighbouring 16-bit floats at the block's largest magnitude (a 64th
    above it), m and d are whole multiples of u: so every m + d * q is a 16-bit float itself."""
    b = x.unflatten(-1, (-1, 32))
    low, high = b.amin(-1), b.amax(-1)
    top = torch.maximum(low.abs(), high.abs()) * (1 + 1 / 64)
    u = ((top.view(torch.int32) & 0x7F800000).view(torch.float32) * 2 ** -10).clamp(min=2 ** -24)
    m = (low / u).round() * u
    d = ((high - low) * (1 / 15) / u).round() * u
    inv = torch.where(d > 0, 1 / d, 0.0)
    q = ((b - m[..., None]) * inv[..., None]).round().clamp(0, 15)
    return q.to(torch.uint8).flatten(-2), d.half(), m.half()


def _filled_pool(g, pages, heads, page, dim):
    gain = torch.ones(heads, dim, device="cuda")
    gain[:, torch.randint(0, dim, (4,), generator=g, device="cuda")] = 5.0  # keys have a few large channels
    shift = torch.randn(heads, dim, generator=g, device="cuda") * 0.5
    shape = (pages, heads, page, dim)
    k = torch.randn(shape, generator=g, device="cuda") * gain[:, None] + shift[:, None]
    kq, kd, km = _quantise(k)
    del k
    return _pack(kq, kd, km, *_quantise(torch.randn(shape, generator=g, device="cuda") * 0.7))


_kept = {}


def _context():
    """A program makes one context and keeps it."""
    if "ctx" not in _kept:
        import bonsai_pot_b200 as bp
        _kept["ctx"] = bp.PagedContext(device=torch.cuda.current_device())
    return _kept["ctx"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    dtype, dim = DTYPES[case["dtype"]], case["head_dim"]
    if case["op"] in ("rope", "append"):
        n = case["n"]
        heads = case["n_head"] if case["op"] == "rope" else 2 * case["n_kv_head"]
        # the operator's heads lie in a fused projection's output beside others
        fused = torch.randn(n, heads + 4, dim, generator=g, device="cuda").mul_(1.5).to(dtype)
        n_pos = 4 * n + 512
        s["table"] = _rope_table(n_pos, case["rot"], 4.0 if n > 4096 else 1.0)
        s["positions"] = torch.randint(0, n_pos, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["w_norm"] = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype) if case["norm"] else None
    if case["op"] == "rope":
        s["x"] = fused[:, :heads]
        s["out"] = torch.empty(n, heads, dim, device="cuda", dtype=dtype)
    elif case["op"] == "append":
        hkv, page = case["n_kv_head"], case["page"]
        s["k"], s["v"] = fused[:, 4:4 + hkv], fused[:, 4 + hkv:4 + 2 * hkv]
        s["pages"] = -(-n // page) + 8
        s["pool"] = torch.zeros(s["pages"], hkv, page * dim * 5 // 4, device="cuda", dtype=torch.uint8)
        s["slots"] = torch.randperm(s["pages"] * page, generator=g, device="cuda")[:n]
        s["k_out"], s["v_out"] = (torch.empty(n, hkv, dim, device="cuda", dtype=dtype) for _ in range(2))
    else:
        q_len, kv_len = _lengths(case)
        page, n = case["page"], sum(q_len)
        need = [-(-x // page) for x in kv_len]
        s["pages"], s["max_q"], s["max_kv"] = sum(need) + 3, max(q_len), max(kv_len)
        s["pool"] = _filled_pool(g, s["pages"], case["n_kv_head"], page, dim)
        order = torch.randperm(s["pages"], generator=g, device="cuda", dtype=torch.int32)
        s["page_table"] = torch.zeros(case["n_req"], max(max(need), 1), device="cuda", dtype=torch.int32)
        at = 0
        for i, k in enumerate(need):
            s["page_table"][i, :k] = order[at:at + k]
            at += k
        s["q_start"] = torch.tensor([sum(q_len[:i]) for i in range(len(q_len) + 1)], device="cuda", dtype=torch.int32)
        s["kv_len"] = torch.tensor(kv_len, device="cuda", dtype=torch.int32)
        s["queries"] = torch.randn(n, case["n_head"], dim, generator=g, device="cuda").to(dtype)
        s["out"] = torch.empty_like(s["queries"])
    if own:
        import bonsai_pot_b200 as bp
        s["ctx"] = _context()
        if "pool" in s:
            s["cache"] = bp.KV4Pool(s["pool"], s["pages"], case["page"], case["n_kv_head"], dim)
        if "table" in s:
            s["rope"] = bp.RopeTable(s["table"], layout=case["layout"])
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _unpack(pool, heads, page, dim):
    """pool [.., heads, bytes] -> K and V f32 [.., heads, page, dims].

    A page of a head: K codes [page][dims / 2 bytes], K d [page][blocks] f16, K m, then the same of V. Row of K: four chunks c of
    one 32-bit word per block b; bits 4 j of it are dim 32 b + 8 c + 2 j, bits 16 + 4 j the one behind it. Row of V: eight chunks
    c of 16 bits per block b; bits 4 i are dim 32 b + 4 c + i."""
    lead, nb, half = pool.shape[:-1], dim // 32, page * dim * 5 // 8

    def one(part):
        codes = part[..., :page * dim // 2]
        scales = part[..., page * dim // 2:].contiguous().view(torch.float16).unflatten(-1, (2, page, nb)).float()
        nibbles = torch.stack([codes & 15, codes >> 4], -1)
        return nibbles, scales[..., 0, :, :, None], scales[..., 1, :, :, None]

    k, d, m = one(pool[..., :half])
    k = k.reshape(*lead, page, 4, nb, 2, 2, 2).movedim(-5, -4).movedim(-3, -1).reshape(*lead, page, nb, 32)
    keys = (k.float() * d + m).flatten(-2)
    v, d, m = one(pool[..., half:])
    v = v.reshape(*lead, page, 2, -1)
    v = torch.where(_swapped(torch.arange(page, device="cuda"), dim)[:, None, None], v.flip(-2), v)
    v = v.reshape(*lead, page, 8, nb, 2, 2).movedim(-4, -3).reshape(*lead, page, nb, 32)
    return keys, (v.float() * d + m).flatten(-2)


def _norm(x, w):
    """RMS norm of the last axis in 32 bits; the squares of neighbours are added, then pairs, then fours, as the operator defines it
    (its 4-bit codes depend on the last bit)."""
    dim = x.shape[-1]
    if dim & (dim - 1):
        mean = (x * x).mean(-1, keepdim=True)
    else:
        t = (x * x).view(*x.shape[:-1], *([2] * 6), -1)
        t = t[..., 0] if dim == 64 else t.sum(-1) if dim == 128 else t[..., 0::2].add(t[..., 1::2]).sum(-1)
        mean = (t.sum(-1).sum(-1).sum(-1).sum(-1).sum(-1).sum(-1) / dim)[..., None]
    return x * (mean + EPS).sqrt().reciprocal() * w.float()


def _rotate(x, table, positions, layout, inverse=False):
    rot = table.shape[1] * 2
    row = table[positions.long()][:, None]
    cos, sin = row[..., 0], row[..., 1]
    if inverse:
        sin = -sin
    head, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _rope_plain(s):
    x = s["x"].float()
    if s["norm"]:
        x = _norm(x, s["w_norm"])
    s["out"].copy_(_rotate(x, s["table"], s["positions"], s["layout"], s["inverse"]))
    return s["out"]


def _append_plain(s):
    heads, page, dim = s["n_kv_head"], s["page"], s["head_dim"]
    k = s["k"].float()
    if s["norm"]:
        k = _norm(k, s["w_norm"])
    k = _rotate(k, s["table"], s["positions"], s["layout"])
    nb, size = dim // 32, page * dim // 2
    where, tok = s["slots"] // page, s["slots"] % page
    for base, x in ((0, k), (page * dim * 5 // 8, s["v"].float())):
        q, d, m = _quantise(x.clamp(-64512, 64512))
        codes = _v_codes(q, _swapped(tok, dim)[:, None].expand(q.shape[:-1])) if base else _k_codes(q)
        s["pool"][..., base:base + size].unflatten(-1, (page, dim // 2))[where, :, tok] = codes
        scales = s["pool"][..., base + size:base + size + 4 * page * nb].unflatten(-1, (2, page, 2 * nb))
        scales[where, :, :, tok] = torch.stack([d, m], -2).view(torch.uint8)
    # read back
    keys, values = _unpack(s["pool"], heads, page, dim)
    s["k_out"].copy_(keys[where, :, tok])
    s["v_out"].copy_(values[where, :, tok])
    return {"k": s["k_out"], "v": s["v_out"]}


def _attend_plain(s):
    heads, hkv, page, dim, n_req = s["n_head"], s["n_kv_head"], s["page"], s["head_dim"], s["n_req"]
    group, max_q = heads // hkv, s["max_q"]
    tables = s["page_table"].long()
    keys, values = _unpack(s["pool"][tables], hkv, page, dim)  # [requests, pages, heads, page, dims]
    keys, values = (t.movedim(2, 1).reshape(n_req, hkv, -1, dim) for t in (keys, values))
    start = s["q_start"].long()
    q_len, kv_len = start[1:] - start[:-1], s["kv_len"].long()
    i = torch.arange(max_q, device="cuda")
    at = (start[:-1, None] + i).clamp(max=s["queries"].shape[0] - 1)
    q = s["queries"][at].float()  # [requests, max_q, heads, dims]; rows behind a request's own are not read below
    q = q.view(n_req, max_q, hkv, group, dim).permute(0, 2, 3, 1, 4).reshape(n_req, hkv, group * max_q, dim)
    scores = (q @ keys.transpose(-1, -2)) * dim ** -0.5
    scores = scores.view(n_req, hkv, group, max_q, -1)
    pos = (kv_len - q_len)[:, None] + i  # each query's place among its request's keys
    j = torch.arange(keys.shape[2], device="cuda")
    seen = (j <= pos[..., None]) & (j < kv_len[:, None, None])
    if s["window"]:
        seen &= j > pos[..., None] - s["window"]
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p.view(n_req, hkv, group * max_q, -1) @ values
    out = out.view(n_req, hkv, group, max_q, dim) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n_req, max_q, heads, dim)
    s["out"].copy_(out[i < q_len[:, None]])
    return s["out"]


def run(s):
    if not own:
        return {"rope": _rope_plain, "append": _append_plain, "attend": _attend_plain}[s["op"]](s)
    ctx = s["ctx"]
    if s["op"] == "rope":
        ctx.rope(s["x"], s["out"], s["positions"], s["rope"], w_norm=s["w_norm"], eps=EPS, inverse=s["inverse"])
        return s["out"]
    if s["op"] == "append":
        ctx.append(s["cache"], s["k"], s["v"], s["positions"], s["slots"], s["rope"], w_k_norm=s["w_norm"], eps=EPS)
        ctx.read(s["cache"], s["slots"], s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"]}
    ctx.attention(s["cache"], s["queries"], s["out"], s["q_start"], s["kv_len"], s["page_table"], max_q=s["max_q"], max_kv=s["max_kv"], window=s["window"])
    return s["out"]


def _pairs(q, kv, window):
    """(visible pairs, keys that some query sees) of one request of q queries at the end of kv keys."""
    if kv == 0:
        return 0, 0
    w = window or kv
    full = sum(min(kv - q + i + 1, w) for i in range(q))
    return full, min(kv, w + q - 1)


def work(case):
    dim = case["head_dim"]
    if case["op"] == "rope":
        values = case["n"] * case["n_head"] * dim
        return {"bytes": 4 * values + case["n"] * (4 * case["rot"] + 4), "flops": 3 * values * case["rot"] // dim}
    if case["op"] == "append":
        values = 2 * case["n"] * case["n_kv_head"] * dim  # read once, written and read as codes, written once
        return {"bytes": values * (2 + 0.625 + 0.625 + 2) + case["n"] * (4 * case["rot"] + 12), "flops": 8 * values}
    q_len, kv_len = _lengths(case)
    pairs = [_pairs(q, kv, case["window"]) for q, kv in zip(q_len, kv_len)]
    keys = sum(k for _, k in pairs)
    return {"bytes": keys * case["n_kv_head"] * dim * 1.25 + 4 * sum(q_len) * case["n_head"] * dim, "flops": 4 * dim * case["n_head"] * sum(p for p, _ in pairs)}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------

def _turn64(x, table, positions, layout, sign):
    rot, y = 2 * table.shape[1], x.clone()
    z = torch.complex(table[..., 0].double(), sign * table[..., 1].double())[positions.long()][:, None]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    w = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _norm64(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()


def _grid64(x):
    """The values that the 4-bit blocks stand for."""
    b = x.clamp(-64512, 64512).unflatten(-1, (-1, 32))
    low, high = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
    u = torch.exp2(torch.frexp(torch.maximum(-low, high) * 65 / 64).exponent.double().clamp(min=-13) - 11)
    m, d = (low / u).round() * u, ((high - low) / 15 / u).round() * u
    return (m + d * torch.where(d > 0, (b - m) / d, 0.0).round().clamp(0, 15)).flatten(-2)


def _page64(pool, page, dim, token):
    """K and V [heads, dims] in 64 bits of one token of every page: pool [pages, heads, bytes]."""
    nb, half, found = dim // 32, page * dim * 5 // 8, []
    for base, chunks in ((0, 4), (half, 8)):
        width = dim // 2 // chunks // nb
        row = pool[..., base + token * dim // 2:base + (token + 1) * dim // 2].long()
        if chunks == 8 and dim == 128 and token & 2:
            row = torch.cat([row[..., 32:], row[..., :32]], -1)
        d, m = (pool[..., at:at + 2 * nb].contiguous().view(torch.float16).double() for at in
                (base + page * dim // 2 + 2 * nb * token, base + page * dim // 2 + 2 * nb * (page + token)))
        out = torch.empty(*pool.shape[:-1], dim, dtype=torch.float64, device="cuda")
        for c in range(chunks):
            for b in range(nb):
                word = sum(row[..., (c * nb + b) * width + i] << (8 * i) for i in range(width))
                for i in range(2 * width):
                    at = 32 * b + 8 * c + (2 * i if i < 4 else 2 * i - 7) if chunks == 4 else 32 * b + 4 * c + i
                    out[..., at] = m[..., b] + d[..., b] * ((word >> (4 * i)) & 15)
        found.append(out)
    return found


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "attend":
        name = "x" if case["op"] == "rope" else "k"
        x = s[name].double()
        if case["norm"]:
            x = _norm64(x, s["w_norm"])
        x = _turn64(x, s["table"], s["positions"], case["layout"], -1 if case.get("inverse") else 1)
        return x if case["op"] == "rope" else {"k": _grid64(x), "v": _grid64(s["v"].double())}
    q_len, kv_len = _lengths(case)
    page, dim, hkv = case["page"], case["head_dim"], case["n_kv_head"]
    group, at, out = case["n_head"] // hkv, 0, []
    for r, (nq, nk) in enumerate(zip(q_len, kv_len)):
        q = s["queries"][at:at + nq].double().view(nq, hkv, group, dim)
        at += nq
        if nk == 0:
            out.append(torch.zeros(nq, hkv * group, dim, dtype=torch.float64, device="cuda"))
            continue
        pool = s["pool"][s["page_table"][r, :-(-nk // page)].long()]
        both = [_page64(pool, page, dim, t) for t in range(page)]
        keys, values = (torch.stack([b[i] for b in both], 1).flatten(0, 1)[:nk] for i in (0, 1))
        place = torch.arange(nk - nq, nk, device="cuda")[:, None]
        j = torch.arange(nk, device="cuda")
        hidden = (j > place) | (j <= place - case["window"] if case["window"] else j < 0)
        rows = torch.empty(nq, hkv, group, dim, dtype=torch.float64, device="cuda")
        for h in range(hkv):
            for k in range(group):
                p = torch.softmax((q[:, h, k] @ keys[:, h].T / dim ** 0.5).masked_fill(hidden, float("-inf")), -1)
                rows[:, h, k] = p @ values[:, h]
        out.append(rows.flatten(1, 2))
    return torch.cat(out)
