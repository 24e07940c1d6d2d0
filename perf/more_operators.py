"""Pages of a 4-bit cache that requests share, copy, give back and choose among.

  turnover  rows of a page table are given back, then every row grows by some tokens: pages, positions and slots for them
  fork      rows become copies of other rows: whole pages are shared, a page that is filled in part is copied in all layers
  compact   pages at the back of a pool move into the holes at its front, in all layers, and the tables follow
  shared    attention of requests that have a long prefix in common, over the prefix and over each request's own keys
  sparse    the pages just filled get a summary; each query's best pages are chosen by it; attention over those alone

A cache page holds `page` tokens; a block is 32 consecutive dims of one head, a value is m + d * q with 16-bit d and m per
block and a whole q of 0 .. 15 (`_quantise` says which). `_unpack` says where a pool's bytes hold them.
"""
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
I32 = torch.int32


def listed():
    return [
        # a step of a serving loop: three requests have ended and make room for short prompts, the others get a token each
        dict(name="turnover_step_64", op="turnover", rows=64, page=32, kv=8000, back=3, prompt=300, token=1, spare=900),
        # prompts of many tokens in a pool that is almost full
        dict(name="turnover_prompts_24", op="turnover", rows=24, page=16, kv=30000, back=16, prompt=2047, token=0, spare=30),
        # a few answers to one question
        dict(name="fork_answers_4", op="fork", parents=1, children=4, page=32, kv=700, n_kv_head=8, head_dim=128, layers=36, spare=90),
        # a batch of beams over conversations of all lengths, narrow heads
        dict(name="fork_beams_64", op="fork", parents=8, children=64, page=64, kv=4099, n_kv_head=8, head_dim=64, layers=36, spare=200),
        # a few pages between two steps
        dict(name="compact_some_16", op="compact", rows=12, page=32, kv=1000, n_pages=300, most=16, n_kv_head=8, head_dim=128, layers=36),
        # all of a pool, before its back is given to something else
        dict(name="compact_all_2000", op="compact", rows=40, page=32, kv=4000, n_pages=2000, most=1000, n_kv_head=8, head_dim=128, layers=36),
        # eight answers to one question
        dict(name="shared_answers_8", op="shared", n_req=8, n_prefix=1, alone=0, prefix=2048, q=1, ragged=False, kv=100, n_head=32, n_kv_head=8, head_dim=128, page=16, dtype="f16"),
        # conversations behind two long instructions, one of them not begun
        dict(name="shared_batch_64", op="shared", n_req=64, n_prefix=2, alone=0, prefix=8191, q=1, ragged=False, kv=1000, n_head=32, n_kv_head=8, head_dim=128, page=32, dtype="bf16"),
        # chunks of a few prompts behind a long document
        dict(name="shared_chunks_4x512", op="shared", n_req=4, n_prefix=1, alone=0, prefix=16384, q=512, ragged=True, kv=1030, n_head=32, n_kv_head=8, head_dim=128, page=64, dtype="bf16"),
        # one token of a long context
        dict(name="sparse_token_32768", op="sparse", n_req=1, q=1, ragged=False, kv_min=32768, kv=32768, chosen=64, n_head=32, n_kv_head=8, head_dim=128, page=32, dtype="f16"),
        # drafted tokens of a few requests, narrow heads
        dict(name="sparse_draft_16x5", op="sparse", n_req=16, q=5, ragged=True, kv_min=40, kv=8191, chosen=48, n_head=40, n_kv_head=8, head_dim=64, page=16, dtype="bf16"),
        # a batch of long contexts
        dict(name="sparse_batch_32", op="sparse", n_req=32, q=1, ragged=False, kv_min=0, kv=32768, chosen=32, n_head=32, n_kv_head=8, head_dim=128, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["turnover", "fork", "compact", "shared", "shared", "sparse", "sparse"])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([16, 32, 64])
    n_head, n_kv_head, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (16, 16, 64), (24, 8, 128), (40, 8, 64), (32, 4, 128), (16, 1, 128), (14, 2, 64)])
    if op == "turnover":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, page=page, kv=_log(rng, 20, min(30000, 480000 // rows)), back=rng.randint(0, min(rows, 16)), prompt=_log(rng, 1, 2000), token=rng.choice([0, 1, 1, 4]), spare=_log(rng, 1, 1000))
    if op == "fork":
        parents = _log(rng, 1, 8)
        return dict(op=op, parents=parents, children=_log(rng, 1, 30), page=page, kv=_log(rng, 20, 4000), n_kv_head=min(n_kv_head, 8), head_dim=head_dim,
                    layers=rng.choice([1, 2, 16, 36]), spare=_log(rng, 8, 200))
    if op == "compact":
        n_pages = _log(rng, 8, 1000)
        return dict(op=op, rows=_log(rng, 1, 40), page=page, kv=_log(rng, 20, 4000), n_pages=n_pages, most=_log(rng, 1, n_pages), n_kv_head=min(n_kv_head, 8), head_dim=head_dim,
                    layers=rng.choice([1, 2, 16, 36]))
    kind = rng.choice(["token", "token", "draft", "chunk"])
    n_req = _log(rng, 1, 64 if kind == "token" else 16 if kind == "draft" else 4)
    q = 1 if kind == "token" else rng.randint(2, 8) if kind == "draft" else _log(rng, 16, 1200 // n_req if op == "shared" else 400 // n_req)
    ragged = rng.random() < 0.6
    if op == "shared":
        return dict(op=op, n_req=n_req, n_prefix=min(n_req, rng.choice([1, 1, 2, 5])), alone=rng.choice([0, 0, 1]), prefix=_log(rng, 16, 16384 if kind != "token" else 8191), q=q, ragged=ragged,
                    kv=_log(rng, q, 1200), n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, page=page, dtype=dtype)
    n_req, kv = min(n_req, 32), max(q, _log(rng, 50, 32768 if kind != "chunk" else 8191))
    return dict(op=op, n_req=n_req, q=q, ragged=ragged, kv_min=rng.choice([0, 1, kv // 8, kv]), kv=kv, chosen=_log(rng, 3, max(3, min(100, 65536 // (n_req * q * page)))),
                n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, page=page, dtype=dtype)


def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _ceil(a, b):
    return -(-a // b)


def _lengths(case):
    """(queries, own keys) of each request: the first has kv keys, the second kv_min (none, of a request that has not begun), the others lie between
    a sixteenth of kv and kv. There are no more queries than keys unless there is no key at all."""
    rng = _rng(case)
    n, least, hi = case["n_req"], case.get("kv_min", 0), case["kv"]
    lo = max(1, least, hi // 16)
    kv = [hi] + [least if i == 1 else _log(rng, lo, hi) for i in range(1, n)]
    q = [rng.randint(1, case["q"]) if case["ragged"] and i else case["q"] for i in range(n)]
    return [min(a, b) if b else a for a, b in zip(q, kv)], kv


def _prefixes(case):
    """Where the requests of each prefix begin (the last entry: where the last one's end), and the prefixes' lengths."""
    rng = _rng(case)
    n, k, first = case["n_req"], case["n_prefix"], min(case["alone"], case["n_req"] - case["n_prefix"])
    start = [first + (n - first) * i // k for i in range(k)] + [n]
    return start, [case["prefix"]] + [_log(rng, max(1, case["prefix"] // 8), case["prefix"]) for _ in range(k - 1)]


def _rows(case):
    """Tokens of each row before the call, and (turnover) how many each gets, (fork) which row each child copies."""
    rng = _rng(case)
    if case["op"] == "turnover":
        kv = [case["kv"]] + [_log(rng, max(1, case["kv"] // 16), case["kv"]) for _ in range(case["rows"] - 1)]
        back = sorted(rng.sample(range(case["rows"]), case["back"]))
        new = [rng.randint(max(1, case["prompt"] // 4), case["prompt"]) if r in back else case["token"] for r in range(case["rows"])]
        return kv, back, new
    if case["op"] == "fork":
        kv = [case["kv"]] + [_log(rng, max(1, case["kv"] // 8), case["kv"]) for _ in range(case["parents"] - 1)]
        return kv + [0] * case["children"], [rng.randrange(case["parents"]) for _ in range(case["children"])], None
    kv = [case["kv"]] + [_log(rng, max(1, case["kv"] // 8), case["kv"]) for _ in range(case["rows"] - 1)]
    left = int(0.6 * case["n_pages"])  # rows that would fill more than six tenths of the pool stay shorter
    for i, n in enumerate(kv):
        kv[i] = min(n, left * case["page"])
        left -= _ceil(kv[i], case["page"])
    return kv, None, None


# ---- what a user's program has in hand ------------------------------------------------------------------------------

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
    """Keys have a few large channels, and drift along a page's tokens less than from page to page."""
    gain = torch.ones(heads, dim, device="cuda")
    gain[:, torch.randint(0, dim, (4,), generator=g, device="cuda")] = 5.0
    shape = (pages, heads, page, dim)
    k = torch.randn(shape, generator=g, device="cuda") * gain[:, None]
    k += torch.randn((pages, heads, 1, dim), generator=g, device="cuda") * 0.5
    kq, kd, km = _quantise(k)
    del k
    return _pack(kq, kd, km, *_quantise(torch.randn(shape, generator=g, device="cuda") * 0.7))


def _summary(pool, heads, page, dim):
    """What `sparse` keeps of each page and head: codes int8 [pages, heads, 2, dims], scale f32 [pages, heads]. code * scale is the smallest such
    number that is no smaller than any key of the page in that dim (0), or than any negated key (1)."""
    keys, _ = _unpack(pool, heads, page, dim)
    ends = torch.stack([keys.amax(-2), -keys.amin(-2)], -2)
    top = ends.abs().amax((-1, -2))
    scale = (top.view(torch.int32) & 0x7F800000).view(torch.float32).clamp(2 ** -24, 2 ** 16) * 2 ** -6
    scale = torch.where(top > 127 * scale, 2 * scale, scale)
    return (ends / scale[..., None, None]).ceil().clamp(-127, 127).to(torch.int8), scale


_kept = {}


def _context():
    """A program makes one context and keeps it."""
    if "ctx" not in _kept:
        import bonsai_pot_b200 as bp
        _kept["ctx"] = bp.PagedContext(device=torch.cuda.current_device())
    return _kept["ctx"]


def _tensor(values, dtype=I32):
    return torch.tensor(values, device="cuda", dtype=dtype)


def _tables(s, case, g):
    """One int32 buffer [table, lengths, reference counts] before the call, and one that the call works on."""
    kv, other, new = _rows(case)
    page, n_rows = case["page"], len(kv)
    need = [_ceil(n, page) for n in kv]
    if case["op"] == "turnover":
        after = [_ceil(new[r] if r in other else kv[r] + new[r], page) for r in range(n_rows)]
        s["pages"] = sum(need) + sum(max(a - b, 0) for a, b in zip(after, need)) + case["spare"]
        width = max(max(need), max(after))
        s["rows"], s["n_new"] = _tensor(other), _tensor(new)
        n_out = sum(new) + 5  # the program's buffers are a little longer than a step needs
        s["q_start"] = torch.zeros(n_rows + 1, device="cuda", dtype=I32)
        s["positions"], s["slots"] = torch.zeros(n_out, device="cuda", dtype=I32), torch.zeros(n_out, device="cuda", dtype=torch.int64)
    elif case["op"] == "fork":
        s["pages"], width = sum(need) + case["children"] + case["spare"], max(need)
        s["parents"], s["children_rows"] = _tensor(other), torch.arange(case["parents"], n_rows, device="cuda", dtype=I32)
        n_lists = case["children"]
    else:
        s["pages"], width = case["n_pages"], max(max(need), 1)
        n_lists = case["most"]
    width += 3
    # full pages of every other row are those of the row before it, as after a fork
    order = torch.randperm(s["pages"], generator=g, device="cuda", dtype=I32)
    table, refs, at = torch.zeros(n_rows, width, device="cuda", dtype=I32), torch.zeros(s["pages"], device="cuda", dtype=I32), 0
    for r, k in enumerate(need):
        both = min(kv[r], kv[r - 1]) // page if r % 2 and case["op"] != "fork" else 0
        table[r, :both] = table[r - 1, :both]
        table[r, both:k] = order[at:at + k - both]
        refs[table[r, :k].long()] += 1
        at += k - both
    s["saved"] = torch.cat([table.flatten(), _tensor(kv), refs])
    s["live"] = s["saved"].clone()
    ends = (n_rows * width, n_rows * width + n_rows)
    s["table"], s["kv_len"], s["refs"] = s["live"][:ends[0]].view(n_rows, width), s["live"][ends[0]:ends[1]], s["live"][ends[1]:]
    if case["op"] != "turnover":
        s["src"], s["dst"] = (torch.full((n_lists,), -1, device="cuda", dtype=I32) for _ in range(2))
        s["pool"] = torch.randint(0, 256, (case["layers"], s["pages"], case["n_kv_head"], page * case["head_dim"] * 5 // 4), generator=g, device="cuda", dtype=torch.uint8)


def _placed(s, name, lengths, page, order, at):
    """A page table of `lengths`, its pages taken from `order` on."""
    need = [_ceil(n, page) for n in lengths]
    s[name] = torch.zeros(len(need), max(max(need), 1), device="cuda", dtype=I32)
    for i, k in enumerate(need):
        s[name][i, :k] = order[at:at + k]
        at += k
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    page = case["page"]
    if case["op"] in ("turnover", "fork", "compact"):
        _tables(s, case, g)
    else:
        q_len, kv_len = _lengths(case)
        dim, hkv, n = case["head_dim"], case["n_kv_head"], sum(q_len)
        start, prefix = _prefixes(case) if case["op"] == "shared" else ([0], [])
        s["pages"] = sum(_ceil(k, page) for k in kv_len + prefix) + 3
        s["pool"] = _filled_pool(g, s["pages"], hkv, page, dim)
        order = torch.randperm(s["pages"], generator=g, device="cuda", dtype=I32)
        at = _placed(s, "page_table", kv_len, page, order, 0)
        s["max_q"], s["max_kv"] = max(q_len), max(kv_len)
        s["q_start"] = _tensor([sum(q_len[:i]) for i in range(len(q_len) + 1)])
        s["kv_len"] = _tensor(kv_len)
        s["queries"] = torch.randn(n, case["n_head"], dim, generator=g, device="cuda").to(DTYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["queries"])
        if case["op"] == "shared":
            _placed(s, "prefix_table", prefix, page, order, at)
            s["prefix_start"], s["prefix_len"], s["max_prefix"] = _tensor(start), _tensor(prefix), max(prefix)
        else:
            s["codes"], s["scales"] = _summary(s["pool"], hkv, page, dim)
            # pages that the new tokens have filled: their summaries are not there yet
            filled = [s["page_table"][r, (k - q) // page:k // page] for r, (q, k) in enumerate(zip(q_len, kv_len))]
            s["filled"] = torch.cat(filled + [_tensor([-1])])
            s["codes"][s["filled"][:-1].long()] = 0
            s["chosen_pages"] = torch.zeros(n, hkv, case["chosen"], device="cuda", dtype=I32)
            s["chosen_keys"] = torch.zeros(n, device="cuda", dtype=I32)
    if own:
        import bonsai_pot_b200 as bp
        s["ctx"] = _context()
        if "pool" in s:
            pools = s["pool"] if s["pool"].dim() == 4 else s["pool"][None]
            s["cache"] = [bp.KV4Pool(p, s["pages"], page, case["n_kv_head"], case["head_dim"]) for p in pools]
            s["pools"] = bp.KV4Pools(s["cache"])
        if "refs" in s:
            s["tables"] = bp.PageTables(s["table"], s["kv_len"], s["refs"], page)
        if "codes" in s:
            s["summary"] = bp.BlockSummary(s["codes"], s["scales"])
        if case["op"] == "shared":
            s["work"] = torch.empty(s["ctx"].shared_work(sum(q_len), case["n_head"], case["head_dim"]), device="cuda", dtype=torch.float32)
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
    v = v.reshape(*lead, page, 2, dim // 2)
    v = torch.where(_swapped(torch.arange(page, device="cuda"), dim)[:, None, None], v.flip(-2), v)
    v = v.reshape(*lead, page, 8, nb, 2, 2).movedim(-4, -3).reshape(*lead, page, nb, 32)
    return keys, (v.float() * d + m).flatten(-2)


def _held(s):
    """Which entries of the table are pages of their row."""
    return torch.arange(s["table"].shape[1], device="cuda") < ((s["kv_len"] + s["page"] - 1) // s["page"])[:, None]


def _give_back(s, rows):
    held = _held(s)[rows]
    s["refs"].scatter_add_(0, torch.where(held, s["table"][rows], 0).flatten().long(), -held.flatten().to(I32))
    s["kv_len"].index_fill_(0, rows, 0)


def _free_first(s):
    """Pages nobody holds, lowest first (behind them the others)."""
    return torch.sort((s["refs"] != 0).to(I32), stable=True)[1].to(I32)


def _turnover_plain(s):
    page, table = s["page"], s["table"]
    _give_back(s, s["rows"].long())
    before = (s["kv_len"] + page - 1) // page
    kv = s["kv_len"] + s["n_new"]
    need = (kv + page - 1) // page - before
    i = torch.arange(table.shape[1], device="cuda")
    fresh = (i >= before[:, None]) & (i < (before + need)[:, None])
    rank = (need.cumsum(0) - need - before)[:, None] + i
    pages = _free_first(s)[rank.clamp(0, s["pages"] - 1)]
    table.copy_(torch.where(fresh, pages, table))
    s["refs"].scatter_add_(0, torch.where(fresh, pages, 0).flatten().long(), fresh.flatten().to(I32))
    s["q_start"][1:] = s["n_new"].cumsum(0)
    t = torch.arange(s["positions"].shape[0], device="cuda", dtype=I32)
    row = torch.searchsorted(s["q_start"][1:].contiguous(), t, right=True)
    real = row < table.shape[0]
    row = row.clamp(max=table.shape[0] - 1)
    at = torch.where(real, s["kv_len"][row] + t - s["q_start"][row], 0)
    s["positions"].copy_(torch.where(real, at, -1))
    s["slots"].copy_(torch.where(real, table[row, (at // page).long()].long() * page + at % page, -1))
    s["kv_len"].copy_(kv)
    return {k: s[k] for k in ("table", "kv_len", "refs", "q_start", "positions", "slots")}


def _copy_plain(s):
    there = s["dst"] >= 0
    s["pool"][:, s["dst"][there].long()] = s["pool"][:, s["src"][there].long()]


def _fork_plain(s):
    page, table = s["page"], s["table"]
    parents, children = s["parents"].long(), s["children_rows"].long()
    _give_back(s, children)
    kv = s["kv_len"][parents]
    full, part = (kv // page).long(), kv % page > 0
    i = torch.arange(table.shape[1], device="cuda")
    both = i < full[:, None]
    lines = torch.where(both, table[parents], table[children])
    rank = part.to(I32).cumsum(0) - part.to(I32)
    fresh = _free_first(s)[rank]
    last = (i == full[:, None]) & part[:, None]
    table[children] = torch.where(last, fresh[:, None], lines)
    held = both | last
    s["refs"].scatter_add_(0, torch.where(held, table[children], 0).flatten().long(), held.flatten().to(I32))
    s["kv_len"][children] = kv
    s["src"].copy_(torch.where(part, table[parents].gather(1, full[:, None])[:, 0], -1))
    s["dst"].copy_(torch.where(part, fresh, -1))
    _copy_plain(s)
    return {k: s[k] for k in ("table", "kv_len", "refs", "src", "dst", "pool")}


def _compact_plain(s):
    n, most = s["pages"], s["most"]
    low = _free_first(s)[:most]
    high = n - 1 - torch.sort((s["refs"].flip(0) == 0).to(I32), stable=True)[1].to(I32)[:most]
    moves = (high > low) & (s["refs"][high] != 0) & (s["refs"][low] == 0)
    to = torch.arange(n + 1, device="cuda", dtype=I32)
    to.scatter_(0, torch.where(moves, high, n).long(), torch.where(moves, low, n))
    s["table"].copy_(torch.where(_held(s), to[s["table"].long()], s["table"]))
    refs = torch.where(to[:n] == torch.arange(n, device="cuda"), s["refs"], 0)
    refs.scatter_add_(0, torch.where(moves, low, 0).long(), torch.where(moves, s["refs"][high], 0))
    s["refs"].copy_(refs)
    s["src"].copy_(torch.where(moves, high, -1))
    s["dst"].copy_(torch.where(moves, low, -1))
    _copy_plain(s)
    return {k: s[k] for k in ("table", "refs", "src", "dst", "pool")}


def _by_request(s, max_q):
    """Queries f32 [requests, KV heads, group, max_q, dims] (rows behind a request's own are of no use), and each request's number of them."""
    hkv, dim = s["n_kv_head"], s["head_dim"]
    start = s["q_start"].long()
    at = (start[:-1, None] + torch.arange(max_q, device="cuda")).clamp(max=s["queries"].shape[0] - 1)
    return s["queries"][at].float().unflatten(2, (hkv, -1)).movedim(1, 3), start[1:] - start[:-1]


def _shared_plain(s):
    hkv, page, dim, max_q = s["n_kv_head"], s["page"], s["head_dim"], s["max_q"]
    q, q_len = _by_request(s, max_q)
    n_req, group = q.shape[0], q.shape[2]
    which = torch.searchsorted(s["prefix_start"], torch.arange(n_req, device="cuda", dtype=I32), right=True) - 1  # -1: no prefix
    parts, values = [], []
    i = torch.arange(max_q, device="cuda")
    for name in ("prefix_table", "page_table"):
        k, v = (t.movedim(2, 1).flatten(2, 3) for t in _unpack(s["pool"][s[name].long()], hkv, page, dim))  # [tables, heads, keys, dims]
        j = torch.arange(k.shape[2], device="cuda")
        if name == "prefix_table":
            k, v = k[which], v[which]
            seen = (j < torch.where(which >= 0, s["prefix_len"][which], 0)[:, None])[:, None]
        else:
            at = (s["kv_len"] - q_len)[:, None] + i
            seen = (j <= at[..., None]) & (j < s["kv_len"][:, None, None])
        scores = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (group, max_q)) * dim ** -0.5
        parts.append(scores.masked_fill(~seen[:, None, None], float("-inf")))
        values.append(v)
    top = torch.maximum(parts[0].amax(-1, keepdim=True), parts[1].amax(-1, keepdim=True))
    top = torch.where(top.isinf(), 0.0, top)
    total, out = 0.0, 0.0
    for scores, v in zip(parts, values):
        p = torch.exp(scores - top)
        total = total + p.sum(-1, keepdim=True)
        out = out + (p.flatten(2, 3) @ v).unflatten(2, (group, max_q))
    out = (out / torch.where(total > 0, total, 1.0)).movedim(3, 1).flatten(2, 3)
    s["out"].copy_(out[i < q_len[:, None]])
    return s["out"]


def _sparse_plain(s):
    hkv, page, dim, max_q, chosen = s["n_kv_head"], s["page"], s["head_dim"], s["max_q"], s["chosen"]
    filled = s["filled"][:-1].long()
    s["codes"][filled], s["scales"][filled] = _summary(s["pool"][filled], hkv, page, dim)
    # each query's number of keys and of pages
    q, q_len = _by_request(s, max_q)
    i = torch.arange(max_q, device="cuda")
    real = i < q_len[:, None]
    n_keys = torch.where(s["kv_len"][:, None] > 0, (s["kv_len"] - q_len)[:, None] + i + 1, 0).clamp(min=0)
    n_pages = (n_keys + page - 1) // page
    # scores: whole numbers below 2^24 (255 * 127 * 256 at most), times a power of two
    parts = torch.stack([q.clamp(min=0), (-q).clamp(min=0)], -2)  # [requests, KV heads, group, max_q, 2, dims]
    total = parts[:, :, 0]
    for h in range(1, q.shape[2]):  # in this order, as the operator defines it
        total = total + parts[:, :, h]
    top = total.amax((-1, -2))
    unit = (top.view(torch.int32) & 0x7F800000).view(torch.float32).clamp(2.0 ** -100, 2.0 ** 127) * 2 ** -7
    query = (total / unit[..., None, None]).round().clamp(max=255).flatten(-2)
    table = s["page_table"].long()
    scores = query @ s["codes"][table].float().movedim(2, 1).flatten(-2).transpose(-1, -2)  # [requests, KV heads, max_q, pages]
    scores = scores * s["scales"][table].movedim(2, 1)[:, :, None]
    b = torch.arange(table.shape[1], device="cuda")
    last = n_pages[:, None, :, None]
    scores = torch.where((b < 1) | (b >= last - 1), float("inf"), scores).masked_fill(b >= last, float("-inf"))
    best = torch.sort(scores, dim=-1, descending=True, stable=True)[1][..., :chosen]
    k = torch.arange(best.shape[-1], device="cuda")
    best = torch.where(k < last, best, table.shape[1]).sort(-1)[0]  # in the order of the keys
    pages = torch.where(k < last, torch.cat([table, table[:, :1]], 1)[:, None, None].expand(*best.shape[:3], -1).gather(-1, best), -1)
    s["chosen_pages"].fill_(-1)
    s["chosen_pages"][..., :best.shape[-1]] = pages.movedim(2, 1)[real].to(I32)
    s["chosen_keys"].copy_(((n_pages.clamp(max=chosen) - n_pages) * page + n_keys)[real])
    # attention over them
    rows = s["chosen_pages"].clamp(min=0).long()
    heads = torch.arange(hkv, device="cuda")[:, None]
    keys, values = (t.flatten(2, 3) for t in _unpack(s["pool"][rows, heads], hkv, page, dim))  # [tokens, KV heads, keys, dims]
    q = s["queries"].float().unflatten(1, (hkv, -1))
    weights = (q @ keys.transpose(-1, -2)) * dim ** -0.5
    j = torch.arange(keys.shape[2], device="cuda")
    weights = weights.masked_fill(j >= s["chosen_keys"][:, None, None, None], float("-inf"))
    top = weights.amax(-1, keepdim=True)
    p = torch.exp(weights - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    s["out"].copy_((p @ values / torch.where(total > 0, total, 1.0)).flatten(1, 2))
    return {k: s[k] for k in ("codes", "scales", "chosen_pages", "chosen_keys", "out")}


def run(s):
    op = s["op"]
    if op in ("turnover", "compact"):
        s["live"].copy_(s["saved"])  # a pass begins with the same tables
    if not own:
        return {"turnover": _turnover_plain, "fork": _fork_plain, "compact": _compact_plain, "shared": _shared_plain, "sparse": _sparse_plain}[op](s)
    ctx = s["ctx"]
    if op == "turnover":
        ctx.release(s["tables"], s["rows"])
        ctx.grow(s["tables"], s["n_new"], s["q_start"], s["positions"], s["slots"])
        return {k: s[k] for k in ("table", "kv_len", "refs", "q_start", "positions", "slots")}
    if op == "fork":
        ctx.release(s["tables"], s["children_rows"])
        ctx.fork(s["tables"], s["parents"], s["children_rows"], s["src"], s["dst"])
        ctx.copy_pages(s["pools"], s["src"], s["dst"])
        return {k: s[k] for k in ("table", "kv_len", "refs", "src", "dst", "pool")}
    if op == "compact":
        ctx.compact(s["tables"], s["src"], s["dst"])
        ctx.copy_pages(s["pools"], s["src"], s["dst"])
        return {k: s[k] for k in ("table", "refs", "src", "dst", "pool")}
    cache = s["cache"][0]
    if op == "shared":
        ctx.attention_shared(cache, s["queries"], s["out"], s["q_start"], s["kv_len"], s["page_table"], s["prefix_start"], s["prefix_len"], s["prefix_table"], s["work"],
                             max_q=s["max_q"], max_kv=s["max_kv"], max_prefix=s["max_prefix"])
        return s["out"]
    ctx.summarise(cache, s["summary"], s["filled"])
    ctx.select(cache, s["summary"], s["queries"], s["chosen_pages"], s["chosen_keys"], s["q_start"], s["kv_len"], s["page_table"], max_q=s["max_q"], max_kv=s["max_kv"], first=1, last=1)
    ctx.attention_selected(cache, s["queries"], s["out"], s["chosen_pages"], s["chosen_keys"])
    return {k: s[k] for k in ("codes", "scales", "chosen_pages", "chosen_keys", "out")}


def work(case):
    op, page = case["op"], case["page"]
    if op in ("turnover", "fork", "compact"):
        kv, other, new = _rows(case)
        need = [_ceil(n, page) for n in kv]
        if op == "turnover":  # entries given back and their counts, counts of pages looked through once, entries and counts of new ones, the tokens' indices
            kept = [0 if r in other else n for r, n in enumerate(kv)]
            fresh = sum(_ceil(k + n, page) - _ceil(k, page) for k, n in zip(kept, new))
            return {"bytes": 12 * sum(need[r] for r in other) + 4 * sum(need) + 8 * fresh + 12 * (sum(new) + 5) + 16 * len(kv), "flops": 0}
        size = case["n_kv_head"] * page * case["head_dim"] * 5 // 4 * case["layers"]
        if op == "fork":
            copied = sum(1 for p in other if kv[p] % page)
            return {"bytes": 2 * copied * size + 16 * sum(need[p] for p in other) + 24 * len(other), "flops": 0}
        used = sum(need)  # (rows of a pair share some: no more than this)
        moved = min(case["most"], int(used * (1 - used / case["n_pages"])))
        return {"bytes": 2 * moved * size + 8 * used + 4 * case["n_pages"] + 16 * moved, "flops": 0}
    dim, hkv, heads = case["head_dim"], case["n_kv_head"], case["n_head"]
    q_len, kv_len = _lengths(case)
    rows = 4 * sum(q_len) * heads * dim
    if op == "shared":
        start, prefix = _prefixes(case)
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(q_len, kv_len) if k)
        pairs += sum(p * sum(q_len[start[i]:start[i + 1]]) for i, p in enumerate(prefix))
        return {"bytes": (sum(kv_len) + sum(prefix)) * hkv * dim * 1.25 + rows, "flops": 4 * dim * heads * pairs}
    filled = sum(k // page - (k - q) // page for q, k in zip(q_len, kv_len) if k)
    seen = [_ceil(k, page) for k in kv_len]  # summaries of each request's pages are read once; each token's chosen pages (those of one request's tokens may be the same ones)
    chosen = sum(min(case["chosen"], n) for n in seen) * page
    flops = sum(4 * dim * hkv * q * n + 4 * dim * heads * q * min(case["chosen"], n) * page for q, n in zip(q_len, seen))
    return {"bytes": filled * page * hkv * dim * 0.625 + (filled + sum(seen)) * hkv * (2 * dim + 4) + chosen * hkv * dim * 1.25 + rows + 4 * sum(q_len) * hkv * case["chosen"], "flops": flops}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------

def _page64(pool, page, dim, token):
    """K and V [.., dims] in 64 bits of one token of every page: pool [.., bytes]."""
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


def _keys64(s, pages):
    """K and V [heads, keys, dims] in 64 bits of some pages, one behind the other."""
    pool = s["pool"][pages.long()]
    both = [_page64(pool, s["page"], s["head_dim"], t) for t in range(s["page"])]
    return [torch.stack([b[i] for b in both], 2).movedim(1, 0).flatten(1, 2) for i in (0, 1)]


def _exact_shared(case, s):
    q_len, kv_len = _lengths(case)
    start, prefix = _prefixes(case)
    dim, hkv, page = case["head_dim"], case["n_kv_head"], case["page"]
    group, at, out, heads_of = case["n_head"] // hkv, 0, [], {}
    for r, (nq, nk) in enumerate(zip(q_len, kv_len)):
        q = s["queries"][at:at + nq].double().view(nq, hkv, group, dim)
        at += nq
        k, v = (t[:, :nk] for t in _keys64(s, s["page_table"][r, :_ceil(nk, page)]))
        before = 0
        for i, n in enumerate(prefix):
            if start[i] <= r < start[i + 1]:
                if i not in heads_of:
                    heads_of = {i: [t[:, :n] for t in _keys64(s, s["prefix_table"][i, :_ceil(n, page)])]}
                k, v, before = torch.cat([heads_of[i][0], k], 1), torch.cat([heads_of[i][1], v], 1), n
        rows = torch.zeros(nq, hkv, group, dim, dtype=torch.float64, device="cuda")
        j = torch.arange(before + nk, device="cuda")
        hidden = j > torch.arange(nk - nq, nk, device="cuda").clamp(min=-1)[:, None] + before
        if before + nk:
            for h in range(hkv):
                for g in range(group):
                    rows[:, h, g] = torch.softmax((q[:, h, g] @ k[h].T / dim ** 0.5).masked_fill(hidden, float("-inf")), -1) @ v[h]
        out.append(rows.nan_to_num(0.0).flatten(1, 2))
    return torch.cat(out)


def _exact_sparse(case, s):
    q_len, kv_len = _lengths(case)
    dim, hkv, page, most = case["head_dim"], case["n_kv_head"], case["page"], case["chosen"]
    out, at = torch.zeros(s["queries"].shape, dtype=torch.float64, device="cuda"), 0
    for r, (nq, nk) in enumerate(zip(q_len, kv_len)):
        k, v = _keys64(s, s["page_table"][r, :_ceil(nk, page)]) if nk else (None, None)
        if nk:
            ends = torch.stack([k.unflatten(1, (-1, page)).amax(2), -k.unflatten(1, (-1, page)).amin(2)], 2)  # [heads, pages, 2, dims]
            big = ends.abs().amax((-1, -2))
            unit = torch.exp2(torch.frexp(big).exponent.double().clamp(-23, 17) - 7)
            unit = torch.where(big > 127 * unit, 2 * unit, unit)[..., None, None]
            ends = (ends / unit).ceil().clamp(-127, 127) * unit
        for i in range(nq):
            sees = nk - nq + 1 + i if nk else 0
            q = s["queries"][at].double().view(hkv, -1, dim)
            n = _ceil(sees, page)
            for h in range(hkv if sees > 0 else 0):
                up = torch.stack([q[h].clamp(min=0).float().cumsum(0)[-1], (-q[h]).clamp(min=0).float().cumsum(0)[-1]]).double()
                unit = 2.0 ** (torch.frexp(up.max()).exponent.double() - 8)
                score = ((up / unit).round().clamp(max=255) * ends[h, :n]).sum((-1, -2))
                score[0] = score[n - 1] = float("inf")
                best = sorted(range(n), key=lambda b, z=score.tolist(): (-z[b], b))[:most]
                tokens = torch.cat([torch.arange(b * page, min((b + 1) * page, sees), device="cuda") for b in sorted(best)])
                p = torch.softmax(q[h] @ k[h, tokens].T / dim ** 0.5, -1)
                out[at].view(hkv, -1, dim)[h] = p @ v[h, tokens]
            at += 1
    return {"codes": None, "scales": None, "chosen_pages": None, "chosen_keys": None, "out": out}


def exact(case, seed):
    if case["op"] in ("turnover", "fork", "compact"):
        return None  # whole numbers all of them
    s = prepare(case, seed)
    return _exact_shared(case, s) if case["op"] == "shared" else _exact_sparse(case, s)
