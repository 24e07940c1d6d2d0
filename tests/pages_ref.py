"""Page tables, summaries of pages, the choice among them and attention in two parts from their definitions (include/bonsai_pages.h), in
numpy; nothing here comes from the package."""
import numpy as np

F = np.float32


class Tables:
    """table [rows, pages], kv [rows], refs [pages of the pool]; every call returns whether something was refused."""

    def __init__(self, table, kv, refs, page):
        self.table, self.kv, self.refs, self.page = table.copy(), kv.copy(), refs.copy(), page

    def pages(self, n):
        return -(-int(n) // self.page)

    def entries(self, r):
        return self.table[r, :self.pages(self.kv[r])]

    def grow(self, n_new, n_out):
        start = np.concatenate([[0], np.cumsum(np.maximum(n_new, 0))])
        pos, slots, bad = np.full(n_out, -1), np.full(n_out, -1), False
        free, rank = np.flatnonzero(self.refs == 0), 0
        old, plan = self.kv.copy(), []
        for r, n in enumerate(n_new):
            fits = n >= 0 and old[r] >= 0 and start[r] + n <= n_out and self.pages(old[r] + n) <= self.table.shape[1]
            need = self.pages(old[r] + n) - self.pages(old[r]) if fits else 0
            plan.append((fits and (need == 0 or rank + need <= len(free)), rank, need))
            rank += need
        for r, (ok, rank, need) in enumerate(plan):
            bad |= not ok
            if not ok:
                continue
            at = self.pages(old[r])
            self.table[r, at:at + need] = free[rank:rank + need]
            self.refs[free[rank:rank + need]] = 1
            self.kv[r] += n_new[r]
            t = np.arange(old[r], self.kv[r])
            pos[start[r]:start[r + 1]] = t
            slots[start[r]:start[r + 1]] = self.table[r, t // self.page].astype(np.int64) * self.page + t % self.page
        return bad, start, pos, slots

    def release(self, rows):
        for r in rows:
            if r >= 0:
                np.subtract.at(self.refs, self.entries(r), 1)
                self.kv[r] = 0

    def fork(self, parents, children):
        free, rank, bad = np.flatnonzero(self.refs == 0), 0, False
        src, dst = np.full(len(parents), -1), np.full(len(parents), -1)
        for i, (p, c) in enumerate(zip(parents, children)):
            if p < 0 or c < 0:
                continue
            full, part = self.kv[p] // self.page, self.kv[p] % self.page > 0
            if part and rank >= len(free):
                bad = True
                continue
            self.table[c, :full] = self.table[p, :full]
            np.add.at(self.refs, self.table[p, :full], 1)
            if part:
                src[i], dst[i] = self.table[p, full], free[rank]
                self.table[c, full] = dst[i]
                self.refs[dst[i]] = 1
                rank += 1
            self.kv[c] = self.kv[p]
        return bad, src, dst

    def compact(self, most):
        free, used = np.flatnonzero(self.refs == 0), np.flatnonzero(self.refs > 0)[::-1]
        src, dst, to = np.full(most, -1), np.full(most, -1), np.arange(len(self.refs))
        for i in range(min(most, len(free), len(used))):
            if used[i] > free[i]:
                src[i], dst[i] = used[i], free[i]
                to[used[i]] = free[i]
                self.refs[free[i]], self.refs[used[i]] = self.refs[used[i]], 0
        for r in range(len(self.kv)):
            e = self.entries(r)
            e[:] = to[e]
        return src, dst


def summary(keys):
    """keys [.., tokens, dims] -> codes int8 [.., 2, dims], scale [..]."""
    with np.errstate(invalid="ignore"):
        some = ~np.isnan(keys).all(-2)
        hi = np.where(some, np.fmax.reduce(keys, -2), 0)
        lo = np.where(some, np.fmin.reduce(keys, -2), 0)
    ends = np.stack([hi, -lo], -2).astype(np.float64)
    top = np.abs(ends).max((-1, -2))
    e = np.clip(np.where(np.isinf(top), 16, np.frexp(np.where(np.isinf(top), 1, top))[1] - 1), -24, 16)
    e = np.where(top == 0, -24, e)
    scale = 2.0 ** (e - 6)
    scale = np.where(top > 127 * scale, 2 * scale, scale)
    return np.clip(np.ceil(ends / scale[..., None, None]), -127, 127).astype(np.int8), scale.astype(F)


def scores(q, codes, scale):
    """q [group, dims] as binary32 of one token and KV head; codes [pages, 2, dims], scale [pages]: exact."""
    up, down = np.zeros(q.shape[1], F), np.zeros(q.shape[1], F)
    for x in q.astype(F):
        up = up + np.fmax(x, F(0))
        down = down + np.fmax(-x, F(0))
    top = float(max(up.max(), down.max()))
    e = max(np.frexp(top)[1] - 1, -100) if top > 0 else -100
    both = np.minimum(np.rint(np.stack([up, down]).astype(np.float64) * 2.0 ** (7 - e)), 255)
    return (both[None] * codes.astype(np.float64)).sum((1, 2)) * scale.astype(np.float64)


def choose(score, first, last, chosen):
    """Indices of the chosen pages, ascending, from the scores of all that are seen."""
    n = len(score)
    s = score.copy()
    s[:first] = np.inf
    s[n - last:] = np.inf
    return np.sort(np.argsort(-s, kind="stable")[:chosen])


def softmax_over(q, keys, values, seen, scale):
    """q [n, heads, dim], keys and values [m, KV heads, dim], seen [n, m]: the outputs and sum p |v| / sum p."""
    heads, hkv = q.shape[1], keys.shape[1]
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    if keys.shape[0] == 0:
        return out, weight
    for h in range(heads):
        k, v = keys[:, h // (heads // hkv)], values[:, h // (heads // hkv)]
        s = np.where(seen, q[:, h] @ k.T * scale, -np.inf)
        top = s.max(-1, keepdims=True)
        p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
        total = p.sum(-1, keepdims=True)
        p = p / np.where(total > 0, total, 1)
        out[:, h], weight[:, h] = p @ v, p @ np.abs(v)
    return out, weight


def shared_seen(nq, n_prefix, nk):
    """[queries, prefix and own keys]: all of the prefix, own keys causally up to the last one."""
    own = np.arange(nk)[None] <= np.arange(nk - nq, nk)[:, None]
    return np.concatenate([np.ones((nq, n_prefix), bool), own], 1)
