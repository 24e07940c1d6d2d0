"""The paged 4-bit operators from their definitions, in numpy: bit for bit in binary32 where the format fixes every step
(quantisation), in binary64 elsewhere. Nothing here comes from the package."""
import numpy as np

F = np.float32


def bf16_bits(x):
    """binary32 -> bfloat16 bits, ties to even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b >> 16) & 1) + 0x7FFF
    out = ((b + r) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def table(n_pos, rot, base=1e6, scaling=None, factor=1.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=0):
    i = np.arange(rot // 2, dtype=np.float64)
    mscale = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    theta = base ** (-2 * i / rot)
    if scaling == "linear":
        theta = theta / factor
    if scaling == "yarn":
        turns = lambda beta: rot * np.log(orig_ctx / (beta * 2 * np.pi)) / (2 * np.log(base))  # noqa: E731
        low, high = max(np.floor(turns(beta_fast)), 0), min(np.ceil(turns(beta_slow)), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        theta = theta / factor * ramp + theta * (1 - ramp)
        mscale = 0.1 * np.log(factor) + 1 if factor > 1 else 1.0
    a = np.arange(n_pos, dtype=np.float64)[:, None] * theta
    return (np.stack([np.cos(a), np.sin(a)], -1) * mscale).astype(np.float32)


def pairs(rot, layout):
    i = np.arange(rot // 2)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def rotate(x, tab, positions, layout, inverse=False):
    """x [n, heads, dim] in its own precision (every operation rounded by itself)."""
    y = x.copy()
    p1, p2 = pairs(2 * tab.shape[1], layout)
    c = tab[positions][:, None, :, 0].astype(x.dtype)
    s = tab[positions][:, None, :, 1].astype(x.dtype) * x.dtype.type(-1 if inverse else 1)
    a, b = x[..., p1], x[..., p2]
    y[..., p1] = a * c - b * s
    y[..., p2] = b * c + a * s
    return y


def norm64(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def norm32(x, w, eps):
    """As the cache defines it: a binary tree over neighbours."""
    s = x * x
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    r = F(1) / np.sqrt(s * F(1 / x.shape[-1]) + F(eps))
    return (x * r) * w


def quantise(x):
    """binary32 [.., dim] -> codes uint8 [.., dim], d, m float16 [.., dim / 32]."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        b = np.clip(x, F(-64512), F(64512)).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
        lo, hi = b.min(-1), b.max(-1)
        top = np.maximum(np.abs(lo), np.abs(hi)) * F(65 / 64)
        u = np.maximum((top.view(np.uint32) & 0x7F800000).view(np.float32) * F(2 ** -10), F(2 ** -24))
        m = np.rint(lo / u) * u
        d = np.rint((hi - lo) * F(1 / 15) / u) * u
        inv = np.where(d > 0, F(1) / d, F(0))
        q = np.clip(np.rint((b - m[..., None]) * inv[..., None]), 0, 15)
        return np.nan_to_num(q).astype(np.uint8).reshape(x.shape), d.astype(np.float16), m.astype(np.float16)


def dequantise(q, d, m):
    b = q.reshape(*q.shape[:-1], q.shape[-1] // 32, 32).astype(np.float64)
    return (b * d.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]).reshape(q.shape)


class Pool:
    """A pool's bytes as views that the tests write and read token by token."""

    def __init__(self, n_pages, page, heads, dim, fill=0):
        self.page, self.heads, self.dim, self.nb = page, heads, dim, dim // 32
        self.bytes = np.full((n_pages, heads, page * dim * 5 // 4), fill, np.uint8)

    def place(self, kind, slot):
        """(codes, d, m) byte views [heads, ..] of a slot; kind 0 = K, 1 = V."""
        rec = self.bytes[slot // self.page]
        t, base, row = slot % self.page, kind * self.page * self.dim * 5 // 8, self.dim // 2
        at = base + self.page * row
        d = rec[:, at + 2 * self.nb * t:at + 2 * self.nb * (t + 1)]
        at += 2 * self.nb * self.page
        return rec[:, base + row * t:base + row * (t + 1)], d, rec[:, at + 2 * self.nb * t:at + 2 * self.nb * (t + 1)]

    def where(self, kind, slot):
        """For every dim: byte of the row, bit in it."""
        dim = np.arange(self.dim)
        b, r = dim // 32, dim % 32
        if kind == 0:
            byte, bit = (r // 8) * 4 * self.nb + 4 * b, 4 * (r % 8 // 2) + 16 * (r % 2)
        else:
            byte, bit = (r // 4) * 2 * self.nb + 2 * b, 4 * (r % 4)
            if self.dim == 128 and slot % self.page & 2:
                byte = byte ^ 32
        return byte + bit // 8, bit % 8

    def write(self, kind, slots, q, d, m):
        """Tokens [n, heads, ..] at `slots`."""
        rows = np.zeros((2, len(slots), self.heads, self.dim // 2), np.uint8)
        for odd in range(2):  # slot 2 stands for those whose place has bit 1 set
            byte, bit = self.where(kind, 2 * odd)
            for i in range(self.dim):
                rows[odd, :, :, byte[i]] |= q[:, :, i] << np.uint8(bit[i])
        d, m = np.ascontiguousarray(d).view(np.uint8), np.ascontiguousarray(m).view(np.uint8)
        for i, slot in enumerate(slots):
            codes, dv, mv = self.place(kind, int(slot))
            codes[:], dv[:], mv[:] = rows[slot % self.page >> 1 & 1, i], d[i], m[i]

    def read(self, kind, slot):
        codes, dv, mv = self.place(kind, slot)
        byte, bit = self.where(kind, slot)
        q = (codes[:, byte] >> bit.astype(np.uint8)) & 15
        return dequantise(q, np.ascontiguousarray(dv).view(np.float16), np.ascontiguousarray(mv).view(np.float16))


def attention(q, keys, values, scale, window=0):
    """One request: q [nq, heads, dim], keys and values [nk, kv heads, dim], binary64. Returns the outputs and, for every output,
    sum p |v| / sum p, by which its rounding errors are bounded."""
    nq, heads, dim = q.shape
    nk, hkv, _ = keys.shape
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    if nk == 0:
        return out, weight
    place = np.arange(nk - nq, nk)[:, None]
    j = np.arange(nk)[None]
    seen = j <= place
    if window:
        seen &= j > place - window
    for h in range(heads):
        s = q[:, h] @ keys[:, h // (heads // hkv)].T * scale
        s = np.where(seen, s, -np.inf)
        top = s.max(-1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        p = np.where(seen, p, 0.0)
        total = p.sum(-1, keepdims=True)
        p = p / np.where(total > 0, total, 1.0)
        out[:, h] = p @ values[:, h // (heads // hkv)]
        weight[:, h] = p @ np.abs(values[:, h // (heads // hkv)])
    return out, weight
