"""What a text decoder writes with, on numpy: the rotation in 64 bits, the 4-bit
cache byte by byte, its attention in 64 bits with the sizes of its sums."""
from __future__ import annotations

import numpy as np

import decoder_plain as R
from ppocr_native_amd import decoder as D

STEP = R.STEP


# ----------------------------------------------------------------- the rotation

def frequencies(rotary, base=10000.0):
    return (base ** (-np.arange(rotary // 2) * 2.0 / max(rotary, 1))).astype(np.float32)


def turned(x, positions, freqs, rotary, pairs):
    """x [rows][heads][dim] as float64, turned; and the sizes |x1| + |x2| of each value's two terms."""
    out, size = x.copy(), np.zeros_like(x)
    half = rotary // 2
    one = 2 * np.arange(half) if pairs else np.arange(half)
    two = one + (1 if pairs else half)
    angle = np.asarray(positions, np.float64)[:, None, None] * freqs.astype(np.float64)
    a, b = x[..., one], x[..., two]
    out[..., one], out[..., two] = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    size[..., one] = size[..., two] = np.abs(a) + np.abs(b)
    return out, size


def turned_bound(want, size, t):
    """Half a step of t; in f32 a cosine or sine is off by half a step of at most 1, a product by half a step of its own
    and the sum by half of its: 1.5 of 2^-24 of |x1| + |x2| each for two terms and their sum, 4 in all."""
    return R.half_step(want, t) * (1 + 2.0 ** -10) + size * 4 * 2.0 ** -24


# ------------------------------------------------------------- the 4-bit cache

def padded(dim):
    return next(p for p in (32, 64, 96, 128, 192, 256) if p >= dim)


class Cache4:
    """A cache of given texts on the host, as bytes: pages shuffled, 0xAB (whose scales are numbers) or, `nan`, NaN
    scales in all that no text holds, table entries past a text's pages far out of range."""

    def __init__(self, rng, lengths, page, heads, dim, group, spare=2, nan=False, gap=0):
        need = [-(-n // page) for n in lengths]
        self.pages, self.page, self.heads, self.dim, self.group = sum(need) + spare, page, heads, dim, group
        self.p = padded(dim)
        self.size = group if group and group < self.p else self.p
        self.groups = -(-self.p // self.size)
        self.width = max(need + [1])
        self.table = np.full((len(lengths), self.width), 2 ** 30, np.int32)
        order = rng.permutation(self.pages)
        for b, n in enumerate(need):
            self.table[b, :n], order = order[:n], order[n:]
        codes, few = page * self.p // 2, page * 2 * self.groups
        self.at = np.cumsum([0, codes, few, few, codes, few, few])
        self.chunk = int(self.at[-1])
        assert D.kv4_page_bytes(page, heads, dim, group) == heads * self.chunk
        self.stride = heads * self.chunk + gap
        self.data = np.full((self.pages, self.stride), 0xAB, np.uint8)
        if nan:
            for view in self.few():
                view[...] = np.nan

    def plane(self, i, cut=None):
        at = self.at if cut is None else cut
        d = self.data[:, :self.heads * self.chunk].reshape(self.pages, self.heads, self.chunk)
        return d[:, :, at[i]:at[i + 1]]

    def few(self):
        """Views of K's scales and minima and V's: [page][head][token][group]."""
        return [self.plane(i).view(np.float16).reshape(self.pages, self.heads, self.page, self.groups) for i in (1, 2, 4, 5)]

    def place(self, b, i):
        return self.table[b, i // self.page], i % self.page

    def dims(self, slot):
        """Where in a chunk the bytes of a token's dims 0, 2, 4, ... lie, of K and of V."""
        d = np.arange(0, self.p, 2)
        c = self.p // 32
        k = slot * (self.p // 2) + 4 * (c * (d % 32 // 8) + d // 32) + d % 8 // 2
        v = self.at[3] + slot // 4 * (2 * self.p) + 4 * (c * (d % 32 // 2) + d // 32) + slot % 4
        return k, v

    def set(self, b, i, n, s, m):
        """Token i of text b: codes n [2][heads][P], scales and minima [2][heads][groups] in f16."""
        page, slot = self.place(b, i)
        chunk = self.data[page, :self.heads * self.chunk].reshape(self.heads, self.chunk)
        for part, at in enumerate(self.dims(slot)):
            chunk[:, at] = n[part][:, 0::2] | n[part][:, 1::2] << 4
        for part, (views, rows) in enumerate(zip((self.few()[0::2], self.few()[1::2]), (s, m))):
            for kv in range(2):
                views[kv][page, :, slot] = rows[kv]

    def get(self, b, i):
        """(n s, m) of K and of V [2][heads][dim] as float64 of token i of text b."""
        page, slot = self.place(b, i)
        chunk = self.data[page, :self.heads * self.chunk].reshape(self.heads, self.chunk)
        of = np.arange(self.dim) // self.size
        out = []
        for part, at in enumerate(self.dims(slot)):
            n = np.stack((chunk[:, at] & 15, chunk[:, at] >> 4), -1).reshape(self.heads, -1)[:, :self.dim].astype(np.float64)
            s, m = (self.few()[2 * part + j][page, :, slot].astype(np.float64)[:, of] for j in (0, 1))
            out.append((n * s, m))
        return out

    def fill(self, rng, lengths):
        """Any codes, scales over three decades, minima either side of 0, for the texts' tokens."""
        for b, length in enumerate(lengths):
            for i in range(length):
                s = (10.0 ** rng.uniform(-3, 0, (2, self.heads, self.groups)) / 4).astype(np.float16)
                m = rng.normal(0, 1, s.shape).astype(np.float16)
                self.set(b, i, rng.integers(0, 16, (2, self.heads, self.p)).astype(np.uint8), s, m)

    def upload(self):
        self.gpu, self.gpu_table = R.on_gpu(self.data), R.on_gpu(self.table)
        tight = self.stride == self.heads * self.chunk
        return D.Kv4Cache(self.gpu.addr, self.pages, self.page, self.heads, self.dim, self.group,
                          0 if tight else self.stride)

    def back(self):
        return R.back(self.gpu, np.uint8, self.data.shape)


def quantised(x, p, size):
    """Codes [..][P], scales and minima [..][groups] (f16) of x [..][dim] in f32, rounded as is documented."""
    x = np.asarray(x, np.float32)
    dim, f = x.shape[-1], np.float32
    groups = -(-p // size)
    n = np.zeros(x.shape[:-1] + (p,), np.uint8)
    s, m = (np.zeros(x.shape[:-1] + (groups,), np.float16) for _ in range(2))
    with np.errstate(all="ignore"):
        for g in range(groups):
            part = x[..., g * size:(g + 1) * size]
            if part.shape[-1] == 0:
                continue
            bad = ~np.isfinite(part).all(-1)
            part = np.clip(np.where(np.isnan(part), 0, part), f(-65504), f(65504))
            low, high = part.min(-1), part.max(-1)
            m[..., g] = (low + f(0)).astype(np.float16)  # (the least of -0 and 0 is either: 0)
            base = m[..., g].astype(f)
            s[..., g] = (np.maximum((high - base) * f(1 / 15), f(0)) + f(0)).astype(np.float16)
            scale = s[..., g].astype(f)
            q = np.clip(np.rint((part - base[..., None]) * (f(1) / scale)[..., None]), 0, 15)
            q = np.where(((scale == 0) | bad)[..., None], 0, q)
            n[..., g * size:g * size + part.shape[-1]] = q.astype(np.uint8)
            s[..., g] = np.where(bad, np.float16(np.nan), s[..., g])
            m[..., g] = np.where(bad, np.float16(0), m[..., g])
    assert dim <= p
    return n, s, m


def attend4(q, keys, values, seen, scale):
    """One query q [dim] over keys and values, each (n s, m) [tokens][dim], of the tokens `seen`: (y, sizes, reach) as
    decoder_plain.attend's, with the sizes of the sums as they are taken: |n s| + |m|."""
    k, v = keys[0] + keys[1], values[0] + values[1]
    if not seen.any():
        return np.zeros(q.shape), np.zeros(q.shape), 0.0
    z = (k[seen] @ q) * scale
    e = np.exp(z - z.max())
    e /= e.sum()
    reach = ((np.abs(keys[0]) + np.abs(keys[1]))[seen] @ np.abs(q)).max() * abs(scale)
    return e @ v[seen], e @ (np.abs(values[0]) + np.abs(values[1]))[seen], reach


def attend4_bound(y, size, reach, t):
    """decoder_plain.attention_bound without rounded weights; two more steps of the largest |q| a term (q in f16 parts
    of 2^-22 in all) are within its 16 of a logit, and two parts of a weight, cut at 2^-21, within its 24."""
    return R.attention_bound(y, size, np.asarray(reach), t, False)
