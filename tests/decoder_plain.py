"""The decoder layers in 64 bits on numpy, number types, and tolerances.

A rounding to a type is off by at most half a step, `eps / 2` of the value.
The kernels sum in f32 (24 bits; the matrix products may cut instead of round,
so a step is counted as 2^-23). Roundings of a sum are independent: n of them
come to about sqrt(n) steps of the largest partial sum, and a tolerance takes
16 (four standard deviations, 0.29 sqrt(n) steps each, of 200 roundings) times
the sum of the terms' sizes.
"""
from __future__ import annotations

import numpy as np

from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import DeviceArray

EPS = {D.F32: 2.0 ** -23, D.BF16: 2.0 ** -7, D.F16: 2.0 ** -10, D.E4M3: 2.0 ** -3}
STEP = 2.0 ** -23
# The smallest numbers' step: below 2^-14 in F16 (2^-126 in BF16 and F32) numbers are multiples of it, so that a
# rounding there is off by up to half of it however small the value (F16: 6.98e-6 = 117.1 steps, stored as 117).
LEAST = {D.F32: 2.0 ** -149, D.BF16: 2.0 ** -133, D.F16: 2.0 ** -24}
REAL = [D.F32, D.BF16, D.F16]


def stored(a, t) -> np.ndarray:
    """The nearest values of type t, as stored."""
    a = np.asarray(a, np.float32)
    if t == D.F32:
        return a.copy()
    if t == D.F16:
        return a.astype(np.float16)
    bits = a.view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    out[np.isnan(a)] = 0x7FC0
    return out


def values(raw, t) -> np.ndarray:
    """Stored values as float64."""
    if t == D.BF16:
        return (np.asarray(raw, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if t == D.E4M3:
        raw = np.asarray(raw, np.uint8)
        e, m = (raw >> 3 & 15).astype(np.int32), (raw & 7).astype(np.float64)
        v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
        v = np.where((raw & 127) == 127, np.nan, v)
        return np.where(raw & 128, -v, v)
    if t == D.I8:
        return np.asarray(raw).view(np.int8).astype(np.float64)
    return np.asarray(raw).astype(np.float64)


def dtype(t):
    return {D.F32: np.float32, D.BF16: np.uint16, D.F16: np.float16, D.E4M3: np.uint8, D.I8: np.uint8}[t]


def on_gpu(a) -> DeviceArray:
    """The array on the GPU; a guard of 0xAB bytes behind it."""
    a = np.ascontiguousarray(a)
    d = DeviceArray(a.nbytes + 64)
    d.upload(np.concatenate([a.view(np.uint8).reshape(-1), np.full(64, 0xAB, np.uint8)]))
    return d


def back(d: DeviceArray, like, shape) -> np.ndarray:
    """What is on the GPU, after a check of the guard."""
    n = int(np.prod(shape)) * np.dtype(like).itemsize
    raw = d.download(n + 64, np.uint8)
    assert (raw[n:] == 0xAB).all(), "written past the end"
    return raw[:n].view(like).reshape(shape)


def half_step(want, t):
    return np.maximum(np.abs(want) * EPS[t], LEAST[t]) / 2


def close(got, want, bound):
    bad = ~(np.abs(got - want) <= bound) & ~(np.isnan(got) & np.isnan(want)) & ~(np.isinf(want) & (got == want))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


def norm(x, residual, weight, t, eps):
    """(h as stored, y)."""
    h = stored(x, t)
    if residual is not None:
        h = stored(values(h, t).astype(np.float32) + values(stored(residual, t), t).astype(np.float32), t)
    hv = values(h, t)
    return h, hv / np.sqrt((hv * hv).mean(-1, keepdims=True) + eps) * values(stored(weight, t), t)


def product(x, q, scales, zeros, group):
    """(y, the terms' sizes as the kernel sums them); x, scales as float64, q [n][k]."""
    k = x.shape[1]
    of = np.arange(k) // group
    z = np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64)
    w = (q - z[:, of]) * scales[:, of]
    size = (32.0 + q + z[:, of]) * np.abs(scales[:, of])
    return x @ w.T, np.abs(x) @ size.T


def packed(q) -> np.ndarray:
    """Weights 0 .. 15 two to a byte."""
    q = np.asarray(q, np.uint8)
    if q.shape[1] % 2:
        q = np.concatenate([q, np.zeros((q.shape[0], 1), np.uint8)], 1)
    return np.ascontiguousarray(q[:, 0::2] | q[:, 1::2] << 4)


def attend(q, k, v, seen, scale):
    """One head: q [rows][dim], k, v [keys][dim], seen [rows][keys] -> (y, the
    sizes sum p |v|, the largest sum |q k| scale). Unseen keys are left out."""
    y, size, reach = np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], 1))
    for i in range(q.shape[0]):
        on = seen[i]
        if not on.any():
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = (k[on] @ q[i]) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            y[i], size[i] = p @ v[on], p @ np.abs(v[on])
            reach[i] = (np.abs(k[on]) @ np.abs(q[i])).max() * abs(scale)
    return y, size, reach


def attention_bound(y, size, reach, t, rounded):
    """Half a step of y; of the weights, where they are rounded to t, in the
    product with v and in their sum (e_i: a weight's relative error, at most
    half a step; sum p (1 + e) v / sum p (1 + e) = y + sum p e (v - y) but for
    e^2, and sum p |v - y| <= sum p |v| + |y|); and a weight's relative error from its logarithm's, 16 steps of sum |q k| scale,
    twice (in the sum too), with 8 steps of its exponential."""
    steps = (2 * 16 * reach + 8 + 16) * STEP
    return half_step(y, t) + size * steps + ((size + np.abs(y)) * EPS[t] / 2 if rounded else 0)


def window_seen(places, keys, window, sinks):
    """seen[row][key] for queries at `places`."""
    p, j = np.asarray(places)[:, None], np.arange(keys)[None]
    near = (j > p - window) if window else np.ones_like(j > p)
    return (j <= p) & (near | (j < sinks))


class Pages:
    """A paged cache of given texts on the GPU: pages shuffled, NaN in all that
    no text holds, table entries past a text's pages far out of range."""

    def __init__(self, rng, lengths, page, heads, dim, t, strides=(0, 0, 0), shape=None, spare=2):
        need = [-(-n // page) for n in lengths]
        self.pages, self.page, self.heads, self.dim, self.t = sum(need) + spare, page, heads, dim, t
        self.width = max(need + [1])
        self.table = np.full((len(lengths), self.width), 2 ** 30, np.int32)
        order = rng.permutation(self.pages)
        for b, n in enumerate(need):
            self.table[b, :n], order = order[:n], order[n:]
        self.shape = shape or (self.pages, page, heads, dim)
        nan = stored(np.full(self.shape, np.nan, np.float32), t)
        self.host = [nan.copy(), nan.copy()]
        self.strides = strides
        self.k, self.v = [stored(rng.normal(0, 1, (n, heads, dim)), t) for n in lengths], \
            [stored(rng.normal(0, 1, (n, heads, dim)), t) for n in lengths]
        for b, n in enumerate(lengths):
            for i in range(n):
                self.put(b, i, self.k[b][i], self.v[b][i])

    def at(self, b, i):
        return self.table[b, i // self.page], i % self.page

    def put(self, b, i, k, v):
        page, slot = self.at(b, i)
        for host, row in zip(self.host, (k, v)):
            if self.strides == (0, 0, 0):
                host[page, slot] = row
            else:  # [page][head][token][dim + gap]
                host[page, :, slot, :self.dim] = row

    def upload(self):
        self.gpu = [on_gpu(h) for h in self.host]
        self.gpu_table = on_gpu(self.table)
        return D.KvCache(self.gpu[0].addr, self.gpu[1].addr, self.pages, self.page, self.heads, self.dim, self.t,
                         *self.strides)
