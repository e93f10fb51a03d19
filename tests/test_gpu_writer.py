"""The append with the rotation of positions and the cache in 4 bits on the GPU,
against the same in 64 bits and byte by byte."""
import numpy as np
import pytest

import decoder_plain as R
import writer_plain as W
from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import DeviceArray, synchronize
from test_gpu_decoder import Graph, _stream, pages_of

pytestmark = pytest.mark.gpu


def addr(d):
    return 0 if d is None else d.addr


# ------------------------------------------- rotation with the plain cache

def run_rotated(t, lengths, new, page, heads, kv, dim, rotary, pairs, layout="tokens", gap=0, far=None, in_place=False,
                queries=True):
    rng = np.random.default_rng(dim * 7 + rotary + page)
    p = pages_of(rng, lengths, page, kv, dim, t, layout)
    cache = p.upload()
    rows = sum(new)
    wide = lambda n: np.concatenate([R.stored(rng.normal(0, 1, (rows, n * dim)), t), np.full((rows, gap), 7, R.dtype(t))], 1)  # noqa: E731
    q, k, v = wide(heads), wide(kv), wide(kv)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    places = np.concatenate([np.arange(n) + length - n for n, length in zip(new, lengths)] + [np.zeros(0)]).astype(np.int64)
    positions = places if far is None else places + far
    freqs = W.frequencies(rotary)
    dq, dk, dv = R.on_gpu(q), R.on_gpu(k), R.on_gpu(v)
    do = dq if in_place else R.on_gpu(np.full(q.shape, 7, R.dtype(t)))
    dl, ds, df = R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(starts), R.on_gpu(freqs)
    dp = None if far is None else R.on_gpu(positions.astype(np.int32))
    print(f"rotated append, type {t}, new {new[:6]}, page {page}, heads {heads}/{kv} of {dim}, turned {rotary} pairs {pairs} "
          f"{layout} gap {gap} far {far}", flush=True)
    D.kv_append_rotated(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, len(lengths), rows,
                        freqs=df.addr if rotary else 0, rotary=rotary, pairs=pairs, positions=addr(dp),
                        q=dq.addr if queries else 0, q_out=do.addr if queries else 0, heads=heads if queries else 0,
                        starts=0 if new == [1] * len(new) else ds.addr, q_stride=heads * dim + gap,
                        q_out_stride=heads * dim + gap, k_stride=kv * dim + gap, v_stride=kv * dim + gap)
    synchronize()
    cut = lambda a, n: a[:, :n * dim].reshape(rows, n, dim)  # noqa: E731
    if queries:
        got = R.back(do, R.dtype(t), q.shape)
        assert np.array_equal(got[:, heads * dim:], np.full((rows, gap), 7, R.dtype(t)))
        want, size = W.turned(R.values(cut(q, heads), t), positions, freqs, rotary, pairs)
        R.close(R.values(cut(got, heads), t), want, W.turned_bound(want, size, t) * (size > 0))
    want, size = W.turned(R.values(cut(k, kv), t), positions, freqs, rotary, pairs)
    text = np.repeat(np.arange(len(new)), new)
    for i in range(rows):  # v exactly, and k as it was found, so that all else must be as it was
        p.put(text[i], places[i], cut(k, kv)[i], cut(v, kv)[i])
    got_k, got_v = (R.back(g, R.dtype(t), h.shape) for g, h in zip(p.gpu, p.host))
    assert np.array_equal(got_v.view(np.uint8), p.host[1].view(np.uint8))
    found = np.zeros((rows, kv, dim), R.dtype(t))
    for i in range(rows):
        at, slot = p.at(text[i], places[i])
        found[i] = got_k[at, slot] if layout == "tokens" else got_k[at, :, slot, :dim]
        p.put(text[i], places[i], found[i], cut(v, kv)[i])
    assert np.array_equal(got_k.view(np.uint8), p.host[0].view(np.uint8))
    R.close(R.values(found, t), want, W.turned_bound(want, size, t) * (size > 0))


SHAPES = [(16, 4, 2, 64, 64, False), (16, 4, 2, 64, 64, True), (7, 3, 3, 96, 32, False), (64, 8, 1, 128, 128, False),
          (1, 2, 2, 15, 14, True), (5, 2, 1, 15, 6, False), (24, 6, 2, 80, 40, True), (16, 2, 2, 256, 256, False),
          (16, 5, 5, 2, 2, True), (16, 2, 1, 129, 128, False), (16, 3, 1, 1, 0, False), (16, 40, 8, 128, 64, False),
          (16, 4, 4, 72, 24, True), (16, 4, 4, 72, 16, False)]


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("page,heads,kv,dim,rotary,pairs", SHAPES)
def test_rotated_append(t, page, heads, kv, dim, rotary, pairs):
    lengths, new = [page * 3 + 1, 5, 40, 1, 9], [3, 5, 40, 1, 0]
    run_rotated(t, lengths, new, page, heads, kv, dim, rotary, pairs)
    run_rotated(t, lengths, new, page, heads, kv, dim, rotary, pairs, "heads", gap=3, far=2 ** 20 + 3, in_place=True)
    run_rotated(t, [5, 70, 1], [1, 1, 1], page, heads, kv, dim, rotary, pairs, queries=False)


def test_rotated_append_many_texts():
    # More starts than a wave looks at in one step, most texts without a row.
    for batch in (63, 64, 65, 200, 5000):
        new = [1 if i % 7 == 3 or i == batch - 1 else 0 for i in range(batch)]
        new[batch // 2] = 9
        run_rotated(D.F16, [n + 20 for n in new], new, 16, 2, 1, 32, 32, False)


@pytest.mark.parametrize("positions", [[2 ** 31 - 1, -1, -2 ** 31, 0, 123456789]])
def test_rotation_of_far_positions(positions):
    # Angles far from 0, of either sign: what f32 angles would have no digit of.
    rows, dim = len(positions), 64
    rng = np.random.default_rng(2)
    p = R.Pages(rng, [1] * rows, 16, 1, dim, D.F32)
    cache = p.upload()
    k = rng.normal(0, 1, (rows, 1, dim)).astype(np.float32)
    freqs = np.concatenate([W.frequencies(62), [3.0]]).astype(np.float32)
    dk, dl, df, dp = R.on_gpu(k), R.on_gpu(np.ones(rows, np.int32)), R.on_gpu(freqs), R.on_gpu(np.array(positions, np.int32))
    do = R.on_gpu(k)
    print("rotation, far positions", flush=True)
    D.kv_append_rotated(dk.addr, dk.addr, cache, p.gpu_table.addr, p.width, dl.addr, rows, rows, freqs=df.addr,
                        rotary=dim, positions=dp.addr, q=dk.addr, q_out=do.addr, heads=1)
    synchronize()
    want, size = W.turned(k.astype(np.float64), positions, freqs, dim, False)
    R.close(R.back(do, np.float32, k.shape).astype(np.float64), want, W.turned_bound(want, size, D.F32))


def test_rotated_append_leaves_what_is_out_of_range():
    # As kv_append: places below 0, past the table and in pages that do not exist are written nowhere; the queries of
    # these rows are turned all the same, rows of no text are left.
    rng = np.random.default_rng(3)
    p = R.Pages(rng, [20, 20, 20, 20], 16, 1, 8, D.F32)
    p.table[2, 1], p.table[3, 1] = -1, p.pages
    cache = p.upload()
    k = rng.normal(0, 1, (10, 1, 8)).astype(np.float32)
    dk, dl, df = R.on_gpu(k), R.on_gpu(np.array([1, 33, 18, 18], np.int32)), R.on_gpu(W.frequencies(8))
    ds = R.on_gpu(np.array([1, 3, 5, 7, 10], np.int32))  # row 0 is no text's, the last text's third row is past the rows
    do = R.on_gpu(np.full((10, 1, 8), 7, np.float32))
    print("rotated append out of range", flush=True)
    D.kv_append_rotated(dk.addr, dk.addr, cache, p.gpu_table.addr, p.width, dl.addr, 4, 9, freqs=df.addr, rotary=8,
                        starts=ds.addr, q=dk.addr, q_out=do.addr, heads=1)
    synchronize()
    out = R.back(do, np.float32, k.shape)
    assert (out[[0, 9]] == 7).all()
    places = np.array([-1, 0, 31, 32, 16, 17, 15, 16])
    want, size = W.turned(k[1:9].astype(np.float64), places, W.frequencies(8), 8, False)
    R.close(out[1:9].astype(np.float64), want, W.turned_bound(want, size, D.F32))
    p.put(0, 0, out[2], k[2])
    p.put(1, 31, out[3], k[3])
    p.host[0][p.table[3, 0], 15], p.host[1][p.table[3, 0], 15] = out[7], k[7]
    assert np.array_equal(R.back(p.gpu[0], np.float32, p.host[0].shape), p.host[0], equal_nan=True)
    assert np.array_equal(R.back(p.gpu[1], np.float32, p.host[1].shape), p.host[1], equal_nan=True)


@pytest.mark.parametrize("starts", [(0, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1), (3, 2)])
@pytest.mark.parametrize("four", [False, True])
def test_starts_far_out(starts, four):
    # Only the rows there are count, however many the starts tell of: row i + 1 of a text of 2^31 - 1 has place i then.
    rng = np.random.default_rng(4)
    k = rng.normal(0, 1, (6, 1, 8)).astype(np.float32)
    dk, ds = R.on_gpu(k), R.on_gpu(np.array(starts, np.int32))
    dl = R.on_gpu(np.array([2 ** 31 - 1], np.int32))
    print(f"rotated append, starts {starts}, 4 bits {four}", flush=True)
    p = W.Cache4(rng, [20], 16, 1, 8, 0) if four else R.Pages(rng, [20], 16, 1, 8, D.F32)
    cache = p.upload()
    (D.kv4_append if four else D.kv_append_rotated)(dk.addr, dk.addr, cache, p.gpu_table.addr, p.width, dl.addr, 1, 6,
                                                    starts=ds.addr)
    synchronize()
    if starts[1] > starts[0]:
        for i in range(6):
            if four:
                n, s, m = W.quantised(k[i], 32, 32)
                p.set(0, i, np.stack([n, n]), np.stack([s, s]), np.stack([m, m]))
            else:
                p.put(0, i, k[i], k[i])
    if four:
        assert np.array_equal(p.back(), p.data)
    else:
        for gpu, want in zip(p.gpu, p.host):
            assert np.array_equal(R.back(gpu, np.float32, want.shape), want, equal_nan=True)


# ------------------------------------------------------------ the 4-bit cache

DIMS4 = [(1, 0), (15, 0), (32, 0), (40, 32), (64, 0), (64, 32), (80, 64), (80, 32), (96, 0), (100, 32), (128, 0), (128, 64),
         (128, 32), (130, 32), (150, 64), (192, 64), (192, 0), (200, 32), (256, 0), (256, 64), (256, 32)]


def rows_like(rng, shape):
    """Values of several sizes; groups of one value, of zeros, past f16, and tiny ones among them."""
    x = rng.normal(0, 1, shape) * 10.0 ** rng.uniform(-2, 2, shape[:-1] + (1,))
    x = x.astype(np.float32).reshape(-1, shape[-1])
    x[::11] = 3.25
    x[5::13] = 0
    x[7::17] *= 1e4
    x[8::17] *= 1e-8
    return x.reshape(shape)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group", DIMS4)
def test_append4_and_read(t, dim, group):
    # Every byte as the formula gives it; what is not written stays. Then read back, rounded once.
    rng = np.random.default_rng(dim + group)
    for page, heads, gap, lengths, new in ((16, 3, 0, [50, 5, 38, 1, 9, 23], [7, 5, 38, 1, 0, 2]),
                                           (48, 5, 32, [33, 100, 4], [1, 1, 1])):
        p = W.Cache4(rng, lengths, page, heads, dim, group, gap=gap)
        cache = p.upload()
        rows = sum(new)
        k, v = (R.stored(np.concatenate([rows_like(rng, (rows, heads, dim)).reshape(rows, -1), np.zeros((rows, 3))], 1), t)
                for _ in range(2))
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        dk, dv, dl, ds = R.on_gpu(k), R.on_gpu(v), R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(starts)
        print(f"4-bit append, type {t}, {heads} heads of {dim} in groups of {group}, page {page}, new {new}", flush=True)
        D.kv4_append(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, len(new), rows, type=t,
                     starts=0 if new == [1, 1, 1] else ds.addr, k_stride=heads * dim + 3, v_stride=heads * dim + 3)
        synchronize()
        at = 0
        for b, n in enumerate(new):
            for i in range(lengths[b] - n, lengths[b]):
                parts = [W.quantised(R.values(x[at, :heads * dim], t).reshape(heads, dim), p.p, p.size) for x in (k, v)]
                p.set(b, i, *(np.stack([a[j] for a in parts]) for j in range(3)))
                at += 1
        got = p.back()
        assert np.array_equal(got, p.data), np.argwhere(got != p.data)[:5].tolist()
        # All of each text, and one row more than the texts have.
        whole = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        total = int(whole[-1])
        out = [R.on_gpu(np.full((total + 1, heads * dim + 5), 7, R.dtype(t))) for _ in range(2)]
        dw = R.on_gpu(whole)
        D.kv4_read(out[0].addr, out[1].addr, cache, p.gpu_table.addr, p.width, dl.addr, len(new), total + 1,
                   starts=dw.addr, type=t, k_stride=heads * dim + 5, v_stride=heads * dim + 5)
        synchronize()
        for part, d in enumerate(out):
            got = R.back(d, R.dtype(t), (total + 1, heads * dim + 5))
            assert (got[:, heads * dim:] == 7).all() and (got[total] == 7).all()
            want = np.concatenate([sum(p.get(b, i)[part]).reshape(1, -1) for b, n in enumerate(lengths) for i in range(n)])
            R.close(R.values(got[:total, :heads * dim], t), want, R.half_step(want, t))


def test_append4_of_infinities():
    # A group with an infinity or NaN has the scale NaN and codes 0; its neighbours are as they would be.
    rng = np.random.default_rng(9)
    heads, dim = 2, 128
    p = W.Cache4(rng, [6], 16, heads, dim, 32)
    cache = p.upload()
    k, v = (rng.normal(0, 1, (6, heads, dim)).astype(np.float32) for _ in range(2))
    k[1, 0, 5], k[2, 1, 127], v[3, 1, 64], v[5, 0, 33] = np.inf, np.nan, -np.inf, np.nan
    dk, dv, dl, ds = R.on_gpu(k), R.on_gpu(v), R.on_gpu(np.array([6], np.int32)), R.on_gpu(np.array([0, 6], np.int32))
    print("4-bit append of infinities", flush=True)
    D.kv4_append(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, 1, 6, starts=ds.addr)
    D.kv4_read(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, 1, 6, starts=ds.addr)
    synchronize()
    for x, d in ((k, dk), (v, dv)):
        got = R.back(d, np.float32, x.shape)
        n, s, m = W.quantised(x, 128, 32)
        want = n.astype(np.float64) * np.repeat(s.astype(np.float64), 32, -1) + np.repeat(m.astype(np.float64), 32, -1)
        assert np.isnan(want).sum() == 64
        assert np.array_equal(np.isnan(got), np.isnan(want))
        R.close(got.astype(np.float64), want, R.half_step(np.nan_to_num(want), D.F32))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group,rotary,pairs", [(64, 0, 64, False), (64, 32, 64, True), (15, 0, 14, False),
                                                    (15, 0, 6, True), (128, 64, 128, False), (96, 32, 32, True),
                                                    (80, 64, 40, False), (100, 32, 50, False), (256, 32, 256, False),
                                                    (192, 0, 96, True), (128, 32, 48, False)])
def test_append4_rotated(t, dim, group, rotary, pairs):
    # k turned in f32, then held: each value is half a scale off its group's line at most, and the line ends where the
    # largest value does but for the scale's rounding (15 times half a step) and the minimum's.
    rng = np.random.default_rng(dim + rotary)
    heads, kv, page, far = 6, 3, 16, 900000
    lengths, new = [50, 5, 38, 9], [7, 5, 38, 2]
    p = W.Cache4(rng, lengths, page, kv, dim, group)
    cache = p.upload()
    rows = sum(new)
    q, k, v = (R.stored(rng.normal(0, 1, (rows, n, dim)), t) for n in (heads, kv, kv))
    places = np.concatenate([np.arange(n) + length - n for n, length in zip(new, lengths)])
    freqs = W.frequencies(rotary)
    dq, dk, dv, df = R.on_gpu(q), R.on_gpu(k), R.on_gpu(v), R.on_gpu(freqs)
    dl, ds = R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    dp, do = R.on_gpu((places + far).astype(np.int32)), R.on_gpu(np.zeros_like(q))
    print(f"4-bit append, type {t}, heads of {dim} in groups of {group}, {rotary} turned, pairs {pairs}", flush=True)
    D.kv4_append(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, 4, rows, type=t, starts=ds.addr,
                 freqs=df.addr, rotary=rotary, pairs=pairs, positions=dp.addr, q=dq.addr, q_out=do.addr, heads=heads)
    synchronize()
    want, size = W.turned(R.values(q, t), places + far, freqs, rotary, pairs)
    R.close(R.values(R.back(do, R.dtype(t), q.shape), t), want, W.turned_bound(want, size, t) * (size > 0))
    want, size = W.turned(R.values(k, t), places + far, freqs, rotary, pairs)
    p.data[...] = p.back()
    at = 0
    for b, n in enumerate(new):
        for i in range(lengths[b] - n, lengths[b]):
            (ks, km), (vs, vm) = p.get(b, i)
            page_, slot = p.place(b, i)
            s, m = (np.repeat(p.few()[j][page_, :, slot].astype(np.float64), p.size, -1)[:, :dim] for j in (0, 1))
            R.close(ks + km, want[at], s / 2 + 15 * s * 2.0 ** -11 + np.abs(m) * 2.0 ** -10 + size[at] * 4 * 2.0 ** -24 + 1e-7)
            n4, s4, m4 = W.quantised(R.values(v[at], t), p.p, p.size)
            of = np.arange(dim) // p.size
            assert np.array_equal(vs + vm, n4[:, :dim] * s4.astype(np.float64)[:, of] + m4.astype(np.float64)[:, of])
            at += 1


def test_read4_of_pages_that_do_not_exist():
    # NaN there and past the table's row; rows at places below 0 and of no text are left.
    rng = np.random.default_rng(3)
    p = W.Cache4(rng, [20, 20, 20], 16, 2, 40, 32)
    p.fill(rng, [20, 20, 20])
    p.table[1, 1], p.table[2, 1] = -1, p.pages
    cache = p.upload()
    lengths, count = [2, 18, 34], [4, 18, 5]
    rows = sum(count)
    out = [R.on_gpu(np.full((rows + 3, 2, 40), 7, np.float32)) for _ in range(2)]
    dl, ds = R.on_gpu(np.array(lengths, np.int32)), R.on_gpu((1 + np.concatenate([[0], np.cumsum(count)])).astype(np.int32))
    print("4-bit read of bad pages", flush=True)
    D.kv4_read(out[0].addr, out[1].addr, cache, p.gpu_table.addr, p.width, dl.addr, 3, rows + 2, starts=ds.addr)
    synchronize()
    for part, d in enumerate(out):
        got = R.back(d, np.float32, (rows + 3, 2, 40))
        assert (got[[0, 1, 2, rows + 1, rows + 2]] == 7).all()  # text 0's places -2 and -1, and rows of no text
        assert np.array_equal(got[3:5], np.stack([sum(p.get(0, i)[part]) for i in range(2)]).astype(np.float32))
        assert np.array_equal(got[5:21], np.stack([sum(p.get(1, i)[part]) for i in range(16)]).astype(np.float32))
        assert np.isnan(got[21:28]).all()  # text 1's page 1, and text 2's places 29 .. 33: a page past the cache's, and past the row


# ----------------------------------------------------- attention in 4 bits

def run_attend4(lengths, page, heads, kv, dim, group, t, window=0, sinks=0, work=1 << 22, gap=0, longest=0, scale=None,
                seed=0, cut=None):
    rng = np.random.default_rng(dim + page + seed)
    p = W.Cache4(rng, lengths, page, kv, dim, group, nan=True, gap=64 if gap else 0)
    p.fill(rng, lengths)
    if cut:
        cut(p)
    cache = p.upload()
    batch, scale = len(lengths), 1.3 * dim ** -0.5 if scale is None else scale
    q = R.stored(rng.normal(0, 2, (batch, heads * dim + gap)), t)
    dq, dl = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32))
    dy, dw = R.on_gpu(np.zeros((batch, heads * dim + gap), R.dtype(t))), R.on_gpu(np.full(max(work, 4), 0xFF, np.uint8))
    print(f"4-bit attention {lengths} page {page} heads {heads}/{kv} of {dim} in {group} type {t} window {window} sinks "
          f"{sinks} work {work}", flush=True)
    D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, batch, heads, scale=scale, type=t,
                    window=window, sinks=sinks, longest=longest, workspace=dw.addr if work else 0, workspace_bytes=work,
                    q_stride=heads * dim + gap, y_stride=heads * dim + gap)
    synchronize()
    R.back(dw, np.uint8, (max(work, 4),))
    y = R.back(dy, R.dtype(t), (batch, heads * dim + gap))
    assert not y[:, heads * dim:].any()
    got = R.values(y[:, :heads * dim], t).reshape(batch, heads, dim)
    per = heads // kv
    for b, n in enumerate(lengths):
        seen = R.window_seen([n - 1], n, window, sinks)[0]
        parts = [p.get(b, i) for i in range(n)]
        for h in range(heads):
            k, v = ([np.array([x[part][j][h // per] for x in parts]).reshape(n, dim) for j in (0, 1)] for part in (0, 1))
            qh = R.values(q[b, h * dim:(h + 1) * dim], t)
            want, size, reach = W.attend4(qh, k, v, seen, scale)
            R.close(got[b, h], want, W.attend4_bound(want, size, reach, t))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group", DIMS4)
def test_attend4(t, dim, group):
    run_attend4([1, 0, 130, 16, 33], 16, 4, 2, dim, group, t)
    run_attend4([250, 31], 48, 3, 1, dim, group, t, work=0, gap=5)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 1), (17, 1), (40, 2), (7, 7)])
def test_attend4_heads(t, heads, kv):
    run_attend4([70, 200], 32, heads, kv, 64, 32, t)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (33, 4), (100, 1), (64, 60), (300, 4), (40, 200)])
def test_attend4_window(t, window, sinks):
    run_attend4([300, 1, 97, 64, 0], 16, 4, 2, 64, 0, t, window, sinks)
    run_attend4([300, 129], 48, 4, 2, 128, 64, t, window, sinks, work=0)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("work,longest", [(1 << 22, 0), (1 << 14, 0), (0, 0), (1 << 22, 40)])
def test_attend4_long(t, work, longest):
    run_attend4([2100, 3, 700], 16, 2, 1, 96, 32, t, work=work, longest=longest)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-20, 30.0])
def test_attend4_scales(t, scale):
    run_attend4([100, 5], 16, 2, 1, 64, 32, t, scale=scale)


@pytest.mark.parametrize("factor", [1e-7, 1e-3, 1e3, 8000.0])
def test_attend4_scales_of_v(factor):
    # V's scales as small and as large as F16 has them, growing from tile to tile: weights times scales stay in range.
    def cut(p):
        s, m = p.few()[2:]
        with np.errstate(all="ignore"):
            s[...] = np.where(np.isnan(s), s, (s.astype(np.float64) * factor * 4).astype(np.float16))
        m[...] = np.where(np.isnan(m), m, np.float16(0))
    for t in R.REAL:
        run_attend4([400, 90], 16, 2, 1, 64, 32, t, cut=cut)


def test_attend4_bad_pages():
    # A seen page that does not exist, and a length past the table, give NaN in their text alone.
    rng = np.random.default_rng(5)
    lengths = [100, 100, 100, 100]
    for work in (0, 1 << 20):
        p = W.Cache4(rng, lengths, 16, 1, 64, 0)
        p.fill(rng, lengths)
        p.table[1, 3], p.table[2, 6] = -1, p.pages
        cache = p.upload()
        q = rng.normal(0, 1, (4, 64)).astype(np.float32)
        dq, dy, dw = R.on_gpu(q), R.on_gpu(np.zeros((4, 64), np.float32)), R.on_gpu(np.zeros(max(work, 4), np.uint8))
        dl = R.on_gpu(np.array([100, 100, 100, 113], np.int32))
        print(f"4-bit attention, bad pages, work {work}", flush=True)
        D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 4, 1, scale=0.1,
                        workspace=dw.addr if work else 0, workspace_bytes=work)
        synchronize()
        y = R.back(dy, np.float32, (4, 64))
        assert np.isfinite(y[0]).all() and np.isnan(y[1:]).all()
        D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 4, 1, scale=0.1, window=4,
                        sinks=16, workspace=dw.addr if work else 0, workspace_bytes=work)
        synchronize()
        y = R.back(dy, np.float32, (4, 64))
        assert np.isfinite(y[:2]).all() and np.isnan(y[2:]).all()  # text 1's page 3 is not seen


def test_attend4_of_what_is_not_finite():
    # A NaN scale in a seen key gives NaN in its text's head, in a seen value in its group's dims; an infinity or NaN
    # in a query gives NaN in that head.
    rng = np.random.default_rng(6)
    p = W.Cache4(rng, [70, 70, 70], 16, 2, 64, 32)
    p.fill(rng, [70, 70, 70])
    page, slot = p.place(0, 40)
    p.few()[0][page, 1, slot, 0] = np.nan
    page, slot = p.place(1, 69)
    p.few()[2][page, 0, slot, 1] = np.nan
    cache = p.upload()
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    q[2, 1, 3], q[2, 2, 63] = np.inf, np.nan
    dq, dy, dl = R.on_gpu(q), R.on_gpu(np.zeros_like(q)), R.on_gpu(np.full(3, 70, np.int32))
    print("4-bit attention, not finite", flush=True)
    D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 3, 4, scale=0.1)
    synchronize()
    bad = np.isnan(R.back(dy, np.float32, q.shape))
    want = np.zeros_like(bad)
    want[0, 2:], want[1, :2, 32:], want[2, 1:3] = True, True, True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("f", [1e-30, 1e30, 2.0 ** -140])
def test_attend4_of_large_and_small_queries(f):
    # The scale that makes the products what they were: q of any size, down to the numbers below 2^-126.
    rng = np.random.default_rng(7)
    p = W.Cache4(rng, [90], 16, 1, 64, 0)
    p.fill(rng, [90])
    cache = p.upload()
    q = (np.round(rng.normal(0, 8, (2, 64))) * f).astype(np.float32)
    scale = float(np.float32(min(0.02 / f, 3e38)))
    dq, dy, dl = R.on_gpu(q), R.on_gpu(np.zeros_like(q)), R.on_gpu(np.array([90], np.int32))
    print(f"4-bit attention, q times {f}", flush=True)
    D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 1, 2, scale=scale)
    synchronize()
    got = R.back(dy, np.float32, q.shape).astype(np.float64)
    parts = [p.get(0, i) for i in range(90)]
    k, v = ([np.array([x[part][j][0] for x in parts]) for j in (0, 1)] for part in (0, 1))
    for h in range(2):
        want, size, reach = W.attend4(q[h].astype(np.float64), k, v, np.ones(90, bool), scale)
        R.close(got[h], want, W.attend4_bound(want, size, reach, D.F32))


def test_cache4_far_offsets():
    # Pages whose bytes lie past 2^32 of the first.
    rng = np.random.default_rng(8)
    page, heads, dim, group = 16, 2, 64, 32
    stride = 3 << 30
    near = W.Cache4(rng, [70], page, heads, dim, group, spare=0)
    near.table[0] = rng.permutation(5)
    far = DeviceArray(4 * stride + 65536)
    cache = D.Kv4Cache(far.addr, 5, page, heads, dim, group, stride)
    k, v = (rng.normal(0, 1, (70, heads, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 1, (1, heads, dim)).astype(np.float32)
    dk, dv, dq, dy = R.on_gpu(k), R.on_gpu(v), R.on_gpu(q), R.on_gpu(np.zeros_like(q))
    dt, dl, ds = R.on_gpu(near.table), R.on_gpu(np.array([70], np.int32)), R.on_gpu(np.array([0, 70], np.int32))
    print("4-bit cache, far offsets", flush=True)
    D.kv4_append(dk.addr, dv.addr, cache, dt.addr, 5, dl.addr, 1, 70, starts=ds.addr)
    D.kv4_attention(dq.addr, cache, dt.addr, 5, dl.addr, dy.addr, 1, heads, scale=0.1)
    D.kv4_read(dk.addr, dv.addr, cache, dt.addr, 5, dl.addr, 1, 70, starts=ds.addr)
    synchronize()
    for i in range(70):
        parts = [W.quantised(x[i], near.p, near.size) for x in (k, v)]
        near.set(0, i, *(np.stack([a[j] for a in parts]) for j in range(3)))
    parts = [near.get(0, i) for i in range(70)]
    for part, d in enumerate((dk, dv)):
        assert np.array_equal(R.back(d, np.float32, k.shape), np.stack([sum(x[part]) for x in parts]).astype(np.float32))
    got = R.back(dy, np.float32, q.shape).astype(np.float64)
    for h in range(heads):
        kk, vv = ([np.array([x[part][j][h] for x in parts]) for j in (0, 1)] for part in (0, 1))
        want, size, reach = W.attend4(q[0, h].astype(np.float64), kk, vv, np.ones(70, bool), 0.1)
        R.close(got[0, h], want, W.attend4_bound(want, size, reach, D.F32))


# ---------------------------------------------- many rows, and long texts

@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv,dim,rotary,pairs", [(4, 2, 64, 64, False), (5, 1, 40, 16, True), (70, 2, 128, 64, False),
                                                       (2, 1, 15, 14, False)])
def test_rotated_append_many_rows(t, heads, kv, dim, rotary, pairs):
    # More rows than the compute units have: odd counts, texts that end between two rows of a workgroup.
    run_rotated(t, [1100, 3, 9, 200], [1023, 1, 0, 3], 16, heads, kv, dim, rotary, pairs, "heads", in_place=True)
    run_rotated(t, [600, 701], [600, 423], 48, heads, kv, dim, rotary, pairs, gap=8, far=1000, queries=False)


def test_rotated_append_many_rows_of_no_text():
    # Rows before the first text, between those of a start that goes back, and behind the last are left.
    rng = np.random.default_rng(4)
    rows, dim = 1101, 32
    p = R.Pages(rng, [600, 600], 16, 1, dim, D.F16)
    cache = p.upload()
    k = R.stored(rng.normal(0, 1, (rows, 1, dim)), D.F16)
    dk, dl, df = R.on_gpu(k), R.on_gpu(np.array([500, 510], np.int32)), R.on_gpu(W.frequencies(dim))
    ds, do = R.on_gpu(np.array([3, 503, 1013], np.int32)), R.on_gpu(np.full(k.shape, 7, np.float16))
    print("rotated append, many rows of no text", flush=True)
    D.kv_append_rotated(dk.addr, dk.addr, cache, p.gpu_table.addr, p.width, dl.addr, 2, rows, freqs=df.addr, rotary=dim,
                        starts=ds.addr, q=dk.addr, q_out=do.addr, heads=1)
    synchronize()
    out = R.back(do, np.float16, k.shape)
    assert (out[:3] == 7).all() and (out[1013:] == 7).all()
    places = np.concatenate([np.arange(500), np.arange(510)])
    want, size = W.turned(k[3:1013].astype(np.float64), places, W.frequencies(dim), dim, False)
    R.close(out[3:1013].astype(np.float64), want, W.turned_bound(want, size, D.F16))
    for i, (b, at) in enumerate([(0, i) for i in range(500)] + [(1, i) for i in range(510)]):
        p.put(b, at, out[3 + i], k[3 + i])
    for got, held in zip(p.gpu, p.host):
        assert np.array_equal(R.back(got, np.float16, held.shape).view(np.uint16), held.view(np.uint16))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group", DIMS4)
def test_attend4_eight_heads(t, dim, group):
    # Five to eight query heads a key head: two columns each.
    run_attend4([1, 0, 130, 16, 33], 16, 16, 2, dim, group, t)
    run_attend4([250, 31], 48, 5, 1, dim, group, t, work=0, gap=5)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group", DIMS4)
def test_attend4_sixteen_heads(t, dim, group):
    run_attend4([1, 0, 130, 16, 33], 16, 11, 1, dim, group, t)
    run_attend4([250, 31], 48, 20, 1, dim, group, t, work=0, gap=5)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads", [2, 6, 9])
def test_attend4_long_without_parts(t, heads):
    # More tokens than a workgroup looks pages up for at once, in one part.
    run_attend4([4097, 8300], 16, heads, 1, 32, 0, t, work=0)
    run_attend4([9000], 16, heads, 1, 32, 0, t, 4500, 20, work=0)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv", [(2, 1), (3, 3), (14, 2)])
def test_attend4_many_texts(t, heads, kv):
    # Texts of very different lengths, whose parts share out the card's workgroups: more texts than a wave has lanes.
    rng = np.random.default_rng(heads)
    lengths = [int(x) for x in rng.integers(0, 40, 150)]
    lengths[3], lengths[70], lengths[149], lengths[64] = 2500, 1300, 900, 0
    run_attend4(lengths, 16, heads, kv, 32, 0, t, work=1 << 26)
    run_attend4(lengths, 16, heads, kv, 32, 32, t, 600, 20, work=1 << 26)
    run_attend4(lengths, 16, heads, kv, 32, 0, t, work=150 * heads * 34 * 4 * 3)  # three parts a text at most


def test_attend4_more_texts_than_are_added_up():
    lengths = [0, 1, 2, 17] * 300
    lengths[5], lengths[1030], lengths[1199] = 1500, 2100, 700
    run_attend4(lengths, 16, 2, 1, 32, 0, D.F16, work=1 << 26)


@pytest.mark.parametrize("longest", [1000, 2000])
def test_attend4_longer_than_said(longest):
    # Texts longer than `longest`, whose parts go by the lengths that there are.
    lengths = [3, 40, 2500, 0, 700] * 30
    run_attend4(lengths, 16, 4, 4, 32, 0, D.F16, longest=longest, work=1 << 27)


def test_attend4_captured_with_lengths_that_change():
    # The parts of a captured call go by the lengths of each replay: as eager calls, bit for bit.
    rng = np.random.default_rng(8)
    batch, heads, dim = 150, 4, 64
    most = rng.integers(1, 1500, batch)
    p = W.Cache4(rng, most.tolist(), 32, heads, dim, 32)
    p.fill(rng, most.tolist())
    cache = p.upload()
    q = R.stored(rng.normal(0, 2, (batch, heads * dim)), D.BF16)
    dq, dl = R.on_gpu(q), DeviceArray(4 * batch)
    size = D.kv4_attention_workspace(cache, batch, heads, 1500)
    out = [R.on_gpu(np.zeros(q.shape, q.dtype)) for _ in range(2)]
    work = [R.on_gpu(np.full(size, 0xFF, np.uint8)) for _ in range(2)]

    def call(i, stream=0):
        D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, out[i].addr, batch, heads, scale=0.1,
                        type=D.BF16, longest=1500, workspace=work[i].addr, workspace_bytes=size, stream=stream)

    s = _stream()
    dl.upload(most.astype(np.int32))
    call(0, s.value)
    synchronize()
    graph = Graph(s, lambda: call(0, s.value))
    for i in range(5):
        lengths = np.where(rng.random(batch) < 0.3, 0, rng.integers(0, most + 1)) if i else np.minimum(most, 5)
        dl.upload(lengths.astype(np.int32))
        print(f"captured 4-bit attention, replay {i}", flush=True)
        graph.launch()
        synchronize()
        call(1)
        synchronize()
        one, other = (R.back(o, q.dtype, q.shape) for o in out)
        assert np.array_equal(one.view(np.uint16), other.view(np.uint16))
        assert not one[lengths == 0].any() and one[lengths > 0].astype(np.float32).any(-1).all()


# -------------------------- the 4-bit append's queries, in every kind of row

def run_append4(t, lengths, new, page, heads, kv, dim, group, rotary, pairs, gap=0, in_place=False, far=None, held=None,
                change=None, first=0, behind=0):
    """Texts of `lengths` tokens get `new` rows, behind `first` rows of no text and before `behind` of them. What is in
    range is held: k near its line, v as the formula has it; every other byte stays; all texts' queries are turned."""
    rng = np.random.default_rng(dim * 3 + rotary + len(new))
    p = W.Cache4(rng, held or lengths, page, kv, dim, group)
    if change:
        change(p)
    cache = p.upload()
    rows = first + sum(new) + behind
    wide = lambda n: np.concatenate([R.stored(rng.normal(0, 1, (rows, n * dim)), t), np.full((rows, gap), 7, R.dtype(t))], 1)  # noqa: E731
    q, k, v = wide(heads), wide(kv), wide(kv)
    starts = (first + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
    text = np.repeat(np.arange(len(new)), new)
    places = np.concatenate([np.arange(n) + length - n for n, length in zip(new, lengths)]).astype(np.int64)
    positions = np.zeros(rows, np.int64)
    positions[first:first + len(places)] = places + (far or 0)
    freqs = W.frequencies(rotary)
    dq, dk, dv, df = R.on_gpu(q), R.on_gpu(k), R.on_gpu(v), R.on_gpu(freqs)
    do = dq if in_place else R.on_gpu(np.full(q.shape, 7, R.dtype(t)))
    dl, ds, dp = R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(starts), R.on_gpu(positions.astype(np.int32))
    single = new == [1] * len(new) and rows == len(new)
    print(f"4-bit append, type {t}, lengths {lengths[:6]}, new {new[:6]}, heads {heads}/{kv} of {dim} in {group}, {rotary} "
          f"turned, pairs {pairs}, gap {gap}, in place {in_place}, far {far}", flush=True)
    D.kv4_append(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, len(new), rows, type=t,
                 starts=0 if single else ds.addr, freqs=df.addr, rotary=rotary, pairs=pairs,
                 positions=0 if far is None else dp.addr, q=dq.addr, q_out=do.addr, heads=heads,
                 q_stride=heads * dim + gap, q_out_stride=heads * dim + gap, k_stride=kv * dim + gap,
                 v_stride=kv * dim + gap)
    synchronize()
    own = slice(first, first + len(places))
    out = R.back(do, R.dtype(t), q.shape)
    cut = lambda a, n: R.values(a[own, :n * dim].reshape(-1, n, dim), t)  # noqa: E731
    left = q if in_place else np.full_like(q, 7)
    for a, b in ((out[:, heads * dim:], left[:, heads * dim:]), (out[:first], left[:first]),
                 (out[own.stop:], left[own.stop:])):
        assert np.array_equal(a, b)
    want, size = W.turned(cut(q, heads), positions[own], freqs, rotary, pairs)
    R.close(cut(out, heads), want, W.turned_bound(want, size, t) * (size > 0))
    want, size = W.turned(cut(k, kv), positions[own], freqs, rotary, pairs)
    rest, got = p.data.copy(), p.back()
    p.data[...] = got
    of = np.arange(dim) // p.size
    for i, (b, at) in enumerate(zip(text, places)):
        if at < 0 or at // page >= p.width or not 0 <= p.table[b, at // page] < p.pages:
            continue
        (ks, km), (vs, vm) = p.get(b, at)
        page_, slot = p.place(b, at)
        s, m = (p.few()[j][page_, :, slot].astype(np.float64)[:, of] for j in (0, 1))
        R.close(ks + km, want[i], s / 2 + 15 * s * 2.0 ** -11 + np.abs(m) * 2.0 ** -10 + size[i] * 4 * 2.0 ** -24 + 1e-7)
        n4, s4, m4 = W.quantised(cut(v, kv)[i], p.p, p.size)
        assert np.array_equal(vs, n4[:, :dim] * s4.astype(np.float64)[:, of])
        assert np.array_equal(vm, m4.astype(np.float64)[:, of])
        # This token's bytes may differ from what was there.
        for x, y in zip(rest[page_, :kv * p.chunk].reshape(kv, -1), got[page_, :kv * p.chunk].reshape(kv, -1)):
            for bytes_ in p.dims(slot):
                x[bytes_] = y[bytes_]
            for j in (1, 2, 4, 5):
                at_ = p.at[j] + slot * 2 * p.groups
                x[at_:at_ + 2 * p.groups] = y[at_:at_ + 2 * p.groups]
    assert np.array_equal(got, rest)


TURNS4 = [(128, 64, 128, False), (64, 0, 32, False), (96, 32, 48, False), (40, 0, 40, True), (15, 0, 14, False),
          (15, 0, 6, True), (72, 32, 24, False), (256, 32, 256, False)]


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group,rotary,pairs", TURNS4)
def test_append4_of_places_below_0(t, dim, group, rotary, pairs):
    # A text of fewer tokens than rows: a finished one of length 0 with its one row, or a prompt whose length was cut.
    turn = (dim, group, rotary, pairs)
    run_append4(t, [5, 0, 7, 0], [1, 1, 1, 1], 16, 4, 2, *turn)
    run_append4(t, [5, 0, -40, 16], [1, 1, 1, 1], 16, 4, 2, *turn, gap=3, in_place=True, far=1000, held=[5, 1, 1, 16])
    run_append4(t, [3, 0, 20, 2], [40, 17, 3, 2], 16, 4, 2, *turn, first=2, behind=3)
    run_append4(t, [1, 33], [17, 34], 48, 6, 1, *turn, in_place=True, far=50)


@pytest.mark.parametrize("t", R.REAL)
def test_append4_leaves_what_is_out_of_range(t):
    # As the plain cache's: places past the table and in pages that do not exist are written nowhere; the queries of
    # these rows are turned all the same.
    def change(p):
        p.table[2, 1], p.table[3, 1] = -1, p.pages
    for in_place in (False, True):
        run_append4(t, [1, 33, 18, 18], [2, 2, 4, 5], 16, 2, 1, 8, 0, 8, False, held=[20] * 4, change=change, first=1,
                    behind=1, in_place=in_place)
        run_append4(t, [40, 33, 18, 18], [1] * 4, 16, 4, 2, 64, 32, 64, False, held=[20] * 4, change=change,
                    in_place=in_place)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim,group,rotary,pairs", TURNS4)
def test_append4_of_a_token_a_text(t, dim, group, rotary, pairs):
    # The newest token of each text, turned with its queries, in place or not, rows with gaps.
    lengths = [1, 16, 17, 40, 5, 100, 33]
    for in_place, gap, far in ((False, 0, None), (True, 5, None), (True, 0, 2 ** 20 + 1), (False, 8, 300)):
        run_append4(t, lengths, [1] * 7, 16, 6, 3, dim, group, rotary, pairs, gap=gap, in_place=in_place, far=far)
    run_append4(t, [70, 49, 4], [9, 17, 4], 48, 40, 8, dim, group, rotary, pairs, gap=8, in_place=True)


# ------------------------------------- attention: scales of V of very different sizes

def check_attend4(p, lengths, q, t, scale, work=1 << 22):
    """Attention over the cache as it is, of q [texts][heads][dim] (as stored), against 64 bits."""
    cache = p.upload()
    batch, heads, dim = q.shape
    dq, dl, dy = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(np.zeros_like(q))
    dw = R.on_gpu(np.full(max(work, 4), 0xFF, np.uint8))
    print(f"4-bit attention {lengths}, heads {heads}/{p.heads} of {dim} in {p.group} type {t} scale {scale} work {work}",
          flush=True)
    D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, batch, heads, scale=scale, type=t,
                    workspace=dw.addr if work else 0, workspace_bytes=work)
    synchronize()
    got = R.values(R.back(dy, q.dtype, q.shape), t)
    for b, n in enumerate(lengths):
        parts = [p.get(b, i) for i in range(n)]
        for h in range(heads):
            k, v = ([np.array([x[part][j][h * p.heads // heads] for x in parts]).reshape(n, dim) for j in (0, 1)]
                    for part in (0, 1))
            want, size, reach = W.attend4(R.values(q[b, h], t), k, v, np.ones(n, bool), scale)
            R.close(got[b, h], want, W.attend4_bound(want, size, reach, t))


def spread_v(p, lengths, ratio, tokens=(), group=None):
    """V's scales `ratio` times as large for some tokens of each text, or in one group of each head; its minima 0, so
    that outputs are sums of weights times scales times codes alone."""
    for b, n in enumerate(lengths):
        for i in range(n):
            page, slot = p.place(b, i)
            s, m = p.few()[2][page, :, slot], p.few()[3][page, :, slot]
            large = (i in tokens) | (np.arange(p.groups) == group)
            s[...] = s.astype(np.float64) * np.where(large, 8000.0, 8000.0 / ratio)
            m[...] = 0


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads", [2, 6, 11])
@pytest.mark.parametrize("ratio", [2.0 ** 16, 2.0 ** 22, 2.0 ** 26])
def test_attend4_of_a_group_with_large_scales(t, heads, ratio):
    # A group's bits are its own: another group of the same head has scales up to 2^26 times as large.
    lengths = [400, 90, 33]
    for dim, group, work in ((64, 0, 1 << 22), (64, 1, 0), (128, 2, 1 << 22)):
        rng = np.random.default_rng(dim + group)
        p = W.Cache4(rng, lengths, 16, 1, dim, 32, nan=True)
        p.fill(rng, lengths)
        spread_v(p, lengths, ratio, group=group)
        check_attend4(p, lengths, R.stored(rng.normal(0, 1, (3, heads, dim)), t), t, dim ** -0.5, work)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads", [2, 6, 11])
@pytest.mark.parametrize("where", [[0, 1, 200], [63, 64, 399], list(range(0, 400, 7))])
def test_attend4_of_large_scales_without_weight(t, heads, where):
    # Tokens whose scales are 2^26 times the others', but whose keys give them weights of e^-30 beside these (and
    # that may come first): the others keep their bits.
    lengths = [400, 401]
    for group, work in ((32, 1 << 22), (0, 0)):
        rng = np.random.default_rng(group + 3)
        p = W.Cache4(rng, lengths, 16, 1, 64, group, nan=True)
        p.fill(rng, lengths)
        spread_v(p, lengths, 2.0 ** 26, tokens=where)
        for b, n in enumerate(lengths):
            for i in range(n):  # keys the same in all dims: the score is that times the query's sum
                page, slot = p.place(b, i)
                p.few()[0][page, :, slot] = 0
                p.few()[1][page, :, slot] = -1.0 if i in where else (i % 5) / 32
        check_attend4(p, lengths, R.stored(1 + rng.integers(0, 2, (2, heads, 64)), t), t, 20 / 64, work)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads", [2, 6, 11])
@pytest.mark.parametrize("scale", [1e4, 1e6, -3.3e7, 1e9, 7e12, 1e20, 1e30])
def test_attend4_of_very_large_scores(t, heads, scale):
    # Products of q with keys that f32 holds exactly, times a scale that makes scores of 10^6 and more of them: all
    # weight goes to the keys whose product is the largest, in equal parts, wherever they lie.
    lengths, dim = [300, 301, 40], 64
    for work, group in ((1 << 22, 32), (0, 0)):
        rng = np.random.default_rng(heads)
        p = W.Cache4(rng, lengths, 16, 1, dim, group, nan=True)
        p.fill(rng, lengths)
        keys = [rng.integers(-3, 3, n) for n in lengths]
        for b, n in enumerate(lengths):
            keys[b][rng.integers(0, n, 3)] = 3
            keys[b][rng.integers(0, n, 3)] = -4
            for i in range(n):
                page, slot = p.place(b, i)
                p.few()[0][page, :, slot] = 0
                p.few()[1][page, :, slot] = keys[b][i]
        q = R.stored(rng.integers(1, 7, (3, heads, dim)), t)
        cache = p.upload()
        dq, dl, dy = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(np.zeros_like(q))
        dw = R.on_gpu(np.full(max(work, 4), 0xFF, np.uint8))
        print(f"4-bit attention, scale {scale}, heads {heads} type {t} group {group} work {work}", flush=True)
        D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 3, heads, scale=scale, type=t,
                        workspace=dw.addr if work else 0, workspace_bytes=work)
        synchronize()
        got = R.values(R.back(dy, q.dtype, q.shape), t)
        for b, n in enumerate(lengths):
            best = np.nonzero(keys[b] == (keys[b].max() if scale > 0 else keys[b].min()))[0]
            v = [p.get(b, i)[1] for i in best]
            want = np.mean([n_ + m for n_, m in v], 0)[0]
            size = np.mean([np.abs(n_) + np.abs(m) for n_, m in v], 0)[0]
            for h in range(heads):  # the scores of the best are equal: no error of theirs counts
                R.close(got[b, h], want, W.attend4_bound(want, size, 0.0, t))


@pytest.mark.parametrize("heads", [4, 8, 16])
@pytest.mark.parametrize("dim,group", [(64, 0), (128, 32)])
def test_attend4_of_f32_is_not_off_to_one_side(heads, dim, group):
    # Values that are all the same number: what is left is the weights' rounding into two F16 parts. Cut, these would
    # be less by 2^-22 (1/2 + 1/8 + 1/32 ...) of 1 .. 2 on average, 0.92 steps of 2^-23 of the result; rounded, by
    # nothing. An output's other roundings (its sums' over 10 tiles of a column) come to two steps, independent from
    # text to text and head to head: the mean of 256 or more is within 4 * 2 / 16 = 0.5 steps.
    rng = np.random.default_rng(heads)
    lengths = [300] * 64
    p = W.Cache4(rng, lengths, 16, 1, dim, group)
    p.data[...] = rng.integers(0, 256, p.data.shape)
    ks, km, vs, vm = p.few()
    ks[...], km[...], vs[...], vm[...] = rng.uniform(0.01, 0.2, ks.shape), rng.normal(0, 1, km.shape), 0.0713, 0
    p.plane(3)[...] = 0xFF
    cache = p.upload()
    q = rng.normal(0, 1, (64, heads, dim)).astype(np.float32)
    dq, dl, dy = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(np.zeros_like(q))
    print(f"4-bit attention of equal values, heads {heads} of {dim} in {group}", flush=True)
    D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 64, heads, scale=0.3)
    synchronize()
    want = 15 * float(np.float16(0.0713))
    off = (R.back(dy, np.float32, q.shape).astype(np.float64) / want - 1) / R.STEP
    assert abs(off.mean()) < 0.5, off.mean()


# ------------------------------------------------ values next to F16's largest

LARGEST = [(0.0, 65504.0), (-65504.0, 65504.0), (-65504.0, 0.0), (65000.0, 65504.0), (65504.0, 65504.0), (-3.0, 65488.0)]


@pytest.mark.parametrize("dim,group", [(64, 0), (128, 32), (40, 32)])
def test_read4_of_the_largest_values(dim, group):
    # Finite rows come back finite in F16 where code 15 stands for 65520 or 65536; in BF16 and F32 as they are held.
    rng = np.random.default_rng(dim)
    rows = len(LARGEST)
    p = W.Cache4(rng, [rows], 16, 2, dim, group)
    cache = p.upload()
    k, v = (np.stack([rng.uniform(low, high, (2, dim)) for low, high in LARGEST]).astype(np.float16) for _ in range(2))
    for x in (k, v):  # each group has both ends
        for i, (low, high) in enumerate(LARGEST):
            x[i, :, ::8], x[i, :, 3::8] = low, high
    dk, dv, dl, ds = R.on_gpu(k), R.on_gpu(v), R.on_gpu(np.array([rows], np.int32)), R.on_gpu(np.array([0, rows], np.int32))
    print(f"4-bit read of the largest values, heads of {dim} in {group}", flush=True)
    D.kv4_append(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, 1, rows, starts=ds.addr, type=D.F16)
    for t in R.REAL:
        out = [R.on_gpu(np.full((rows, 2, dim), 7, R.dtype(t))) for _ in range(2)]
        D.kv4_read(out[0].addr, out[1].addr, cache, p.gpu_table.addr, p.width, dl.addr, 1, rows, starts=ds.addr, type=t)
        synchronize()
        for x, d in ((k, out[0]), (v, out[1])):
            n, s, m = W.quantised(x, p.p, p.size)
            of = np.arange(dim) // p.size
            want = n[..., :dim] * s.astype(np.float64)[..., of] + m.astype(np.float64)[..., of]
            assert want.max() > 65504
            got = R.values(R.back(d, R.dtype(t), (rows, 2, dim)), t)
            assert np.isfinite(got).all()
            want = np.minimum(want, 65504) if t == D.F16 else want
            R.close(got, want, R.half_step(want, t))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("work", [0, 1 << 20])
@pytest.mark.parametrize("dim,group", [(64, 0), (128, 32)])
def test_attend4_of_the_largest_values(t, work, dim, group):
    # Means of values that are held as 65520 or 65536: finite in F16, too.
    rng = np.random.default_rng(dim)
    n = len(LARGEST)
    for lengths in ([n, 1, 2], [2000, 1, 1500]):
        p = W.Cache4(rng, lengths, 16, 1, dim, group, nan=True)
        p.fill(rng, lengths)
        for b, length in enumerate(lengths):
            for i in range(length):
                x = np.full((1, dim), LARGEST[i % 2][1], np.float32)
                x[:, ::8] = LARGEST[i % 2][0]
                _, s, m = W.quantised(x, p.p, p.size)
                page, slot = p.place(b, i)
                p.few()[2][page, :, slot], p.few()[3][page, :, slot] = s, m
        p.plane(3)[...] = 0xFF
        cache = p.upload()
        q = R.stored(rng.normal(0, 1, (3, 2, dim)), t)
        dq, dl, dy = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(np.zeros_like(q))
        dw = R.on_gpu(np.full(max(work, 4), 0xFF, np.uint8))
        print(f"4-bit attention of the largest values, type {t} heads of {dim} in {group} work {work}", flush=True)
        D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 3, 2, scale=0.1, type=t,
                        workspace=dw.addr if work else 0, workspace_bytes=work)
        synchronize()
        got = R.values(R.back(dy, q.dtype, q.shape), t)
        for b, length in enumerate(lengths):
            parts = [p.get(b, i) for i in range(length)]
            k, v = ([np.array([x[part][j][0] for x in parts]) for j in (0, 1)] for part in (0, 1))
            for h in range(2):
                want, size, reach = W.attend4(R.values(q[b, h], t), k, v, np.ones(length, bool), 0.1)
                assert want.max() > 65504 and np.isfinite(got[b, h]).all()
                want = np.minimum(want, 65504) if t == D.F16 else want
                R.close(got[b, h], want, W.attend4_bound(want, size, reach, t))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,dim,group", [(32, 128, 64), (16, 64, 0)])
def test_attend4_again(t, heads, dim, group):
    # The same call gives the same bits, whatever the workspace and the output held before and whatever ran between.
    rng = np.random.default_rng(dim)
    lengths = [4000] + [int(x) for x in rng.integers(1, 4000, 31)]
    p = W.Cache4(rng, lengths, 64, 8, dim, group)
    p.data[...] = rng.integers(0, 256, p.data.shape, np.uint8)
    ks, km, vs, vm = p.few()
    ks[...], vs[...] = rng.uniform(0.05, 0.3, (2,) + ks.shape)
    km[...], vm[...] = rng.normal(-2, 0.5, (2,) + km.shape)
    cache = p.upload()
    q = R.stored(rng.normal(0, 2, (32, heads, dim)), t)
    dq, dl = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32))
    size = D.kv4_attention_workspace(cache, 32, heads, 4000)
    assert size
    print(f"4-bit attention again, type {t} heads {heads} of {dim}", flush=True)
    got = []
    for i in range(6):
        dy, dw = R.on_gpu(np.full(q.shape, i, q.dtype)), R.on_gpu(np.full(size, (0, 255, 127, 60, 1, 0)[i], np.uint8))
        D.kv4_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 32, heads, scale=dim ** -0.5, type=t,
                        longest=4000, workspace=dw.addr, workspace_bytes=size)
        if i % 2:
            D.kv4_read(dy.addr, dy.addr, cache, p.gpu_table.addr, p.width, dl.addr, 0, 0, type=t)
        synchronize()
        got.append(R.back(dy, q.dtype, q.shape).copy())
    assert all(np.array_equal(g.view(np.uint8), got[0].view(np.uint8)) for g in got)
    assert np.isfinite(R.values(got[0], t)).all()
