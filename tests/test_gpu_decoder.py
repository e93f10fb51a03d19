"""The decoder layers on the GPU against the same operators in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import decoder_plain as R
from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import hip, synchronize

pytestmark = pytest.mark.gpu
STEP = R.STEP


# ------------------------------------------------------------------- the norm

def run_norm(x, residual, weight, t, y_type=None, group=0, eps=1e-6, gap=0, in_place=False):
    """(h, y raw, scales) of the kernel; rows `gap` values apart."""
    rows, c = x.shape
    y_type = t if y_type is None else y_type
    wide = lambda a: np.concatenate([R.stored(a, t), np.zeros((rows, gap), R.dtype(t))], 1)  # noqa: E731
    dx, dr = R.on_gpu(wide(x)), None if residual is None else R.on_gpu(wide(residual))
    dw = R.on_gpu(R.stored(weight, t))
    dh = dr if in_place else R.on_gpu(np.zeros((rows, c + gap), R.dtype(t)))
    dy = R.on_gpu(np.zeros((rows, c + gap), R.dtype(y_type)))
    groups = -(-c // group) if group else 1
    ds = R.on_gpu(np.zeros((rows, groups), np.float32))
    print(f"norm {rows}x{c} type {t} -> {y_type} group {group} gap {gap}", flush=True)
    D.rms_norm(dx.addr, dw.addr, dy.addr, rows, c, residual=0 if dr is None else dr.addr, sum=dh.addr,
               scales=ds.addr, type=t, y_type=y_type, group=group, eps=eps, x_stride=c + gap,
               residual_stride=c + gap, sum_stride=c + gap, y_stride=c + gap)
    synchronize()
    return (R.back(dh, R.dtype(t), (rows, c + gap))[:, :c], R.back(dy, R.dtype(y_type), (rows, c + gap)),
            R.back(ds, np.float32, (rows, groups)))


NORM_SIZES = [(1, 1), (3, 7), (5, 120), (2, 512), (9, 513), (1, 1000), (3, 2048), (2, 2055), (4, 4096), (1, 5003),
              (2, 8192), (1, 16390), (1, 32768), (2, 33001)]


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("rows,c", NORM_SIZES)
def test_norm(t, rows, c):
    rng = np.random.default_rng(c)
    x, r, w = rng.normal(0, 1, (rows, c)), rng.normal(0, 2, (rows, c)), rng.normal(1, 0.2, c)
    for residual, gap in ((r, 0), (None, 3), (r, 5)):
        h, y, _ = run_norm(x, residual, w, t, gap=gap, in_place=residual is not None and gap == 5)
        want_h, want = R.norm(x, residual, w, t, 1e-6)
        assert np.array_equal(h.view(np.uint8), want_h.view(np.uint8))  # one rounding of an f32 sum
        # Half a step of y; the sum of squares is positive, so 16 steps of it, half that after the root.
        R.close(R.values(y[:, :c], t), want, R.half_step(want, t) + np.abs(want) * 12 * STEP)
        assert not y[:, c:].any()  # the gap is left as it was


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("y_type", [D.E4M3, D.I8])
@pytest.mark.parametrize("rows,c,group", [(3, 7, 0), (5, 120, 32), (2, 513, 64), (3, 4096, 0), (2, 4096, 128),
                                          (2, 1000, 128), (1, 33001, 0), (1, 33001, 32), (2, 20000, 64)])
def test_norm_8_bits(t, y_type, rows, c, group):
    rng = np.random.default_rng(c + group)
    x, w = rng.normal(0, 1, (rows, c)) * 10.0 ** rng.uniform(-3, 3, (rows, c)), rng.normal(1, 0.2, c)
    x[-1, :min(c, 140)] = 0  # groups of zeros
    _, y, scales = run_norm(x, None, w, t, y_type=y_type, group=group, gap=group and 3)
    _, want = R.norm(x, None, w, t, 1e-6)
    size = group or c
    top = 448.0 if y_type == D.E4M3 else 127.0
    most = np.stack([np.abs(want[:, i:i + size]).max(1) for i in range(0, c, size)], 1)
    R.close(scales.astype(np.float64), most / top, most / top * 16 * STEP)
    spread = np.repeat(scales.astype(np.float64), size, 1)[:, :c]
    got = R.values(y[:, :c], y_type) * spread
    # Half a step: of the code in E4M3 (or of its smallest numbers, 2^-9), of the integers in I8.
    half = np.maximum(np.abs(want) * R.EPS[D.E4M3] / 2, spread * 2.0 ** -10) if y_type == D.E4M3 else spread / 2
    R.close(got, want, half * (1 + 2.0 ** -10) + np.abs(want) * 32 * STEP)
    assert not y[:, c:].any()
    assert np.abs(R.values(y[:, :c], y_type)).max() == top


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("c", [300, 33001])
def test_norm_infinities(t, c):
    x, w = np.ones((4, c)), np.ones(c)
    x[1, 5], x[2, 170] = np.nan, np.inf
    _, y, _ = run_norm(x, None, w, t)
    with np.errstate(all="ignore"):
        _, want = R.norm(x, None, w, t, 1e-6)
    R.close(R.values(y, t), want, np.abs(want) * R.EPS[t])
    for y_type in (D.E4M3, D.I8):
        _, y, s = run_norm(x, None, w, t, y_type=y_type, group=128)
        # The NaN makes its whole row NaN; the infinity makes the others 0 and itself NaN.
        assert np.isfinite(s[[0, 3]]).all() and np.isnan(s[1]).all()
        assert np.isnan(s[2, 1]) and not s[2, [0, 2]].any()
        v = y[2, 128:256]
        assert (v == (0x7F if y_type == D.E4M3 else 0)).all()


# ---------------------------------------------------------------- the product

def run_product(rng, m, n, k, group, x_type, scale_type, y_type, zeros, bias, x_group=0, gap=0):
    x = rng.normal(0, 1, (m, k))
    groups = -(-k // group)
    q = rng.integers(0, 16, (n, k))
    scales = R.stored(rng.uniform(0.5, 1.5, (n, groups)) / 64, scale_type)
    z = rng.integers(0, 16, (n, groups)).astype(np.uint8) if zeros else None
    b = R.stored(rng.normal(0, 1, n), y_type) if bias else None
    xs, xv = None, None
    if x_type in (D.E4M3, D.I8):
        xg = groups if x_group else 1
        xs = rng.uniform(0.01, 0.02, (m, xg)).astype(np.float32)
        raw = rng.integers(0, 256, (m, k)).astype(np.uint8)
        if x_type == D.E4M3:
            raw[(raw & 127) == 127] = 0x40
        xv = R.values(raw, x_type) * np.repeat(xs.astype(np.float64), x_group or k, 1)[:, :k]
    else:
        raw = R.stored(x, x_type)
        xv = R.values(raw, x_type)
    dx = R.on_gpu(np.concatenate([raw, np.zeros((m, gap), raw.dtype)], 1))
    dq, ds, dz = R.on_gpu(R.packed(q)), R.on_gpu(scales), None if z is None else R.on_gpu(z)
    db, dxs = None if b is None else R.on_gpu(b), None if xs is None else R.on_gpu(xs)
    dy = R.on_gpu(np.zeros((m, n + gap), R.dtype(y_type)))
    addr = lambda d: 0 if d is None else d.addr  # noqa: E731
    print(f"product {m}x{k}->{n} group {group} x {x_type} scales {scale_type} y {y_type} zeros {zeros}", flush=True)
    D.q4_product(dx.addr, dq.addr, ds.addr, dy.addr, m, n, k, group=group, zeros=addr(dz), bias=addr(db),
                 x_scales=addr(dxs), x_group=x_group, x_type=x_type, scale_type=scale_type, y_type=y_type,
                 x_stride=k + gap, y_stride=n + gap)
    synchronize()
    y = R.back(dy, R.dtype(y_type), (m, n + gap))
    assert not y[:, n:].any()
    want, size = R.product(xv, q, R.values(scales, scale_type), z, group)
    if b is not None:
        want = want + R.values(b, y_type)
    R.close(R.values(y[:, :n], y_type), want, R.half_step(want, y_type) + 16 * STEP * size)


PRODUCT_SIZES = [(1, 1, 1), (1, 16, 32), (2, 40, 100), (3, 17, 127), (5, 33, 257), (16, 64, 128), (17, 50, 384),
                 (33, 100, 200), (1, 300, 4096), (64, 31, 1030), (70, 48, 513), (1, 77, 16001), (4, 1000, 65)]


@pytest.mark.parametrize("x_type", [D.F32, D.BF16, D.F16, D.E4M3, D.I8])
@pytest.mark.parametrize("m,n,k", PRODUCT_SIZES)
def test_product(x_type, m, n, k):
    rng = np.random.default_rng(m * 100 + n)
    y_type = x_type if x_type in R.REAL else D.BF16
    for group, scale_type, zeros, bias, gap in ((32, D.F32, True, False, 0), (64, D.BF16, False, True, 5),
                                                (128, D.F16, True, True, 0)):
        run_product(rng, m, n, k, group, x_type, scale_type, y_type, zeros, bias, gap=gap)
        if x_type in (D.E4M3, D.I8):
            run_product(rng, m, n, k, group, x_type, scale_type, D.F32, zeros, bias, x_group=group)


@pytest.mark.parametrize("x_type", [D.F32, D.BF16, D.F16, D.E4M3])
@pytest.mark.parametrize("m,n,k,group", [(3, 9000, 96, 32), (17, 8300, 200, 128), (2, 16500, 130, 64), (40, 5000, 64, 32),
                                         (16, 32, 4160, 32), (16, 1000, 2100, 32)])
def test_product_many_tiles(x_type, m, n, k, group):
    # Two and four tiles a workgroup, blocks of rows, several chunks of x.
    y_type = x_type if x_type in R.REAL else D.F16
    run_product(np.random.default_rng(n), m, n, k, group, x_type, D.F16, y_type, True, False,
                x_group=group if x_type == D.E4M3 else 0)


def test_product_at_any_address():
    # Weights, scales and x that start at any address of their own type's alignment.
    m, n, k = 3, 50, 512
    rng = np.random.default_rng(6)
    q, x = rng.integers(0, 16, (n, k)), R.stored(rng.normal(0, 1, (m, k)), D.F16)
    s = R.stored(rng.uniform(0.5, 1.5, (n, 8)) / 64, D.BF16)
    for off in (1, 2, 4, 16):
        dq = R.on_gpu(np.concatenate([np.zeros(off, np.uint8), R.packed(q).reshape(-1)]))
        ds, dx = (R.on_gpu(np.concatenate([np.zeros(1, a.dtype), a.reshape(-1)])) for a in (s, x))
        dy = R.on_gpu(np.zeros((m, n), np.float32))
        print(f"product with weights {off} bytes off", flush=True)
        D.q4_product(dx.addr + 2, dq.addr + off, ds.addr + 2, dy.addr, m, n, k, group=64, x_type=D.F16,
                     scale_type=D.BF16, y_type=D.F32)
        synchronize()
        want, size = R.product(R.values(x, D.F16), q, R.values(s, D.BF16), None, 64)
        R.close(R.back(dy, np.float32, (m, n)).astype(np.float64), want,
                R.half_step(want, D.F32) + 16 * STEP * size)


def test_product_keeps_rows_apart():
    # A NaN or infinity in one row of x leaves the others' results alone, and q's bytes past an odd row's end do not matter.
    m, n, k = 5, 40, 131
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (m, k))
    x[1, 7], x[3, 130] = np.nan, np.inf
    q, s = rng.integers(0, 16, (n, k)), np.full((n, 5), 1 / 64, np.float32)
    bytes_ = R.packed(q)
    bytes_[:, -1] |= 0xF0
    for t in R.REAL:
        dx, dq, ds = R.on_gpu(R.stored(x, t)), R.on_gpu(bytes_), R.on_gpu(s)
        dy = R.on_gpu(np.zeros((m, n), R.dtype(t)))
        print(f"product rows apart, type {t}", flush=True)
        D.q4_product(dx.addr, dq.addr, ds.addr, dy.addr, m, n, k, group=32, x_type=t, scale_type=D.F32, y_type=t)
        synchronize()
        y = R.values(R.back(dy, R.dtype(t), (m, n)), t)
        assert np.isnan(y[1]).all() and np.isnan(y[3]).all()
        rest = [0, 2, 4]
        want, size = R.product(R.values(R.stored(x, t), t)[rest], q, s.astype(np.float64), None, 32)
        R.close(y[rest], want, R.half_step(want, t) + 16 * STEP * size)


# ------------------------------------------------------------------ the cache

LAYOUTS = ["tokens", "heads"]


def pages_of(rng, lengths, page, heads, dim, t, layout):
    if layout == "tokens":
        return R.Pages(rng, lengths, page, heads, dim, t)
    need = sum(-(-n // page) for n in lengths) + 2  # [page][head][token][dim + 3]
    return R.Pages(rng, lengths, page, heads, dim, t, (heads * page * (dim + 3), dim + 3, page * (dim + 3)),
                   (need, heads, page, dim + 3))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page,heads,dim", [(16, 2, 64), (1, 1, 15), (7, 3, 96), (64, 1, 129)])
def test_append(t, layout, page, heads, dim):
    rng = np.random.default_rng(page + dim)
    lengths, new = [page * 3 + 1, 5, 40, 1, 9], [3, 5, 40, 1, 0]
    p = pages_of(rng, lengths, page, heads, dim, t, layout)
    cache = p.upload()
    before = [h.copy() for h in p.host]
    rows = sum(new)
    k, v = (R.stored(rng.normal(0, 1, (rows + 2, heads, dim)), t) for _ in range(2))
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    at = 0
    for b, n in enumerate(new):
        for i in range(n):
            p.put(b, lengths[b] - n + i, k[at], v[at])
            at += 1
    dk, dv, dl, ds = R.on_gpu(k), R.on_gpu(v), R.on_gpu(np.array(lengths, np.int32)), R.on_gpu(starts)
    print(f"append page {page} heads {heads} dim {dim} type {t} {layout}", flush=True)
    D.kv_append(dk.addr, dv.addr, cache, p.gpu_table.addr, p.width, dl.addr, 5, rows, starts=ds.addr)
    synchronize()
    for gpu, want, old in zip(p.gpu, p.host, before):
        got = R.back(gpu, R.dtype(t), want.shape)
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
        assert not np.array_equal(got.view(np.uint8), old.view(np.uint8))
    # One token a text, and the rows a stride apart.
    p2 = pages_of(rng, lengths, page, heads, dim, t, layout)
    cache = p2.upload()
    wide = np.zeros((5, heads * dim + 4), R.dtype(t))
    wide[:, :heads * dim] = k[:5].reshape(5, -1)
    dk, dv = R.on_gpu(wide), R.on_gpu(v[:5])
    D.kv_append(dk.addr, dv.addr, cache, p2.gpu_table.addr, p2.width, dl.addr, 5, 5, k_stride=heads * dim + 4)
    synchronize()
    for b in range(5):
        p2.put(b, lengths[b] - 1, k[b], v[b])
    for gpu, want in zip(p2.gpu, p2.host):
        assert np.array_equal(R.back(gpu, R.dtype(t), want.shape).view(np.uint8), want.view(np.uint8))


def test_append_leaves_what_is_out_of_range():
    # Lengths of nothing, places past the table and pages that do not exist are written nowhere.
    rng = np.random.default_rng(3)
    p = R.Pages(rng, [20, 20, 20, 20], 16, 1, 8, D.F32)
    p.table[2, 1], p.table[3, 1] = -1, p.pages
    cache = p.upload()
    k = rng.normal(0, 1, (8, 1, 8)).astype(np.float32)
    dk, dl = R.on_gpu(k), R.on_gpu(np.array([1, 33, 18, 18], np.int32))
    ds = R.on_gpu(np.array([0, 2, 4, 6, 9], np.int32))  # the last text's third row is past the rows
    print("append out of range", flush=True)
    D.kv_append(dk.addr, dk.addr, cache, p.gpu_table.addr, p.width, dl.addr, 4, 8, starts=ds.addr)
    synchronize()
    p.put(0, 0, k[1], k[1])   # text 0: places -1 and 0
    p.put(1, 31, k[2], k[2])  # text 1: places 31 and 32, the table's end
    p.host[0][p.table[3, 0], 15] = p.host[1][p.table[3, 0], 15] = k[6]  # text 3: places 15, 16, 17
    assert np.array_equal(R.back(p.gpu[0], np.float32, p.host[0].shape), p.host[0], equal_nan=True)
    assert np.array_equal(R.back(p.gpu[1], np.float32, p.host[1].shape), p.host[1], equal_nan=True)


@pytest.mark.parametrize("starts", [(0, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1), (3, 2)])
def test_append_starts_far_out(starts):
    # Only the rows there are count, however many the starts tell of; and a
    # length that all those would have puts row 0 at place 0 again.
    p = R.Pages(np.random.default_rng(4), [20], 16, 1, 8, D.F32)
    cache = p.upload()
    k = np.random.default_rng(5).normal(0, 1, (6, 1, 8)).astype(np.float32)
    dk, ds = R.on_gpu(k), R.on_gpu(np.array(starts, np.int32))
    dl = R.on_gpu(np.array([2 ** 31 - 1], np.int32))
    print(f"append, starts {starts}", flush=True)
    D.kv_append(dk.addr, dk.addr, cache, p.gpu_table.addr, p.width, dl.addr, 1, 6, starts=ds.addr)
    synchronize()
    if starts[1] > starts[0]:
        for i in range(6):
            p.put(0, i, k[i], k[i])
    for gpu, want in zip(p.gpu, p.host):
        assert np.array_equal(R.back(gpu, np.float32, want.shape), want, equal_nan=True)


# ------------------------------------------------------ the decode attention

def run_paged(rng, lengths, page, heads, kv_heads, dim, t, window=0, sinks=0, layout="tokens", work=1 << 22, gap=0,
              longest=0, scale=None):
    p = pages_of(rng, lengths, page, kv_heads, dim, t, layout)
    cache = p.upload()
    batch, scale = len(lengths), 1.3 * dim ** -0.5 if scale is None else scale
    q = R.stored(rng.normal(0, 2, (batch, heads * dim + gap)), t)
    dq, dl = R.on_gpu(q), R.on_gpu(np.array(lengths, np.int32))
    dy, dw = R.on_gpu(np.zeros((batch, heads * dim + gap), R.dtype(t))), R.on_gpu(np.full(max(work, 4), 0xFF, np.uint8))
    print(f"paged {lengths} page {page} heads {heads}/{kv_heads} dim {dim} type {t} window {window} sinks {sinks} "
          f"{layout} work {work}", flush=True)
    D.paged_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, batch, heads, scale=scale,
                      window=window, sinks=sinks, longest=longest, workspace=dw.addr if work else 0,
                      workspace_bytes=work, q_stride=heads * dim + gap, y_stride=heads * dim + gap)
    synchronize()
    R.back(dw, np.uint8, (max(work, 4),))
    y = R.back(dy, R.dtype(t), (batch, heads * dim + gap))
    assert not y[:, heads * dim:].any()
    got = R.values(y[:, :heads * dim], t).reshape(batch, heads, dim)
    per = heads // kv_heads
    for b, n in enumerate(lengths):
        k, v = R.values(p.k[b], t), R.values(p.v[b], t)
        seen = R.window_seen([n - 1], n, window, sinks)
        for h in range(heads):
            qh = R.values(q[b, h * dim:(h + 1) * dim], t)[None]
            y, size, reach = R.attend(qh, k[:, h // per], v[:, h // per], seen, scale)
            R.close(got[b, h:h + 1], y, R.attention_bound(y, size, reach, t, False))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 8, 15), (3, 1, 128), (40, 2, 96), (6, 2, 256), (5, 5, 1),
                                                (2, 1, 80)])
@pytest.mark.parametrize("page", [16, 64, 7])
def test_paged(t, heads, kv_heads, dim, page):
    rng = np.random.default_rng(dim + page)
    run_paged(rng, [1, 0, 130, 16, 33, 700], page, heads, kv_heads, dim, t)
    run_paged(rng, [250, 31], page, heads, kv_heads, dim, t, layout="heads", work=0, gap=5)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [80, 88, 96, 104, 136, 184, 192, 200])
@pytest.mark.parametrize("page", [16, 24])
def test_paged_dims(t, dim, page):
    # Head sizes between the powers of two.
    rng = np.random.default_rng(dim)
    run_paged(rng, [700, 1, 95, 0, 33], page, 6, 2, dim, t)
    run_paged(rng, [700, 1, 95, 0, 33], page, 6, 2, dim, t, 50, 3, layout="heads")


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("page", [16, 48, 1, 5])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 4), (32, 32), (33, 40), (500, 70), (64, 1000), (100000, 3)])
def test_paged_window(t, page, window, sinks):
    rng = np.random.default_rng(window + sinks)
    run_paged(rng, [1, 39, 41, 64, 300, 801], page, 4, 2, 64, t, window, sinks)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("work,longest", [(0, 0), (1 << 15, 0), (1 << 22, 0), (1 << 22, 9000), (1 << 22, 50)])
def test_paged_long(t, work, longest):
    # Split over many parts, over as many as a small workspace takes, over none; `longest` only guides.
    run_paged(np.random.default_rng(5), [9000, 17, 0, 4100], 32, 4, 1, 64, t, work=work, longest=longest)


def test_paged_window_over_evicted_pages():
    # Pages that only unseen tokens lie in may be gone from the table.
    rng = np.random.default_rng(2)
    for page in (16, 10):
        p = R.Pages(rng, [400], page, 1, 64, D.F16)
        for slot in range(1, 300 // page):
            p.table[0, slot] = -1
        cache = p.upload()
        q = R.stored(rng.normal(0, 2, (1, 1, 64)), D.F16)
        dq, dl, dy = R.on_gpu(q), R.on_gpu(np.array([400], np.int32)), R.on_gpu(np.zeros((1, 64), np.float16))
        print(f"paged over evicted pages of {page}", flush=True)
        D.paged_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 1, 1, scale=0.125, window=90,
                          sinks=4)
        synchronize()
        y, size, reach = R.attend(R.values(q[0], D.F16), R.values(p.k[0], D.F16)[:, 0], R.values(p.v[0], D.F16)[:, 0],
                                  R.window_seen([399], 400, 90, 4), 0.125)
        R.close(R.values(R.back(dy, np.float16, (1, 64)), D.F16), y, R.attention_bound(y, size, reach, D.F16, False))


@pytest.mark.parametrize("t", [D.F32, D.F16])
def test_cache_far_offsets(t):
    # Pages further apart than 32 bits of values: append and attention.
    heads, dim, page, stride = 2, 64, 16, (1 << 30) + 64
    rng = np.random.default_rng(1)
    size = np.dtype(R.dtype(t)).itemsize
    far = [R.DeviceArray(size * (4 * stride + 65536)) for _ in range(2)]
    cache = D.KvCache(far[0].addr, far[1].addr, 5, page, heads, dim, t, stride, heads * dim, dim)
    table = np.array([[4, 2, 3]], np.int32)
    k, v = (R.stored(rng.normal(0, 1, (40, heads, dim)), t) for _ in range(2))
    q = R.stored(rng.normal(0, 2, (1, heads, dim)), t)
    dk, dv, dq, dt = R.on_gpu(k), R.on_gpu(v), R.on_gpu(q), R.on_gpu(table)
    dl, ds = R.on_gpu(np.array([40], np.int32)), R.on_gpu(np.array([0, 40], np.int32))
    dy = R.on_gpu(np.zeros((heads, dim), R.dtype(t)))
    print("a cache past 32 bits", flush=True)
    D.kv_append(dk.addr, dv.addr, cache, dt.addr, 3, dl.addr, 1, 40, starts=ds.addr)
    D.paged_attention(dq.addr, cache, dt.addr, 3, dl.addr, dy.addr, 1, heads, scale=0.125)
    synchronize()
    got = R.values(R.back(dy, R.dtype(t), (heads, dim)), t)
    for h in range(heads):
        y, s, reach = R.attend(R.values(q[:, h], t), R.values(k[:, h], t), R.values(v[:, h], t),
                               np.ones((1, 40), bool), 0.125)
        R.close(got[h:h + 1], y, R.attention_bound(y, s, reach, t, False))


@pytest.mark.parametrize("page", [16, 10])
@pytest.mark.parametrize("work", [0, 1 << 22])
def test_paged_bad_pages(page, work):
    # A seen token in a page that does not exist, or a length past the table, gives NaN in that text alone.
    rng = np.random.default_rng(4)
    lengths = [600, 600, 600, 600, 600]
    p = R.Pages(rng, lengths, page, 1, 64, D.F32)
    p.table[1, 3], p.table[3, 599 // page] = p.pages, -5
    cache = p.upload()
    q = rng.normal(0, 1, (5, 1, 64)).astype(np.float32)
    given = np.array([600, 600, p.width * page + 1, 600, -7], np.int32)
    dq, dl, dy = R.on_gpu(q), R.on_gpu(given), R.on_gpu(np.zeros((5, 64), np.float32))
    dw = R.on_gpu(np.zeros(max(work, 4), np.uint8))
    print(f"paged with bad pages of {page}, work {work}", flush=True)
    D.paged_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 5, 1, scale=0.125,
                      workspace=dw.addr if work else 0, workspace_bytes=work)
    synchronize()
    y = R.back(dy, np.float32, (5, 64))
    assert np.isnan(y[1:4]).all() and np.isfinite(y[0]).all() and not y[4].any()


# ------------------------------------------------------ the prompt attention

def run_prompt(rng, nq, nk, heads, kv_heads, dim, t, window, sinks, fused=False, poison=(), scale=None, odd=0):
    """`fused`: q, k and v in one buffer, a row's behind one another, `odd` values more. `poison`: (text, key) whose k
    and v are NaN."""
    rows_q, rows_k = int(sum(nq)), int(sum(nk))
    scale = 1.2 * dim ** -0.5 if scale is None else scale
    q, k, v = (R.stored(rng.normal(0, s, (n + 3, h, dim)), t)
               for n, h, s in ((rows_q, heads, 2), (rows_k, kv_heads, 1), (rows_k, kv_heads, 1)))
    nan = R.stored(np.full(dim, np.nan, np.float32), t)
    cq, ck = (np.concatenate([[0], np.cumsum(n)]).astype(np.int32) for n in (nq, nk))
    k[rows_k:], v[rows_k:] = nan, nan
    for b, j in poison:
        k[ck[b] + j], v[ck[b] + j] = nan, nan
    y0 = R.stored(np.full((rows_q + 3, heads, dim), 77.0), t)
    dy, dcq, dck = R.on_gpu(y0), R.on_gpu(cq), R.on_gpu(ck)
    print(f"prompt {nq} of {nk} heads {heads}/{kv_heads} dim {dim} type {t} window {window} sinks {sinks} "
          f"fused {fused}", flush=True)
    if fused:
        both = np.concatenate([a.reshape(a.shape[0], -1) for a in (q, k, v)] + [np.zeros((rows_q + 3, odd), R.dtype(t))], 1)
        d, width, size = R.on_gpu(both), both.shape[1], np.dtype(R.dtype(t)).itemsize
        at = [d.addr, d.addr + heads * dim * size, d.addr + (heads + kv_heads) * dim * size]
        strides = dict(q_stride=width, k_stride=width, v_stride=width)
    else:
        d = [R.on_gpu(a) for a in (q, k, v)]
        at, strides = [a.addr for a in d], {}
    D.window_attention(*at, dy.addr, dcq.addr, dck.addr, len(nq), rows_q + 3, rows_k + 3, heads, kv_heads, dim, type=t,
                       scale=scale, window=window, sinks=sinks, **strides)
    synchronize()
    y = R.back(dy, R.dtype(t), y0.shape)
    assert np.array_equal(y[rows_q:].view(np.uint8), y0[rows_q:].view(np.uint8))  # rows behind the last text
    got, per = R.values(y[:rows_q], t), heads // kv_heads
    for b in range(len(nq)):
        seen = R.window_seen(np.arange(nq[b]) + nk[b] - nq[b], nk[b], window, sinks)
        for h in range(heads):
            qh, kh, vh = (R.values(a[c[b]:c[b + 1], i], t) for a, c, i in ((q, cq, h), (k, ck, h // per),
                                                                           (v, ck, h // per)))
            want, size, reach = R.attend(qh, kh, vh, seen, scale)
            R.close(got[cq[b]:cq[b + 1], h], want, R.attention_bound(want, size, reach, t, t != D.F32))


PROMPTS = [([1], [1]), ([80] * 3, [80] * 3), ([5, 0, 64, 1, 33], [5, 0, 64, 1, 33]), ([3, 70, 9], [200, 70, 140]),
           ([130, 20], [40, 7]), ([257], [300])]


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 15), (4, 2, 64), (3, 1, 128), (2, 2, 200), (2, 1, 80)])
@pytest.mark.parametrize("nq,nk", PROMPTS)
def test_prompt(t, heads, kv_heads, dim, nq, nk):
    rng = np.random.default_rng(dim + sum(nq))
    for window, sinks in ((0, 0), (20, 4)):
        run_prompt(rng, nq, nk, heads, kv_heads, dim, t, window, sinks)
    if nq == nk:
        run_prompt(rng, nq, nk, heads, kv_heads, dim, t, 33, 0, fused=True)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 16), (17, 40), (64, 64), (100, 300), (65, 5), (128, 129),
                                          (5000, 2)])
def test_prompt_window(t, window, sinks):
    run_prompt(np.random.default_rng(window), [290, 70], [400, 70], 2, 1, 64, t, window, sinks)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [15, 64])
@pytest.mark.parametrize("window", [0, 31, 200])
def test_prompt_ragged_texts(t, dim, window):
    # Texts of very different lengths, empty ones among them: every block of every text once, in any order.
    rng = np.random.default_rng(17)
    nq = [0, 400, 1, 33, 0, 290, 128, 64, 129, 5, 0]
    run_prompt(rng, nq, [n + i % 3 for i, n in enumerate(nq)], 4, 2, dim, t, window, 3)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("window", [149, 150, 151, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 40])
def test_prompt_window_of_all(t, window):
    # A window as long as the text, or longer, is none.
    rng = np.random.default_rng(12)
    run_prompt(rng, [150, 20], [150, 3], 4, 2, 64, t, window, 0)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [8, 20, 32, 64, 96, 128, 256])
def test_prompt_any_stride(t, dim):
    # Rows that do not start at 16 bytes, and rows that do.
    for odd in (1, 0):
        run_prompt(np.random.default_rng(dim), [100, 40], [100, 40], 4, 2, dim, t, 30, 3, fused=True, odd=odd)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_scales_below_0_and_0(t, scale):
    for dim in (64, 15):
        run_prompt(np.random.default_rng(dim), [70, 5], [70, 9], 2, 1, dim, t, 20, 2, scale=scale)
    run_paged(np.random.default_rng(3), [90, 1, 0], 16, 2, 1, 64, t, scale=scale)
    run_paged(np.random.default_rng(3), [90, 1, 0], 16, 2, 1, 64, t, 20, 2, scale=scale)


def test_prompt_many_texts():
    # More texts than a wave has lanes, some of them empty.
    rng = np.random.default_rng(7)
    nq = rng.integers(0, 9, 200).tolist()
    run_prompt(rng, nq, nq, 2, 1, 64, D.F16, 4, 1)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [64, 128, 30])
def test_prompt_nan_in_unseen_keys(t, dim):
    # A NaN key reaches the queries that see it and no others, also inside a tile.
    for window, sinks, at in ((0, 0, 150), (40, 3, 37), (40, 3, 1), (9, 0, 260)):
        run_prompt(np.random.default_rng(at), [290, 40], [290, 40], 2, 1, dim, t, window, sinks, poison=[(0, at), (1, 20)])


# --------------------------------------------------- a run of them, and graphs

class Step:
    """One step of a decoder block on the GPU: norm in 8 bits, q | k | v by a
    4-bit product, append, attention, an output product, the next norm."""

    def __init__(self, rng, batch=3, held=70, heads=4, kv=2, dim=32, t=D.BF16, width=160):
        self.a = dict(batch=batch, heads=heads, kv=kv, dim=dim, t=t, width=width)
        self.wide = (heads + 2 * kv) * dim
        self.lengths = np.array([held + 9 * b for b in range(batch)], np.int32)
        self.pages = R.Pages(rng, list(self.lengths + 8), 16, kv, dim, t)
        self.cache = self.pages.upload()
        up = R.on_gpu
        self.x, self.res = rng.normal(0, 1, (batch, width)), rng.normal(0, 1, (batch, width))
        self.dx, self.dres = up(R.stored(self.x, t)), up(R.stored(self.res, t))
        self.w1, self.w2 = R.stored(rng.normal(1, 0.1, width), t), R.stored(rng.normal(1, 0.1, width), t)
        self.dw1, self.dw2 = up(self.w1), up(self.w2)
        self.q1, self.q2 = rng.integers(0, 16, (self.wide, width)), rng.integers(0, 16, (width, heads * dim))
        self.s1 = (rng.uniform(0.5, 1.5, (self.wide, 5)) / 60).astype(np.float32)
        self.s2 = (rng.uniform(0.5, 1.5, (width, 4)) / 60).astype(np.float32)
        self.dq1, self.dq2, self.ds1, self.ds2 = up(R.packed(self.q1)), up(R.packed(self.q2)), up(self.s1), up(self.s2)
        zeros = lambda *s, t=t: up(np.zeros(s, R.dtype(t)))  # noqa: E731
        self.y8, self.sc = zeros(batch, width, t=D.E4M3), up(np.zeros((batch, 5), np.float32))
        self.h, self.qkv, self.o = zeros(batch, width), zeros(batch, self.wide), zeros(batch, heads * dim)
        self.p, self.y = zeros(batch, width), zeros(batch, width)
        self.h2 = zeros(batch, width)
        self.dl = up(self.lengths)
        self.work = up(np.zeros(1 << 20, np.uint8))

    def run(self, stream=0):
        a, s = self.a, dict(stream=stream)
        n, t, kv, dim, heads, width = a["batch"], a["t"], a["kv"], a["dim"], a["heads"], a["width"]
        D.rms_norm(self.dx.addr, self.dw1.addr, self.y8.addr, n, width, residual=self.dres.addr, sum=self.h.addr,
                   scales=self.sc.addr, type=t, y_type=D.E4M3, group=32, **s)
        D.q4_product(self.y8.addr, self.dq1.addr, self.ds1.addr, self.qkv.addr, n, self.wide, width, group=32,
                     x_scales=self.sc.addr, x_group=32, x_type=D.E4M3, scale_type=D.F32, y_type=t, **s)
        k = self.qkv.addr + 2 * heads * dim
        D.kv_append(k, k + 2 * kv * dim, self.cache, self.pages.gpu_table.addr, self.pages.width, self.dl.addr, n, n,
                    k_stride=self.wide, v_stride=self.wide, **s)
        D.paged_attention(self.qkv.addr, self.cache, self.pages.gpu_table.addr, self.pages.width, self.dl.addr,
                          self.o.addr, n, heads, scale=dim ** -0.5, q_stride=self.wide, workspace=self.work.addr,
                          workspace_bytes=1 << 20, **s)
        D.q4_product(self.o.addr, self.dq2.addr, self.ds2.addr, self.p.addr, n, width, heads * dim, group=32, x_type=t,
                     scale_type=D.F32, y_type=t, **s)
        D.rms_norm(self.p.addr, self.dw2.addr, self.y.addr, n, width, residual=self.h.addr, sum=self.h2.addr, type=t, **s)

    def outputs(self):
        a = self.a
        return [R.back(d, R.dtype(a["t"]), s).copy() for d, s in
                ((self.qkv, (a["batch"], self.wide)), (self.o, (a["batch"], a["heads"] * a["dim"])),
                 (self.y, (a["batch"], a["width"])), (self.pages.gpu[0], self.pages.host[0].shape))]

    def check(self):
        """Each layer's output against 64 bits on the layer's own stored inputs."""
        a = self.a
        n, t, kv, dim, heads, width = a["batch"], a["t"], a["kv"], a["dim"], a["heads"], a["width"]
        qkv, o, y, _ = self.outputs()
        _, yv = R.norm(self.x, self.res, R.values(self.w1, t), t, 1e-6)
        y8 = R.values(R.back(self.y8, np.uint8, (n, width)), D.E4M3)
        sc = np.repeat(R.back(self.sc, np.float32, (n, 5)).astype(np.float64), 32, 1)[:, :width]
        R.close(y8 * sc, yv, np.maximum(np.abs(yv) / 16, sc * 2.0 ** -10) * 1.001)
        want, size = R.product(y8 * sc, self.q1, self.s1.astype(np.float64), None, 32)
        R.close(R.values(qkv, t), want, R.half_step(want, t) + 16 * STEP * size)
        for b in range(n):
            length = int(self.lengths[b])
            new = qkv[b, heads * dim:].reshape(2, kv, dim)
            k, v = self.pages.k[b][:length].copy(), self.pages.v[b][:length].copy()
            k[-1], v[-1] = new
            for h in range(heads):
                q = R.values(qkv[b, h * dim:(h + 1) * dim], t)[None]
                g = h // (heads // kv)
                w, s, reach = R.attend(q, R.values(k[:, g], t), R.values(v[:, g], t), np.ones((1, length), bool),
                                       dim ** -0.5)
                R.close(R.values(o[b, h * dim:(h + 1) * dim], t)[None], w, R.attention_bound(w, s, reach, t, False))
        p = R.values(R.back(self.p, R.dtype(t), (n, width)), t)
        want, size = R.product(R.values(o, t), self.q2, self.s2.astype(np.float64), None, 32)
        R.close(p, want, R.half_step(want, t) + 16 * STEP * size)
        h = R.values(R.back(self.h, R.dtype(t), (n, width)), t)
        _, want = R.norm(p, h, R.values(self.w2, t), t, 1e-6)
        R.close(R.values(y, t), want, R.half_step(want, t) + np.abs(want) * 12 * STEP)


@pytest.mark.parametrize("t", [D.BF16, D.F16])
def test_a_step_of_a_block(t):
    step = Step(np.random.default_rng(8), t=t)
    print("a step of a decoder block", flush=True)
    step.run()
    synchronize()
    step.check()


def _stream():
    s = C.c_void_p()
    assert hip().hipStreamCreate(C.byref(s)) == 0
    return s


class Graph:
    """What `make` queues on `stream`, captured."""

    def __init__(self, stream, make):
        h = hip()
        graph, self.exec = C.c_void_p(), C.c_void_p()
        assert h.hipStreamBeginCapture(stream, 2) == 0
        try:
            make()
        finally:
            rc = h.hipStreamEndCapture(stream, C.byref(graph))
        assert rc == 0
        h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
        h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
        assert h.hipGraphInstantiate(C.byref(self.exec), graph, None, None, 0) == 0
        self.stream = stream

    def launch(self):
        assert hip().hipGraphLaunch(self.exec, self.stream) == 0


def test_a_step_captured():
    # A captured step, replayed while the texts grow: as the eager calls, bit for bit, each time.
    s = _stream()
    a, b = Step(np.random.default_rng(9)), Step(np.random.default_rng(9))
    a.run(s.value)  # eager once before the capture
    synchronize()
    a.check()
    g = Graph(s, lambda: a.run(s.value))
    b.run()
    for i in range(4):
        for step in (a, b):
            step.lengths += 1
            step.dl.upload(step.lengths)
        print(f"captured step, replay {i}", flush=True)
        g.launch()
        synchronize()
        b.run()
        synchronize()
        for x, y in zip(a.outputs(), b.outputs()):
            assert np.array_equal(x.view(np.uint8), y.view(np.uint8))


def test_two_threads_at_once():
    # Calls and refusals from two threads: each its own results and reasons.
    import threading
    steps, said = [Step(np.random.default_rng(40 + i), held=100 + 200 * i) for i in range(2)], [[], []]

    def work(i):
        for n in range(20):
            steps[i].run()
            try:
                D.q4_product(16, 16, 16, 16, 1, 1, 1, group=1000 + i)
            except Exception as e:
                said[i].append(str(e))

    print("two threads", flush=True)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    synchronize()
    for i in range(2):
        steps[i].check()
        assert len(said[i]) == 20 and all(f"groups of {1000 + i} " in s for s in said[i])


def test_two_streams_at_once():
    # The same steps on two streams, each with its own buffers, give what they give alone.
    s = [_stream(), _stream()]
    steps = [Step(np.random.default_rng(20 + i), held=500 + 300 * i) for i in range(2)]
    print("two streams", flush=True)
    for _ in range(5):
        for one, at in zip(steps, s):
            one.run(at.value)
    synchronize()
    got = [one.outputs() for one in steps]
    for one, outs in zip(steps, got):
        one.run()
        synchronize()
        one.check()
        for x, y in zip(outs, one.outputs()):
            assert np.array_equal(x.view(np.uint8), y.view(np.uint8))


def test_after_another_calls_error():
    # What another call of the thread's failed at is not these calls' failure.
    step = Step(np.random.default_rng(31))
    print("after an error", flush=True)
    assert hip().hipSetDevice(10 ** 6) != 0
    step.run()
    synchronize()
    step.check()
    hip().hipGetLastError()
