"""The decoder layers on the GPU where numbers or shapes are at an edge: weights
far below the largest, infinities that are seen, sums that leave f32's range,
codes next to a rounding's border, tiles and heads of every kernel, a first
call inside a capture."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import decoder_plain as R
from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import synchronize
from test_gpu_decoder import run_product, run_prompt

pytestmark = pytest.mark.gpu
STEP = R.STEP


# ------------------------------------------- attention: given keys and values

def paged(q, k, v, t, scale, kv_heads=1, page=16, work=1 << 20):
    """q [heads][dim] of one text, k and v [keys][kv heads][dim], stored -> y [heads][dim] as float64."""
    heads, dim = q.shape
    n = k.shape[0]
    p = R.Pages(np.random.default_rng(1), [n], page, kv_heads, dim, t)
    for i in range(n):
        p.put(0, i, k[i], v[i])
    cache = p.upload()
    dq, dl, dy = R.on_gpu(q), R.on_gpu(np.array([n], np.int32)), R.on_gpu(np.zeros((heads, dim), R.dtype(t)))
    dw = R.on_gpu(np.zeros(max(work, 4), np.uint8))
    print(f"paged {n} keys, {heads}/{kv_heads} heads of {dim}, type {t}, work {work}", flush=True)
    D.paged_attention(dq.addr, cache, p.gpu_table.addr, p.width, dl.addr, dy.addr, 1, heads, scale=scale,
                      workspace=dw.addr if work else 0, workspace_bytes=work)
    synchronize()
    return R.values(R.back(dy, R.dtype(t), (heads, dim)), t)


def prompt(q, k, v, t, scale, odd=0, window=0, sinks=0):
    """q [rows][heads][dim], k and v [rows][1][dim] of one text, stored; rows of k and v `odd` values apart (1: the
    kernel that takes any address) -> y as float64."""
    rows, heads, dim = q.shape
    wide = lambda a: R.on_gpu(np.concatenate([a.reshape(len(a), -1), np.zeros((len(a), odd), a.dtype)], 1))  # noqa: E731
    dq, dk, dv, dy = R.on_gpu(q), wide(k), wide(v), R.on_gpu(np.zeros(q.shape, R.dtype(t)))
    ds, dt = R.on_gpu(np.array([0, rows], np.int32)), R.on_gpu(np.array([0, len(k)], np.int32))
    print(f"prompt {rows} of {len(k)} keys, {heads} heads of {dim}, type {t}, odd {odd}", flush=True)
    D.window_attention(dq.addr, dk.addr, dv.addr, dy.addr, ds.addr, dt.addr, 1, rows, len(k), heads, 1, dim,
                       type=t, scale=scale, window=window, sinks=sinks, k_stride=dim + odd, v_stride=dim + odd)
    synchronize()
    return R.values(R.back(dy, R.dtype(t), q.shape), t)


# --------------------------------------- one key far ahead of all the others

def far_ahead(t, dim, heads, keys):
    """Keys 1, 2, ... at the same score, key 0 between 13 and 18.3 nats ahead of them (another distance a head), its
    value 0: what comes out is the others' alone."""
    rng = np.random.default_rng(dim)
    q = np.zeros((heads, dim))
    q[:, 3] = np.linspace(13, 18.3, heads)
    k = np.zeros((keys, 1, dim))
    k[0, 0, 3] = 1.0
    v = rng.uniform(500, 1500, (keys, 1, dim))
    v[0] = 0
    return tuple(R.stored(a, t) for a in (q, k, v))


# F16's smallest step is 2^-24: a weight that goes into the product as F16 is off by up to 2^-25 of the unit it is
# held in. The decode attention's unit is 2^-14 of the row's largest weight, the prompt attention's 2^-13 of a
# reference that the largest is at most 2^2 above (so never more than 2^-13 of the largest): 2^-39 and 2^-38 of the
# largest, which the sum of weights is not below.
LEAST_DECODE, LEAST_PROMPT = 2.0 ** -39, 2.0 ** -38


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [64, 128, 80, 30])
@pytest.mark.parametrize("work", [0, 1 << 20])
def test_decode_of_small_weights(t, dim, work):
    q, k, v = far_ahead(t, dim, 8, 2000)
    got = paged(q, k, v, t, 1.0, work=work)
    qv, kv, vv = R.values(q, t), R.values(k, t)[:, 0], R.values(v, t)[:, 0]
    y, size, reach = R.attend(qv, kv, vv, np.ones((8, 2000), bool), 1.0)
    least = LEAST_DECODE * np.abs(vv).sum(0)[None] if t == D.F16 else 0
    R.close(got, y, R.attention_bound(y, size, reach, t, False) + least)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [64, 128, 96, 30])
@pytest.mark.parametrize("odd", [0, 1])
def test_prompt_of_small_weights(t, dim, odd):
    # Every query sees key 0 and all before it: the one ahead comes in the first tile.
    q1, k, v = far_ahead(t, dim, 4, 700)
    q = np.repeat(q1[None], 700, 0)
    got = prompt(q, k, v, t, 1.0, odd)
    seen = R.window_seen(np.arange(700), 700, 0, 0)
    kv, vv = R.values(k, t)[:, 0], R.values(v, t)[:, 0]
    sums = np.cumsum(np.abs(vv), 0)
    for h in range(4):
        y, size, reach = R.attend(R.values(q[:, h], t), kv, vv, seen, 1.0)
        least = LEAST_PROMPT * (sums + np.arange(1, 701)[:, None] * np.abs(y)) if t == D.F16 else 0
        R.close(got[:, h], y, R.attention_bound(y, size, reach, t, t != D.F32) + least)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("odd", [0, 1])
def test_prompt_of_growing_scores(t, odd):
    # Scores that rise by a little from key to key: the running maximum follows in steps, in every tile.
    rng = np.random.default_rng(3)
    keys, dim = 600, 64
    q, k = np.zeros((keys, 2, dim)), np.zeros((keys, 1, dim))
    q[:, 0, 5], q[:, 1, 5] = 1.0, -1.0
    k[:, 0, 5] = np.arange(keys) * 0.02
    q, k, v = R.stored(q, t), R.stored(k, t), R.stored(rng.normal(0, 1, (keys, 1, dim)), t)
    got = prompt(q, k, v, t, 1.0, odd)
    seen = R.window_seen(np.arange(keys), keys, 0, 0)
    kv, vv = R.values(k, t)[:, 0], R.values(v, t)[:, 0]
    for h in range(2):
        y, size, reach = R.attend(R.values(q[:, h], t), kv, vv, seen, 1.0)
        least = LEAST_PROMPT * np.cumsum(np.abs(vv) + np.abs(y), 0) if t == D.F16 else 0
        R.close(got[:, h], y, R.attention_bound(y, size, reach, t, t != D.F32) + least)


# ---------------------------------------------- infinities in values that are seen

def with_infinities(v, t, at):
    """Infinities in values `at` and behind: columns that come out as inf, -inf, and NaN (both, or a NaN)."""
    v = np.asarray(R.values(v, t), np.float32)
    n = len(v)
    for i, d, x in ((0, 1, np.inf), (0, 2, -np.inf), (3, 2, -np.inf), (5, 7, np.inf), (6, 7, -np.inf), (2, 9, np.nan)):
        if at + i < n:
            v[at + i, 0, d] = x
    return R.stored(v, t)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [64, 128, 80, 30])
@pytest.mark.parametrize("keys,at,work", [(1, 0, 0), (40, 10, 0), (70, 68, 0), (3000, 1700, 0), (3000, 1700, 1 << 20)])
def test_decode_of_infinities(t, dim, keys, at, work):
    rng = np.random.default_rng(keys)
    q, k = R.stored(rng.normal(0, 2, (4, dim)), t), R.stored(rng.normal(0, 1, (keys, 1, dim)), t)
    v = with_infinities(R.stored(rng.normal(0, 1, (keys, 1, dim)), t), t, at)
    got = paged(q, k, v, t, dim ** -0.5, work=work)
    with np.errstate(invalid="ignore"):
        y, size, reach = R.attend(R.values(q, t), R.values(k, t)[:, 0], R.values(v, t)[:, 0],
                                  np.ones((4, keys), bool), dim ** -0.5)
        assert np.isinf(y[:, 1]).all() and np.isinf(y[:, 2]).all()
        R.close(got, y, R.attention_bound(y, size, reach, t, False))


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [64, 128, 96, 30])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("window,sinks,at", [(0, 0, 0), (0, 0, 100), (30, 4, 2), (30, 4, 100), (200, 0, 30)])
def test_prompt_of_infinities(t, dim, odd, window, sinks, at):
    rng = np.random.default_rng(at + dim)
    rows = 290
    q, k = R.stored(rng.normal(0, 2, (rows, 2, dim)), t), R.stored(rng.normal(0, 1, (rows, 1, dim)), t)
    v = with_infinities(R.stored(rng.normal(0, 1, (rows, 1, dim)), t), t, at)
    got = prompt(q, k, v, t, dim ** -0.5, odd, window, sinks)
    seen = R.window_seen(np.arange(rows), rows, window, sinks)
    with np.errstate(invalid="ignore"):
        for h in range(2):
            y, size, reach = R.attend(R.values(q[:, h], t), R.values(k, t)[:, 0], R.values(v, t)[:, 0], seen,
                                      dim ** -0.5)
            assert np.isinf(y).any() and np.isfinite(y).any()
            R.close(got[:, h], y, R.attention_bound(y, size, reach, t, t != D.F32))


# -------------------------------------------------- products of very large numbers

@pytest.mark.parametrize("t", [D.F32, D.BF16, D.F16])
@pytest.mark.parametrize("m,n,k,group,zeros", [(1, 40, 256, 128, False), (5, 100, 300, 32, True),
                                               (17, 33, 1030, 64, True), (3, 9001, 640, 128, False)])
def test_product_of_large_x(t, m, n, k, group, zeros):
    # Groups of like signs whose sums of x (16 + q) pass f32's largest where those of x (q - z) do not, values that
    # round past bf16's largest, and beside them ordinary rows, and rows with an infinity or NaN.
    rng = np.random.default_rng(n)
    x = rng.normal(0, 1, (m, k))
    big = 3.0e38 if t == D.BF16 else 65504.0 if t == D.F16 else 3.4e38
    x[0] = rng.uniform(0.2, 0.9, k) * big
    if m > 2:
        x[2, 3], x[2, k - 1] = big, -big
    if m > 4:
        x[3, 7], x[4, k // 2] = np.inf, np.nan
    raw = R.stored(x, t)
    groups = -(-k // group)
    q, s = rng.integers(0, 16, (n, k)), R.stored(rng.uniform(0.5, 1.5, (n, groups)) / 2 ** 14, D.F32)
    z = rng.integers(0, 16, (n, groups)).astype(np.uint8) if zeros else None
    b = R.stored(rng.normal(0, 1, n), t)
    dx, dq, ds, db = (R.on_gpu(a) for a in (raw, R.packed(q), s, b))
    dz = R.on_gpu(z) if zeros else None
    dy = R.on_gpu(np.zeros((m, n), R.dtype(t)))
    print(f"product of large x {m}x{k}->{n} type {t}", flush=True)
    D.q4_product(dx.addr, dq.addr, ds.addr, dy.addr, m, n, k, group=group, zeros=dz.addr if zeros else 0,
                 bias=db.addr, x_type=t, scale_type=D.F32, y_type=t)
    synchronize()
    got = R.values(R.back(dy, R.dtype(t), (m, n)), t)
    rows = [i for i in range(m) if i not in (3, 4)] if m > 4 else list(range(m))
    want, size = R.product(R.values(raw, t)[rows], q, s.astype(np.float64), z, group)
    want = want + R.values(b, t)
    assert np.abs(want).max() < R.values(R.stored([big], t), t)[0]  # all of it can be told
    R.close(got[rows], want, R.half_step(want, t) + 16 * STEP * size)
    if m > 4:
        assert np.isnan(got[3:5]).all()


def test_product_that_overflows():
    # A sum past f32's largest is an infinity.
    x, q = np.full((2, 64), 3e38, np.float32), np.full((20, 64), 15)
    x[1] = 1
    q[::2] = 0
    s = np.full((20, 2), 1, np.float32)
    dx, dq, ds, dy = R.on_gpu(x), R.on_gpu(R.packed(q)), R.on_gpu(s), R.on_gpu(np.zeros((2, 20), np.float32))
    print("product that overflows", flush=True)
    D.q4_product(dx.addr, dq.addr, ds.addr, dy.addr, 2, 20, 64, group=32)
    synchronize()
    y = R.back(dy, np.float32, (2, 20))
    assert (y[0, ::2] == -np.inf).all() and (y[0, 1::2] == np.inf).all()
    assert (y[1, ::2] == -512).all() and (y[1, 1::2] == 448).all()


# ------------------------------------------------------ codes of 8 bits of the norm

@pytest.mark.parametrize("y_type", [D.E4M3, D.I8])
@pytest.mark.parametrize("rows,c,group", [(64, 16384, 0), (64, 16384, 128), (3, 40000, 0), (500, 2000, 32)])
def test_norm_codes_are_the_nearest(y_type, rows, c, group):
    # The same norm in F32 tells y. A scale is max |y| times 1 / 448 (127): two roundings, of half a step each, so at
    # most 2^-23 (1 + 2^-24) off. A code is that of y / scale, which is rounded to f32 once before: next to a code's
    # border it may fall to the other side by half a step of f32.
    rng = np.random.default_rng(c)
    x, w = rng.normal(0, 1, (rows, c)).astype(np.float32), rng.normal(1, 0.2, c).astype(np.float32)
    groups, size, top = -(-c // group) if group else 1, group or c, 448.0 if y_type == D.E4M3 else 127.0
    dx, dw, dy = R.on_gpu(x), R.on_gpu(w), R.on_gpu(np.zeros((rows, c), np.float32))
    d8, ds = R.on_gpu(np.zeros((rows, c), np.uint8)), R.on_gpu(np.zeros((rows, groups), np.float32))
    print(f"norm codes {rows}x{c} type {y_type} group {group}", flush=True)
    D.rms_norm(dx.addr, dw.addr, dy.addr, rows, c)
    D.rms_norm(dx.addr, dw.addr, d8.addr, rows, c, scales=ds.addr, y_type=y_type, group=group)
    synchronize()
    y = R.back(dy, np.float32, (rows, c)).astype(np.float64)
    s = R.back(ds, np.float32, (rows, groups))
    most = np.stack([np.abs(y[:, i:i + size]).max(1) for i in range(0, c, size)], 1)
    assert int((np.abs(s - most / top) > most / top * STEP * (1 + STEP / 2)).sum()) == 0
    quotient = y / np.repeat(s.astype(np.float64), size, 1)[:, :c]
    step = np.ones_like(quotient)
    if y_type == D.E4M3:
        step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(quotient), 1e-30))), -6) - 3)
    got = R.values(R.back(d8, np.uint8, (rows, c)), y_type)
    assert int((np.abs(got - quotient) > step / 2 + np.abs(quotient) * STEP / 2).sum()) == 0


# ------------------------------------------------ the product's kernels of several tiles

# Tiles a workgroup takes: 2 and 4 of each type of x, 8 of f32 (test_decoder_tiles.py holds these sizes to that);
# last strips that are cut; rows of weights of 16-, 4- and 1-byte alignment; more blocks of rows than one.
TILES = [(1, 6000, 520, 32), (5, 9003, 640, 64), (16, 17001, 1030, 128), (17, 8215, 530, 32), (40, 6001, 513, 64),
         (3, 40005, 600, 32), (16, 17000, 1088, 32), (9, 17100, 576, 128), (2, 17500, 520, 64)]


@pytest.mark.parametrize("x_type", [D.F32, D.BF16, D.F16, D.E4M3, D.I8])
@pytest.mark.parametrize("m,n,k,group", TILES)
def test_product_of_several_tiles(x_type, m, n, k, group):
    y_type = x_type if x_type in R.REAL else D.BF16
    run_product(np.random.default_rng(n), m, n, k, group, x_type, D.F32 if group == 64 else D.F16, y_type, group != 64,
                group == 128, x_group=group if x_type not in R.REAL and m % 2 else 0, gap=3 if group == 32 else 0)


# ------------------------------- the prompt attention's heads side by side, and head sizes

HEADS = [(4, 1), (8, 2), (8, 1), (6, 1), (7, 1)]  # four, two or one of a key head's in a workgroup


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv_heads", HEADS)
@pytest.mark.parametrize("nq,nk", [([1], [1]), ([5, 0, 64, 1, 33], [5, 0, 64, 1, 33]), ([3, 70, 9], [200, 70, 140]),
                                   ([130, 20], [40, 7]), ([257], [300])])
def test_prompt_heads(t, heads, kv_heads, nq, nk):
    for window, sinks in ((0, 0), (20, 4)):
        run_prompt(np.random.default_rng(heads), nq, nk, heads, kv_heads, 64, t, window, sinks)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("dim", [40, 104, 128, 136, 160, 192, 256])
def test_prompt_dims(t, dim):
    # Head sizes in the kernels for those up to 64, 96, 128, 192 and 256, four query heads to a key head.
    rng = np.random.default_rng(dim)
    run_prompt(rng, [150, 0, 33], [150, 4, 60], 4, 1, dim, t, 0, 0)
    run_prompt(rng, [150, 0, 33], [150, 4, 60], 4, 1, dim, t, 50, 3)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 40), (64, 64), (100, 300), (128, 129), (5000, 2)])
def test_prompt_heads_window(t, window, sinks):
    run_prompt(np.random.default_rng(window), [290, 70], [400, 70], 4, 1, 64, t, window, sinks)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("window", [0, 31, 200])
def test_prompt_heads_ragged_texts(t, window):
    nq = [0, 400, 1, 33, 0, 290, 128, 64, 31, 5, 0]
    run_prompt(np.random.default_rng(18), nq, [n + i % 3 for i, n in enumerate(nq)], 4, 1, 64, t, window, 3)


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 64), (8, 1, 128), (6, 1, 192), (4, 1, 96)])
def test_prompt_heads_nan_in_unseen_keys(t, heads, kv_heads, dim):
    for window, sinks, at in ((0, 0, 150), (40, 3, 1), (9, 0, 260)):
        run_prompt(np.random.default_rng(at), [290, 40], [290, 40], heads, kv_heads, dim, t, window, sinks,
                   poison=[(0, at), (1, 20)])


# ------------------------------------------------------------ a first call inside a capture

FIRST = """
import ctypes as C
import conftest
import numpy as np
import decoder_plain as R
import test_gpu_decoder as T
from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import hip, synchronize

t, rows, heads, dim = D.BF16, 150, 4, 64
rng = np.random.default_rng(2)
steps = [T.Step(np.random.default_rng(9), t=t) for _ in range(2)]
q, k, v = (R.on_gpu(R.stored(rng.normal(0, 1, (rows, h, dim)), t)) for h in (heads, 1, 1))
y = [R.on_gpu(np.zeros((rows, heads, dim), np.uint16)) for _ in range(2)]
starts = R.on_gpu(np.array([0, rows], np.int32))


def run(i, stream):
    steps[i].run(stream)
    D.window_attention(q.addr, k.addr, v.addr, y[i].addr, starts.addr, starts.addr, 1, rows, rows, heads, 1, dim,
                       scale=0.125, type=t, stream=stream)


h = hip()
stream, graph, ready = T._stream(), C.c_void_p(), C.c_void_p()
assert h.hipStreamBeginCapture(stream, 0) == 0  # the global mode: nothing unsafe in any thread
run(0, stream.value)
assert h.hipStreamEndCapture(stream, C.byref(graph)) == 0
h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
assert h.hipGraphInstantiate(C.byref(ready), graph, None, None, 0) == 0
for i in range(3):
    assert h.hipGraphLaunch(ready, stream) == 0
    synchronize()
    run(1, 0)
    synchronize()
    steps[0].check()
    for a, b in zip(steps[0].outputs() + [R.back(y[0], np.uint16, (rows, heads, dim))],
                    steps[1].outputs() + [R.back(y[1], np.uint16, (rows, heads, dim))]):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    print("replay", i, flush=True)
print("the same", flush=True)
"""


def test_first_calls_inside_a_capture():
    # In a process of its own, whose first calls of these layers are captured.
    print("first calls inside a capture", flush=True)
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=Path(__file__).parent, capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("the same\n"), (r.returncode, r.stdout[-500:], r.stderr[-2000:])
