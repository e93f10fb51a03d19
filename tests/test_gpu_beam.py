"""Beam search on the GPU: the choice against 64 bits, the reordering against
plain steps, byte by byte; and a whole search that writes with the 4-bit cache."""
import numpy as np
import pytest

import beam_plain as B
import decoder_plain as R
import writer_plain as W
from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import DeviceArray, synchronize

pytestmark = pytest.mark.gpu
STEP = R.STEP


class Select:
    """One call's buffers, with guards behind every output."""

    def __init__(self, x, base, keep, t, ended=None, end=-1, gap=0):
        self.batch, self.beams, self.vocab = x.shape
        self.keep, self.t, self.end = keep, t, end
        self.x = R.stored(np.concatenate([x, np.full(x.shape[:2] + (gap,), 1e4)], -1), t)
        self.base, self.ended = np.asarray(base, np.float32), ended
        self.stride = self.vocab + gap
        self.dx, self.db = R.on_gpu(self.x), R.on_gpu(self.base)
        self.de = None if ended is None else R.on_gpu(np.asarray(ended, np.uint8))
        n = (self.batch, keep)
        self.out = [R.on_gpu(np.full(n, 7, d)) for d in (np.float32, np.int32, np.int32, np.uint8)]
        self.bytes = D.beam_select_workspace(self.batch, self.beams, self.vocab, keep)
        self.work = R.on_gpu(np.full(self.bytes, 0xFF, np.uint8))

    def run(self, stream=0):
        print(f"select {self.keep} of {self.batch} x {self.beams} x {self.vocab}, type {self.t}, ended "
              f"{self.ended is not None}", flush=True)
        D.beam_select(self.dx.addr, self.db.addr, *(o.addr for o in self.out[:3]), self.batch, self.beams, self.vocab,
                      self.keep, type=self.t, ended=0 if self.de is None else self.de.addr, out_ended=self.out[3].addr,
                      end=self.end, stride=self.stride, workspace=self.work.addr, workspace_bytes=self.bytes, stream=stream)

    def outputs(self):
        R.back(self.work, np.uint8, (self.bytes,))
        return [R.back(o, d, (self.batch, self.keep)) for o, d in zip(self.out, (np.float32, np.int32, np.int32, np.uint8))]

    def check(self):
        got = self.outputs()
        for b in range(self.batch):
            x = R.values(self.x[b, :, :self.vocab], self.t)
            want, near = B.choose(x, self.base[b].astype(np.float64), self.keep,
                                  None if self.ended is None else self.ended[b], self.end)
            # Sums of f32 exponentials are off by 16 steps at most, and so is their logarithm: scores of one beam keep
            # their distances exactly, those of two beams are apart by more than twice that (as the inputs are made), or equal.
            score = got[0][b].astype(np.float64)
            R.close(score, want[0], np.abs(want[0]) * STEP / 2 + 17 * STEP)
            for j in range(1, 4):
                assert np.array_equal(got[j][b], want[j]), (j, got[j][b], want[j], want[0])
        return got


SIZES = [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 50, 3), (1, 4, 18385, 4), (3, 2, 2049, 7), (2, 8, 8191, 8), (1, 5, 8193, 16),
         (2, 1, 40000, 33), (1, 32, 3000, 32), (5, 4, 333, 64), (1, 128, 700, 128), (2, 7, 100000, 5), (40, 3, 1000, 6),
         (700, 2, 9000, 4), (1, 2, 7, 40)]


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("batch,beams,vocab,keep", SIZES)
def test_select(t, batch, beams, vocab, keep):
    rng = np.random.default_rng(vocab + keep)
    for ended, gap in ((False, 0), (True, 3)):
        x = rng.normal(0, 2, (batch, beams, vocab))
        base = -rng.uniform(0, 6, (batch, beams))
        e = rng.random((batch, beams)) < 0.4 if ended else None
        s = Select(x, base, keep, t, e, vocab // 2 if ended else -1, gap)
        s.run()
        synchronize()
        s.check()


@pytest.mark.parametrize("t", R.REAL)
def test_select_ties(t):
    # Equal logits, in one beam and over beams: the lower beam, then the lower token.
    rng = np.random.default_rng(1)
    for vocab, keep in ((100, 10), (9000, 128), (40000, 20)):
        x = np.round(rng.normal(0, 1, (2, 3, vocab)))
        x[0] = 0  # nothing but ties
        x[1, 2] = x[1, 1]
        base = np.array([[-1, -1, -1], [-2, -1, -1]])
        s = Select(x, base, keep, t)
        s.run()
        synchronize()
        s.check()
    x = np.zeros((1, 2, 3000))
    x[0, :, ::2] = -0.0  # 0 and -0 are one number
    s = Select(x, np.zeros((1, 2)), 9, t)
    s.run()
    synchronize()
    s.check()


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("keep", [1, 8, 128])
def test_select_of_sorted_logits(t, keep):
    # Sorted logits, where a part's first bound leaves most of it: the bound is halved in on. Rising, falling, and few
    # values many times.
    for vocab in (8192, 30000):
        up = np.arange(vocab) * (8.0 / vocab)
        for x in (up, up[::-1], np.floor(up * 4) / 4, np.where(np.arange(vocab) % 256 < 224, 1.0, 0.0)):
            s = Select(np.stack([x, x - 1])[None].copy(), np.array([[0.0, -3.0]]), keep, t)
            s.run()
            synchronize()
            s.check()


def test_select_among_many_equal_choices():
    # More equal candidates than a workgroup lists, by scores alone and at one score: beams of low and of high first
    # parts, so that the groups' least is low.
    for low in (0.0, 6.0):
        x = np.full((1, 32, 160000), 6.0, np.float32)
        x[0, :, :10000] = low
        x[0, 3, 20000:20010] = 6.5
        s = Select(x, np.zeros((1, 32)), 128, D.F32)
        s.run()
        synchronize()
        s.check()
    rng = np.random.default_rng(4)
    x = rng.normal(0, 1, (1, 32, 160000)).astype(np.float32)
    x[0, :, :10000] -= 20
    s = Select(x, np.zeros((1, 32)), 128, D.F32)
    s.run()
    synchronize()
    s.check()


@pytest.mark.parametrize("t", R.REAL)
def test_select_of_what_is_not_finite(t):
    # Forbidden tokens (-infinity, or the type's lowest value), rows of nothing else, infinities, NaN, dead beams.
    rng = np.random.default_rng(2)
    vocab, keep = 5000, 12
    lowest = {D.F32: -3.4028234663852886e38, D.BF16: -3.3895313892515355e38, D.F16: -65504.0}[t]
    x = rng.normal(0, 2, (8, 4, vocab))
    base = -rng.uniform(0, 3, (8, 4))
    x[0, :, 7:] = -np.inf              # 28 tokens left
    x[1, :, 2:] = -np.inf              # 8 left, fewer than are kept
    x[2] = -np.inf                     # none
    x[3, 1, 40], x[3, 2, 4999], x[3, 0, 0] = np.inf, np.nan, -np.inf
    base[4] = -np.inf                  # no beam is alive
    base[5, 1:] = -np.inf              # a first step
    x[6, :, 3:] = lowest               # the lowest value is a number: kept after the others
    base[7, 0], base[7, 1] = np.nan, 0.0
    s = Select(x, base, keep, t)
    s.run()
    synchronize()
    got = s.check()
    assert (got[2][2] == -1).all() and (got[2][4] == -1).all() and (got[1][5] == 0).all()
    assert (got[2][1][8:] == -1).all() and (got[1][1][8:] == 3).all()
    assert (got[1][3] != 1).all() and (got[1][3] != 2).all()
    # All beams ended: each goes on with the end token, and nothing else.
    s = Select(x[:1], base[:1], 6, t, ended=np.ones((1, 4), np.uint8), end=11)
    s.run()
    synchronize()
    got = s.check()
    assert sorted(got[1][0][:4]) == [0, 1, 2, 3] and (got[2][0][:4] == 11).all() and (got[2][0][4:] == -1).all()


def test_select_at_any_address():
    # Rows that begin at any address of their type, and a stride that is no multiple of 16 bytes.
    rng = np.random.default_rng(3)
    for t in R.REAL:
        x = R.stored(rng.normal(0, 2, (1, 3, 4100)), t)
        size = x.itemsize
        dx = R.on_gpu(np.concatenate([np.zeros(1, x.dtype), np.concatenate([x, np.zeros((1, 3, 1), x.dtype)], -1).reshape(-1)]))
        s = Select(R.values(x, t), np.array([[0.0, -0.5, -0.25]]), 5, t, gap=1)
        D.beam_select(dx.addr + size, s.db.addr, *(o.addr for o in s.out[:3]), 1, 3, 4100, 5, type=t, stride=4101,
                      out_ended=s.out[3].addr, workspace=s.work.addr, workspace_bytes=s.bytes)
        print(f"select at an odd address, type {t}", flush=True)
        synchronize()
        s.check()


# ---------------------------------------------------------------- reordering

def beams_of(rng, batch, beams, page, lengths, extra=2):
    """A page table whose full pages beams of a text share, and spare pages: (table, spare, pages)."""
    width = max(lengths) // page + extra
    table, spare, at = np.full((batch * beams, width), -1, np.int32), [], 0
    for b in range(batch):
        full = lengths[b] // page
        for i in range(beams):
            table[b * beams + i, :full] = np.arange(at, at + full)
        at += full
        for i in range(beams):
            n = min(2, width - full)
            table[b * beams + i, full:full + n] = np.arange(at, at + n)
            spare.append(at + n)
            at += n + 1
    order = rng.permutation(at).astype(np.int32)
    return np.where(table >= 0, order[np.maximum(table, 0)], -1).astype(np.int32), order[np.array(spare)], at


@pytest.mark.parametrize("kind", ["f32", "bf16", "heads", "odd", "4 bits", "4 bits in 32"])
@pytest.mark.parametrize("batch,beams,page,layers", [(1, 4, 16, 1), (3, 5, 32, 2), (2, 2, 48, 40), (1, 1, 16, 1)])
def test_reorder(kind, batch, beams, page, layers):
    rng = np.random.default_rng(batch * 10 + page)
    heads, dim, four = 3, 40, kind.startswith("4")
    lengths = [page * 3 + 5, page * 2, 7][:batch]
    table, spare, pages = beams_of(rng, batch, beams, page, lengths)
    rows = batch * beams
    parents = rng.integers(0, beams, rows).astype(np.int32)
    if rows > 4:
        parents[1], parents[2] = -1, beams  # no beams of their text: they go on from themselves
    frm, want_table, want_spare, copies = B.reorder(parents, table, np.repeat(lengths, beams), spare, beams, page, pages)
    caches, held = [], []
    for _ in range(layers):
        if four:
            size = D.kv4_page_bytes(page, heads, dim, 32 if "32" in kind else 0)
            a = rng.integers(0, 256, (pages, size)).astype(np.uint8)
            d = R.on_gpu(a)
            held.append([(a, d)])
            caches.append(D.Kv4Cache(d.addr, pages, page, heads, dim, 32 if "32" in kind else 0))
            continue
        t = {"bf16": D.BF16, "odd": D.F16}.get(kind, D.F32)
        wide = dim + 3 if kind == "odd" else dim
        shape = {"heads": (pages, heads, page, dim), "odd": (pages, page, heads, wide)}.get(kind, (pages, page, heads, dim))
        pair = [rng.integers(0, 100, shape).astype(R.dtype(t)) for _ in range(2)]
        on = [R.on_gpu(a) for a in pair]
        held.append(list(zip(pair, on)))
        strides = {"heads": (heads * page * dim, dim, page * dim), "odd": (page * heads * wide, heads * wide, wide)}.get(kind, (0, 0, 0))
        caches.append(D.KvCache(on[0].addr, on[1].addr, pages, page, heads, dim, t, *strides))
    history = rng.integers(0, 1000, (rows, 33)).astype(np.int32)
    state = rng.integers(0, 256, (rows, 70007)).astype(np.uint8)
    dh, ds = R.on_gpu(history), R.on_gpu(state)
    oh, os_ = R.on_gpu(np.zeros_like(history)), R.on_gpu(np.full((rows, 70010), 7, np.uint8))
    dp, dt, dl, dsp = R.on_gpu(parents), R.on_gpu(table), R.on_gpu(np.repeat(np.array(lengths, np.int32), beams)), R.on_gpu(spare)
    ot, osp = R.on_gpu(np.full_like(table, 9)), R.on_gpu(np.full_like(spare, 9))
    print(f"reorder {batch} x {beams} beams, page {page}, {layers} layers, {kind}", flush=True)
    D.beam_reorder(caches, dp.addr, dt.addr, ot.addr, table.shape[1], dl.addr, dsp.addr, osp.addr, batch, beams,
                   states=[D.BeamState(dh.addr, oh.addr, 4 * 33), D.BeamState(ds.addr, os_.addr, 70007, 70007, 70010)])
    synchronize()
    assert np.array_equal(R.back(ot, np.int32, table.shape), want_table)
    assert np.array_equal(R.back(osp, np.int32, spare.shape), want_spare)
    assert np.array_equal(R.back(oh, np.int32, history.shape), history[frm])
    got = R.back(os_, np.uint8, (rows, 70010))
    assert np.array_equal(got[:, :70007], state[frm]) and (got[:, 70007:] == 7).all()
    for layer in held:
        for a, d in layer:
            want = a.copy()
            for src, dst, n in copies:
                if four:
                    n = -(-n // 4) * 4
                    w = W.Cache4.__new__(W.Cache4)
                    p = W.padded(dim)
                    groups = p // 32 if "32" in kind else 1
                    sizes = [page * p // 2, page * 2 * groups, page * 2 * groups] * 2
                    chunk, at = sum(sizes), 0
                    one, two = want[dst].reshape(heads, chunk), a[src].reshape(heads, chunk)
                    for size in sizes:
                        one[:, at:at + size * n // page] = two[:, at:at + size * n // page]
                        at += size
                elif kind == "heads":
                    want[dst][:, :n] = a[src][:, :n]
                elif kind == "odd":
                    want[dst][:n, :, :dim] = a[src][:n, :, :dim]
                else:
                    want[dst][:n] = a[src][:n]
            assert np.array_equal(R.back(d, a.dtype, a.shape), want)


def test_reorder_of_pages_that_do_not_exist():
    # A parent's page that is none is taken over as it is; a spare page that is none is not written to.
    page, pages = 16, 6
    table = np.array([[0, -1], [0, 1], [0, 2]], np.int32)
    spare = np.array([3, 4, 99], np.int32)
    parents = np.array([0, 0, 1], np.int32)
    a = np.arange(pages * page * 8, dtype=np.float32).reshape(pages, page, 1, 8)
    on = [R.on_gpu(a), R.on_gpu(a)]
    dp, dt, dsp, dl = R.on_gpu(parents), R.on_gpu(table), R.on_gpu(spare), R.on_gpu(np.full(3, 20, np.int32))
    ot, osp = R.on_gpu(np.zeros_like(table)), R.on_gpu(np.zeros_like(spare))
    for lengths in (20, 100, 16, 0, -5):
        dl.upload(np.full(3, lengths, np.int32))
        print(f"reorder, bad pages, {lengths} tokens", flush=True)
        D.beam_reorder([D.KvCache(on[0].addr, on[1].addr, pages, page, 1, 8, D.F32)], dp.addr, dt.addr, ot.addr, 2,
                       dl.addr, dsp.addr, osp.addr, 1, 3)
        synchronize()
        _, want, left, _ = B.reorder(parents, table, [lengths] * 3, spare, 3, page, pages)
        assert np.array_equal(R.back(ot, np.int32, table.shape), want)
        assert np.array_equal(R.back(osp, np.int32, spare.shape), left)
        assert all(np.array_equal(R.back(d, np.float32, a.shape), a) for d in on)


def test_reorder_states_alone():
    rng = np.random.default_rng(1)
    a = rng.integers(0, 256, (6, 1 << 21)).astype(np.uint8)
    parents = np.array([2, 0, 0, 1, 1, 2], np.int32)
    d, o, dp = R.on_gpu(a), R.on_gpu(np.zeros_like(a)), R.on_gpu(parents)
    print("reorder, states alone", flush=True)
    D.beam_reorder([], dp.addr, 0, 0, 0, 0, 0, 0, 2, 3, states=[D.BeamState(d.addr, o.addr, 1 << 21)])
    synchronize()
    assert np.array_equal(R.back(o, np.uint8, a.shape), a[[2, 0, 0, 4, 4, 5]])


@pytest.mark.parametrize("base", [-1e9, -3e38, 1e9])
def test_select_of_scores_that_32_bits_do_not_tell_apart(base):
    # Scores so far from 0 that all candidates' are one number in 32 bits, many more than a workgroup lists; logits are
    # whole numbers of 1/8, so that in 64 bits each keeps its place (1e9), or all are equal and the logits decide (3e38).
    rng = np.random.default_rng(5)
    x = rng.permutation(131072).reshape(1, 1, -1) / 8.0
    s = Select(x, np.full((1, 1), base), 128, D.F32)
    s.run()
    synchronize()
    s.check()


@pytest.mark.parametrize("t", R.REAL)
@pytest.mark.parametrize("beams,vocab,keep", [(1, 131072, 128), (32, 20000, 128), (3, 131072, 64), (2, 300, 5)])
def test_select_of_infinite_scores(t, beams, vocab, keep):
    # A score of +infinity: every continuation of its beam has it, more than a workgroup lists, and the lower beam, the
    # larger logit and the lower token decide. A beam that has ended goes on with its end token at that.
    rng = np.random.default_rng(beams)
    x = rng.normal(0, 2, (2, beams, vocab))
    base = np.full((2, beams), np.inf)
    base[1, :beams // 2] = -1
    s = Select(x, base, keep, t)
    s.run()
    synchronize()
    got = s.check()
    assert (got[0] == np.inf).all() or beams == 2
    ended = np.zeros((2, beams), np.uint8)
    ended[:, 0] = 1
    s = Select(x, base, keep, t, ended=ended, end=5)
    s.run()
    synchronize()
    s.check()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("layers", [2, 60])
def test_reorder_of_caches_with_fewer_pages(four, layers):
    # A page is there if all caches have it, however many launches they take: the last layer's has fewer. What one cache
    # copies all do, and the tables say.
    rng = np.random.default_rng(layers)
    batch, beams, page, heads, dim = 3, 4, 16, 2, 32
    lengths = [40, 21, 70]
    table, spare, pages = beams_of(rng, batch, beams, page, lengths)
    rows, fewer = batch * beams, pages - 9
    parents = rng.integers(0, beams, rows).astype(np.int32)
    frm, want_table, want_spare, copies = B.reorder(parents, table, np.repeat(lengths, beams), spare, beams, page, fewer)
    assert copies and len(copies) < len(B.reorder(parents, table, np.repeat(lengths, beams), spare, beams, page, pages)[3])
    caches, held = [], []
    size = D.kv4_page_bytes(page, heads, dim, 0) if four else page * heads * dim * 4
    for i in range(layers):
        n = fewer if i == layers - 1 else pages
        arrays = [rng.integers(0, 256, (n, size)).astype(np.uint8) for _ in range(1 if four else 2)]
        on = [R.on_gpu(a) for a in arrays]
        held += list(zip(arrays, on))
        caches.append(D.Kv4Cache(on[0].addr, n, page, heads, dim, 0) if four else
                      D.KvCache(on[0].addr, on[1].addr, n, page, heads, dim, D.F32))
    dp, dt, dsp = R.on_gpu(parents), R.on_gpu(table), R.on_gpu(spare)
    dl = R.on_gpu(np.repeat(np.array(lengths, np.int32), beams))
    ot, osp = R.on_gpu(np.full_like(table, 9)), R.on_gpu(np.full_like(spare, 9))
    print(f"reorder, fewer pages in the last of {layers} layers, 4 bits {four}", flush=True)
    D.beam_reorder(caches, dp.addr, dt.addr, ot.addr, table.shape[1], dl.addr, dsp.addr, osp.addr, batch, beams)
    synchronize()
    assert np.array_equal(R.back(ot, np.int32, table.shape), want_table)
    assert np.array_equal(R.back(osp, np.int32, spare.shape), want_spare)
    for a, d in held:
        want = a.copy()
        for src, dst, n in copies:
            if four:  # of each head's planes the tokens in use, up to the next multiple of four
                n, at, chunk = -(-n // 4) * 4, 0, size // heads
                one, two = want[dst].reshape(heads, chunk), a[src].reshape(heads, chunk)
                for part in [page * 16, page * 2, page * 2] * 2:
                    one[:, at:at + part * n // page] = two[:, at:at + part * n // page]
                    at += part
            else:
                want[dst, :n * heads * dim * 4] = a[src, :n * heads * dim * 4]
        assert np.array_equal(R.back(d, np.uint8, a.shape), want)
