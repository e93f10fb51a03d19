"""A whole beam search as a program runs it: each step appends the beams' newest
tokens, turned, to a paged cache (in 4 bits, or plain), attends over it, makes
logits of that, chooses, and reorders caches and histories; eager, and captured
as two graphs that take turns."""
import numpy as np
import pytest

import beam_plain as B
import decoder_plain as R
import writer_plain as W
from ppocr_native_amd import decoder as D
from ppocr_native_amd.devmem import synchronize
from test_gpu_decoder import Graph, _stream

pytestmark = pytest.mark.gpu

BATCH, BEAMS, PAGE, KV, HEADS, DIM, ROTARY, VOCAB, STEPS, END, LAYERS = 2, 3, 16, 2, 4, 64, 32, 500, 40, 7, 2
ROWS = BATCH * BEAMS


class Search:
    """The buffers of a search. Sides 0 and 1 of tables, spare pages and histories take turns."""

    def __init__(self, seed, four):
        rng = np.random.default_rng(seed)
        self.four, self.t = four, D.F32
        self.prompt = rng.integers(0, VOCAB, (BATCH, 21))
        # What a layer makes of a token: here each token's q, k and v are given, as a network without a past would make them.
        self.q, self.k, self.v = (rng.normal(0, 1, (LAYERS, VOCAB, n, DIM)).astype(np.float32) for n in (HEADS, KV, KV))
        self.freqs = W.frequencies(ROTARY)
        most = -(-(self.prompt.shape[1] + STEPS) // PAGE)
        self.pages = BATCH * 2 + ROWS * (most + 1)
        order = rng.permutation(self.pages).astype(np.int32)
        shared = order[:BATCH * 2].reshape(BATCH, 2)
        rest = order[BATCH * 2:].reshape(ROWS, most + 1)
        table = rest[:, :most].copy()
        full = self.prompt.shape[1] // PAGE
        table[:, :full] = np.repeat(shared[:, :full], BEAMS, 0)  # the prompts' full pages are shared
        self.width = most
        up = R.on_gpu
        self.table = [up(table), up(np.zeros_like(table))]
        self.spare = [up(rest[:, most].copy()), up(np.zeros(ROWS, np.int32))]
        self.history = [up(np.zeros((ROWS, STEPS + 32), np.int32)) for _ in range(2)]
        self.lengths = np.full(ROWS, self.prompt.shape[1], np.int32)
        self.dl, self.df = up(self.lengths), up(self.freqs)
        rows4 = lambda n: [up(np.zeros((ROWS, n, DIM), np.float32)) for _ in range(LAYERS)]  # noqa: E731
        self.dq, self.dk, self.dv, self.dqo, self.dy = rows4(HEADS), rows4(KV), rows4(KV), rows4(HEADS), rows4(HEADS)
        self.wq = rng.integers(0, 16, (VOCAB, HEADS * DIM))
        self.ws = (np.full((VOCAB, HEADS * DIM // 64), 0.02)).astype(np.float32)
        self.dwq, self.dws = up(R.packed(self.wq)), up(self.ws)
        self.logits = up(np.zeros((ROWS, VOCAB), np.float32))
        base = np.full((BATCH, BEAMS), -np.inf, np.float32)
        base[:, 0] = 0
        self.scores, self.ended = [up(base), up(base)], [up(np.zeros(ROWS, np.uint8)), up(np.zeros(ROWS, np.uint8))]
        self.parents, self.tokens = up(np.zeros(ROWS, np.int32)), up(np.zeros(ROWS, np.int32))
        self.bytes = D.beam_select_workspace(BATCH, BEAMS, VOCAB, BEAMS)
        self.work, self.work2 = up(np.zeros(self.bytes, np.uint8)), up(np.zeros(1 << 20, np.uint8))
        if four:
            size = D.kv4_page_bytes(PAGE, KV, DIM, 32)
            self.data = [up(np.zeros((self.pages, size), np.uint8)) for _ in range(LAYERS)]
            self.caches = [D.Kv4Cache(d.addr, self.pages, PAGE, KV, DIM, 32) for d in self.data]
        else:
            self.data = [[up(np.zeros((self.pages, PAGE, KV, DIM), np.float32)) for _ in range(2)] for _ in range(LAYERS)]
            self.caches = [D.KvCache(k.addr, v.addr, self.pages, PAGE, KV, DIM) for k, v in self.data]
        self.write_prompts(table)

    def write_prompts(self, table):
        """The prompts' tokens into the cache: full pages once a text, the last, partial page for each beam."""
        n = self.prompt.shape[1]
        starts, lengths = R.on_gpu((np.arange(ROWS + 1) * n).astype(np.int32)), self.dl
        tokens = np.repeat(self.prompt, BEAMS, 0).reshape(-1)
        for i in range(LAYERS):
            k, v = R.on_gpu(self.k[i][tokens]), R.on_gpu(self.v[i][tokens])
            # (Beams share their full pages: all write the same there, one text's beams one after the other.)
            for r in range(ROWS):
                at = r * n * KV * DIM * 4
                (D.kv4_append if self.four else D.kv_append_rotated)(
                    k.addr + at, v.addr + at, self.caches[i], self.table[0].addr + 4 * r * self.width, self.width,
                    lengths.addr + 4 * r, 1, n, starts=starts.addr, freqs=self.df.addr, rotary=ROTARY)
            synchronize()
        h = np.zeros((ROWS, STEPS + 32), np.int32)
        h[:, :n] = np.repeat(self.prompt, BEAMS, 0)
        self.history[0].upload(h)

    def put_tokens(self, tokens):
        """What the layers make of the newest tokens, each of them one place further on."""
        self.lengths += 1
        self.dl.upload(self.lengths)
        for i in range(LAYERS):
            self.dq[i].upload(self.q[i][tokens]), self.dk[i].upload(self.k[i][tokens]), self.dv[i].upload(self.v[i][tokens])

    def step(self, side, stream=0):
        s = dict(stream=stream)
        table = self.table[side].addr
        for i in range(LAYERS):
            turn = dict(freqs=self.df.addr, rotary=ROTARY, q=self.dq[i].addr, q_out=self.dqo[i].addr, heads=HEADS, **s)
            seen = dict(scale=DIM ** -0.5, longest=100, workspace=self.work2.addr, workspace_bytes=1 << 20, **s)
            if self.four:
                D.kv4_append(self.dk[i].addr, self.dv[i].addr, self.caches[i], table, self.width, self.dl.addr, ROWS, ROWS, **turn)
                D.kv4_attention(self.dqo[i].addr, self.caches[i], table, self.width, self.dl.addr, self.dy[i].addr, ROWS, HEADS, **seen)
            else:
                D.kv_append_rotated(self.dk[i].addr, self.dv[i].addr, self.caches[i], table, self.width, self.dl.addr, ROWS, ROWS, **turn)
                D.paged_attention(self.dqo[i].addr, self.caches[i], table, self.width, self.dl.addr, self.dy[i].addr, ROWS, HEADS, **seen)
        D.q4_product(self.dy[LAYERS - 1].addr, self.dwq.addr, self.dws.addr, self.logits.addr, ROWS, VOCAB, HEADS * DIM,
                     group=64, **s)
        D.beam_select(self.logits.addr, self.scores[side].addr, self.scores[1 - side].addr, self.parents.addr,
                      self.tokens.addr, BATCH, BEAMS, VOCAB, BEAMS, ended=self.ended[side].addr,
                      out_ended=self.ended[1 - side].addr, end=END, workspace=self.work.addr, workspace_bytes=self.bytes, **s)
        D.beam_reorder(self.caches, self.parents.addr, table, self.table[1 - side].addr, self.width, self.dl.addr,
                       self.spare[side].addr, self.spare[1 - side].addr, BATCH, BEAMS,
                       states=[D.BeamState(self.history[side].addr, self.history[1 - side].addr, 4 * (STEPS + 32))], **s)

    def note(self, side):
        """The chosen tokens, written down behind their beams' histories."""
        synchronize()
        h = R.back(self.history[1 - side], np.int32, (ROWS, STEPS + 32)).copy()
        tokens = R.back(self.tokens, np.int32, (ROWS,)).copy()
        h[np.arange(ROWS), self.lengths] = tokens
        self.history[1 - side].upload(h)
        return tokens

    # ------------------------------------------------------------- the checks

    def held(self, side):
        """Keys and values [layer][row][token] as the cache has them by side's table, as (n s, m) or (value, 0)."""
        table = R.back(self.table[side], np.int32, (ROWS, self.width))
        out = []
        for i in range(LAYERS):
            if self.four:
                c = W.Cache4(np.random.default_rng(0), [1], PAGE, KV, DIM, 32, spare=self.pages - 1)
                c.data[...] = R.back(self.data[i], np.uint8, c.data.shape)
                c.table = table
                out.append([[c.get(r, j) for j in range(self.lengths[r])] for r in range(ROWS)])
            else:
                k, v = (R.back(d, np.float32, (self.pages, PAGE, KV, DIM)).astype(np.float64) for d in self.data[i])
                out.append([[((k[table[r, j // PAGE], j % PAGE], 0), (v[table[r, j // PAGE], j % PAGE], 0))
                             for j in range(self.lengths[r])] for r in range(ROWS)])
        return out

    def wanted(self, i, token, place):
        """Key and value of a token at a place, as they are to be held: rounded step by step as is documented."""
        f = np.float32
        x = self.k[i][token].copy()
        a = place * self.freqs.astype(np.float64)
        c, s = np.cos(a).astype(f), np.sin(a).astype(f)
        half = ROTARY // 2
        x1, x2 = x[:, :half].copy(), x[:, half:ROTARY].copy()
        x[:, :half], x[:, half:ROTARY] = x1 * c - x2 * s, x2 * c + x1 * s
        out = []
        for row in (x, self.v[i][token]):
            if not self.four:
                out.append(row.astype(np.float64))
                continue
            n, s4, m4 = W.quantised(row, DIM, 32)
            of = np.arange(DIM) // 32
            out.append(n[:, :DIM] * s4.astype(np.float64)[:, of] + m4.astype(np.float64)[:, of])
        return out

    def check_caches(self, side):
        """Each beam's cache holds its own history's tokens, place by place."""
        h = R.back(self.history[side], np.int32, (ROWS, STEPS + 32))
        held = self.held(side)
        for i in range(LAYERS):
            for r in range(ROWS):
                for j in range(self.lengths[r]):
                    for got, want in zip(held[i][r][j], self.wanted(i, h[r, j], j)):
                        assert np.array_equal(got[0] + got[1], want), (i, r, j)

    def check_step(self, side, held):
        """Attention, logits and choice of the step that was just made, each on what it was given."""
        for i in range(LAYERS):
            q, y = (R.back(d, np.float32, (ROWS, HEADS, DIM)).astype(np.float64) for d in (self.dqo[i], self.dy[i]))
            for r in range(ROWS):
                for h in range(HEADS):
                    parts = held[i][r]
                    k, v = ([np.array([np.broadcast_to(x[p][j], (KV, DIM))[h // 2] for x in parts]) for j in (0, 1)] for p in (0, 1))
                    want, size, reach = W.attend4(q[r, h], k, v, np.ones(len(parts), bool), DIM ** -0.5)
                    R.close(y[r, h], want, W.attend4_bound(want, size, reach, D.F32))
        logits = R.back(self.logits, np.float32, (ROWS, VOCAB)).astype(np.float64)
        want, size = R.product(y.reshape(ROWS, -1), self.wq, self.ws.astype(np.float64), None, 64)
        R.close(logits, want, R.half_step(want, D.F32) + 16 * R.STEP * size)
        base, ended = R.back(self.scores[side], np.float32, (BATCH, BEAMS)), R.back(self.ended[side], np.uint8, (BATCH, BEAMS))
        got = [R.back(d, t, (BATCH, BEAMS)) for d, t in ((self.scores[1 - side], np.float32), (self.parents, np.int32),
                                                         (self.tokens, np.int32), (self.ended[1 - side], np.uint8))]
        for b in range(BATCH):
            want, _ = B.choose(logits.reshape(BATCH, BEAMS, VOCAB)[b], base[b].astype(np.float64), BEAMS, ended[b], END)
            R.close(got[0][b].astype(np.float64), want[0], np.abs(want[0]) * R.STEP / 2 + 17 * R.STEP)
            for j in range(1, 4):
                assert np.array_equal(got[j][b], want[j])


def begin(search):
    """The prompts' last tokens are the first to be attended with: they are written once more, at their place."""
    search.lengths -= 1
    return np.repeat(search.prompt[:, -1], BEAMS)


@pytest.mark.parametrize("four", [True, False])
def test_a_search(four):
    search = Search(5, four)
    tokens = begin(search)
    moved = 0
    for i in range(STEPS):
        side = i % 2
        search.put_tokens(tokens)
        print(f"search step {i}, 4 bits {four}", flush=True)
        if i % 8 == 0:  # what the step attends over, found before the pages are copied
            synchronize()
        search.step(side)
        tokens = search.note(side)
        if i % 8 == 0:
            # (The step's own table still names what it attended over: copies went to pages that it does not name.)
            search.check_step(side, search.held(side))
        parents = R.back(search.parents, np.int32, (BATCH, BEAMS))
        moved += int((parents != np.arange(BEAMS)).sum())
        if i % 13 == 12 or i == STEPS - 1:
            search.check_caches(1 - side)
    assert moved > STEPS // 4  # beams did change places


@pytest.mark.parametrize("four", [True, False])
def test_a_captured_search(four):
    # Two graphs, one a side, replayed in turn with the host's work between: as the eager steps, bit for bit.
    s = _stream()
    a, b = Search(6, four), Search(6, four)
    ta = tb = begin(a)
    begin(b)
    graphs = None
    for i in range(STEPS):
        side = i % 2
        a.put_tokens(ta), b.put_tokens(tb)
        b.step(side)
        if i < 2:
            a.step(side, s.value)
        else:
            if graphs is None:
                graphs = [Graph(s, lambda side=side: a.step(side, s.value)) for side in (0, 1)]
            print(f"captured search step {i}, 4 bits {four}", flush=True)
            graphs[side].launch()
        ta, tb = a.note(side), b.note(side)
        assert np.array_equal(ta, tb)
        for x, y in ((a.scores, b.scores), (a.table, b.table), (a.spare, b.spare), (a.history, b.history)):
            assert np.array_equal(x[1 - side].download(x[1 - side].nbytes, np.uint8), y[1 - side].download(y[1 - side].nbytes, np.uint8))
    a.check_caches(STEPS % 2)


def test_two_searches_on_two_streams():
    # Each with its own buffers: as each is alone.
    streams = [_stream(), _stream()]
    pairs = [(Search(7 + i, True), Search(7 + i, True)) for i in range(2)]
    tokens = [begin(p[0]) for p in pairs]
    [begin(p[1]) for p in pairs]
    for i in range(6):
        print(f"two searches, step {i}", flush=True)
        for (one, _), t in zip(pairs, tokens):
            one.put_tokens(t)
        for (one, _), s in zip(pairs, streams):
            one.step(i % 2, s.value)
        synchronize()
        for (_, other), t in zip(pairs, tokens):
            other.put_tokens(t)
            other.step(i % 2)
            synchronize()
        tokens = [one.note(i % 2) for one, _ in pairs]
        assert all(np.array_equal(other.note(i % 2), t) for (_, other), t in zip(pairs, tokens))
