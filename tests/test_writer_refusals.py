"""Calls of what a text decoder writes with that are refused, with their
reasons, before anything reaches a GPU (CPU-only: the addresses are never read)."""
import pytest

from ppocr_native_amd import GpuError, decoder as D
from test_decoder_refusals import A, cache


def cache4(**k):
    a = dict(data=A, pages=4, page_size=16, heads=2, dim=64, group=32)
    a.update(k)
    return D.Kv4Cache(**a)


def rotated(cache=cache(), **k):
    a = dict(k=A, v=A, table=A, table_width=4, lengths=A, batch=2, rows=2, freqs=A, rotary=64, q=A, q_out=A, heads=4)
    a.update(k)
    D.kv_append_rotated(cache=cache, **a)


def append4(cache=cache4(), **k):
    a = dict(k=A, v=A, table=A, table_width=4, lengths=A, batch=2, rows=2, freqs=A, rotary=64, q=A, q_out=A, heads=4,
             type=D.F16)
    a.update(k)
    D.kv4_append(cache=cache, **a)


def read4(cache=cache4(), **k):
    a = dict(k=A, v=A, table=A, table_width=4, lengths=A, batch=2, rows=2, type=D.BF16)
    a.update(k)
    D.kv4_read(cache=cache, **a)


def attend4(cache=cache4(), **k):
    a = dict(q=A, table=A, table_width=4, lengths=A, y=A, batch=2, heads=4, scale=0.1, type=D.F16)
    a.update(k)
    D.kv4_attention(cache=cache, **a)


TURNS = [(dict(rotary=63), "63 dims of heads of 64"), (dict(rotary=66), "66 dims"), (dict(freqs=0), "without frequencies"),
         (dict(q=0), "together"), (dict(q_out=0), "together"), (dict(heads=0), "0 query heads"),
         (dict(heads=3), "3 query heads over 2"), (dict(heads=70000), "70000"), (dict(q=A + 1), "aligned"),
         (dict(q_out=A + 1), "aligned"), (dict(freqs=A + 2), "aligned"), (dict(positions=A + 2), "aligned"),
         (dict(q_stride=255), "strides 255"), (dict(q_out_stride=255), "strides 0, 255")]
ROWS = [(dict(rows=3), "3 rows for 2 texts"), (dict(k=0), "needed"), (dict(v=0), "needed"), (dict(k=A + 1), "aligned"),
        (dict(starts=A + 2), "aligned"), (dict(k_stride=127), "strides 127"), (dict(v_stride=127), "strides 128, 127|strides 0, 127"),
        (dict(batch=70000, rows=70000), "70000 texts"), (dict(rows=1 << 31, starts=A), "rows")]
TABLE = [(dict(table=0), "page table"), (dict(lengths=0), "lengths"), (dict(table_width=0), "0 pages"),
         (dict(table_width=1 << 28), "page table of")]
CACHE4 = [(dict(cache=cache4(**k)), reason) for k, reason in (
    (dict(data=0), "no cache"), (dict(data=A + 8), "aligned"), (dict(pages=0), "0 pages"), (dict(page_size=8), "of 8 tokens"),
    (dict(page_size=24), "multiple of 16"), (dict(page_size=0), "of 0 tokens"), (dict(page_size=1 << 21), "2097152 tokens"),
    (dict(heads=0), "0 heads"), (dict(heads=70000), "70000 heads"), (dict(dim=0), "of 0 values"), (dict(dim=257), "257"),
    (dict(group=16), "groups of 16"), (dict(group=128), "groups of 128"), (dict(page_stride=16), "16 apart"),
    (dict(page_stride=1 << 41), "apart"), (dict(page_stride=(1 << 20) + 8), "multiple of 16"))]


@pytest.mark.parametrize("call,args,reason", [(rotated, *x) for x in TURNS + ROWS + TABLE] + [
    (rotated, dict(cache=cache(type=D.E4M3)), "type 3"), (rotated, dict(cache=cache(dim=257)), "257"),
] + [(append4, *x) for x in TURNS + ROWS + TABLE + CACHE4] + [(append4, dict(type=D.I8), "type 4")] +
    [(read4, *x) for x in ROWS + TABLE + CACHE4] + [(read4, dict(type=9), "type 9")] +
    [(attend4, *x) for x in TABLE + CACHE4] + [
    (attend4, dict(type=D.E4M3), "type 3"), (attend4, dict(heads=3), "3 query heads over 2"),
    (attend4, dict(heads=0), "0 query heads"), (attend4, dict(q=0), "needed"), (attend4, dict(y=0), "needed"),
    (attend4, dict(scale=float("inf")), "scale inf"), (attend4, dict(scale=float("nan")), "scale nan"),
    (attend4, dict(workspace=A + 4, workspace_bytes=1 << 20), "aligned"), (attend4, dict(q_stride=255), "strides 255"),
    (attend4, dict(batch=70000), "70000 texts"),
])
def test_refused(call, args, reason):
    with pytest.raises(GpuError, match=reason):
        call(**args)


@pytest.mark.parametrize("call,args", [(rotated, dict(batch=0)), (rotated, dict(rows=0)), (append4, dict(batch=0)),
                                       (append4, dict(rows=0)), (read4, dict(rows=0)), (attend4, dict(batch=0))])
def test_nothing_to_do(call, args):
    call(**args)


@pytest.mark.parametrize("call", [rotated, append4, read4, attend4])
def test_the_legacy_handle_is_refused(call):
    with pytest.raises(GpuError, match="handle"):
        call(stream=1)


def test_page_bytes():
    # A token's head: P / 2 bytes of codes and 4 of each group's scale and minimum, of K and of V.
    for dim, group, p, groups in ((1, 0, 32, 1), (64, 0, 64, 1), (64, 32, 64, 2), (80, 32, 96, 3), (80, 64, 96, 2),
                                  (128, 64, 128, 2), (130, 32, 192, 6), (200, 64, 256, 4), (32, 64, 32, 1)):
        assert D.kv4_page_bytes(48, 5, dim, group) == 48 * 5 * (p + 8 * groups)
    for size in ((8, 1, 64, 0), (16, 0, 64, 0), (16, 1, 0, 0), (16, 1, 257, 0), (16, 1, 64, 48)):
        assert D.kv4_page_bytes(*size) == 0


def test_workspace4():
    c = cache4(heads=8, dim=128)
    assert D.kv4_attention_workspace(c, 1, 32, 100) == 0  # one part
    n = D.kv4_attention_workspace(c, 1, 32, 16384)
    assert n > 0 and n % (32 * 130 * 4) == 0
    assert D.kv4_attention_workspace(c, 4096, 32, 16384) == 0  # enough texts
    assert D.kv4_attention_workspace(c, 1, 33, 16384) == 0 and D.kv4_attention_workspace(None, 1, 1, 1) == 0


# ------------------------------------------------------------------ beam search

def select(**k):
    a = dict(logits=A, scores=A, out_scores=A, parents=A, tokens=A, batch=2, beams=4, vocab=1000, keep=4, type=D.F16,
             workspace=A, workspace_bytes=1 << 20)
    a.update(k)
    D.beam_select(**a)


def reorder(caches=(cache(),), states=(), **k):
    a = dict(parents=A, table=A, table_out=A + 64, table_width=4, lengths=A, spare=A, spare_out=A + 64, batch=2, beams=3)
    a.update(k)
    D.beam_reorder(list(caches), states=list(states), **a)


@pytest.mark.parametrize("call,args,reason", [
    (select, dict(type=D.E4M3), "type 3"),
    (select, dict(beams=0), "of 0 beams"),
    (select, dict(beams=129), "of 129 beams"),
    (select, dict(keep=0), "0 of 4 beams"),
    (select, dict(keep=129), "129 of 4"),
    (select, dict(vocab=0), "0 tokens"),
    (select, dict(vocab=(1 << 24) + 1), "tokens"),
    (select, dict(batch=70000), "70000 texts"),
    (select, dict(batch=60000, beams=128, vocab=1 << 20), "parts"),
    (select, dict(logits=0), "needed"),
    (select, dict(scores=0), "needed"),
    (select, dict(parents=0), "needed"),
    (select, dict(logits=A + 1), "aligned"),
    (select, dict(tokens=A + 2), "aligned"),
    (select, dict(workspace=A + 8), "aligned"),
    (select, dict(stride=999), "stride 999"),
    (select, dict(end=1000), "end token 1000 of 1000"),
    (select, dict(end=-2), "end token -2"),
    (select, dict(ended=A), "have ended need one"),
    (select, dict(workspace=0), "workspace of"),
    (select, dict(workspace_bytes=100), "not 100"),
    (reorder, dict(beams=0), "0 beams"),
    (reorder, dict(batch=30000), "30000 texts"),
    (reorder, dict(parents=0), "parents"),
    (reorder, dict(parents=A + 2), "parents"),
    (reorder, dict(table=0), "page table"),
    (reorder, dict(table_out=0), "needed"),
    (reorder, dict(table_out=A), "apart"),
    (reorder, dict(spare=0), "needed"),
    (reorder, dict(spare_out=A), "apart"),
    (reorder, dict(spare_out=A + 66), "aligned"),
    (reorder, dict(lengths=0), "lengths"),
    (reorder, dict(caches=[cache(), cache(page_size=32)]), "pages of 16 and 32"),
    (reorder, dict(caches=[cache(dim=300)]), "300"),
    (reorder, dict(caches=[cache4(dim=300)]), "300"),
    (reorder, dict(caches=[cache4(), cache4(page_size=32)]), "pages of 16 and 32"),
    (reorder, dict(states=[D.BeamState(0, A, 4)]), "state 0"),
    (reorder, dict(states=[D.BeamState(A, A, 4)]), "apart"),
    (reorder, dict(states=[D.BeamState(A, A + 64, 8), D.BeamState(A, A + 64, 8, 4)]), "state 1 of 8 bytes"),
    (reorder, dict(states=[D.BeamState(A, A + 64, 8)] * 17), "17 states"),
])
def test_beams_refused(call, args, reason):
    with pytest.raises(GpuError, match=reason):
        call(**args)


def test_beams_nothing_to_do():
    select(batch=0)
    reorder(batch=0)
    reorder(caches=[])
    with pytest.raises(GpuError, match="handle"):
        select(stream=1)
    with pytest.raises(GpuError, match="handle"):
        reorder(stream=1)


def test_select_workspace():
    # For each part of a row, its best and two floats; parts of 2048 to 8192 tokens.
    assert D.beam_select_workspace(1, 4, 1000, 4) == 4 * 5 * 8
    n = D.beam_select_workspace(32, 8, 131072, 8)
    assert n % (256 * 9 * 8) == 0 and 16 <= n // (256 * 9 * 8) <= 64
    assert D.beam_select_workspace(1, 129, 100, 4) == 0 and D.beam_select_workspace(1, 1, 100, 0) == 0


@pytest.mark.parametrize("tokens,heads,strides,refused", [
    (1 << 16, 1 << 15, (1 << 35, 1 << 20, 16), True), (1 << 16, 1 << 15, (1 << 35, 16, 1 << 20), True),
    (1 << 30, 2, (1 << 36, 32, 16), True), ((1 << 16) - 1, 1 << 15, (1 << 35, 1 << 20, 16), False),
    (1 << 16, 1 << 15, (1 << 35, 8, 1 << 19), False), (1 << 16, 1 << 15, (0, 0, 0), False)])
def test_reorder_of_very_many_heads_of_tokens(tokens, heads, strides, refused):
    # Rows of heads that lie apart are counted in 32 bits: from 2^31 on they are refused, and others are not. (The call
    # that is not refused ends at the legacy handle, which is.)
    c = cache(page_size=tokens, heads=heads, dim=8, page_stride=strides[0], token_stride=strides[1], head_stride=strides[2])
    with pytest.raises(GpuError, match="do not lie together" if refused else "handle"):
        reorder(caches=[c], table_width=1, stream=1)
