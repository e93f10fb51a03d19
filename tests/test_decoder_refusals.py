"""Calls of the decoder layers that are refused, with their reasons, before
anything reaches a GPU (CPU-only: the addresses are never read)."""
import pytest

from ppocr_native_amd import GpuError, decoder as D

A = 1 << 20  # an address


def cache(**k):
    a = dict(k=A, v=A, pages=4, page_size=16, heads=2, dim=64, type=D.F16)
    a.update(k)
    return D.KvCache(**a)


def norm(**k):
    a = dict(x=A, weight=A, y=A, rows=2, c=64, type=D.BF16)
    a.update(k)
    D.rms_norm(**a)


def product(**k):
    a = dict(x=A, q=A, scales=A, y=A, m=2, n=32, k=128, group=64)
    a.update(k)
    D.q4_product(**a)


def append(cache=cache(), **k):
    a = dict(k=A, v=A, table=A, table_width=4, lengths=A, batch=2, rows=2)
    a.update(k)
    D.kv_append(cache=cache, **a)


def paged(cache=cache(), **k):
    a = dict(q=A, table=A, table_width=4, lengths=A, y=A, batch=2, heads=4, scale=0.1)
    a.update(k)
    D.paged_attention(cache=cache, **a)


def prompt(**k):
    a = dict(q=A, k=A, v=A, y=A, starts_q=A, starts_k=A, batch=2, rows_q=9, rows_k=9, heads=4, kv_heads=2, dim=64,
             scale=0.1, type=D.F16)
    a.update(k)
    D.window_attention(**a)


@pytest.mark.parametrize("call,args,reason", [
    (norm, dict(type=D.E4M3), "type 3"),
    (norm, dict(type=7), "type 7"),
    (norm, dict(y_type=D.F16), "not 2"),
    (norm, dict(y_type=D.E4M3), "scales"),
    (norm, dict(y_type=D.I8, scales=A, group=16), "16 values"),
    (norm, dict(c=0), "0 values"),
    (norm, dict(c=1 << 31), "values"),
    (norm, dict(x=0), "needed"),
    (norm, dict(weight=0), "needed"),
    (norm, dict(x=A + 1), "aligned"),
    (norm, dict(x_stride=63), "strides 63"),
    (norm, dict(eps=-1.0), "eps -1"),
    (norm, dict(eps=float("nan")), "eps nan"),
    (product, dict(group=0), "0 inputs"),
    (product, dict(group=256), "256 inputs"),
    (product, dict(k=0), "0 inputs"),
    (product, dict(x_type=9), "type 9"),
    (product, dict(scale_type=D.E4M3), "type 3"),
    (product, dict(y_type=D.I8), "type 4"),
    (product, dict(x_type=D.I8), "x_scales"),
    (product, dict(x_type=D.I8, x_scales=A, x_group=32), "each 32 inputs, the weights each 64"),
    (product, dict(q=0), "needed"),
    (product, dict(scales=A + 2), "aligned"),
    (product, dict(x_stride=127), "strides 127"),
    (product, dict(y_stride=31), "strides 0 for 128 inputs, 31"),
    (append, dict(rows=3), "3 rows for 2 texts"),
    (append, dict(k=0), "needed"),
    (append, dict(k=A + 1), "aligned"),
    (append, dict(table=0), "page table"),
    (append, dict(table_width=0), "0 pages"),
    (append, dict(table_width=1 << 28), "page table of"),
    (append, dict(batch=70000, rows=70000), "70000 texts"),
    (append, dict(k_stride=127), "strides 127"),
    (append, dict(cache=cache(type=D.E4M3)), "type 3"),
    (append, dict(cache=cache(dim=257)), "257"),
    (append, dict(cache=cache(dim=0)), "cache of"),
    (append, dict(cache=cache(pages=0)), "0 pages"),
    (append, dict(cache=cache(page_size=0)), "of 0 tokens"),
    (append, dict(cache=cache(k=0)), "no cache"),
    (append, dict(cache=cache(token_stride=64)), "cache strides 0, 64, 0"),
    (paged, dict(heads=3), "3 query heads over 2"),
    (paged, dict(heads=0), "0 query heads"),
    (paged, dict(q=0), "needed"),
    (paged, dict(scale=float("inf")), "scale inf"),
    (paged, dict(workspace=A + 4, workspace_bytes=1 << 20), "aligned"),
    (paged, dict(q_stride=255), "strides 255"),
    (paged, dict(lengths=0), "lengths"),
    (paged, dict(cache=cache(dim=512)), "512"),
    (prompt, dict(type=D.I8), "type 4"),
    (prompt, dict(heads=3), "3 query heads over 2"),
    (prompt, dict(kv_heads=0), "over 0"),
    (prompt, dict(dim=300), "300"),
    (prompt, dict(starts_q=0), "needed"),
    (prompt, dict(v=0), "needed"),
    (prompt, dict(scale=float("nan")), "scale nan"),
    (prompt, dict(v_stride=100), "strides"),
    (prompt, dict(batch=40000), "40000 texts"),
    (prompt, dict(rows_q=1 << 25), "queries"),
    (product, dict(k=1 << 25), "inputs"),
    (product, dict(x_stride=1 << 25), "strides"),
    (product, dict(m=1 << 20, n=1 << 20), "outputs"),
])
def test_refused(call, args, reason):
    with pytest.raises(GpuError, match=reason):
        call(**args)


@pytest.mark.parametrize("call,args", [(norm, dict(rows=0)), (product, dict(m=0)), (product, dict(n=0)),
                                       (append, dict(batch=0)), (append, dict(rows=0)), (paged, dict(batch=0)),
                                       (prompt, dict(batch=0)), (prompt, dict(rows_q=0))])
def test_nothing_to_do(call, args):
    call(**args)


def test_workspace():
    # 8 key heads of 128 values and one text: parts of at least four tiles, each a row of dim + 2 floats a head.
    c = cache(heads=8, dim=128)
    assert D.paged_attention_workspace(c, 1, 32, 100) == 0  # one part
    n = D.paged_attention_workspace(c, 1, 32, 16384)
    assert n > 0 and n % (32 * 130 * 4) == 0
    assert D.paged_attention_workspace(c, 4096, 32, 16384) == 0  # enough texts
    assert D.paged_attention_workspace(c, 1, 33, 16384) == 0 and D.paged_attention_workspace(None, 1, 1, 1) == 0


def test_first_calls_of_two_threads(monkeypatch):
    # The functions are looked up by the first call; one made meanwhile finds all of them or none.
    import threading
    import time
    real = D.lib()

    class Slow:
        def __getattr__(self, name):
            time.sleep(0.02)
            return getattr(real, name)

    monkeypatch.setattr(D, "_fns", {})
    monkeypatch.setattr(D, "lib", Slow)
    got = []

    def call(wait):
        time.sleep(wait)
        got.append(D.paged_attention_workspace(cache(heads=8, dim=128), 1, 32, 16384))

    threads = [threading.Thread(target=call, args=(w,)) for w in (0, 0.05, 0.09)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(got) == 3 and got[0] > 0 and len(set(got)) == 1
