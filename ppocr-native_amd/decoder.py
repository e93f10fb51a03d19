"""The layers of a text decoder on device memory, over the C ABI
(ppocr_hip_rms_norm, ppocr_hip_q4_product, ppocr_hip_kv_append,
ppocr_hip_paged_attention, ppocr_hip_window_attention, the append with the
rotation of positions, the cache in 4 bits ppocr_hip_kv4_*, beam search
ppocr_hip_beam_*): what a program calls that writes or corrects text token by
token after the recogniser.

Arguments are device addresses (integers; 0 = none), sizes, strides in values
(0 = rows without a gap) and a HIP stream (0 = the default stream); see
include/ppocr_hip.h for their meaning. Calls queue their kernels and return;
a refused call raises `GpuError` with the library's reason.
"""
from __future__ import annotations

import ctypes as C
import threading

from . import GpuError, lib

F32, BF16, F16, E4M3, I8 = range(5)

_fns: dict = {}
_ERR = 512


class _Reason(threading.local):
    """A thread's buffer for the reason of a refusal (made once: making it is a good part of a short call)."""

    def __init__(self):
        self.buffer = C.create_string_buffer(_ERR)


_reason = _Reason()


class KvCache(C.Structure):
    """A paged cache of keys and values (`ppocr_kv_cache`): addresses of `k`
    and `v`, `pages` pages of `page_size` tokens of `heads` heads of `dim`
    values, and the strides from page to page, token to token and head to head
    (all 0: [page][token][head][dim])."""

    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("pages", C.c_size_t), ("page_size", C.c_size_t),
                ("heads", C.c_size_t), ("dim", C.c_size_t), ("page_stride", C.c_size_t),
                ("token_stride", C.c_size_t), ("head_stride", C.c_size_t), ("type", C.c_int)]

    def __init__(self, k: int, v: int, pages: int, page_size: int, heads: int, dim: int, type: int = F32,
                 page_stride: int = 0, token_stride: int = 0, head_stride: int = 0):
        super().__init__(k, v, pages, page_size, heads, dim, page_stride, token_stride, head_stride, type)


class Kv4Cache(C.Structure):
    """A paged cache in 4 bits (`ppocr_kv4_cache`): the address of its pages,
    `pages` of them of `page_size` tokens of `heads` heads of `dim` values, a
    scale and a minimum each `group` (32, 64; 0: a head), pages `page_stride`
    bytes apart (0: `kv4_page_bytes`)."""

    _fields_ = [("data", C.c_void_p), ("pages", C.c_size_t), ("page_size", C.c_size_t), ("heads", C.c_size_t),
                ("dim", C.c_size_t), ("group", C.c_size_t), ("page_stride", C.c_size_t)]

    def __init__(self, data: int, pages: int, page_size: int, heads: int, dim: int, group: int = 64,
                 page_stride: int = 0):
        super().__init__(data, pages, page_size, heads, dim, group, page_stride)


class BeamState(C.Structure):
    """A dense state of each beam (`ppocr_beam_state`): rows of `bytes`, at
    addresses `from_` and `to`, strides in bytes (0: `bytes`)."""

    _fields_ = [("from_", C.c_void_p), ("to", C.c_void_p), ("bytes", C.c_size_t), ("from_stride", C.c_size_t),
                ("to_stride", C.c_size_t)]

    def __init__(self, from_: int, to: int, bytes: int, from_stride: int = 0, to_stride: int = 0):
        super().__init__(from_, to, bytes, from_stride, to_stride)


def _functions() -> dict:
    if not _fns:
        L, fns = lib(), {}
        p, n, i, f = C.c_void_p, C.c_size_t, C.c_int, C.c_float
        cache, cache4, end = C.POINTER(KvCache), C.POINTER(Kv4Cache), [p, C.c_char_p, n]
        for name, args in {
            "rms_norm": [p, n, p, n, p, p, n, p, n, p, n, n, i, i, n, f] + end,
            "q4_product": [p, n, p, n, p, p, p, p, p, n, n, n, n, n, i, i, i] + end,
            "kv_append": [p, n, p, n, cache, p, n, p, p, n, n] + end,
            "paged_attention": [p, n, cache, p, n, p, p, n, n, n, f, n, n, n, p, n] + end,
            "window_attention": [p, n, p, n, p, n, p, n, p, p, n, n, n, n, n, n, i, f, n, n] + end,
            "kv_append_rotated": [p, n, p, n, n, p, n, p, n, cache, p, n, p, p, p, p, n, i, n, n] + end,
            "kv4_append": [p, n, p, n, n, p, n, p, n, cache4, p, n, p, p, p, p, n, i, n, n, i] + end,
            "kv4_read": [p, n, p, n, cache4, p, n, p, p, n, n, i] + end,
            "beam_select": [p, n, p, p, p, p, p, p, C.c_int32, n, n, n, n, i, p, n] + end,
            "beam_reorder": [p, n, p, n, p, n, p, p, p, n, p, p, p, n, n] + end,
            "kv4_attention": [p, n, cache4, p, n, p, p, n, n, n, i, f, n, n, n, p, n] + end,
        }.items():
            fn = getattr(L, "ppocr_hip_" + name)
            fn.argtypes, fn.restype = args, i
            fns[name] = fn
        fn = L.ppocr_hip_paged_attention_workspace
        fn.argtypes, fn.restype = [cache, n, n, n], n
        fns["workspace"] = fn
        fn = L.ppocr_hip_kv4_attention_workspace
        fn.argtypes, fn.restype = [cache4, n, n, n], n
        fns["kv4_workspace"] = fn
        fn = L.ppocr_hip_kv4_page_bytes
        fn.argtypes, fn.restype = [n, n, n, n], n
        fns["kv4_page_bytes"] = fn
        fn = L.ppocr_hip_beam_select_workspace
        fn.argtypes, fn.restype = [n, n, n, n], n
        fns["select_workspace"] = fn
        fn = L.ppocr_hip_q4_product_tiles
        fn.argtypes, fn.restype = [n, n, n, i], n
        fns["tiles"] = fn
        _fns.update(fns)  # all at once: another thread may be looking
    return _fns


def _call(name: str, *args) -> None:
    err = _reason.buffer
    if (_fns or _functions())[name](*args, err, _ERR):
        raise GpuError(err.value.decode(errors="replace"))


def rms_norm(x: int, weight: int, y: int, rows: int, c: int, *, residual: int = 0, sum: int = 0, scales: int = 0,
             type: int = F32, y_type: int | None = None, group: int = 0, eps: float = 1e-6, x_stride: int = 0,
             residual_stride: int = 0, sum_stride: int = 0, y_stride: int = 0, stream: int = 0) -> None:
    """h = x + residual (into `sum`), y = h / sqrt(mean(h^2) + eps) * weight,
    in `type`, or in 8 bits (E4M3, I8) with `scales` a row or a group."""
    _call("rms_norm", x, x_stride, residual, residual_stride, weight, sum, sum_stride, y, y_stride, scales, rows, c,
          type, type if y_type is None else y_type, group, eps, stream)


def q4_product(x: int, q: int, scales: int, y: int, m: int, n: int, k: int, *, group: int = 128, zeros: int = 0,
               bias: int = 0, x_scales: int = 0, x_group: int = 0, x_type: int = F32, scale_type: int = F32,
               y_type: int = F32, x_stride: int = 0, y_stride: int = 0, stream: int = 0) -> None:
    """y = x W^T + bias for `m` rows, W[j][i] = scales[j][g] (q[j][i] - zeros[j][g]),
    4 bits a weight, g = i / group."""
    _call("q4_product", x, x_stride, x_scales, x_group, q, scales, zeros, bias, y, y_stride, m, n, k, group, x_type,
          scale_type, y_type, stream)


def q4_product_tiles(m: int, n: int, k: int, x_type: int = F32) -> int:
    """Tiles of 16 outputs that a workgroup of `q4_product` takes: which of its kernels runs."""
    return (_fns or _functions())["tiles"](m, n, k, x_type)


def kv_append(k: int, v: int, cache: KvCache, table: int, table_width: int, lengths: int, batch: int, rows: int, *,
              starts: int = 0, k_stride: int = 0, v_stride: int = 0, stream: int = 0) -> None:
    """Append `rows` rows of keys and values of `batch` texts (`starts`; 0: one
    each) to the cache, to the last places below each text's length."""
    _call("kv_append", k, k_stride, v, v_stride, cache, table, table_width, lengths, starts, batch, rows, stream)


def paged_attention_workspace(cache: KvCache, batch: int, heads: int, longest: int = 0) -> int:
    """Bytes of workspace with which `paged_attention` splits as far as it would."""
    return (_fns or _functions())["workspace"](cache, batch, heads, longest)


def paged_attention(q: int, cache: KvCache, table: int, table_width: int, lengths: int, y: int, batch: int, heads: int,
                    *, scale: float, window: int = 0, sinks: int = 0, longest: int = 0, workspace: int = 0,
                    workspace_bytes: int = 0, q_stride: int = 0, y_stride: int = 0, stream: int = 0) -> None:
    """Attention of one query row a text over its cache, the last `window`
    tokens and first `sinks` of it (window 0: all)."""
    _call("paged_attention", q, q_stride, cache, table, table_width, lengths, y, y_stride, batch, heads, scale, window,
          sinks, longest, workspace, workspace_bytes, stream)


def window_attention(q: int, k: int, v: int, y: int, starts_q: int, starts_k: int, batch: int, rows_q: int, rows_k: int,
                     heads: int, kv_heads: int, dim: int, *, scale: float, type: int = F32, window: int = 0,
                     sinks: int = 0, q_stride: int = 0, k_stride: int = 0, v_stride: int = 0, y_stride: int = 0,
                     stream: int = 0) -> None:
    """Causal attention of prompts with a sliding window and sinks."""
    _call("window_attention", q, q_stride, k, k_stride, v, v_stride, y, y_stride, starts_q, starts_k, batch, rows_q,
          rows_k, heads, kv_heads, dim, type, scale, window, sinks, stream)


def kv_append_rotated(k: int, v: int, cache: KvCache, table: int, table_width: int, lengths: int, batch: int, rows: int,
                      *, freqs: int = 0, rotary: int = 0, pairs: bool = False, positions: int = 0, q: int = 0,
                      q_out: int = 0, heads: int = 0, starts: int = 0, q_stride: int = 0, q_out_stride: int = 0,
                      k_stride: int = 0, v_stride: int = 0, stream: int = 0) -> None:
    """`kv_append` of keys turned by their positions (first `rotary` dims of a
    head, halves apart or in neighbouring `pairs`, angle position * freqs[j]);
    q's rows, turned alike, go to `q_out` (or stay in q, where they are one)."""
    _call("kv_append_rotated", q, q_stride, q_out, q_out_stride, heads, k, k_stride, v, v_stride, cache, table,
          table_width, lengths, starts, positions, freqs, rotary, pairs, batch, rows, stream)


def kv4_page_bytes(page_size: int, heads: int, dim: int, group: int = 64) -> int:
    """Bytes of a page of a cache in 4 bits (0 for sizes that are refused)."""
    return (_fns or _functions())["kv4_page_bytes"](page_size, heads, dim, group)


def kv4_append(k: int, v: int, cache: Kv4Cache, table: int, table_width: int, lengths: int, batch: int, rows: int, *,
               type: int = F32, freqs: int = 0, rotary: int = 0, pairs: bool = False, positions: int = 0, q: int = 0,
               q_out: int = 0, heads: int = 0, starts: int = 0, q_stride: int = 0, q_out_stride: int = 0,
               k_stride: int = 0, v_stride: int = 0, stream: int = 0) -> None:
    """`kv_append_rotated` into a cache in 4 bits, from rows of `type`."""
    _call("kv4_append", q, q_stride, q_out, q_out_stride, heads, k, k_stride, v, v_stride, cache, table, table_width,
          lengths, starts, positions, freqs, rotary, pairs, batch, rows, type, stream)


def kv4_read(k: int, v: int, cache: Kv4Cache, table: int, table_width: int, lengths: int, batch: int, rows: int, *,
             starts: int = 0, type: int = F32, k_stride: int = 0, v_stride: int = 0, stream: int = 0) -> None:
    """The last tokens below each text's length, out of a cache in 4 bits, into `rows` rows of k and v."""
    _call("kv4_read", k, k_stride, v, v_stride, cache, table, table_width, lengths, starts, batch, rows, type, stream)


def kv4_attention_workspace(cache: Kv4Cache, batch: int, heads: int, longest: int = 0) -> int:
    """Bytes of workspace with which `kv4_attention` splits as far as it would."""
    return (_fns or _functions())["kv4_workspace"](cache, batch, heads, longest)


def kv4_attention(q: int, cache: Kv4Cache, table: int, table_width: int, lengths: int, y: int, batch: int, heads: int,
                  *, scale: float, type: int = F32, window: int = 0, sinks: int = 0, longest: int = 0,
                  workspace: int = 0, workspace_bytes: int = 0, q_stride: int = 0, y_stride: int = 0,
                  stream: int = 0) -> None:
    """`paged_attention` over a cache in 4 bits, of queries of `type`."""
    _call("kv4_attention", q, q_stride, cache, table, table_width, lengths, y, y_stride, batch, heads, type, scale,
          window, sinks, longest, workspace, workspace_bytes, stream)


def beam_select_workspace(batch: int, beams: int, vocab: int, keep: int) -> int:
    """Bytes of workspace that `beam_select` needs (0 for sizes that are refused)."""
    return (_fns or _functions())["select_workspace"](batch, beams, vocab, keep)


def beam_select(logits: int, scores: int, out_scores: int, parents: int, tokens: int, batch: int, beams: int,
                vocab: int, keep: int, *, workspace: int, workspace_bytes: int, type: int = F32, ended: int = 0,
                out_ended: int = 0, end: int = -1, stride: int = 0, stream: int = 0) -> None:
    """The `keep` best continuations of each text's beams by one of `vocab`
    tokens, scores[i] + log_softmax(logits[i])[v], the best first."""
    _call("beam_select", logits, stride, scores, ended, out_scores, parents, tokens, out_ended, end, batch, beams, vocab,
          keep, type, workspace, workspace_bytes, stream)


def _array(of, items):
    return items if isinstance(items, C.Array) else (of * len(items))(*items)


def beam_reorder(caches, parents: int, table: int, table_out: int, table_width: int, lengths: int, spare: int,
                 spare_out: int, batch: int, beams: int, *, states=(), stream: int = 0) -> None:
    """Each beam goes on from its parent's state: `caches` (KvCache or Kv4Cache,
    a sequence or a ctypes array of them) with their page table, and dense
    `states` (BeamState)."""
    n = len(caches)
    four = n and isinstance(caches[0], Kv4Cache)
    held, dense = _array(Kv4Cache if four else KvCache, caches) if n else None, _array(BeamState, states) if len(states) else None
    _call("beam_reorder", None if four else held, 0 if four else n, held if four else None, n if four else 0, dense,
          len(states), parents, table, table_out, table_width, lengths, spare, spare_out, batch, beams, stream)
