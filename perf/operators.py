"""The layers of an autoregressive text decoder, as cases to be measured.

A program that reads lines with the recogniser and then has a decoder complete
or correct the text calls these on device memory, one after another: the
root-mean-square norm with the residual's addition (`norm`), products with
4-bit weights (`product`), the append of new keys and values to a paged cache
(`append`), attention of one new token over that cache (`decode`), and
attention of whole prompts with a sliding window and sinks (`prompt`).

Where `own` is false, `run` computes them from elementary torch operations in
32 bits, rounded once at the end.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
WORKSPACE = 32 << 20  # bytes a program keeps for the decode attention's parts


def _decoder():
    """The framework's module of decoder layers."""
    if "ppocr_native_amd" not in sys.modules:
        d = ROOT / "ppocr-native_amd"
        spec = importlib.util.spec_from_file_location("ppocr_native_amd", d / "__init__.py",
                                                      submodule_search_locations=[str(d)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ppocr_native_amd"] = mod
        spec.loader.exec_module(mod)
    from ppocr_native_amd import decoder
    return decoder


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- the cases

def listed() -> list[dict]:
    return [
        # The norm before a layer while one text is written: one row, so the
        # call's latency is what counts.
        {"name": "norm 1x4096 bf16", "op": "norm", "rows": 1, "c": 4096, "type": "bf16", "out": "same", "group": 0,
         "residual": True},
        # The same norm over a long prompt's rows, its output in 8 bits with a
        # scale for each 128 values, for a product that takes 8 bits.
        {"name": "norm 8192x8192 e4m3", "op": "norm", "rows": 8192, "c": 8192, "type": "bf16", "out": "e4m3",
         "group": 128, "residual": True},
        # One text's row through a square layer: the smallest product.
        {"name": "product 1 4096>4096 bf16", "op": "product", "m": 1, "n": 4096, "k": 4096, "group": 128,
         "type": "bf16", "scales": "bf16", "zeros": False},
        # Sixteen texts at once through a wide layer, small groups with zero
        # points of their own.
        {"name": "product 16 4096>28672 f16", "op": "product", "m": 16, "n": 28672, "k": 4096, "group": 32,
         "type": "f16", "scales": "f16", "zeros": True},
        # Five rows in f32, the framework's own type, onto the benchmark's
        # 18385 classes: odd sizes, a last group that is cut off.
        {"name": "product 5 1000>18385 f32", "op": "product", "m": 5, "n": 18385, "k": 1000, "group": 64,
         "type": "f32", "scales": "f32", "zeros": True},
        # Each of 64 texts appends its newest token to the cache.
        {"name": "append 64 tokens", "op": "append", "batch": 64, "most": 1, "page": 16, "held": 250, "kv_heads": 8,
         "dim": 128, "type": "bf16"},
        # Six prompts of up to 1500 tokens go into the cache at once.
        {"name": "append 6 prompts", "op": "append", "batch": 6, "most": 1500, "page": 64, "held": 100, "kv_heads": 8,
         "dim": 128, "type": "f16"},
        # One short text: latency.
        {"name": "decode 1x300 f16", "op": "decode", "batch": 1, "longest": 300, "page": 16, "heads": 12,
         "kv_heads": 4, "dim": 64, "type": "f16", "window": 0, "sinks": 0},
        # A full batch of texts of every length up to 16384.
        {"name": "decode 32x16384 bf16", "op": "decode", "batch": 32, "longest": 16384, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "sinks": 0},
        # Three very long texts of which a window and four sinks are seen.
        {"name": "decode 3x100000 window f32", "op": "decode", "batch": 3, "longest": 100000, "page": 24, "heads": 16,
         "kv_heads": 2, "dim": 128, "type": "f32", "window": 4096, "sinks": 4},
        # Short ragged lines with the recogniser's own eight heads of 15.
        {"name": "prompt 9x160 f32", "op": "prompt", "batch": 9, "longest": 160, "heads": 8, "kv_heads": 8, "dim": 15,
         "type": "f32", "window": 80, "sinks": 4, "past": 0},
        # Two long prompts.
        {"name": "prompt 2x8192 bf16", "op": "prompt", "batch": 2, "longest": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "bf16", "window": 2048, "sinks": 4, "past": 0},
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng: random.Random) -> tuple[int, int]:
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 7, 8]), kv


def _drawn(rng: random.Random) -> dict:
    op = rng.choice(["norm", "product", "product", "append", "decode", "decode", "prompt", "prompt"])
    t = rng.choice(["bf16", "f16", "f32"])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 8192), "c": rng.choice([_log(rng, 60, 16384), 8 * _log(rng, 15, 2048)]),
                "type": t, "out": rng.choice(["same", "same", "e4m3"]), "group": rng.choice([0, 32, 64, 128]),
                "residual": rng.random() < 0.7}
    if op == "product":
        return {"op": op, "m": _log(rng, 1, 64), "n": _log(rng, 100, 28672),
                "k": rng.choice([_log(rng, 100, 16384), 128 * _log(rng, 1, 128)]), "group": rng.choice([32, 64, 128]),
                "type": t, "scales": rng.choice([t, "f32"]), "zeros": rng.random() < 0.6}
    dim = rng.choice([15, 32, 64, 80, 96, 128, 128, 192, 256])
    heads, kv = _heads(rng)
    if op == "append":
        return {"op": op, "batch": _log(rng, 1, 64), "most": rng.choice([1, _log(rng, 2, 1500)]),
                "page": rng.choice([16, 32, 64, 128, rng.randint(1, 100)]), "held": _log(rng, 1, 500), "kv_heads": kv,
                "dim": dim, "type": t}
    if op == "decode":
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        return {"op": op, "batch": _log(rng, 1, 96), "longest": _log(rng, 1, 100000),
                "page": rng.choice([16, 32, 64, 128, rng.randint(1, 100)]), "heads": heads, "kv_heads": kv, "dim": dim,
                "type": t, "window": window, "sinks": rng.choice([0, 1, 4, 60]) if window else 0}
    return {"op": op, "batch": _log(rng, 1, 24), "longest": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv,
            "dim": dim, "type": t, "window": rng.choice([0, _log(rng, 8, 4096), _log(rng, 8, 4096)]),
            "sinks": rng.choice([0, 1, 4, 60]), "past": rng.choice([0, 0, _log(rng, 1, 2000)])}


def _scope(case: dict) -> float:
    """What the plain form keeps in memory at once, in values: a drawn case has no more than the largest listed."""
    if case["op"] == "append":
        return case["batch"] * (case["held"] + case["most"]) * case["kv_heads"] * case["dim"] / (64 * 1500 * 8 * 32)
    if case["op"] == "decode":
        return case["batch"] * case["longest"] * max(case["kv_heads"] * case["dim"], case["heads"]) / (32 * 16384 * 1024)
    if case["op"] == "prompt":
        rows = case["longest"]
        return case["batch"] * case["heads"] * rows * (rows + case["past"]) / (2 * 32 * 8192 * 8192)
    return 0.0


def draw(rng: random.Random) -> dict:
    most = {op: max(max(w["bytes"], w["flops"] / 50) for c in listed() if c["op"] == op for w in [work(c)])
            for op in ("norm", "product", "append", "decode", "prompt")}
    while True:
        case = _drawn(rng)
        w = work(case)
        if _scope(case) <= 1 and max(w["bytes"], w["flops"] / 50) <= most[case["op"]]:
            return case


# --------------------------------------------------- lengths, from the case alone

def _lengths(case: dict, salt: int) -> list[int]:
    """The lengths of a batch's texts: the first is the longest, the others anything down to one token (a prompt's also to none)."""
    rng = random.Random(salt * 1000003 + case["batch"] * 7919 + case["longest"])
    least = 0 if case["op"] == "prompt" else 1
    return [case["longest"]] + [rng.randint(least, case["longest"]) for _ in range(case["batch"] - 1)]


def _news(case: dict) -> tuple[list[int], list[int]]:
    """An append's new tokens and the tokens held before them, for each text."""
    rng = random.Random(case["batch"] * 7919 + case["most"] * 31 + case["held"])
    new = [case["most"]] + [rng.randint(1, case["most"]) for _ in range(case["batch"] - 1)]
    return new, [rng.randint(0, case["held"]) for _ in new]


def _size(t: str) -> int:
    return {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}[t]


def _seen(before: int, window: int, sinks: int) -> int:
    """How many keys a query sees that is number `before` + 1 of its text."""
    n = before + 1
    return n if not window or n <= window else window + min(sinks, n - window)


def work(case: dict) -> dict:
    op = case["op"]
    if op == "norm":
        rows, c, s = case["rows"], case["c"], _size(case["type"])
        per = s + (2 * s if case["residual"] else 0) + (1 if case["out"] == "e4m3" else s)
        scales = 4 * rows * (-(-c // case["group"]) if case["group"] else 1) if case["out"] == "e4m3" else 0
        return {"bytes": rows * c * per + c * s + scales, "flops": 5 * rows * c}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // case["group"])
        return {"bytes": n * ((k + 1) // 2) + n * groups * (_size(case["scales"]) + int(case["zeros"])) +
                (m * k + m * n) * _size(case["type"]), "flops": 2 * m * n * k}
    row = case["kv_heads"] * case["dim"] * _size(case["type"])
    if op == "append":
        return {"bytes": 4 * sum(_news(case)[0]) * row, "flops": 0}
    q = case["heads"] * case["dim"] * _size(case["type"])
    if op == "decode":
        seen = [_seen(n - 1, case["window"], case["sinks"]) for n in _lengths(case, 1)]
        return {"bytes": 2 * sum(seen) * row + 2 * len(seen) * q, "flops": 4 * sum(seen) * case["heads"] * case["dim"]}
    seen, rows, past = 0, 0, case["past"]
    for n in _lengths(case, 2):
        w = case["window"]
        # Sums over positions past .. past + n - 1 of _seen, in closed form.
        full = lambda p: p * (p + 1) // 2  # noqa: E731 - keys seen by positions 0 .. p - 1, nothing hidden
        if not w:
            seen += full(past + n) - full(past)
        else:
            def upto(p):
                if p <= w:
                    return full(p)
                s, more = case["sinks"], p - w
                near = min(more, s)
                return full(w) + more * w + near * (near + 1) // 2 + (more - near) * s
            seen += upto(past + n) - upto(past)
        rows += n
    return {"bytes": 2 * rows * q + 2 * (rows + past * case["batch"]) * row,
            "flops": max(1, 4 * seen * case["heads"] * case["dim"])}


# ---------------------------------------------------------------- the inputs

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(DEV).manual_seed(seed)


def _normal(g, shape, t, scale=1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(TYPES[t])


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(lengths: list[int]) -> list[int]:
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _pages(g, lengths: list[int], page: int, spare: int):
    """A page table for these lengths: the pages in shuffled order, -1 past each text's own."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = torch.tensor(_starts(need)[:-1], device=DEV)[:, None] + torch.arange(max(need + [1]), device=DEV)[None]
    own_page = torch.arange(max(need + [1]), device=DEV)[None] < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(own_page, order[at.clamp(max=pages - 1)], torch.full_like(order[:1], -1))
    return table.to(torch.int32).contiguous(), pages


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    op, t = case["op"], case["type"]
    s = {"case": case}
    if op == "norm":
        rows, c = case["rows"], case["c"]
        # A residual stream: a few channels far larger than the others.
        loud = 1 + 20 * (torch.rand(c, generator=g, device=DEV) < 0.005).float()
        s["x"] = (torch.randn(rows, c, generator=g, device=DEV) * 0.5).to(TYPES[t])
        s["residual"] = (torch.randn(rows, c, generator=g, device=DEV) * 2 * loud).to(TYPES[t]) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(c, generator=g, device=DEV)).to(TYPES[t])
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["y"] = torch.empty(rows, c, dtype=TYPES[t if case["out"] == "same" else "e4m3"], device=DEV)
        groups = -(-c // case["group"]) if case["group"] else 1
        s["scales"] = torch.empty(rows, groups, device=DEV) if case["out"] == "e4m3" else None
        return s
    if op == "product":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        groups = -(-k // group)
        s["x"] = _normal(g, (m, k), t)
        s["q"] = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8)
        s["scales"] = ((0.5 + torch.rand(n, groups, generator=g, device=DEV)) / (4.6 * math.sqrt(k))).to(TYPES[case["scales"]])
        s["zeros"] = torch.randint(4, 12, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        s["y"] = torch.empty(m, n, dtype=TYPES[t], device=DEV)
        return s
    kv, dim = case["kv_heads"], case["dim"]
    if op == "append":
        new, held = _news(case)
        lengths = [a + b for a, b in zip(new, held)]
        s["table"], pages = _pages(g, lengths, case["page"], 3)
        s["lengths"], s["starts"] = _ints(lengths), _ints(_starts(new))
        s["k_cache"] = _normal(g, (pages, case["page"], kv, dim), t)
        s["v_cache"] = _normal(g, (pages, case["page"], kv, dim), t)
        s["k"], s["v"] = _normal(g, (sum(new), kv, dim), t), _normal(g, (sum(new), kv, dim), t)
        return s
    heads = case["heads"]
    s["scale"] = dim ** -0.5
    if op == "decode":
        lengths = _lengths(case, 1)
        s["table"], pages = _pages(g, lengths, case["page"], 3)
        s["lengths"] = _ints(lengths)
        s["longest"] = max(lengths)
        s["k_cache"] = _normal(g, (pages, case["page"], kv, dim), t)
        s["v_cache"] = _normal(g, (pages, case["page"], kv, dim), t)
        s["q"] = _normal(g, (case["batch"], heads, dim), t, 2.0)
        s["y"] = torch.empty_like(s["q"])
        s["work"] = torch.empty(WORKSPACE, dtype=torch.uint8, device=DEV)
        return s
    nq = _lengths(case, 2)
    nk = [n + case["past"] for n in nq]
    s["nq"], s["nk"] = nq, nk
    s["cu_q"], s["cu_k"] = _ints(_starts(nq)), _ints(_starts(nk))
    s["q"] = _normal(g, (sum(nq), heads, dim), t, 2.0)
    s["k"], s["v"] = _normal(g, (sum(nk), kv, dim), t), _normal(g, (sum(nk), kv, dim), t)
    s["y"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------- the plain forms

def _plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    if case["residual"]:
        h = (h + s["residual"].float()).to(s["x"].dtype)
        total, h = h, h.float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    out = {"sum": total} if case["residual"] else {}
    if case["out"] == "same":
        return {**out, "y": y.to(s["x"].dtype)}
    rows, c = y.shape
    group = case["group"] or c
    cut = torch.nn.functional.pad(y, (0, -c % group)).view(rows, -1, group)
    scales = cut.abs().amax(-1) / 448
    y8 = (cut * (1 / scales.clamp(min=1e-38))[..., None]).clamp(-448, 448).view(rows, -1)[:, :c]
    return {**out, "y": y8.to(torch.float8_e4m3fn), "scales": scales}


def _plain_product(s):
    case = s["case"]
    k, group = case["k"], case["group"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), -1).flatten(1)[:, :k].float()
    zeros = s["zeros"].float() if s["zeros"] is not None else torch.full_like(s["scales"], 8, dtype=torch.float32)
    w = (q - zeros.repeat_interleave(group, 1)[:, :k]) * s["scales"].float().repeat_interleave(group, 1)[:, :k]
    return (s["x"].float() @ w.t().contiguous()).to(s["x"].dtype)


def _plain_append(s):
    page = s["case"]["page"]
    rows = torch.arange(s["k"].shape[0], device=DEV)
    text = torch.searchsorted(s["starts"], rows.to(torch.int32), right=True) - 1
    at = (s["lengths"] - s["starts"][1:])[text] + rows
    page_of = s["table"][text, at // page].long()
    s["k_cache"][page_of, at % page] = s["k"]
    s["v_cache"][page_of, at % page] = s["v"]
    return s["k_cache"], s["v_cache"]


def _attend(q, k, v, hidden, scale):
    """Softmax attention of q [batch, kv heads, rows, dim] over k, v [batch, kv heads, keys, dim], none of the `hidden` keys seen; a row that sees none gives zeros."""
    p = torch.matmul(q * scale, k.transpose(-1, -2).contiguous())
    p.masked_fill_(hidden, -math.inf)
    most = p.amax(-1, keepdim=True)
    p.sub_(most.masked_fill_(most == -math.inf, 0)).exp_()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_decode(s):
    case = s["case"]
    b, kv, dim = case["batch"], case["kv_heads"], case["dim"]
    tokens = torch.arange(s["longest"], device=DEV)
    page_of = s["table"].clamp(min=0).long()[:, tokens // case["page"]]
    k = s["k_cache"][page_of, tokens % case["page"]].transpose(1, 2).float()
    v = s["v_cache"][page_of, tokens % case["page"]].transpose(1, 2).float()
    n = s["lengths"][:, None]
    hidden = tokens >= n
    if case["window"]:
        hidden = hidden | ((tokens < n - case["window"]) & (tokens >= case["sinks"]))
    y = _attend(s["q"].float().view(b, kv, -1, dim), k, v, hidden[:, None, None], s["scale"])
    return y.reshape(b, -1, dim).to(s["q"].dtype)


def _plain_prompt(s):
    case = s["case"]
    b, heads, kv, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    nq, nk = s["cu_q"].diff()[:, None], s["cu_k"].diff()[:, None]
    iq, ik = torch.arange(max(s["nq"]), device=DEV), torch.arange(max(s["nk"]), device=DEV)
    rows, keys = (s["cu_q"][:-1, None] + iq), (s["cu_k"][:-1, None] + ik)
    q = s["q"][rows.clamp(max=s["q"].shape[0] - 1)].float().view(b, -1, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    k = s["k"][keys.clamp(max=s["k"].shape[0] - 1)].float().transpose(1, 2)
    v = s["v"][keys.clamp(max=s["v"].shape[0] - 1)].float().transpose(1, 2)
    at = (nk - nq + iq)[:, :, None]
    hidden = (ik > at) | (ik >= nk[..., None])
    if case["window"]:
        hidden = hidden | ((ik <= at - case["window"]) & (ik >= case["sinks"]))
    hidden = hidden[:, None].expand(b, heads // kv, -1, -1).reshape(b, 1, -1, ik.numel())
    y = _attend(q.reshape(b, kv, -1, dim), k, v, hidden, s["scale"])
    y = y.view(b, kv, heads // kv, -1, dim).permute(0, 3, 1, 2, 4).reshape(b, -1, heads, dim)
    return y[iq < nq].to(s["q"].dtype)


# ----------------------------------------------------------------- one pass

def _own(s):
    D = _decoder()
    case = s["case"]
    op, t = case["op"], getattr(D, case["type"].upper())
    ptr = lambda x: x.data_ptr() if x is not None else 0  # noqa: E731
    if op == "norm":
        D.rms_norm(ptr(s["x"]), ptr(s["weight"]), ptr(s["y"]), case["rows"], case["c"], residual=ptr(s["residual"]),
                   sum=ptr(s["sum"]), scales=ptr(s["scales"]), type=t, y_type=t if case["out"] == "same" else D.E4M3,
                   group=case["group"], eps=1e-6, stream=_stream())
        return {k: s[k] for k in ("sum", "y", "scales") if s[k] is not None}
    if op == "product":
        D.q4_product(ptr(s["x"]), ptr(s["q"]), ptr(s["scales"]), ptr(s["y"]), case["m"], case["n"], case["k"],
                     group=case["group"], zeros=ptr(s["zeros"]), x_type=t, y_type=t,
                     scale_type=getattr(D, case["scales"].upper()), stream=_stream())
        return s["y"]
    if op in ("append", "decode"):
        if "cache" not in s:
            s["cache"] = D.KvCache(ptr(s["k_cache"]), ptr(s["v_cache"]), s["k_cache"].shape[0], case["page"],
                                   case["kv_heads"], case["dim"], type=t)
    if op == "append":
        D.kv_append(ptr(s["k"]), ptr(s["v"]), s["cache"], ptr(s["table"]), s["table"].shape[1], ptr(s["lengths"]),
                    case["batch"], s["k"].shape[0], starts=ptr(s["starts"]), stream=_stream())
        return s["k_cache"], s["v_cache"]
    if op == "decode":
        D.paged_attention(ptr(s["q"]), s["cache"], ptr(s["table"]), s["table"].shape[1], ptr(s["lengths"]), ptr(s["y"]),
                          case["batch"], case["heads"], scale=s["scale"], window=case["window"], sinks=case["sinks"],
                          longest=s["longest"], workspace=ptr(s["work"]), workspace_bytes=WORKSPACE, stream=_stream())
        return s["y"]
    D.window_attention(ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["y"]), ptr(s["cu_q"]), ptr(s["cu_k"]), case["batch"],
                       s["q"].shape[0], s["k"].shape[0], case["heads"], case["kv_heads"], case["dim"], type=t,
                       scale=s["scale"], window=case["window"], sinks=case["sinks"], stream=_stream())
    return s["y"]


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "product": _plain_product, "append": _plain_append, "decode": _plain_decode,
            "prompt": _plain_prompt}[state["case"]["op"]](state)


# ------------------------------------------------------------------ in 64 bits

def _one_text(q, k, v, first, window, sinks, scale):
    """Queries at positions first, first + 1, ... of a text over its keys k, v: [rows, heads, dim], all f64, 512 rows at a time."""
    rows, heads, dim = q.shape
    per = heads // k.shape[1]
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    out = torch.zeros_like(q)
    j = torch.arange(k.shape[0], device=DEV)
    for a in range(0, rows, 512):
        part = q[a:a + 512]
        p = torch.arange(first + a, first + a + part.shape[0], device=DEV)[:, None]
        ok = j[None] <= p
        if window:
            ok = ok & ((j[None] > p - window) | (j[None] < sinks))
        for h in range(k.shape[1]):
            z = torch.einsum("rgd,dk->grk", part[:, h * per:(h + 1) * per], kt[h]) * scale
            z = torch.where(ok, z, torch.full_like(z[:1, :1, :1], -math.inf))
            e = torch.where(ok, torch.exp(z - z.max(-1, keepdim=True).values.clamp(min=-1e300)), torch.zeros_like(z[:1, :1, :1]))
            total = e.sum(-1, keepdim=True)
            e = e / torch.where(total > 0, total, torch.ones_like(total))
            out[a:a + 512, h * per:(h + 1) * per] = torch.einsum("grk,kd->rgd", e, vt[h])
    return out


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        out, h = {}, s["x"].double()
        if case["residual"]:
            out["sum"] = h + s["residual"].double()
            h = out["sum"].to(s["x"].dtype).double()  # the norm is of the stored sum
        y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["c"] + 1e-6) * s["weight"].double()
        if case["out"] == "same":
            return {**out, "y": y}
        size = case["group"] or case["c"]
        scales = torch.stack([part.abs().max(-1).values for part in y.split(size, -1)], -1) / 448
        spread = scales.repeat_interleave(size, -1)[:, :case["c"]]
        return {**out, "y": y / spread, "scales": scales}
    if op == "product":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        out = torch.empty(m, n, dtype=torch.float64, device=DEV)
        for a in range(0, n, 4096):
            raw = s["q"][a:a + 4096].to(torch.int64)
            w = torch.empty(raw.shape[0], 2 * raw.shape[1], dtype=torch.float64, device=DEV)
            w[:, 0::2], w[:, 1::2] = (raw % 16).double(), (raw // 16).double()
            of = torch.arange(k, device=DEV) // group
            w = w[:, :k] - (s["zeros"][a:a + 4096].double()[:, of] if case["zeros"] else 8.0)
            out[:, a:a + 4096] = s["x"].double() @ (w * s["scales"][a:a + 4096].double()[:, of]).t()
        return out
    if op == "append":
        new, held = _news(case)
        table = s["table"].tolist()
        at = [table[b][(held[b] + i) // case["page"]] * case["page"] + (held[b] + i) % case["page"]
              for b in range(case["batch"]) for i in range(new[b])]
        at = torch.tensor(at, device=DEV)
        out = []
        for cache, rows in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
            flat = cache.double().flatten(0, 1).clone()
            flat[at] = rows.double()
            out.append(flat.view(cache.shape))
        return tuple(out)
    if op == "decode":
        out = []
        for b, n in enumerate(_lengths(case, 1)):
            at = torch.arange(n, device=DEV)
            if case["window"]:
                at = at[(at >= n - case["window"]) | (at < case["sinks"])]
            page = s["table"][b].long()[at // case["page"]]
            k, v = s["k_cache"][page, at % case["page"]].double(), s["v_cache"][page, at % case["page"]].double()
            out.append(_one_text(s["q"][b:b + 1].double(), k, v, at.numel() - 1, 0, 0, s["scale"]))
        return torch.cat(out)
    out, a, c = [], 0, 0
    for nq, nk in zip(s["nq"], s["nk"]):
        if nq:
            out.append(_one_text(s["q"][a:a + nq].double(), s["k"][c:c + nk].double(), s["v"][c:c + nk].double(), nk - nq,
                                 case["window"], case["sinks"], s["scale"]))
        a, c = a + nq, c + nk
    return torch.cat(out)
