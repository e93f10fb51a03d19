"""What a text decoder needs to write with, as cases to be measured.

A program that has a decoder write text behind the recogniser calls these on
device memory between the layers' products: the rotation of queries and keys
by their positions with the append of keys and values to a paged cache
(`append`), the same into a cache held in 4 bits, and the reading of tokens
back from it for a prompt's attention (`store4`), attention of one new token
over that cache (`attend4`), the choice of the next tokens by beam search
(`select`), and the reordering of the beams' caches and histories after it
(`reorder`).

Where `own` is false, `run` computes them from elementary torch operations in
32 bits (angles, and scores next to a border, in 64), rounded once at the end.

A 4-bit cache is bytes [page][key head][chunk], a chunk the planes

    K codes   [token][4 quarters][P / 32][4]   scales [token][group]   minima [token][group]
    V codes   [token / 4][16][P / 32][4]       scales [token][group]   minima [token][group]

with scales and minima in f16 and heads padded to P = 32, 64, 96, 128, 192 or
256 values. A code byte holds two neighbouring dims, the even one in its low
bits: byte j of quarter q, block c of a token's K has dims 32 c + 8 q + 2 j,
byte t of column i, block c of four tokens' V has dims 32 c + 2 i of the t-th
of them. A code n stands for n scale + minimum.
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
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WORKSPACE = 64 << 20  # bytes a program keeps for the parts of a split cache and of the beams' vocabularies


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
        # Each of 64 texts appends its newest token, turned by its position: latency.
        {"name": "append 64 tokens", "op": "append", "batch": 64, "most": 1, "page": 16, "held": 250, "far": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "pairs": False, "type": "bf16"},
        # Six prompts of up to 1500 tokens go into the cache at once.
        {"name": "append 6 prompts", "op": "append", "batch": 6, "most": 1500, "page": 64, "held": 100, "far": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "pairs": False, "type": "f16"},
        # Lines in f32, the framework's own type, a third of each head turned in neighbouring pairs, and positions far
        # past the places: the program has dropped the texts' oldest pages.
        {"name": "append 9 lines far", "op": "append", "batch": 9, "most": 160, "page": 24, "held": 60, "far": 700000,
         "heads": 8, "kv_heads": 8, "dim": 96, "rotary": 32, "pairs": True, "type": "f32"},
        # The newest tokens of 64 texts into a 4-bit cache, and back as they are held.
        {"name": "store4 64 tokens", "op": "store4", "batch": 64, "most": 1, "page": 16, "held": 250, "far": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "pairs": False, "type": "bf16", "group": 64,
         "read": "new"},
        # Four chunks of prompts into a 4-bit cache; all that their texts hold then comes back as rows, for the
        # attention of the chunks' queries.
        {"name": "store4 4 chunks", "op": "store4", "batch": 4, "most": 4096, "page": 64, "held": 4000, "far": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "pairs": False, "type": "f16", "group": 32,
         "read": "all"},
        # One short text over its 4-bit cache: latency.
        {"name": "attend4 1x300 f16", "op": "attend4", "batch": 1, "longest": 300, "page": 16, "heads": 12,
         "kv_heads": 4, "dim": 64, "group": 0, "type": "f16", "window": 0, "sinks": 0},
        # A full batch of texts of every length up to 16384.
        {"name": "attend4 32x16384 bf16", "op": "attend4", "batch": 32, "longest": 16384, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "group": 64, "type": "bf16", "window": 0, "sinks": 0},
        # Three very long texts of which a window and four sinks are seen, small groups, heads of 96.
        {"name": "attend4 3x100000 window f32", "op": "attend4", "batch": 3, "longest": 100000, "page": 48, "heads": 16,
         "kv_heads": 2, "dim": 96, "group": 32, "type": "f32", "window": 4096, "sinks": 4},
        # A text's first step over the benchmark's 18385 classes: one live beam gives four.
        {"name": "select 1x4 of 18385 first", "op": "select", "batch": 1, "beams": 4, "vocab": 18385, "keep": 4,
         "type": "f32", "first": True, "ended": False, "masked": 0.0},
        # Many texts of eight beams over a large vocabulary, some beams ended, some tokens forbidden.
        {"name": "select 32x8 of 131072", "op": "select", "batch": 32, "beams": 8, "vocab": 131072, "keep": 8,
         "type": "bf16", "first": False, "ended": True, "masked": 0.1},
        # One text's four beams and one layer of cache: latency.
        {"name": "reorder 4 beams", "op": "reorder", "batch": 1, "beams": 4, "layers": 1, "longest": 100, "page": 16,
         "kv_heads": 8, "dim": 64, "steps": 100, "type": "f32"},
        # Sixteen texts of four beams, twelve layers.
        {"name": "reorder 16x4 beams, 12 layers", "op": "reorder", "batch": 16, "beams": 4, "layers": 12,
         "longest": 600, "page": 64, "kv_heads": 8, "dim": 128, "steps": 600, "type": "bf16"},
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng: random.Random) -> tuple[int, int]:
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 7, 8]), kv


def _drawn(rng: random.Random) -> dict:
    op = rng.choice(["append", "append", "store4", "store4", "attend4", "attend4", "attend4", "select", "select", "reorder"])
    t = rng.choice(["bf16", "f16", "f32"])
    if op == "select":
        beams = _log(rng, 1, 32)
        return {"op": op, "batch": _log(rng, 1, 64), "beams": beams, "vocab": _log(rng, 50, 160000),
                "keep": rng.choice([beams, beams, 2 * beams, _log(rng, 1, 32)]), "type": t, "first": rng.random() < 0.2,
                "ended": rng.random() < 0.4, "masked": rng.choice([0.0, 0.0, 0.1, 0.95])}
    dim = rng.choice([15, 32, 64, 80, 96, 128, 128, 192, 256])
    heads, kv = _heads(rng)
    if op == "reorder":
        return {"op": op, "batch": _log(rng, 1, 32), "beams": _log(rng, 2, 16), "layers": _log(rng, 1, 40),
                "longest": _log(rng, 1, 4000), "page": rng.choice([16, 32, 64, rng.randint(1, 100)]), "kv_heads": kv,
                "dim": dim, "steps": _log(rng, 10, 2000), "type": t}
    if op == "attend4":
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        return {"op": op, "batch": _log(rng, 1, 96), "longest": _log(rng, 1, 100000),
                "page": 16 * rng.choice([1, 2, 4, 8, rng.randint(1, 12)]), "heads": heads, "kv_heads": kv, "dim": dim,
                "group": rng.choice([0, 32, 64]), "type": t, "window": window,
                "sinks": rng.choice([0, 1, 4, 60]) if window else 0}
    case = {"op": op, "batch": _log(rng, 1, 64), "most": rng.choice([1, _log(rng, 2, 4096)]),
            "page": rng.choice([16, 32, 64, 128, rng.randint(1, 100)]), "held": _log(rng, 1, 4000),
            "far": rng.choice([0, 0, _log(rng, 1, 1 << 24)]), "heads": heads, "kv_heads": kv, "dim": dim,
            "rotary": rng.choice([dim // 2 * 2, dim // 2 * 2, dim // 4 * 2]), "pairs": rng.random() < 0.5, "type": t}
    if op == "store4":
        case["page"] = 16 * max(1, case["page"] // 16)
        case.update(group=rng.choice([0, 32, 64]), read=rng.choice(["new", "all"]))
    return case


def _scope(case: dict) -> float:
    """What the plain form keeps in memory at once, in values: a drawn case has no more than the largest listed."""
    op = case["op"]
    if op in ("append", "store4"):
        return case["batch"] * (case["held"] + case["most"]) * case["kv_heads"] * case["dim"] / (64 * 2000 * 8 * 64)
    if op == "attend4":
        return case["batch"] * case["longest"] * max(case["kv_heads"] * case["dim"], case["heads"]) / (32 * 16384 * 1024)
    if op == "reorder":
        pages = case["batch"] * (case["longest"] / case["page"] + 3 * case["beams"])
        return case["layers"] * pages * case["page"] * case["kv_heads"] * case["dim"] / (12 * 350 * 64 * 8 * 128)
    return 0.0


def draw(rng: random.Random) -> dict:
    most = {op: max(max(w["bytes"], w["flops"] / 50) for c in listed() if c["op"] == op for w in [work(c)])
            for op in ("append", "store4", "attend4", "select", "reorder")}
    while True:
        case = _drawn(rng)
        w = work(case)
        if _scope(case) <= 1 and max(w["bytes"], w["flops"] / 50) <= most[case["op"]]:
            return case


# ------------------------------------------- sizes and lengths, from the case alone

def _lengths(case: dict) -> list[int]:
    """The lengths of a batch's texts: the first is the longest, the others anything down to one token."""
    rng = random.Random(1000003 + case["batch"] * 7919 + case["longest"])
    return [case["longest"]] + [rng.randint(1, case["longest"]) for _ in range(case["batch"] - 1)]


def _news(case: dict) -> tuple[list[int], list[int]]:
    """An append's new tokens and the tokens held before them, for each text."""
    rng = random.Random(case["batch"] * 7919 + case["most"] * 31 + case["held"])
    new = [case["most"]] + [rng.randint(1, case["most"]) for _ in range(case["batch"] - 1)]
    return new, [rng.randint(0, case["held"]) for _ in new]


def _parents(case: dict) -> list[int]:
    """Which beam of its text each beam goes on from: good beams have several heirs, some beams none."""
    rng = random.Random(case["batch"] * 101 + case["beams"])
    return [min(rng.randrange(case["beams"]), rng.randrange(case["beams"])) for _ in range(case["batch"] * case["beams"])]


def _size(t: str) -> int:
    return {"f32": 4, "bf16": 2, "f16": 2}[t]


def _padded(dim: int) -> int:
    return next(p for p in (32, 64, 96, 128, 192, 256) if p >= dim)


def _groups(case: dict) -> int:
    return -(-case["dim"] // case["group"]) if case["group"] else 1


def _held_bytes(case: dict) -> int:
    """Bytes of a token's keys and values in a 4-bit cache, of one head."""
    return _padded(case["dim"]) + 8 * _groups(case)


def _seen(before: int, window: int, sinks: int) -> int:
    """How many keys a query sees that is number `before` + 1 of its text."""
    n = before + 1
    return n if not window or n <= window else window + min(sinks, n - window)


def work(case: dict) -> dict:
    op = case["op"]
    if op == "select":
        rows = case["batch"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * _size(case["type"]) + 5) + case["batch"] * case["keep"] * 13,
                "flops": 3 * rows * case["vocab"]}
    row = case["kv_heads"] * case["dim"] * _size(case["type"])
    if op == "reorder":
        tokens = sum(_lengths(case)[i // case["beams"]] % case["page"] for i, p in enumerate(_parents(case))
                     if p != i % case["beams"])
        rows = case["batch"] * case["beams"]
        width = case["longest"] // case["page"] + 2
        return {"bytes": 4 * tokens * row * case["layers"] + 8 * rows * (width + 1 + case["steps"]), "flops": 0}
    q = case["heads"] * case["dim"] * _size(case["type"])
    if op == "attend4":
        seen = sum(_seen(n - 1, case["window"], case["sinks"]) for n in _lengths(case))
        return {"bytes": seen * case["kv_heads"] * _held_bytes(case) + 2 * case["batch"] * q,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    new, held = _news(case)
    turned = 3 * sum(new) * (case["heads"] + case["kv_heads"]) * case["rotary"]
    if op == "append":
        return {"bytes": sum(new) * (2 * q + 4 * row), "flops": turned}
    back = sum(new) + (sum(held) if case["read"] == "all" else 0)
    return {"bytes": sum(new) * (2 * q + 2 * row) + (sum(new) + back) * case["kv_heads"] * _held_bytes(case) + back * 2 * row,
            "flops": turned + 4 * (sum(new) + back) * case["kv_heads"] * case["dim"]}


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


def _keys(g, shape, t) -> torch.Tensor:
    """Keys as layers make them: a few channels of each head stand off zero."""
    off = 3 * torch.randn(shape[-2:], generator=g, device=DEV) * (torch.rand(shape[-2:], generator=g, device=DEV) < 0.05)
    return (torch.randn(shape, generator=g, device=DEV) + off).to(TYPES[t])


def _frequencies(rotary: int) -> torch.Tensor:
    return (10000.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) * 2 / max(rotary, 1))).float().to(DEV)


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    op, t = case["op"], case["type"]
    s = {"case": case}
    if op == "select":
        return _prepare_select(s, g)
    if op == "reorder":
        return _prepare_reorder(s, g)
    kv, dim, heads, page = case["kv_heads"], case["dim"], case["heads"], case["page"]
    if op == "attend4":
        lengths = _lengths(case)
        s["table"], pages = _pages(g, lengths, page, 3)
        s["lengths"], s["longest"], s["scale"] = _ints(lengths), max(lengths), dim ** -0.5
        s["data"] = _cache4(case, pages)
        _fill4(s["data"], case, g)
        s["q"] = _normal(g, (case["batch"], heads, dim), t, 2.0)
        s["y"] = torch.empty_like(s["q"])
        s["work"] = torch.empty(WORKSPACE, dtype=torch.uint8, device=DEV)
        return s
    new, held = _news(case)
    lengths = [a + b for a, b in zip(new, held)]
    s["table"], pages = _pages(g, lengths, page, 3)
    s["lengths"], s["starts"] = _ints(lengths), _ints(_starts(new))
    s["freqs"] = _frequencies(case["rotary"])
    s["positions"] = _ints([case["far"] + h + i for n, h in zip(new, held) for i in range(n)]) if case["far"] else None
    s["q"] = _normal(g, (sum(new), heads, dim), t, 2.0)
    s["k"], s["v"] = _keys(g, (sum(new), kv, dim), t), _normal(g, (sum(new), kv, dim), t)
    s["q_out"] = torch.empty_like(s["q"])
    if op == "append":
        s["k_cache"] = _normal(g, (pages, page, kv, dim), t)
        s["v_cache"] = _normal(g, (pages, page, kv, dim), t)
        return s
    s["data"] = _cache4(case, pages)
    _fill4(s["data"], case, g)
    back = new if case["read"] == "new" else lengths
    s["back"] = _ints(_starts(back))
    s["k_back"] = torch.empty(sum(back), kv, dim, dtype=TYPES[t], device=DEV)
    s["v_back"] = torch.empty_like(s["k_back"])
    return s


def _prepare_select(s, g):
    case = s["case"]
    b, n, v, t = case["batch"], case["beams"], case["vocab"], case["type"]
    # A network's logits: a few tokens stand out in each row.
    x = torch.randn(b, n, v, generator=g, device=DEV) * 2 + torch.randn(b, n, 1, generator=g, device=DEV)
    bump = torch.randint(0, v, (b, n, 6), generator=g, device=DEV)
    x.scatter_add_(2, bump, 6 * torch.rand(b, n, 6, generator=g, device=DEV))
    s["logits"] = x.to(TYPES[t])
    if case["masked"]:
        # Tokens that a grammar forbids; half of them at the type's lowest value instead of -infinity.
        r = torch.rand(b, n, v, generator=g, device=DEV)
        s["logits"].masked_fill_(r < case["masked"], -math.inf)
        s["logits"].masked_fill_(r < case["masked"] / 2, torch.finfo(TYPES[t]).min)
    s["scores"] = -torch.rand(b, n, generator=g, device=DEV).mul_(8).sort(-1).values.contiguous()
    if case["first"]:
        s["scores"][:, 1:] = -math.inf
    s["ended"] = (torch.rand(b, n, generator=g, device=DEV) < 0.3).to(torch.uint8) if case["ended"] else None
    keep = case["keep"]
    s["out_scores"] = torch.empty(b, keep, device=DEV)
    s["parents"] = torch.empty(b, keep, dtype=torch.int32, device=DEV)
    s["tokens"] = torch.empty(b, keep, dtype=torch.int32, device=DEV)
    s["out_ended"] = torch.empty(b, keep, dtype=torch.uint8, device=DEV)
    s["work"] = torch.empty(WORKSPACE, dtype=torch.uint8, device=DEV)
    return s


def _prepare_reorder(s, g):
    case = s["case"]
    b, n, page, t = case["batch"], case["beams"], case["page"], case["type"]
    lengths = [x for x in _lengths(case) for _ in range(n)]
    width = case["longest"] // page + 2
    # A text's beams share its full pages; the page being written, the next one and a spare are each beam's own.
    rows, at, spare = [], 0, []
    for i in range(b):
        full = lengths[i * n] // page
        shared = list(range(at, at + full))
        at += full
        for _ in range(n):
            rows.append(shared + [at, at + 1][:width - full] + [-1] * (width - full - 2))
            spare.append(at + 2)
            at += 3
    order = torch.randperm(at, generator=g, device=DEV).to(torch.int32)
    table = _ints(rows)
    s["table"] = torch.where(table >= 0, order[table.clamp(min=0).long()], table).contiguous()
    s["spare"] = order[torch.tensor(spare, device=DEV)].contiguous()
    s["lengths"], s["parents"] = _ints(lengths), _ints(_parents(case))
    s["table_out"], s["spare_out"] = torch.empty_like(s["table"]), torch.empty_like(s["spare"])
    shape = (case["layers"], at, page, case["kv_heads"], case["dim"])
    s["k_cache"], s["v_cache"] = _normal(g, shape, t), _normal(g, shape, t)
    s["history"] = torch.randint(0, 18385, (b * n, case["steps"]), generator=g, device=DEV, dtype=torch.int32)
    s["history_out"] = torch.empty_like(s["history"])
    return s


# ------------------------------------------------------- a 4-bit cache's planes

def _planes(case: dict):
    """Where a chunk's planes begin: K codes, scales, minima, V codes, scales, minima, and its end."""
    page, codes, few = case["page"], _padded(case["dim"]) // 2, 2 * _groups(case)
    out = [0]
    for size in (codes, few, few) * 2:
        out.append(out[-1] + page * size)
    return out


def _cache4(case: dict, pages: int) -> torch.Tensor:
    return torch.zeros(pages, case["kv_heads"], _planes(case)[-1], dtype=torch.uint8, device=DEV)


def _views(data, case: dict):
    """Views of a cache's planes: codes [pages, heads, token, 4, c, 4], scales and minima [pages, heads, token, group] of K; codes [pages, heads, token / 4, 16, c, 4] and so on of V."""
    at, page, c, groups = _planes(case), case["page"], _padded(case["dim"]) // 32, _groups(case)
    part = [data[..., a:b] for a, b in zip(at, at[1:])]
    few = [part[i].view(torch.float16).unflatten(-1, (page, groups)) for i in (1, 2, 4, 5)]
    return (part[0].unflatten(-1, (page, 4, c, 4)), few[0], few[1], part[3].unflatten(-1, (page // 4, 16, c, 4)),
            few[2], few[3])


def _quantised(x, case: dict):
    """Codes [..., P] (whole numbers as uint8), scales and minima [..., group] in f16 of values [..., dim] in f32."""
    dim, groups, group = case["dim"], _groups(case), case["group"] or case["dim"]
    bad = ~torch.isfinite(x)
    x = x.clamp(-65504, 65504)
    short = groups * group - dim
    pad = torch.nn.functional.pad
    low = pad(x, (0, short), value=math.inf).unflatten(-1, (groups, group)).amin(-1)
    high = pad(x, (0, short), value=-math.inf).unflatten(-1, (groups, group)).amax(-1)
    wrong = pad(bad, (0, short)).unflatten(-1, (groups, group)).any(-1)
    m = low.to(torch.float16)
    scale = ((high - m.float()) * (1 / 15)).to(torch.float16)
    inverse = 1 / scale.float()
    n = ((pad(x, (0, short)).unflatten(-1, (groups, group)) - m.float()[..., None]) * inverse[..., None]).round().clamp(0, 15)
    n = torch.where((scale == 0)[..., None] | wrong[..., None], torch.zeros_like(n), n).flatten(-2)[..., :dim]
    scale = torch.where(wrong, torch.full_like(scale, math.nan), scale)
    return pad(n.to(torch.uint8), (0, _padded(dim) - dim)), scale, m


def _k_bytes(n):
    """[..., P] codes to [..., 4, c, 4] bytes."""
    two = n[..., 0::2] | n[..., 1::2] << 4
    return two.unflatten(-1, (-1, 4, 4)).transpose(-2, -3)


def _v_bytes(n):
    """[..., P] codes of a token to [..., 16, c] bytes."""
    two = n[..., 0::2] | n[..., 1::2] << 4
    return two.unflatten(-1, (-1, 16)).transpose(-1, -2)


def _fill4(data, case: dict, g) -> None:
    """Fills a cache with keys and values as layers make them, some pages at a time."""
    kc, ks, km, vc, vs, vm = _views(data, case)
    step = max(1, (1 << 26) // (case["page"] * case["kv_heads"] * case["dim"]))
    for a in range(0, data.shape[0], step):
        pages = data[a:a + step].shape[0]
        shape = (pages, case["page"], case["kv_heads"], case["dim"])
        n, scale, m = _quantised(_keys(g, shape, "f32").transpose(1, 2), case)
        kc[a:a + step], ks[a:a + step], km[a:a + step] = _k_bytes(n), scale, m
        n, scale, m = _quantised(_normal(g, shape, "f32").transpose(1, 2), case)
        vc[a:a + step] = _v_bytes(n).unflatten(2, (-1, 4)).permute(0, 1, 2, 4, 5, 3)
        vs[a:a + step], vm[a:a + step] = scale, m


def _decoded(n, scale, m, case: dict):
    """Values of codes in natural order [..., P / 2] bytes, scales and minima [..., group]: n scale + minimum in f32."""
    spread = lambda x: x.float().repeat_interleave(case["group"] or case["dim"], -1)[..., :case["dim"]]  # noqa: E731
    n = torch.stack((n & 15, n >> 4), -1).flatten(-2)[..., :case["dim"]].float()
    return n * spread(scale) + spread(m)


def _values(data, case: dict):
    """What the cache stands for: keys and values [pages, page, heads, dim] in f32."""
    kc, ks, km, vc, vs, vm = _views(data, case)
    k = _decoded(kc.transpose(-2, -3).flatten(-3), ks, km, case)
    v = _decoded(vc.permute(0, 1, 2, 5, 4, 3).flatten(-2).flatten(2, 3), vs, vm, case)
    return k.transpose(1, 2), v.transpose(1, 2)


def _values_at(data, case: dict, page_of, slot):
    """The same of some tokens: [tokens, heads, dim]."""
    kc, ks, km, vc, vs, vm = _views(data, case)
    k = kc[page_of, :, slot].transpose(-2, -3).flatten(-3)
    v = vc[page_of, :, slot // 4, :, :, slot % 4].transpose(-1, -2).flatten(-2)
    return (_decoded(k, ks[page_of, :, slot], km[page_of, :, slot], case),
            _decoded(v, vs[page_of, :, slot], vm[page_of, :, slot], case))


# ------------------------------------------------------------- the plain forms

def _places(s):
    """Each new row's text, place in it, page and slot."""
    page = s["case"]["page"]
    rows = torch.arange(s["k"].shape[0], device=DEV)
    text = torch.searchsorted(s["starts"], rows.to(torch.int32), right=True) - 1
    at = (s["lengths"] - s["starts"][1:])[text] + rows
    return at, s["table"][text, at // page].long(), at % page


def _turned(x, positions, freqs, case: dict):
    """x [rows, heads, dim] in f32, its first `rotary` dims turned by the rows' positions."""
    angle = (positions.double()[:, None] * freqs.double())[:, None]
    c, sn = angle.cos().float(), angle.sin().float()
    n = case["rotary"]
    if case["pairs"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat((a * c - b * sn, b * c + a * sn), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _plain_append(s):
    case = s["case"]
    at, page_of, slot = _places(s)
    positions = at if s["positions"] is None else s["positions"]
    q = _turned(s["q"].float(), positions, s["freqs"], case).to(s["q"].dtype)
    k = _turned(s["k"].float(), positions, s["freqs"], case)
    if case["op"] == "append":
        s["k_cache"][page_of, slot] = k.to(s["k"].dtype)
        s["v_cache"][page_of, slot] = s["v"]
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    kc, ks, km, vc, vs, vm = _views(s["data"], case)
    n, scale, m = _quantised(k, case)
    kc[page_of, :, slot], ks[page_of, :, slot], km[page_of, :, slot] = _k_bytes(n), scale, m
    n, scale, m = _quantised(s["v"].float(), case)
    vc[page_of, :, slot // 4, :, :, slot % 4] = _v_bytes(n)
    vs[page_of, :, slot], vm[page_of, :, slot] = scale, m
    rows = torch.arange(s["k_back"].shape[0], device=DEV)
    text = torch.searchsorted(s["back"], rows.to(torch.int32), right=True) - 1
    at = (s["lengths"] - s["back"][1:])[text] + rows
    page_of, slot = s["table"][text, at // case["page"]].long(), at % case["page"]
    k, v = _values_at(s["data"], case, page_of, slot)
    return {"q": q, "k": k.to(s["k"].dtype), "v": v.to(s["v"].dtype)}


def _attend(q, k, v, hidden, scale):
    """Softmax attention of q [batch, kv heads, rows, dim] over k, v [batch, kv heads, keys, dim], none of the `hidden` keys seen; a row that sees none gives zeros."""
    p = torch.matmul(q * scale, k.transpose(-1, -2).contiguous())
    p.masked_fill_(hidden, -math.inf)
    most = p.amax(-1, keepdim=True)
    p.sub_(most.masked_fill_(most == -math.inf, 0)).exp_()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_attend4(s):
    case = s["case"]
    b, kv, dim = case["batch"], case["kv_heads"], case["dim"]
    k, v = _values(s["data"], case)
    tokens = torch.arange(s["longest"], device=DEV)
    page_of = s["table"].clamp(min=0).long()[:, tokens // case["page"]]
    k, v = (x[page_of, tokens % case["page"]].transpose(1, 2) for x in (k, v))
    n = s["lengths"][:, None]
    hidden = tokens >= n
    if case["window"]:
        hidden = hidden | ((tokens < n - case["window"]) & (tokens >= case["sinks"]))
    y = _attend(s["q"].float().view(b, kv, -1, dim), k, v, hidden[:, None, None], s["scale"])
    return y.reshape(b, -1, dim).to(s["q"].dtype)


def _plain_select(s):
    case = s["case"]
    v, keep, beams = case["vocab"], case["keep"], case["beams"]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = s["scores"].double()[..., None] + (x - x.exp().sum(-1, keepdim=True).log())
    if s["ended"] is not None:
        # An ended beam goes on in one way, with the end token (here 2) at no cost.
        over = s["ended"].bool()[..., None]
        x = x.masked_fill(over, -math.inf)
        x[..., 2] = torch.where(over[..., 0], s["scores"].double(), x[..., 2])
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x).flatten(1)
    x, at = x.sort(dim=-1, descending=True, stable=True)
    if x.shape[1] < keep:
        x = torch.nn.functional.pad(x, (0, keep - x.shape[1]), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, keep - at.shape[1]))
    x, at = x[:, :keep], at[:, :keep]
    none = x == -math.inf
    itself = torch.arange(keep, device=DEV).clamp(max=beams - 1)
    parents = torch.where(none, itself, at // v)
    tokens = torch.where(none, -1, at % v)
    ended = (tokens == 2) if s["ended"] is None else (tokens == 2) | (s["ended"].gather(1, parents).bool() & ~none)
    return {"scores": x.float(), "parents": parents.int(), "tokens": tokens.int(), "ended": ended.to(torch.uint8)}


def _plain_reorder(s):
    case = s["case"]
    page, table = case["page"], s["table"]
    row = torch.arange(table.shape[0], device=DEV)
    frm = row // case["beams"] * case["beams"] + s["parents"].long()
    full, part = s["lengths"].long() // page, s["lengths"] % page
    moved = frm != row
    slots = torch.arange(table.shape[1], device=DEV)
    copied = (moved & (part > 0))[:, None]
    out = torch.where(moved[:, None] & (slots < full[:, None]), table[frm], table)
    out = torch.where(copied & (slots == full[:, None]), s["spare"][:, None], out)
    spare = torch.where(copied[:, 0], table[row, full], s["spare"])
    source, into = table[frm, full].long(), s["spare"].long()
    here = (torch.arange(page, device=DEV) < part[:, None]) & copied
    for cache in (s["k_cache"], s["v_cache"]):
        cache[:, into] = torch.where(here[None, :, :, None, None], cache[:, source], cache[:, into])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "table": out, "spare": spare, "history": s["history"][frm]}


# ----------------------------------------------------------------- one pass

def _ptr(x) -> int:
    return x.data_ptr() if x is not None else 0


def _own(s):
    D = _decoder()
    case = s["case"]
    op, t, st = case["op"], getattr(D, case["type"].upper()), _stream()
    if op == "select":
        D.beam_select(_ptr(s["logits"]), _ptr(s["scores"]), _ptr(s["out_scores"]), _ptr(s["parents"]), _ptr(s["tokens"]),
                      case["batch"], case["beams"], case["vocab"], case["keep"], type=t, ended=_ptr(s["ended"]),
                      out_ended=_ptr(s["out_ended"]), end=2, workspace=_ptr(s["work"]), workspace_bytes=WORKSPACE,
                      stream=st)
        return {"scores": s["out_scores"], "parents": s["parents"], "tokens": s["tokens"], "ended": s["out_ended"]}
    if op == "reorder":
        if "caches" not in s:
            s["caches"] = [D.KvCache(_ptr(k), _ptr(v), k.shape[0], case["page"], case["kv_heads"], case["dim"], type=t)
                           for k, v in zip(s["k_cache"], s["v_cache"])]
            s["states"] = [D.BeamState(_ptr(s["history"]), _ptr(s["history_out"]), 4 * case["steps"])]
        D.beam_reorder(s["caches"], _ptr(s["parents"]), _ptr(s["table"]), _ptr(s["table_out"]), s["table"].shape[1],
                       _ptr(s["lengths"]), _ptr(s["spare"]), _ptr(s["spare_out"]), case["batch"], case["beams"],
                       states=s["states"], stream=st)
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "table": s["table_out"], "spare": s["spare_out"],
                "history": s["history_out"]}
    if op != "append" and "cache" not in s:
        s["cache"] = D.Kv4Cache(_ptr(s["data"]), s["data"].shape[0], case["page"], case["kv_heads"], case["dim"],
                                case["group"])
    table, width, lengths = _ptr(s["table"]), s["table"].shape[1], _ptr(s["lengths"])
    if op == "attend4":
        D.kv4_attention(_ptr(s["q"]), s["cache"], table, width, lengths, _ptr(s["y"]), case["batch"], case["heads"],
                        scale=s["scale"], type=t, window=case["window"], sinks=case["sinks"], longest=s["longest"],
                        workspace=_ptr(s["work"]), workspace_bytes=WORKSPACE, stream=st)
        return s["y"]
    turn = dict(freqs=_ptr(s["freqs"]), rotary=case["rotary"], pairs=case["pairs"], positions=_ptr(s["positions"]),
                q=_ptr(s["q"]), q_out=_ptr(s["q_out"]), heads=case["heads"], starts=_ptr(s["starts"]), stream=st)
    if op == "append":
        if "cache" not in s:
            s["cache"] = D.KvCache(_ptr(s["k_cache"]), _ptr(s["v_cache"]), s["k_cache"].shape[0], case["page"],
                                   case["kv_heads"], case["dim"], type=t)
        D.kv_append_rotated(_ptr(s["k"]), _ptr(s["v"]), s["cache"], table, width, lengths, case["batch"],
                            s["k"].shape[0], **turn)
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    D.kv4_append(_ptr(s["k"]), _ptr(s["v"]), s["cache"], table, width, lengths, case["batch"], s["k"].shape[0], type=t,
                 **turn)
    D.kv4_read(_ptr(s["k_back"]), _ptr(s["v_back"]), s["cache"], table, width, lengths, case["batch"],
               s["k_back"].shape[0], starts=_ptr(s["back"]), type=t, stream=st)
    return {"q": s["q_out"], "k": s["k_back"], "v": s["v_back"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "store4": _plain_append, "attend4": _plain_attend4, "select": _plain_select,
            "reorder": _plain_reorder}[state["case"]["op"]](state)


# ------------------------------------------------------------------ in 64 bits

def _exact_turn(x, positions, freqs, rotary, pairs):
    """Each pair of dims as a complex number, times that of its angle."""
    out = x.double().clone()
    half = rotary // 2
    one = torch.arange(half, device=DEV) * (2 if pairs else 1)
    two = one + (1 if pairs else half)
    angle = positions.double()[:, None, None] * freqs.double()
    z = torch.complex(out[..., one], out[..., two]) * torch.polar(torch.ones_like(angle), angle)
    out[..., one], out[..., two] = z.real, z.imag
    return out


def _exact_held(data, case: dict, pages, slots):
    """Keys and values [tokens, heads, dim] in f64 of the tokens at these pages and slots, byte by byte."""
    at, p, groups = _planes(case), _padded(case["dim"]), _groups(case)
    c, heads = p // 32, torch.arange(case["kv_heads"], device=DEV)
    chunk = ((pages[:, None] * case["kv_heads"] + heads) * at[-1])[..., None]
    d = torch.arange(case["dim"], device=DEV)
    t = slots[:, None]
    k_at = at[0] + t * (p // 2) + 4 * (c * (d % 32 // 8) + d // 32) + d % 8 // 2
    v_at = at[3] + t // 4 * (2 * p) + 4 * (c * (d % 32 // 2) + d // 32) + t % 4
    out = []
    for code_at, scale_at, low_at in ((k_at, at[1], at[2]), (v_at, at[4], at[5])):
        take = lambda i: data.flatten()[chunk + i[:, None]]  # noqa: E731
        n = take(code_at) >> (4 * (d % 2)) & 15
        few = []
        for base in (scale_at, low_at):
            i = base + 2 * (t * groups + d // (case["group"] or case["dim"]))
            bits = take(i).int() | take(i + 1).int() << 8
            few.append(bits.to(torch.int16).view(torch.float16).double())
        out.append(n.double() * few[0] + few[1])
    return out


def _exact_quantised(x, case: dict):
    """What values [..., dim] in f64 stand for once they are held."""
    out = torch.empty_like(x)
    size = case["group"] or case["dim"]
    for a in range(0, case["dim"], size):
        part = x[..., a:a + size]
        m = part.min(-1, keepdim=True).values.half().double()
        s = ((part.max(-1, keepdim=True).values - m) / 15).half().double()
        n = torch.where(s > 0, torch.round((part - m) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(s))
        out[..., a:a + size] = n.clamp(0, 15) * s + m
    return out


def _exact_append(s):
    case = s["case"]
    new, held = _news(case)
    page, table = case["page"], s["table"].long().cpu()
    places = torch.tensor([held[b] + i for b in range(case["batch"]) for i in range(new[b])])
    text = torch.tensor([b for b in range(case["batch"]) for _ in range(new[b])])
    positions = (places + case["far"]).to(DEV)
    q = _exact_turn(s["q"], positions, s["freqs"], case["rotary"], case["pairs"])
    k = _exact_turn(s["k"], positions, s["freqs"], case["rotary"], case["pairs"])
    if case["op"] == "append":
        flat = (table[text, places // page] * page + places % page).to(DEV)
        out = {"q": q}
        for name, rows in (("k_cache", k), ("v_cache", s["v"].double())):
            cache = s[name].double().flatten(0, 1)
            cache[flat] = rows
            out[name] = cache.view(s[name].shape)
        return out
    if case["type"] == "f32":
        # A code next to a border between two goes by the last of 32 bits: no value of its own.
        return {"q": q, "k": None, "v": None}
    k, v = _exact_quantised(k, case), _exact_quantised(s["v"].double(), case)
    ks, vs, at = [], [], 0
    for b in range(case["batch"]):
        if case["read"] == "all":
            i = torch.arange(held[b])
            old = _exact_held(s["data"], case, table[b, i // page].to(DEV), (i % page).to(DEV))
            ks.append(old[0]), vs.append(old[1])
        ks.append(k[at:at + new[b]]), vs.append(v[at:at + new[b]])
        at += new[b]
    return {"q": q, "k": torch.cat(ks), "v": torch.cat(vs)}


def _exact_attend4(s):
    case, out = s["case"], []
    per = case["heads"] // case["kv_heads"]
    for b, n in enumerate(_lengths(case)):
        at = torch.arange(n, device=DEV)
        if case["window"]:
            at = at[(at >= n - case["window"]) | (at < case["sinks"])]
        k, v = _exact_held(s["data"], case, s["table"][b].long()[at // case["page"]], at % case["page"])
        q = s["q"][b].double().unflatten(0, (-1, per))  # [kv heads, per, dim]
        z = torch.matmul(q, k.permute(1, 2, 0).contiguous()) * s["scale"]
        e = torch.exp(z - z.max(-1, keepdim=True).values)
        y = torch.matmul(e / e.sum(-1, keepdim=True), v.transpose(0, 1).contiguous())
        out.append(y.flatten(0, 1))
    return torch.stack(out)


def _exact_select(s):
    case = s["case"]
    rows, v, keep = case["beams"], case["vocab"], case["keep"]
    out = {"scores": [], "parents": [], "tokens": [], "ended": []}
    for b in range(case["batch"]):
        found = []  # (score, beam, token), each beam's best
        for i in range(rows):
            base = float(s["scores"][b, i])
            if base == -math.inf:
                continue
            if s["ended"] is not None and int(s["ended"][b, i]):
                found.append((base, i, 2, 1))
                continue
            x = s["logits"][b, i].double()
            p = x - torch.logsumexp(x, 0)
            low = torch.topk(p, min(keep, v)).values[-1]
            at = torch.nonzero((p >= low) & (p > -math.inf)).flatten()[:100000]
            found += [(base + score, i, token, int(token == 2)) for score, token in zip(p[at].tolist(), at.tolist())]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        found = found[:keep]
        found += [(-math.inf, min(j, rows - 1), -1, 0) for j in range(len(found), keep)]
        for k, column in zip(out, zip(*found)):
            out[k].append(list(column))
    return {k: torch.tensor(x, dtype={"scores": torch.float64, "ended": torch.uint8}.get(k, torch.int32), device=DEV)
            for k, x in out.items()}


def _exact_reorder(s):
    case = s["case"]
    n, page, lengths = case["beams"], case["page"], _lengths(case)
    table, spare = s["table"].tolist(), s["spare"].tolist()
    new_table, new_spare = [list(r) for r in table], list(spare)
    frm, source, into = [], [], []
    for r, parent in enumerate(_parents(case)):
        f, length = r // n * n + parent, lengths[r // n]
        frm.append(f)
        if f == r:
            continue
        full, part = divmod(length, page)
        new_table[r][:full] = table[f][:full]
        if part:
            source += [table[f][full] * page + i for i in range(part)]
            into += [spare[r] * page + i for i in range(part)]
            new_table[r][full], new_spare[r] = spare[r], table[r][full]
    out = {}
    for name in ("k_cache", "v_cache"):
        cache = s[name].double().flatten(1, 2)
        cache[:, torch.tensor(into, device=DEV, dtype=torch.long)] = cache[:, torch.tensor(source, device=DEV, dtype=torch.long)]
        out[name] = cache.view(s[name].shape)
    return {**out, "table": _ints(new_table), "spare": _ints(new_spare), "history": s["history"][torch.tensor(frm, device=DEV)]}


def exact(case: dict, seed: int):
    return {"append": _exact_append, "store4": _exact_append, "attend4": _exact_attend4, "select": _exact_select,
            "reorder": _exact_reorder}[case["op"]](prepare(case, seed))
