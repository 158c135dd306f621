"""The operators of a serving step around the 4-bit key/value cache, as cases to time and to check: page
tables, slots and positions from request lengths (`kv4_advance`), the per-head norm and rotation of queries
and keys, to rows (`qk_norm_rope`) or with the keys and values into the cache (`qk_norm_rope_kv4`), attention
through a sliding window beside the first tokens (`attention_kv4_sinks`), and attention of a batch that shares
a prefix (`attention_kv4_prefix`).

The cache is `pages` pages of `page` tokens. A page holds, for each key/value head, one block of
`page * (dim + 8)` bytes: the K codes `[page][dim / 2]` bytes, the V codes the same, then the K and the V
parameters `[page]` 32-bit words each. Channel c of a token is bits 4 * (c % 2) .. +3 of byte c / 2. A
parameter word holds the row's minimum m in its low and its scale s in its high 16 bits, both of the cache's
element type. A code u stands for m + s * u, with

    m = min_c x_c,   s = (max_c x_c - m) / 15 rounded toward zero to the element type,
    u_c = the nearest whole number to (x_c - m) / s, ties to even, in 0 .. 15 (0 where s is 0).

Slot t is token t % page of page t / page.

kv4_advance. `new[b]` rows are appended to sequence b of `lengths[b]` tokens; below 0 the sequence ends, and
its pages go back on the stack `free[0 .. count - 1]` first, in order of sequences and columns. Sequence b
needs ceil((length + new) / page) - ceil(length / page) pages. It is refused (no rows) where its tokens pass the
table; where it needs pages and those that it and the sequences before it ask for are more than are free; or
where the rows that it and the sequences before it ask for pass `rows`. The others take their pages from
the top of the stack, in order of sequences and columns, and their rows are q_starts[b] .. q_starts[b + 1] - 1,
with positions length + 0, 1, .. and the slots of these. Rows past the last carry -1 in both.

qk_norm_rope. Per row and head y = x / sqrt(mean(x^2) + eps) * weight, then pairs of the first `rotary`
channels, (c, c + rotary / 2) or interleaved (2 c, 2 c + 1), turned by the row's position:
(a, b) -> (a cos - b sin, b cos + a sin), cos and sin [position][rotary / 2]. Both are rounded once to the
element type. Into the cache go the rounded keys and the values as they are. A row of position -1 is none: its
rows stay as they were.

Attention. Row i of a sequence's n rows sits at p = length - n + i and sees the keys j <= p. With sinks, of
these the ones with j > p - window or j < sinks. With a prefix, all of the prefix's keys too. A row that sees no key
gives zeros, and -inf as its logsumexp.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

F16, BF16 = "f16", "bf16"
DTYPES = {F16: torch.float16, BF16: torch.bfloat16}
DEV = "cuda"
EPS = 1e-5


def listed():
    return [
        # a decoding step of 64 sequences: a token each, now and then a page, three that end
        {"name": "tables_64", "op": "tables", "batch": 64, "page": 16, "context": 8192, "new": 1,
         "mixed": 0.0, "ended": 0.05, "rows": 64, "short": False, "ragged": 1},
        # continuous batching: 512 sequences, some with prompt chunks, rows padded to a fixed number
        {"name": "tables_512_chunks", "op": "tables", "batch": 512, "page": 64, "context": 6001,
         "new": 2048, "mixed": 0.1, "ended": 0.02, "rows": 129024, "short": True, "ragged": 2},
        # one token's queries and keys, to rows: a launch and its latency
        {"name": "rows_1", "op": "rows", "elem": F16, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "norm": True, "positions": 8192, "cached": False,
         "page": 16, "skip": 0.0},
        # a prompt of odd length without norms, a quarter of the channels rotated in neighbouring pairs
        {"name": "rows_4099_pairs", "op": "rows", "elem": BF16, "tokens": 4099, "heads": 12,
         "kv_heads": 12, "dim": 64, "rotary": 16, "interleaved": True, "norm": False,
         "positions": 5000, "cached": False, "page": 16, "skip": 0.0},
        # a decoding step of 256 sequences, keys and values into the cache
        {"name": "cached_256", "op": "rows", "elem": BF16, "tokens": 256, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "norm": True, "positions": 129024,
         "cached": True, "page": 64, "skip": 0.0},
        # prompts of 31,104 tokens in all into the cache, one row in ten padding
        {"name": "cached_31104", "op": "rows", "elem": BF16, "tokens": 31104, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "norm": True, "positions": 31104,
         "cached": True, "page": 64, "skip": 0.1},
        # one sequence of a long chat through a window of 1,024 and four first tokens: latency
        {"name": "sinks_1x31104", "op": "sinks", "elem": F16, "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "context": 31104, "new": 1, "window": 1024, "sinks": 4, "ragged": 0,
         "mixed": False},
        # a serving step of 64 sequences of up to 20,000 tokens, a window of 4,096, a page of first tokens
        {"name": "sinks_64x20000", "op": "sinks", "elem": BF16, "batch": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "context": 20000, "new": 1, "window": 4096, "sinks": 64, "ragged": 1,
         "mixed": False},
        # a prompt through a window of 2,000, odd sizes
        {"name": "sinks_prompt_8192", "op": "sinks", "elem": F16, "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "context": 8192, "new": 8192, "window": 2000, "sinks": 100,
         "ragged": 0, "mixed": False},
        # four samples of one prompt, ungrouped heads of 64 channels, small pages
        {"name": "prefix_4x4099_mha", "op": "prefix", "elem": F16, "batch": 4, "heads": 12, "kv_heads": 12,
         "dim": 64, "page": 16, "prefix": 4099, "context": 129, "new": 1, "causal": True, "ragged": 3},
        # a serving step of 64 sequences behind one system prompt of 8,192 tokens
        {"name": "prefix_64x8192", "op": "prefix", "elem": BF16, "batch": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "prefix": 8192, "context": 700, "new": 1, "causal": True, "ragged": 4},
        # eight questions of 257 tokens about one document of 31,104
        {"name": "prefix_8x257_31104", "op": "prefix", "elem": BF16, "batch": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 128, "prefix": 31104, "context": 257, "new": 257, "causal": True, "ragged": 0},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["tables", "rows", "rows", "sinks", "sinks", "prefix", "prefix"])
    if op == "tables":
        batch = _log(rng, 1, 900)
        return {"op": op, "batch": batch, "page": rng.choice([16, 32, 64, 128, 256]),
                "context": _log(rng, 1, 9000), "new": _log(rng, 1, 100000 // batch),
                "mixed": rng.choice([0.0, 0.1, 1.0]), "ended": rng.choice([0.0, 0.05, 0.3]),
                "rows": _log(rng, batch, 100000), "short": rng.random() < 0.4,
                "ragged": rng.randrange(1, 1000)}
    dim = rng.choice([64, 128, 128])
    elem = rng.choice([F16, BF16])
    page = rng.choice([16, 32, 64, 128, 256])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    kv_heads = _log(rng, 1, max(1, 32 // group))
    case = {"op": op, "elem": elem, "heads": group * kv_heads, "kv_heads": kv_heads, "dim": dim,
            "page": page}
    if op == "rows":
        tokens = _log(rng, 1, 30000)
        return case | {"tokens": tokens, "rotary": rng.choice([0, 16, 32, 48, 64, dim, dim]),
                       "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.8,
                       "positions": _log(rng, tokens, 100000), "cached": rng.random() < 0.6,
                       "skip": rng.choice([0.0, 0.05, 0.3])}
    kind = rng.choice(["decode", "decode", "verify", "prompt", "mixed"])
    case |= {"batch": 1, "new": 1, "ragged": rng.randrange(1, 1000)}
    if op == "sinks":
        case |= {"window": _log(rng, 1, 5000), "sinks": rng.choice([1, 4, _log(rng, 1, 600)]),
                 "mixed": kind == "mixed"}
        if kind == "decode":
            case["batch"] = _log(rng, 1, 96)
            case["context"] = _log(rng, 1, min(60000, 400000 // case["batch"]))
        elif kind == "verify":
            case["batch"] = _log(rng, 1, 32)
            case["new"] = rng.randrange(2, 17)
            case["context"] = _log(rng, case["new"], 8000)
        elif kind == "prompt":
            case["batch"] = rng.choice([1, 1, 2, 3])
            case["new"] = _log(rng, 17, 4000 // case["batch"])
            case["context"] = case["new"] + rng.choice([0, _log(rng, 1, 4000)])
        else:
            case["batch"] = rng.randrange(2, 12)
            case["new"] = _log(rng, 65, 1024)
            case["context"] = case["new"] + _log(rng, 1, 6000)
        return case
    case["causal"] = rng.random() < 0.8
    if kind in ("decode", "mixed"):
        case["batch"] = _log(rng, 1, 96)
        case["prefix"] = _log(rng, 1, min(30000, 600000 // case["batch"]))
        case["context"] = _log(rng, 1, 2000)
    elif kind == "verify":
        case["batch"] = _log(rng, 1, 32)
        case["new"] = rng.randrange(2, 17)
        case["prefix"] = _log(rng, 1, 10000)
        case["context"] = case["new"] + _log(rng, 1, 1000)
    else:
        case["batch"] = rng.randrange(1, 9)
        case["new"] = _log(rng, 17, 257)
        case["prefix"] = _log(rng, 16, 20000)
        case["context"] = case["new"] + rng.choice([0, _log(rng, 1, 500)])
    return case


def _sequences(case):
    """(new, lengths): each sequence's query rows and its own keys, the same for every seed."""
    r, batch = random.Random(case["ragged"]), case["batch"]
    new = [case["new"]] + [1 if case.get("mixed") else case["new"]] * (batch - 1)
    if not case["ragged"]:
        return new, [case["context"]] * batch
    return new, [case["context"]] + [r.randint(min(case["context"], max(n, case["context"] // 4)),
                                               case["context"]) for n in new[1:]]


def _requests(case):
    """(new, lengths, free): rows asked for by each sequence (-1: it ends), its tokens, free pages."""
    r = random.Random(case["ragged"])
    lengths = [r.randint(case["context"] // 3, case["context"]) for _ in range(case["batch"])]
    new = [-1 if r.random() < case["ended"] else
           r.randint(1, case["new"]) if r.random() < case["mixed"] else 1 for _ in lengths]
    asked = sum(-(-(n + m) // case["page"]) - -(-n // case["page"])
                for n, m in zip(lengths, new) if m > 0)
    return new, lengths, asked * 3 // 4 if case["short"] else asked + 9


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _rows(g, tokens, heads, dim, elem):
    """Keys or values as a projection leaves them: each head's channels have their own size and
    offset, a few of them large."""
    size = 0.5 + _randn(g, heads, dim).abs()
    offset = 0.5 * _randn(g, heads, dim)
    return (_randn(g, tokens, heads, dim) * size + offset).to(DTYPES[elem])


def _filled(g, pages, case):
    """A cache whose every slot holds a quantized row, as bytes."""
    blocks, params = [], []
    for _ in range(2):
        m, s, u = _quantize(_rows(g, pages * case["page"], case["kv_heads"], case["dim"], case["elem"]))
        u = u.to(torch.uint8)
        word = torch.stack([m, s], -1).view(torch.uint8)  # [tokens][heads][4] bytes: m, then s
        for part, a in ((blocks, u[..., 0::2] | (u[..., 1::2] << 4)), (params, word)):
            part.append(a.reshape(pages, case["page"], case["kv_heads"], -1).transpose(1, 2)
                        .reshape(pages, case["kv_heads"], -1))
    return torch.cat(blocks + params, -1).reshape(-1)


def _prepare_tables(case, g):
    new, lengths, free = _requests(case)
    page = case["page"]
    held = [-(-n // page) for n in lengths]
    columns = -(-(case["context"] + case["new"]) // page) + 1
    pages = sum(held) + free + 2
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["batch"], columns), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    stack = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
    stack[:free] = order[at:at + free]
    return {"pages": pages, "columns": columns, "table": table, "free": stack, "new": _ints(new),
            "lengths": _ints(lengths), "count": _ints([free]),
            "lengths_out": _ints([0] * case["batch"]), "count_out": _ints([0]),
            "q_starts": _ints([0] * (case["batch"] + 1)), "slots": _ints([0] * case["rows"]),
            "row_positions": _ints([0] * case["rows"])}


def _prepare_rows(case, g):
    dtype, tokens, dim = DTYPES[case["elem"]], case["tokens"], case["dim"]
    q = _rows(g, tokens, case["heads"], dim, case["elem"]).reshape(tokens, -1)
    k, v = (_rows(g, tokens, case["kv_heads"], dim, case["elem"]).reshape(tokens, -1) for _ in range(2))
    half = case["rotary"] // 2
    angle = (torch.arange(case["positions"], device=DEV, dtype=torch.float64)[:, None]
             * 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / max(half, 1)))
    at = torch.randint(case["positions"], (tokens,), generator=g, device=DEV)
    if tokens > 512:  # of prompts, one token after another
        at = (at[0] + torch.arange(tokens, device=DEV)) % case["positions"]
    skipped = torch.rand(tokens, generator=g, device=DEV) < case["skip"]
    state = {"fused": torch.cat([q, k, v], 1),  # [q | k | v] rows, as one projection writes them
             "q_weight": 1 + 0.2 * _randn(g, dim), "k_weight": 1 + 0.2 * _randn(g, dim),
             "cos": torch.cos(angle).float(), "sin": torch.sin(angle).float(),
             "row_positions": torch.where(skipped, -1, at).to(torch.int32),
             "q_out": torch.zeros_like(q), "k_out": torch.zeros_like(k)}
    if case["cached"]:
        page = case["page"]
        pages = -(-tokens // page) + 3
        order = torch.randperm(pages, generator=g, device=DEV)
        slots = (order[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:tokens]
        state |= {"pages": pages, "slots": torch.where(skipped, -1, slots).to(torch.int32),
                  "cache": torch.zeros(pages * page * case["kv_heads"] * (dim + 8), dtype=torch.uint8,
                                       device=DEV),
                  "v_out": torch.zeros(tokens, case["kv_heads"] * dim, dtype=dtype, device=DEV)}
    return state


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "tables":
        return {"case": case} | _prepare_tables(case, g)
    if case["op"] == "rows":
        return {"case": case} | _prepare_rows(case, g)
    dtype, page = DTYPES[case["elem"]], case["page"]
    new, lengths = _sequences(case)
    shared = case.get("prefix", 0)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + -(-shared // page) + 2
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["batch"], max(1, *held)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    rows = sum(new)
    return {"case": case, "pages": pages, "table": table, "rows": rows,
            "prefix_table": order[at:at + -(-shared // page)].contiguous(),
            "prefix_length": _ints([shared]),
            "cache": _filled(g, pages, case), "lengths": _ints(lengths),
            "q_starts": _ints(np.concatenate([[0], np.cumsum(new)]).tolist()),
            "q": _randn(g, rows, case["heads"] * case["dim"], dtype=dtype),
            "out": torch.zeros(rows, case["heads"] * case["dim"], dtype=dtype, device=DEV),
            "lse": torch.zeros(rows, case["heads"], dtype=torch.float32, device=DEV)}


# ---------------------------------------------------------------- the framework's calls

def _own_tables(H, state, case):
    if "plan" not in state:
        state["plan"] = H.Kv4Cfg(8, 128, case["page"], state["pages"], H.H3_ELEM_BF16)
    H.kv4_advance(state["plan"], case["batch"], state["columns"], case["rows"], state["new"],
                  state["lengths"], state["free"], state["count"], state["table"],
                  state["lengths_out"], state["count_out"], state["q_starts"], state["slots"],
                  state["row_positions"])
    return _tables_out(state)


def _own_rows(H, state, case):
    q_width, width = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    pitch = q_width + 2 * width
    if "plan" not in state:
        elem = {F16: H.H3_ELEM_F16, BF16: H.H3_ELEM_BF16}[case["elem"]]
        qk = H.QkCfg(case["heads"], case["kv_heads"], case["dim"], case["rotary"], case["interleaved"],
                     case["norm"], case["positions"], EPS, elem, pitch, pitch, pitch, q_width, width)
        state["plan"] = (qk, H.Kv4Cfg(case["kv_heads"], case["dim"], case["page"], state["pages"], elem)
                         if case["cached"] else None)
    qk, cfg = state["plan"]
    flat, tokens = state["fused"].view(-1), case["tokens"]
    k, v = flat[q_width:], flat[q_width + width:]
    weights = (state["q_weight"], state["k_weight"]) if case["norm"] else (None, None)
    tables = (state["cos"], state["sin"]) if case["rotary"] else (None, None)
    if not case["cached"]:
        H.qk_norm_rope(qk, tokens, flat, k, *weights, *tables, state["row_positions"], state["q_out"],
                       state["k_out"])
        return {"q": state["q_out"], "k": state["k_out"]}
    H.qk_norm_rope_kv4(qk, cfg, tokens, flat, k, v, *weights, *tables, state["row_positions"],
                       state["slots"], state["q_out"], state["cache"])
    H.kv4_read(cfg, tokens, width, width, state["slots"], state["cache"], state["k_out"], state["v_out"])
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


def _own_attend(H, state, case):
    if "plan" not in state:  # the configs and the workspace a program keeps beside its cache
        elem = {F16: H.H3_ELEM_F16, BF16: H.H3_ELEM_BF16}[case["elem"]]
        cfg = H.Kv4Cfg(case["kv_heads"], case["dim"], case["page"], state["pages"], elem)
        width = case["heads"] * case["dim"]
        acfg = H.Kv4AttentionCfg(case["heads"], width, width, state["table"].shape[1],
                                 case.get("causal", True), case.get("window", 0),
                                 1 / math.sqrt(case["dim"]))
        if case["op"] == "sinks":
            need = H.kv4_sinks_workspace_bytes(cfg, acfg, case["sinks"], case["batch"], state["rows"],
                                               case["new"])
        else:
            need = H.kv4_prefix_workspace_bytes(cfg, acfg, state["prefix_table"].shape[0], case["batch"],
                                                state["rows"], case["new"])
        state["plan"] = (cfg, acfg,
                         torch.empty(need, dtype=torch.uint8, device=DEV) if need else None)
    cfg, acfg, ws = state["plan"]
    if case["op"] == "sinks":
        H.attention_kv4_sinks(cfg, acfg, case["sinks"], case["batch"], state["rows"], case["new"],
                              state["q"], state["cache"], state["table"], state["lengths"],
                              state["q_starts"], state["out"], lse=state["lse"], workspace=ws)
    else:
        H.attention_kv4_prefix(cfg, acfg, state["prefix_table"].shape[0], case["batch"], state["rows"],
                               case["new"], state["q"], state["cache"], state["prefix_table"],
                               state["prefix_length"], state["table"], state["lengths"],
                               state["q_starts"], state["out"], lse=state["lse"], workspace=ws)
    return {"out": state["out"], "lse": state["lse"]}


def _own(state):
    sys.path[:0] = [p for p in [os.path.join(os.getcwd(), "h3-hrx_amd")] if p not in sys.path]
    import h3attn as H

    case = state["case"]
    return {"tables": _own_tables, "rows": _own_rows}.get(case["op"], _own_attend)(H, state, case)


# ---------------------------------------------------------------- the plain form

def _quantize(x):
    """(m, s, u) of rows x [...][dim]: the minimum and the scale in x's type, the codes in f32."""
    y = x.float()
    m, big = y.amin(-1), y.amax(-1)
    wide = (big - m) / 15
    s = wide.to(x.dtype)
    s = torch.where(s.float() > wide, (s.view(torch.int16) - 1).view(x.dtype), s)  # toward zero
    step = s.float()[..., None]
    u = torch.where(step > 0, torch.round((y - m[..., None]) / step), 0.0).clamp(0, 15)
    return m.to(x.dtype), s, u


def _fields(cache, case, pages):
    """The cache's (K codes, V codes, K words, V words), each [pages][heads][page][...]."""
    page, dim = case["page"], case["dim"]
    block = cache.view(pages, case["kv_heads"], page * (dim + 8))
    half = page * dim // 2
    return (block[..., :half].view(pages, -1, page, dim // 2),
            block[..., half:2 * half].view(pages, -1, page, dim // 2),
            block[..., 2 * half:2 * half + 4 * page].view(pages, -1, page, 4),
            block[..., 2 * half + 4 * page:].view(pages, -1, page, 4))


def _values(codes, words, dtype):
    """m + s * u in f32 of code bytes [...][dim / 2] and parameter words [...][4] bytes."""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = words.contiguous().view(dtype).float()
    return p[..., 0:1] + p[..., 1:2] * u


def _nearest(x, dtype):
    """f64 values rounded once to the element type (a cast rounds to f32 on the way)."""
    bits, low = (11, -24) if dtype == torch.float16 else (8, -133)
    _, e = torch.frexp(x)
    unit = torch.exp2((e - bits).clamp(min=low).double())
    return (torch.round(x / unit) * unit).to(dtype)


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    return {"tables": _tables, "rows": _norm_rope}.get(case["op"], _attend)(state, case)


def _tables_out(state):
    return {name: state[name] for name in ("table", "free", "lengths_out", "count_out", "q_starts",
                                           "slots", "row_positions")}


def _tables(state, case):
    page, columns, rows = case["page"], state["columns"], case["rows"]
    new, lengths = state["new"].long(), state["lengths"].long()
    table, free = state["table"], state["free"]
    up = lambda n: (n + page - 1) // page  # noqa: E731
    column = torch.arange(columns, device=DEV)
    # The pages of the sequences that end, onto the stack.
    ends = new < 0
    give = torch.where(ends, up(lengths), 0)
    back = torch.cumsum(give, 0)
    place = state["count"].long() + (back - give)[:, None] + column
    pushed = column < give[:, None]
    free[place[pushed]] = table[pushed]
    count = state["count"].long() + back[-1:]
    # Who gets rows.
    have = torch.where(ends, 0, lengths)
    ask = torch.where(ends, 0, new)
    ask = torch.where(have + ask > columns * page, 0, ask)
    need = up(have + ask) - up(have)
    fits = ((need == 0) | (torch.cumsum(need, 0) <= count)) & (torch.cumsum(ask, 0) <= rows)
    ask, need = torch.where(fits, ask, 0), torch.where(fits, need, 0)
    # Their pages, from the top.
    taken = torch.cumsum(need, 0)
    first = up(have)[:, None]
    filled = (column >= first) & (column < first + need[:, None])
    top = count - 1 - (taken - need)[:, None] - (column - first)
    table[filled] = free[top[filled]]
    state["lengths_out"].copy_(have + ask)
    state["count_out"].copy_(count - taken[-1:])
    ends_at = torch.cumsum(ask, 0)
    state["q_starts"][0] = 0
    state["q_starts"][1:] = ends_at
    row = torch.arange(rows, device=DEV)
    b = torch.searchsorted(ends_at, row, right=True)
    live = b < case["batch"]
    b = b.clamp(max=case["batch"] - 1)
    at = torch.where(live, have[b] + row - (ends_at - ask)[b], 0)
    state["row_positions"].copy_(torch.where(live, at, -1))
    state["slots"].copy_(torch.where(live, table[b, at // page].long() * page + at % page, -1))
    return _tables_out(state)


def _turned(x, weight, state, case):
    """Rows x [tokens][heads][dim], normed and rotated, in f64: what rounds to the next 16-bit value decides
    a cached row's codes."""
    x, half = x.double(), case["rotary"] // 2
    if case["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + float(np.float32(EPS))) * weight.double()
    if not half:
        return x
    at = state["row_positions"].long().clamp(min=0)
    cos, sin = state["cos"][at].double()[:, None], state["sin"][at].double()[:, None]
    turned = x[..., :2 * half]
    a, b = ((turned[..., 0::2], turned[..., 1::2]) if case["interleaved"]
            else (turned[..., :half], turned[..., half:]))
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _norm_rope(state, case):
    dtype, tokens, dim = DTYPES[case["elem"]], case["tokens"], case["dim"]
    q_width, width = case["heads"] * dim, case["kv_heads"] * dim
    q, k, v = state["fused"].split([q_width, width, width], 1)
    live = state["row_positions"] >= 0
    q = _nearest(_turned(q.view(tokens, -1, dim), state["q_weight"], state, case), dtype)
    k = _nearest(_turned(k.view(tokens, -1, dim), state["k_weight"], state, case), dtype)
    state["q_out"][live] = q.flatten(1)[live]
    if not case["cached"]:
        state["k_out"][live] = k.flatten(1)[live]
        return {"q": state["q_out"], "k": state["k_out"]}
    fields = _fields(state["cache"], case, state["pages"])
    slots = state["slots"].long()
    at = slots[live]
    where = at // case["page"], slice(None), at % case["page"]
    for codes, words, x in ((fields[0], fields[2], k), (fields[1], fields[3], v.view(tokens, -1, dim))):
        m, s, u = _quantize(x[live])
        u = u.to(torch.uint8)
        codes[where] = u[..., 0::2] | (u[..., 1::2] << 4)
        words[where] = torch.stack([m, s], -1).view(torch.uint8)
    at = slots.clamp(min=0)
    where = at // case["page"], slice(None), at % case["page"]
    for name, codes, words in (("k_out", fields[0], fields[2]), ("v_out", fields[1], fields[3])):
        back = _values(codes[where], words[where], dtype)
        state[name].copy_(torch.where(live[:, None, None], back, 0.0).to(dtype).flatten(1))
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


def _attend(state, case):
    batch, heads, kv_heads, dim = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    group, most, rows, dtype = heads // kv_heads, case["new"], state["rows"], DTYPES[case["elem"]]
    shared = case.get("prefix", 0)
    fields = _fields(state["cache"], case, state["pages"])

    def gathered(codes, words, pages):
        """[batch][heads][keys][dim] of the pages [batch][columns]."""
        return _values(codes[pages], words[pages], dtype).transpose(1, 2).reshape(
            pages.shape[0], kv_heads, -1, dim)

    table = state["table"].long().clamp(min=0)
    k, v = (gathered(fields[i], fields[i + 2], table) for i in (0, 1))
    own_keys = k.shape[2]
    if shared:
        pages = state["prefix_table"].long()[None]
        k, v = (torch.cat([gathered(fields[i], fields[i + 2], pages)[:, :, :shared]
                           .expand(batch, -1, -1, -1), x], 2) for i, x in ((0, k), (1, v)))
    keys = k.shape[2]
    starts, lengths = state["q_starts"].long(), state["lengths"].long()
    n = starts[1:] - starts[:-1]
    i = torch.arange(most, device=DEV)
    at = (starts[:-1, None] + i).clamp(max=rows - 1)  # [batch][most] rows of q
    q = state["q"].float().view(rows, kv_heads, group, dim)[at]
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, most * group, dim)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1 / math.sqrt(dim))
    j = torch.arange(own_keys, device=DEV)
    p = (lengths - n)[:, None] + i  # each row's own position
    seen = (j < lengths[:, None, None]).expand(batch, most, own_keys)
    if case.get("causal", True):
        seen = seen & (j <= p[..., None])
    if case.get("window"):
        seen = seen & ((j > p[..., None] - case["window"]) | (j < case["sinks"]))
    seen = torch.cat([seen.new_ones(batch, most, shared), seen], 2)
    seen = seen[:, None, :, None, :]  # over heads and the group
    scores = scores.view(batch, kv_heads, most, group, keys).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(batch, kv_heads, most * group, keys), v)
    out = out.view(batch, kv_heads, most, group, dim) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0]
    mine = i < n[:, None]
    state["out"][at[mine]] = (out.permute(0, 2, 1, 3, 4).reshape(batch, most, heads * dim)[mine]
                              .to(dtype))
    state["lse"][at[mine]] = lse.permute(0, 2, 1, 3).reshape(batch, most, heads)[mine]
    return {"out": state["out"], "lse": state["lse"]}


# ---------------------------------------------------------------- what a pass has to do

def _seen(case, n, length):
    """(own keys that some row of a sequence's n rows sees, pairs of a row and a key of its own)."""
    keys, pairs = 0, 0
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    for i in range(n):
        hi = max(0, min(length, length - n + i + 1)) if case.get("causal", True) else length
        lo = max(0, length - n + i + 1 - window) if window else 0
        pairs += max(0, hi - lo) + min(sinks, lo, hi)
        if i == 0:
            keys = min(sinks, lo, hi) - min(lo, length)
    return keys + length, pairs


def work(case):
    if case["op"] == "tables":
        new, lengths, _ = _requests(case)
        pages = sum(-(-n // case["page"]) for n, m in zip(lengths, new) if m < 0)
        grown = sum(-(-(n + m) // case["page"]) - -(-n // case["page"])
                    for n, m in zip(lengths, new) if m > 0)
        return {"bytes": 4 * (4 * case["batch"] + 2 * case["rows"] + 2 * (pages + grown)), "flops": 0}
    dim, kv_heads, heads = case["dim"], case["kv_heads"], case["heads"]
    if case["op"] == "rows":
        row = 2 * (heads + kv_heads) * 2 * dim + 4 * case["rotary"] + 4  # q, k in and out, cos and sin
        if case["cached"]:  # v in, the codes of k and v, and k and v as they are read back
            row += kv_heads * 2 * dim + 4 + 2 * kv_heads * (dim + 8) + 2 * kv_heads * dim
        return {"bytes": case["tokens"] * row, "flops": case["tokens"] * (heads + kv_heads) * dim * 7}
    new, lengths = _sequences(case)
    shared, rows = case.get("prefix", 0), sum(new)
    seen = [_seen(case, n, length) for n, length in zip(new, lengths)]
    return {"bytes": (sum(k for k, _ in seen) + shared) * kv_heads * (dim + 8) + rows * heads * (4 * dim + 4),
            "flops": 4 * (sum(p for _, p in seen) + rows * shared) * heads * dim}


# ---------------------------------------------------------------- the definition in 64 bits

def _rounded(x, elem, how):
    """f64 values rounded by `how` (np.rint, np.floor) to the element type's numbers, as f64."""
    bits, low = (11, -24) if elem == F16 else (8, -133)
    _, e = np.frexp(x)
    unit = np.exp2(np.maximum(e - bits, low).astype(np.float64))
    return how(x / unit) * unit


def _held(x, elem):
    """What rows x (f64) read back as from the cache, before the last rounding."""
    m = x.min(-1, keepdims=True)
    s = _rounded((x.max(-1, keepdims=True) - m) / 15, elem, np.floor)
    with np.errstate(divide="ignore", invalid="ignore"):
        u = np.where(s > 0, np.clip(np.rint((x - m) / s), 0, 15), 0)
    return m + s * u


def _decode64(cache, case, slots):
    """(K, V) of the slots, f64 [slots][heads][dim]: each nibble and its row's parameters by their places."""
    page, dim, heads = case["page"], case["dim"], case["kv_heads"]
    head, c = torch.arange(heads, device=DEV)[:, None], torch.arange(dim, device=DEV)
    block = ((slots // page)[:, None, None] * heads + head) * (page * (dim + 8))
    token = (slots % page)[:, None, None]
    numbers = cache.view(torch.int16).view(DTYPES[case["elem"]])
    got = []
    for part in range(2):
        byte = cache[block + (part * page + token) * (dim // 2) + c // 2].int()
        u = (byte >> (4 * (c % 2)) & 15).double()
        m = (block + page * dim + (part * page + token) * 4) // 2
        got.append(numbers[m].double() + numbers[m + 1].double() * u)
    return got


def _exact_rows(state, case):
    tokens, dim, half = case["tokens"], case["dim"], case["rotary"] // 2
    fused = state["fused"].double().cpu().numpy().reshape(tokens, -1, dim)
    at = state["row_positions"].cpu().numpy()
    turn = (state["cos"].double().cpu().numpy() + 1j * state["sin"].double().cpu().numpy())[np.maximum(at, 0)]
    first = np.arange(half) * 2 if case["interleaved"] else np.arange(half)
    second = first + (1 if case["interleaved"] else half)
    heads, kv = case["heads"], case["kv_heads"]
    got = {}
    for name, x, weight in (("q", fused[:, :heads], state["q_weight"]),
                            ("k", fused[:, heads:heads + kv], state["k_weight"])):
        if case["norm"]:
            rms = np.sqrt(np.square(x).sum(-1, keepdims=True) / dim + float(np.float32(EPS)))
            x = x * weight.double().cpu().numpy() / rms
        y = x.copy()
        pair = (x[..., first] + 1j * x[..., second]) * turn[:, None]
        y[..., first], y[..., second] = pair.real, pair.imag
        got[name] = y
    if case["cached"]:
        got["k"] = _held(_rounded(got["k"], case["elem"], np.rint), case["elem"])
        got["v"] = _held(fused[:, heads + kv:], case["elem"])
    return {name: np.where((at >= 0)[:, None], y.reshape(tokens, -1), 0.0) for name, y in got.items()}


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    state = prepare(case, seed)
    if case["op"] == "rows":
        return _exact_rows(state, case)
    new, lengths = _sequences(case)
    heads, dim, page = case["heads"], case["dim"], case["page"]
    group, shared = heads // case["kv_heads"], case.get("prefix", 0)
    table, prefix_table = state["table"].long(), state["prefix_table"].long()
    out = torch.zeros(state["rows"], heads, dim, dtype=torch.float64)
    lse = torch.full((state["rows"], heads), -math.inf, dtype=torch.float64)
    at = torch.arange(shared, device=DEV)
    before = _decode64(state["cache"], case, prefix_table[at // page] * page + at % page)
    row = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        at = torch.arange(length, device=DEV)
        k, v = _decode64(state["cache"], case, table[b, at // page] * page + at % page)
        j, i = torch.arange(length, device=DEV), torch.arange(n, device=DEV)[:, None] + (length - n)
        hidden = (j > i) if case.get("causal", True) else torch.zeros(n, length, dtype=bool, device=DEV)
        if case.get("window"):
            hidden = hidden | ((j <= i - case["window"]) & (j >= case["sinks"]))
        if shared:
            k, v = torch.cat([before[0], k]), torch.cat([before[1], v])
            hidden = torch.cat([hidden.new_zeros(n, shared), hidden], 1)
        q = state["q"][row:row + n].double().view(n, heads, dim)
        for h in range(heads if len(k) else 0):
            t = (q[:, h] @ k[:, h // group].t().contiguous()) / math.sqrt(dim)
            t[hidden] = -math.inf
            total = torch.logsumexp(t, 1)
            weight = torch.exp(t - torch.where(total == -math.inf, 0.0, total)[:, None])
            out[row:row + n, h] = (weight @ v[:, h // group].contiguous()).cpu()
            lse[row:row + n, h] = total.cpu()
        row += n
    return {"out": out.view(state["rows"], heads * dim), "lse": lse}
