"""The operators of a serving step around the 4-bit cache, restated in numpy in 64 bits: attention with first
tokens or a shared prefix, pages and slots from requested lengths, and the norm and rotation of queries and
keys."""
import numpy as np
import torch

import kv4_plain as P
from kv4_plain import F32, HALF_STEP, from_bits


def visible(n, length, causal, window, sinks, shared):
    """[n][shared + length]: which keys each row sees, the shared ones first."""
    j, p = np.arange(length), length - n + np.arange(n)[:, None]
    seen = np.ones((n, length), bool)
    if causal:
        seen = j <= p
        if window:
            seen = seen & ((j > p - window) | (j < sinks))
    return np.concatenate([np.ones((n, shared), bool), seen], 1)


def attend(cache, acfg, q, table, new, lengths, sinks=0, prefix=None):
    """out [rows][heads][dim], lse [rows][heads] and their error bounds in f64. prefix: (pages, length) of what
    every sequence sees first. An entry that is no page hides its keys; a key whose words are no numbers makes
    the rows that see it NaN.

    The bounds, with h a rounding's half step in the element type: scores are f32 sums of dim exact products
    each, of q (16 + u) and of q, times s and m - 16 s, with a few roundings more: `delta`, (dim + 8) 2^-24 of
    the sums' magnitudes, shifts a score, so changes a weight by twice that, relative. Weights and values are
    rounded to 16 bits at most once each (h max|v| each), out once more; f32 sums have at most keys / 8 terms one after
    the other, and the joins of waves, of parts and of the two kinds of keys 64 at most."""
    c = cache.cfg
    group, dim, rows = acfg.heads // c.kv_heads, c.head_dim, q.shape[0]
    out, lse = np.zeros((rows, acfg.heads, dim)), np.full((rows, acfg.heads), -np.inf)
    out_tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
    qd, half = q.double().numpy(), HALF_STEP[c.elem]
    shared_pages, shared = prefix if prefix else (np.zeros(0, np.int64), 0)

    def slots_of(pages, n):
        j = np.arange(n)
        at = np.asarray(pages, np.int64)[j // c.page_tokens] if n else np.zeros(0, np.int64)
        live = (at >= 0) & (at < c.pages)
        return np.where(live, at, 0) * c.page_tokens + j % c.page_tokens, live

    front, front_live = slots_of(shared_pages, shared)
    first = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        if n == 0:
            continue
        own, own_live = slots_of(table[b], length)
        slots, live = np.concatenate([front, own]), np.concatenate([front_live, own_live])
        seen = visible(n, length, acfg.causal, acfg.window, sinks, shared) & live
        words = cache.words[:, slots]
        fields = [from_bits(((words >> s) & 0xffff).astype(np.uint16), c.elem) for s in (0, 16)]
        bad = ~np.isfinite(fields[0] + fields[1])
        m, s = (np.where(bad, 0, x) for x in fields)
        u = cache.codes[:, slots].astype(np.float64)
        at = slice(first, first + n)
        for g in range(c.kv_heads):
            k = m[0, :, g, None] + s[0, :, g, None] * u[0, :, g]
            v = m[1, :, g, None] + s[1, :, g, None] * u[1, :, g]
            gone = np.repeat((seen & (bad[0, :, g] | bad[1, :, g])).any(1), group)
            mask = np.repeat(seen, group, 0)
            heads = slice(g * group, (g + 1) * group)
            x = qd[at, heads].reshape(n * group, dim)
            keys = mask.sum(1)
            some = keys > 0
            t = np.where(mask, (x @ k.T) * acfg.scale, -np.inf)
            top = np.where(some, t.max(1, initial=-np.inf), 0)
            w = np.exp(t - top[:, None])
            total = np.where(some, w.sum(1), 1)
            o = (w / total[:, None]) @ v
            log = np.where(some, top + np.log(total), -np.inf)
            big = np.where(mask, np.abs(v).max(1, initial=0), 0).max(1, initial=0)
            ms = np.where(mask, np.abs(m[0, :, g]) + 31 * s[0, :, g], 0).max(1, initial=0)
            delta = (dim + 8) * F32 * abs(acfg.scale) * np.abs(x).sum(1) * 2 * ms
            sums = (keys / 8 + 64) * F32
            tol = (half * (np.abs(o) + 2 * big[:, None]) + ((2 * delta + 2 * sums) * 2 * big)[:, None]
                   + 2.0 ** -25)
            ltol = np.where(some, delta + sums + 4 * F32 * (np.abs(np.where(some, log, 0)) + 1), 0)
            o[~some] = tol[~some] = 0
            o[gone], log[gone] = np.nan, np.nan
            out[at, heads], out_tol[at, heads] = (y.reshape(n, group, dim) for y in (o, tol))
            lse[at, heads], lse_tol[at, heads] = (y.reshape(n, group) for y in (log, ltol))
        first += n
    return out, lse, out_tol, lse_tol


# ---------------------------------------------------------------- pages and slots

def advance(cfg, table_stride, rows, asked, lengths, free_pages, free_count, table, prefix=0):
    """kv4_advance one sequence after the other: (free_pages, free_count, table, lengths, q_starts, slots,
    positions) after it."""
    page, limit = cfg.page_tokens, table_stride * cfg.page_tokens
    free, table = free_pages.copy(), table.copy()
    count = min(max(int(free_count), 0), cfg.pages)
    cut = [min(max(int(n), 0), limit) for n in lengths]
    up = lambda n: -(-n // page)  # noqa: E731
    for b, n in enumerate(asked):
        if n < 0:
            for column in range(up(cut[b])):
                if 0 <= table[b, column] < cfg.pages and count < cfg.pages:  # an entry that is no page is none
                    free[count] = table[b, column]
                    count += 1
    out, starts = [], [0]
    slots, positions = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    wanted_pages = wanted_rows = 0
    top = count
    for b, n in enumerate(asked):
        have, n = (0, 0) if n < 0 else (cut[b], int(n))
        if have + n > limit:
            n = 0
        need = up(have + n) - up(have)
        wanted_pages, wanted_rows = wanted_pages + need, wanted_rows + n
        if (need and wanted_pages > count) or wanted_rows > rows:
            n = need = 0
        for i in range(need):
            top -= 1
            table[b, up(have) + i] = free[top]
        for i in range(n):
            at = have + i
            id_ = int(table[b, at // page])
            slots[starts[-1] + i] = id_ * page + at % page if 0 <= id_ < cfg.pages else -1
            positions[starts[-1] + i] = max(int(prefix), 0) + at
        starts.append(starts[-1] + n)
        out.append(have + n)
    return (free, top, table, np.array(out, np.int32), np.array(starts, np.int32), slots, positions)


# ---------------------------------------------------------------- norm and rotation

def nearest(x, elem):
    """f64 values rounded once to the element type, to nearest, ties to even: the 16-bit tensor."""
    bits, low, most = (11, -24, 65520.0) if elem == P.H.H3_ELEM_F16 else (8, -133, 2.0 ** 128 * (1 - 2.0 ** -9))
    with np.errstate(invalid="ignore"):
        _, e = np.frexp(x)
        unit = np.exp2(np.maximum(e.astype(np.float64) - bits, low))
        y = np.rint(x / unit) * unit
    y = np.where(np.abs(x) >= most, np.copysign(np.inf, x), np.where(np.isfinite(x), y, x))
    return torch.from_numpy(y).to(P.DTYPES[elem])  # holds y: exact


def norm_rope(cfg, x, weight, cos, sin, positions):
    """Rows x [tokens][heads][dim] (a 16-bit tensor) normed and rotated, in f64; rows without a position are as
    they were."""
    y = x.double().numpy().copy()
    live = (positions >= 0) & (positions < cfg.positions)
    with np.errstate(all="ignore"):
        if cfg.norm:
            mean = np.square(y).sum(-1, keepdims=True) / cfg.head_dim
            y = y / np.sqrt(mean + float(np.float32(cfg.eps))) * weight.astype(np.float64)
        half = cfg.rotary // 2
        if half:
            first = 2 * np.arange(half) if cfg.interleaved else np.arange(half)
            second = first + (1 if cfg.interleaved else half)
            at = np.where(live, positions, 0)
            c, s = (t[at].astype(np.float64)[:, None] for t in (cos, sin))
            a, b = y[..., first], y[..., second]
            y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    y[~live] = x.double().numpy()[~live]
    return y
