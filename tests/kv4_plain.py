"""The 4-bit key/value cache restated in numpy, in 64 bits: the rows' codes and parameters, the bytes
of the layout, and attention over what they stand for."""
import math

import numpy as np
import torch

import h3attn as H

DTYPES = {H.H3_ELEM_F16: torch.float16, H.H3_ELEM_BF16: torch.bfloat16}
HALF_STEP = {H.H3_ELEM_F16: 2.0 ** -11, H.H3_ELEM_BF16: 2.0 ** -8}  # of a rounding, relative
F32 = 2.0 ** -24


def bits16(x):
    """A 16-bit torch tensor's bit patterns as numpy u16."""
    return x.contiguous().view(torch.int16).numpy().view(np.uint16)


def from_bits(bits, elem):
    """f64 values of u16 bit patterns."""
    t = torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).view(DTYPES[elem])
    return t.double().numpy()


def quantize(x, elem):
    """(words u32, codes u8, near): rows x [...][dim] (a 16-bit tensor) as the cache holds them;
    `near` marks codes within 2^-20 of the border of two."""
    y = x.double().numpy()
    with np.errstate(all="ignore"):
        lo, hi = y.min(-1), y.max(-1)
        bad = ~np.isfinite(y).all(-1)
        lo, hi = np.where(bad, 0, lo), np.where(bad, 0, hi)
        wide = (hi - lo) / 15
        s = bits16(torch.from_numpy(wide).float().to(DTYPES[elem]))
        s = np.where(from_bits(s, elem) > wide, s - 1, s).astype(np.uint16)
        step = from_bits(s, elem)[..., None]
        ratio = np.where(step > 0, (np.where(bad[..., None], 0, y) - lo[..., None]) / step, 0)
    codes = np.clip(np.rint(ratio), 0, 15).astype(np.uint8)
    codes[bad] = 0
    m = bits16(torch.from_numpy(lo).to(DTYPES[elem]))
    words = m.astype(np.uint32) | (s.astype(np.uint32) << 16)
    near = np.abs(ratio - np.floor(ratio) - 0.5) < 2.0 ** -20
    exact_tie = ratio * 2 == np.rint(ratio * 2)
    return np.where(bad, 0x7fff, words).astype(np.uint32), codes, near & ~exact_tie


class Cache:
    """Codes [slots][heads][dim] and words [slots][heads] of K and V, and their bytes."""

    def __init__(self, cfg, rng=None):
        self.cfg, self.slots = cfg, cfg.pages * cfg.page_tokens
        shape = (2, self.slots, cfg.kv_heads)
        self.codes = np.zeros(shape + (cfg.head_dim,), np.uint8)
        self.words = np.zeros(shape, np.uint32)
        if rng is not None:
            self.codes = rng.integers(0, 16, self.codes.shape).astype(np.uint8)

    def put(self, part, slots, x):
        """Rows x [len(slots)][heads][dim] quantized into part 0 (K) or 1 (V)."""
        words, codes, near = quantize(x, self.cfg.elem)
        ok = (slots >= 0) & (slots < self.slots)
        self.words[part, slots[ok]] = words[ok]
        self.codes[part, slots[ok]] = codes[ok]
        return near

    def bytes(self):
        c = self.cfg
        parts = [self.codes[p][..., 0::2] | (self.codes[p][..., 1::2] << 4) for p in (0, 1)]
        parts += [np.ascontiguousarray(self.words[p][..., None]).view(np.uint8) for p in (0, 1)]
        parts = [a.reshape(c.pages, c.page_tokens, c.kv_heads, -1).transpose(0, 2, 1, 3)
                 .reshape(c.pages, c.kv_heads, -1) for a in parts]
        return np.concatenate(parts, -1).reshape(-1)

    def values(self, part, slots):
        """f64 rows [len(slots)][heads][dim] that the slots stand for."""
        w = self.words[part, slots]
        m = from_bits((w & 0xffff).astype(np.uint16), self.cfg.elem)
        s = from_bits((w >> 16).astype(np.uint16), self.cfg.elem)
        with np.errstate(invalid="ignore"):
            return m[..., None] + s[..., None] * self.codes[part, slots]


def span(n, length, i, causal, window):
    if not causal:
        return 0, length
    p = length - n + i
    hi = max(0, min(length, p + 1))
    return min(hi, max(0, p + 1 - window) if window else 0), hi


def attend(cache, acfg, q, table, new, lengths):
    """out [rows][heads][dim], lse [rows][heads] and their error bounds, in f64, of the sequences'
    rows one after the other in q [rows][heads][dim] (a 16-bit tensor). A table entry that is no page
    hides its keys.

    The bounds. Scores: q (16 + u) and sum(q) are f32 sums of dim exact products each (relative
    error dim 2^-24 of the sum of magnitudes), times s and m - 16 s, a few roundings more; `delta`
    is that over the row's keys, a shift of a score, so twice a relative error of a weight.
    Probabilities and values are rounded to 16 bits at most once each (a half-step of max|v| each),
    out once more; sums of f32 add 2^-24 a term, of at most keys / 8 terms one after the other."""
    c = cache.cfg
    group, dim = acfg.heads // c.kv_heads, c.head_dim
    rows = q.shape[0]
    out, lse = np.zeros((rows, acfg.heads, dim)), np.full((rows, acfg.heads), -np.inf)
    out_tol, lse_tol = np.zeros((rows, acfg.heads, dim)), np.zeros((rows, acfg.heads))
    qd = q.double().numpy()
    half = HALF_STEP[c.elem]
    row = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        j = np.arange(length)
        pages = table[b, j // c.page_tokens].astype(np.int64) if length else np.zeros(0, np.int64)
        live = (pages >= 0) & (pages < c.pages)
        slots = np.where(live, pages, 0) * c.page_tokens + j % c.page_tokens
        k, v = cache.values(0, slots), cache.values(1, slots)
        kw = cache.words[0, slots]
        ms = np.abs(from_bits((kw & 0xffff).astype(np.uint16), c.elem)) + 31 * from_bits(
            (kw >> 16).astype(np.uint16), c.elem)  # [keys][heads]: |m| + 31 s
        for i in range(n):
            lo, hi = span(n, length, i, acfg.causal, acfg.window)
            at = j[lo:hi][live[lo:hi]]
            if not len(at):
                continue
            for h in range(acfg.heads):
                g = h // group
                t = (k[at, g] @ qd[row + i, h]) * acfg.scale
                total = np.logaddexp.reduce(t)
                p = np.exp(t - total)
                out[row + i, h] = p @ v[at, g]
                lse[row + i, h] = total
                delta = ((dim + 8) * F32 * abs(acfg.scale) * np.abs(qd[row + i, h]).sum()
                         * 2 * ms[at, g].max())
                sums = (len(at) / 8 + 64) * F32
                biggest = np.abs(v[at, g]).max()
                out_tol[row + i, h] = (half * (np.abs(out[row + i, h]) + 2 * biggest)
                                       + (2 * delta + 2 * sums) * 2 * biggest + 2.0 ** -25)
                lse_tol[row + i, h] = delta + sums + 4 * F32 * (abs(total) + 1)
        row += n
    return out, lse, out_tol, lse_tol


def attend_all(cache, acfg, q, table, new, lengths, kernel):
    """As `attend` over whole matrices, for many rows and heads, with the bounds of one kernel: "few" (tiles
    of 4 to 32 rows) or "rows" (of 256; along a line too). A row that sees a key whose row of K or of V holds a
    NaN or an infinity (a word that is none) has NaN in out and lse.

    The bounds, with h a rounding's half step in the element type, w_j a row's weights (they sum to 1),
    b the largest |v| it sees and n its keys:
    - scores, sums and lse as in `attend`: (2 delta + 2 sums) 2 b of out;
    - out once more rounded: h |out|;
    - few: p s is rounded once, a weight of u - 8: h sum_j w_j s_j |u_j - 8|. In f16 it is held 2^8 / S times, S the
      power of two from the largest s that any row of the tile has met (at most twice that s), and the largest p of a
      part is 1 or more: below the normal numbers it is off by 2^-25, n S 2^-33 8 in all. The f32 sums are of
      p s (16 + u), less 24 p s: 64 sum_j w_j s_j to the terms' roundings;
    - rows: p and v are rounded once each: 2 h (1 + 2^-8) sum_j w_j |v_j|. In f16, p is off by 2^-25 below the normal
      numbers, while a row's sum is 2^7 or more: n b 2^-32 in all; and v by 2^-25."""
    c = cache.cfg
    group, dim = acfg.heads // c.kv_heads, c.head_dim
    rows = q.shape[0]
    out, lse = np.zeros((rows, acfg.heads, dim)), np.full((rows, acfg.heads), -np.inf)
    out_tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
    qd = q.double().numpy()
    h, f16 = HALF_STEP[c.elem], c.elem == H.H3_ELEM_F16
    first = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        j = np.arange(length)
        pages = table[b, j // c.page_tokens].astype(np.int64) if length else np.zeros(0, np.int64)
        live = (pages >= 0) & (pages < c.pages)
        slots = np.where(live, pages, 0) * c.page_tokens + j % c.page_tokens
        spans = [span(n, length, i, acfg.causal, acfg.window) for i in range(n)]
        seen = np.array([(j >= lo) & (j < hi) for lo, hi in spans], bool).reshape(n, length) & live
        part = cache.words[:, slots]
        fields = [from_bits(((part >> s) & 0xffff).astype(np.uint16), c.elem) for s in (0, 16)]
        bad = ~np.isfinite(fields[0] + fields[1])            # [K, V][keys][heads]
        m, s = (np.where(bad, 0, x) for x in fields)
        u = cache.codes[:, slots].astype(np.float64)
        for g in range(c.kv_heads):
            k = m[0, :, g, None] + s[0, :, g, None] * u[0, :, g]
            v = m[1, :, g, None] + s[1, :, g, None] * u[1, :, g]
            nan = (seen & (bad[0, :, g] | bad[1, :, g])).any(1)
            heads = slice(g * group, (g + 1) * group)
            at = slice(first, first + n)
            x = qd[at, heads].reshape(n * group, dim)
            mask = np.repeat(seen, group, 0)
            keys = mask.sum(1)
            some = keys > 0
            t = np.where(mask, (x @ k.T) * acfg.scale, -np.inf)
            top = np.where(some, t.max(1, initial=-np.inf), 0)
            w = np.exp(t - top[:, None])
            total = np.where(some, w.sum(1), 1)
            w /= total[:, None]
            o = w @ v
            big = np.where(mask, np.abs(v).max(1, initial=0), 0).max(1, initial=0)
            ms = np.where(mask, np.abs(m[0, :, g]) + 31 * s[0, :, g], 0).max(1, initial=0)
            delta = (dim + 8) * F32 * abs(acfg.scale) * np.abs(x).sum(1) * 2 * ms
            sums = (keys / 8 + 64) * F32
            if kernel == "few":
                held = w @ (s[1, :, g, None] * np.abs(u[1, :, g] - 8))
                more = 64 * (w @ s[1, :, g])
                unit = 2 * s[1, seen.any(0), g].max(initial=0) * 2.0 ** -30 * keys if f16 else 0 * keys
            else:
                held, more = 2 * (1 + 2.0 ** -8) * (w @ np.abs(v)), 0
                unit = keys * big * 2.0 ** -32 + 2.0 ** -25 if f16 else 0 * keys
            tol = ((h * held + ((2 * delta + 2 * sums) * 2 * big + sums * more + unit)[:, None]) * (1 + h)
                   + h * np.abs(o) + (2.0 ** -25 if f16 else 0))
            log = np.where(some, top + np.log(total), -np.inf)
            ltol = np.where(some, delta + sums + 4 * F32 * (np.abs(top + np.log(total)) + 1), 0)
            gone = np.repeat(nan, group)
            o[~some] = tol[~some] = 0
            o[gone], log[gone] = np.nan, np.nan
            out[at, heads], out_tol[at, heads] = (y.reshape(n, group, dim) for y in (o, tol))
            lse[at, heads], lse_tol[at, heads] = (y.reshape(n, group) for y in (log, ltol))
        first += n
    return out, lse, out_tol, lse_tol


def rows(rng, shape, elem):
    """Rows whose channels differ in size and offset."""
    dim = shape[-1]
    x = rng.standard_normal(shape) * (0.3 + np.abs(rng.standard_normal(dim))) \
        + 0.5 * rng.standard_normal(dim)
    return torch.from_numpy(x).to(DTYPES[elem])


def softmax_scale(dim):
    return float(np.float32(1 / math.sqrt(dim)))


def within(got, want, tol):
    """got (f64) equals want to tol, infinities and NaNs in the same places."""
    same = np.isnan(got) == np.isnan(want)
    fine = np.isfinite(want)
    assert same.all(), f"{(~same).sum()} NaNs differ"
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
    over = np.abs(got[fine] - want[fine]) - tol[fine]
    assert not len(over) or over.max() <= 0, (
        f"{(over > 0).sum()} of {over.size} past their bound, the worst by {over.max():.3g}")
