"""kv4_write and kv4_read where the arithmetic of a row is hard: scales against exact fractions, rows and words
that hold no numbers."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16


def toward_zero(x, elem):
    """The element type's bits of a Fraction x >= 0 rounded toward zero, by halving the range of its bits (the
    order of the numbers >= 0 is that of their bits)."""
    lo, hi = 0, 0x7bff if elem == F16 else 0x7f7f
    while lo < hi:
        mid = (lo + hi + 1) // 2
        if Fraction(float(P.from_bits(np.array([mid], np.uint16), elem)[0])) <= x:
            lo = mid
        else:
            hi = mid - 1
    return lo


def written(dev, elem, x, page=16):
    """The words [rows] and codes [rows][dim] of rows x [rows][dim] (16-bit tensor) as kv4_write leaves them."""
    n, dim = x.shape
    pages = -(-n // page)
    cfg = H.Kv4Cfg(1, dim, page, pages, elem)
    cache = torch.zeros(H.kv4_cache_bytes(cfg), dtype=torch.uint8, device=dev)
    slots = torch.arange(n, dtype=torch.int32, device=dev)
    x = x.to(dev)
    H.kv4_write(cfg, n, dim, dim, x, x, slots, cache)
    back = torch.empty(2, n, dim, dtype=x.dtype, device=dev)
    H.kv4_read(cfg, n, dim, dim, slots, cache, back[0], back[1])
    assert torch.equal(back[0].view(torch.int16), back[1].view(torch.int16))
    raw = cache.cpu().numpy().reshape(pages, page * (dim + 8))
    half = page * dim // 2
    codes = raw[:, :half].reshape(-1, dim // 2)[:n]
    words = np.ascontiguousarray(raw[:, 2 * half:2 * half + 4 * page]).view(np.uint32).reshape(-1)[:n]
    return words, np.stack([codes & 15, codes >> 4], -1).reshape(n, dim), back[0].cpu()


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_are_rounded_toward_zero_from_the_exact_range(dev, elem, dim):
    """Rows whose max - min is no 32-bit float: rounded to one it can be 15 times a number of the type that the
    exact range stays below."""
    small = [2.0 ** -24, 2.0 ** -16, 3 * 2.0 ** -20] if elem == F16 else [2.0 ** -133, 2.0 ** -40, 3 * 2.0 ** -30]
    ends = []
    for s in (1.0, 1.0078125, 1.9921875, 0.0625, 96.0, 1.5):  # 15 s is a number of both types where s is short
        top = 15 * s
        for e in small:
            ends += [(e, top), (-top, -e), (-e, top), (-top, e), (0.0, top), (-top, 0.0)]
    for e in small:
        ends += [(e, 16 * e), (-e, 14 * e), (3 * e, 3.0), (-e, e)]
    rng = np.random.default_rng(dim)
    a = torch.from_numpy(rng.standard_normal(200) * 2.0 ** rng.uniform(-12, 4, 200)).to(P.DTYPES[elem]).double()
    b = torch.from_numpy(rng.standard_normal(200) * 2.0 ** rng.uniform(-12, 4, 200)).to(P.DTYPES[elem]).double()
    ends += [(min(x, y), max(x, y)) for x, y in zip(a.tolist(), b.tolist())]
    x = torch.tensor(ends, dtype=torch.float64)
    x = torch.stack([x[:, 0], x[:, 1]], 1).repeat(1, dim // 2).to(P.DTYPES[elem])
    ends = [(float(r.double().min()), float(r.double().max())) for r in x]
    words, codes, back = written(dev, elem, x)
    for i, (lo, hi) in enumerate(ends):
        want = toward_zero((Fraction(hi) - Fraction(lo)) / 15, elem)
        assert words[i] >> 16 == want, (lo, hi, hex(words[i] >> 16), hex(want))
        m, s = (Fraction(float(P.from_bits(np.array([w], np.uint16), elem)[0]))
                for w in (words[i] & 0xffff, words[i] >> 16))
        assert m == Fraction(lo) and m + int(codes[i].max()) * s <= Fraction(hi), (lo, hi)
        assert lo <= float(back[i].double().min()) and float(back[i].double().max()) <= hi, (lo, hi)


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_hold_no_number(dev, elem, dim):
    """Every kind of NaN and infinity, in every lane's channels and several in a row, beside rows of numbers:
    0x7fff and codes 0, NaN when read back; the other rows as ever."""
    top = 0x7c00 if elem == F16 else 0x7f80
    kinds = [top, top | 0x8000, top | 1, top | 0x8001, 0x7fff, 0xffff, (0x7fff + top) // 2 + 1]
    rng = np.random.default_rng(dim)
    x = P.rows(rng, (600, dim), elem)
    bits = x.view(torch.int16).numpy().view(np.uint16)
    bad = np.arange(600) % 3 == 1
    for i in np.flatnonzero(bad):
        for c in rng.choice(dim, 1 + i % 4, replace=False):
            bits[i, c] = kinds[(i // 3 + c) % len(kinds)]
    bits[4] = 0xffff
    words, codes, back = written(dev, elem, x)
    want, want_codes, near = P.quantize(x, elem)
    assert (words == want).all() and (words[bad] == 0x7fff).all() and (codes[bad] == 0).all()
    assert (codes != want_codes).sum() <= near.sum()
    assert back[bad].isnan().all() and back[~bad].isfinite().all()


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_words_that_are_no_numbers_read_back_as_nan(dev, elem, dim):
    """Words that no written row has: either half a NaN or an infinity."""
    one, top = (0x3c00, 0x7c00) if elem == F16 else (0x3f80, 0x7f80)
    words = [one | (x << 16) for x in (top, top + 1, 0x7fff, 0x8000 | top, 0xffff)]
    words += [x | (one << 16) for x in (top, top + 1, 0x7fff, 0x8000 | top, 0xffff)] + [one | (one << 16)] * 6
    cfg = H.Kv4Cfg(1, dim, 16, 1, elem)
    plain = P.Cache(cfg, np.random.default_rng(1))
    plain.words[:, :, 0] = np.array(words, np.uint32)
    slots = torch.arange(16, dtype=torch.int32, device=dev)
    back = torch.empty(2, 16, dim, dtype=P.DTYPES[elem], device=dev)
    H.kv4_read(cfg, 16, dim, dim, slots, torch.from_numpy(plain.bytes()).to(dev), back[0], back[1])
    for part in (0, 1):
        y = back[part].cpu().double().numpy()
        assert np.isnan(y[:10]).all()
        assert (y[10:] == 1 + plain.codes[part, 10:, 0]).all()
