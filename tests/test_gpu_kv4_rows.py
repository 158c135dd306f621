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
