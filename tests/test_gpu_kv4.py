"""The 4-bit key/value cache on the GPU: kv4_write and kv4_read against the numpy restatement byte for
byte, attention_kv4 against 64-bit attention over what the cache stands for (kv4_plain.py, which
derives the bounds)."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16
STALE = 0x7fff7fff  # a word whose minimum and scale are NaN, where nothing may look


def poisoned(cfg, dev):
    t = torch.full((H.kv4_cache_bytes(cfg) + 64,), 0xA5, dtype=torch.uint8, device=dev)
    return t


# ---------------------------------------------------------------- write and read

@pytest.mark.parametrize("elem,dim,heads,page,tokens,pad", [
    (F16, 128, 8, 16, 1, 0), (BF16, 128, 8, 64, 37, 0), (F16, 64, 3, 32, 130, 24),
    (BF16, 64, 1, 16, 7, 8), (F16, 128, 5, 256, 300, 1024), (BF16, 128, 2, 1024, 515, 8),
    (F16, 128, 1, 32, 20011, 16), (BF16, 64, 3, 16, 40003, 0),        # two rows a lane
    (BF16, 128, 1, 64, 131111, 8), (F16, 64, 5, 128, 131079, 0)])
def test_write_and_read_match_the_definition(dev, elem, dim, heads, page, tokens, pad):
    rng = np.random.default_rng(dim * tokens + heads)
    pages = tokens // page + 3
    cfg = H.Kv4Cfg(heads, dim, page, pages, elem)
    plain = P.Cache(cfg)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    slots[rng.random(tokens) < 0.2] = -1
    if tokens > 5:
        slots[4] = pages * page  # one past the last slot
        slots[5] = -2 ** 31
    k, v = (P.rows(rng, (tokens, heads, dim), elem) for _ in range(2))
    # Rows in a wider buffer, K and V at their own pitches.
    width = heads * dim
    kb = torch.full((tokens, width + pad), float("nan"), dtype=P.DTYPES[elem])
    vb = torch.full((tokens, width + 2 * pad), float("nan"), dtype=P.DTYPES[elem])
    kb[:, :width], vb[:, :width] = k.reshape(tokens, width), v.reshape(tokens, width)
    cache = poisoned(cfg, dev)
    dslots = torch.from_numpy(slots).to(dev)
    H.kv4_write(cfg, tokens, width + pad, width + 2 * pad, kb.to(dev), vb.to(dev), dslots, cache)
    got = cache.cpu().numpy()
    # What no slot names keeps its bytes.
    plain.codes[:] = np.where(np.arange(dim) % 2 == 0, 0x5, 0xA)
    plain.words[:] = 0xA5A5A5A5
    near = plain.put(0, slots, k).sum() + plain.put(1, slots, v).sum()
    want = np.concatenate([plain.bytes(), np.full(64, 0xA5, np.uint8)])
    differ = (got != want).sum()
    assert differ <= near, f"{differ} bytes differ, {near} codes lie at a border"

    back = torch.full((2, tokens, width + pad), 7.0, dtype=P.DTYPES[elem], device=dev)
    H.kv4_read(cfg, tokens, width + pad, width + pad, dslots, cache, back[0], back[1])
    back = back.cpu()
    assert (back[:, :, width:] == 7.0).all()
    ok = (slots >= 0) & (slots < pages * page)
    for part in (0, 1):
        y = back[part, :, :width].double().numpy().reshape(tokens, heads, dim)
        assert (y[~ok] == 0).all()
        value = plain.values(part, slots[ok])
        # one rounding in f32 and one to the element type
        tol = P.HALF_STEP[elem] * np.abs(value) * (1 + 2.0 ** -12) + 2.0 ** -25
        if not near:
            P.within(y[ok], value, tol)
        # and no further from the row than half a step and what the scale lost in rounding
        x = (k, v)[part].double().numpy()[ok]
        step = (x.max(-1) - x.min(-1))[..., None] / 15
        P.within(y[ok], x, step * (0.5 + 15 * 2 * P.HALF_STEP[elem]) + tol + 15 * 2.0 ** -24)


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_of_extreme_values(dev, elem, dim):
    """Constant rows, zeros of both signs, the type's largest and smallest values, NaN, infinities."""
    big = torch.finfo(P.DTYPES[elem]).max
    tiny = 2.0 ** -24 if elem == F16 else 2.0 ** -133
    x = torch.zeros(12, dim, dtype=torch.float64)
    x[1] = 3.25
    x[2, ::2] = -0.0
    x[3, 0], x[3, 1] = big, -big / 2
    x[4, 5] = big
    x[5, 7] = tiny
    x[6, 3] = 20 * tiny
    x[7, 9] = float("nan")
    x[8, 11] = float("inf")
    x[9, 13] = -float("inf")
    x[10] = torch.arange(dim) % 16
    x[11] = -(torch.arange(dim) % 31) * 0.5
    x = x.to(P.DTYPES[elem]).reshape(12, 1, dim)
    cfg = H.Kv4Cfg(1, dim, 16, 1, elem)
    slots = torch.arange(12, dtype=torch.int32, device=dev)
    cache = torch.zeros(H.kv4_cache_bytes(cfg), dtype=torch.uint8, device=dev)
    H.kv4_write(cfg, 12, dim, dim, x.to(dev), x.flip(0).contiguous().to(dev), slots, cache)
    plain = P.Cache(cfg)
    near = plain.put(0, np.arange(12), x).sum() + plain.put(1, np.arange(12), x.flip(0)).sum()
    got, want = cache.cpu().numpy(), plain.bytes()
    # Zeros of both signs may leave either as the minimum: 0x8000 for 0x0000.
    i = np.flatnonzero(got != want)
    zero_sign = (i >= 16 * dim) & ((got[i] ^ want[i]) == 0x80) & (got[i] & 0x7f == 0)
    assert (~zero_sign).sum() <= near
    back = torch.empty(2, 12, dim, dtype=P.DTYPES[elem], device=dev)
    H.kv4_read(cfg, 12, dim, dim, slots, cache, back[0], back[1])
    y = back[0].cpu().double().numpy()
    ref = x.reshape(12, dim).double().numpy()
    wrong = ~np.isfinite(ref).all(1)
    assert np.isnan(y[wrong]).all() and np.isfinite(y[~wrong]).all()
    assert (y[~wrong] >= ref[~wrong].min(1)[:, None]).all()
    assert (y[~wrong] <= ref[~wrong].max(1)[:, None]).all()
    assert (y[1] == 3.25).all() and (y[10] == ref[10]).all()


# ---------------------------------------------------------------- attention

class Call:
    """A cache, its table and the rows of some sequences, on the host and on the GPU."""

    def __init__(self, dev, elem, dim, heads, kv_heads, page, new, lengths, causal=1, window=0,
                 seed=0, pad=0, columns=0, out_pad=0):
        rng = self.rng = np.random.default_rng(seed + 17 * dim + sum(lengths))
        held = [-(-n // page) for n in lengths]
        columns = max(1, *held, columns)
        pages = sum(held) + 2
        self.cfg = H.Kv4Cfg(kv_heads, dim, page, pages, elem)
        self.width = heads * dim
        self.acfg = H.Kv4AttentionCfg(heads, self.width + pad, self.width + out_pad, columns, causal,
                                      window, P.softmax_scale(dim))
        order = rng.permutation(pages)
        self.table = np.full((len(new), columns), -7, np.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.new, self.lengths = list(new), list(lengths)
        self.plain = P.Cache(self.cfg, rng)
        self.plain.words[:] = STALE
        for b, n in enumerate(lengths):
            j = np.arange(n)
            slots = self.table[b, j // page] * page + j % page
            for part in (0, 1):
                self.plain.put(part, slots, P.rows(rng, (n, kv_heads, dim), elem))
        self.rows = sum(new)
        self.q = torch.from_numpy(rng.standard_normal((self.rows, heads, dim))).to(P.DTYPES[elem])
        self.dev = dev

    def run(self, workspace=True, max_q=None, stream=None, extra=0, starts=None):
        """(out, lse) in f64, after checking that nothing past the rows was written."""
        dev, a, c = self.dev, self.acfg, self.cfg
        rows = self.rows + extra
        q = torch.full((rows, a.q_stride), float("nan"), dtype=P.DTYPES[c.elem])
        q[:self.rows, :self.width] = self.q.reshape(self.rows, self.width)
        out = torch.full((rows + 1, a.out_stride), 5.0, dtype=P.DTYPES[c.elem], device=dev)
        lse = torch.full((rows + 1, a.heads), 9.0, dtype=torch.float32, device=dev)
        if starts is None:
            starts = np.concatenate([[0], np.cumsum(self.new)])
        max_q = max_q or max(1, *self.new)
        need = H.kv4_workspace_bytes(c, a, len(self.new), rows, max_q)
        ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=dev) if workspace else None
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
        args = (q.to(dev), put(self.plain.bytes()), put(self.table),
                put(np.array(self.lengths, np.int32)), put(starts.astype(np.int32)))
        torch.cuda.synchronize()
        H.attention_kv4(c, a, len(self.new), rows, max_q, *args, out, lse, ws, stream)
        torch.cuda.synchronize()
        if ws is not None:
            assert (ws[need:] == 0xFF).all()
        assert (out[self.rows:] == 5.0).all() and (out[:, self.width:] == 5.0).all()
        assert (lse[self.rows:] == 9.0).all()
        return (out[:self.rows, :self.width].cpu().double().numpy().reshape(self.rows, a.heads, -1),
                lse[:self.rows].cpu().double().numpy())

    def want(self):
        return P.attend(self.plain, self.acfg, self.q, self.table, self.new, self.lengths)

    def check(self, **how):
        out, lse, out_tol, lse_tol = self.want()
        got_out, got_lse = self.run(**how)
        P.within(got_lse, lse, lse_tol)
        P.within(got_out, out, out_tol)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 255, 257]


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens_at_every_edge(dev, elem, dim, page):
    Call(dev, elem, dim, 4, 2, page, [1] * len(EDGES), EDGES).check()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 6), (3, 1), (10, 2), (14, 2), (16, 1),
                                            (32, 2), (33, 1), (71, 1)])
def test_head_layouts(dev, heads, kv_heads):
    Call(dev, F16 if heads % 2 else BF16, 128, heads, kv_heads, 32, [1, 2, 3], [70, 1, 300],
         pad=8 * heads, out_pad=16).check()


@pytest.mark.parametrize("elem,dim,page,new,lengths,window", [
    (F16, 128, 16, [5, 1, 9, 3], [5, 100, 40, 2], 0),       # rows before the first key: empty
    (BF16, 64, 32, [7, 16, 0, 1], [90, 16, 33, 0], 0),
    (F16, 128, 64, [4, 4], [200, 67], 1),
    (BF16, 128, 16, [6, 2, 30], [260, 131, 30], 33),
    (F16, 64, 256, [33, 70], [33, 500], 64),
    (BF16, 128, 128, [130, 1, 64], [300, 77, 64], 0),
    (F16, 128, 16, [129, 200], [129, 431], 100),
    (F16, 64, 64, [65], [65], 0),
    (BF16, 64, 16, [257, 1], [257, 1000], 0)])
def test_ragged_rows_and_windows(dev, elem, dim, page, new, lengths, window):
    Call(dev, elem, dim, 4, 2, page, new, lengths, window=window).check()


@pytest.mark.parametrize("elem,dim", [(F16, 128), (BF16, 64)])
def test_every_row_sees_every_key(dev, elem, dim):
    Call(dev, elem, dim, 8, 2, 32, [40, 1, 150, 3], [77, 512, 100, 0], causal=0).check()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths", [
    (F16, 128, 4, 1, 16, [1], [9001]), (BF16, 128, 8, 8, 128, [1, 2], [5000, 3333]),
    (F16, 64, 12, 2, 64, [3], [12345]), (BF16, 64, 2, 1, 16, [1, 1, 1], [8191, 1, 4097]),
    (F16, 128, 4, 1, 64, [70], [2500])])
def test_long_keys_in_parts_and_in_one(dev, elem, dim, heads, kv_heads, page, new, lengths):
    call = Call(dev, elem, dim, heads, kv_heads, page, new, lengths)
    assert H.kv4_workspace_bytes(call.cfg, call.acfg, len(new), call.rows, max(new)) > 0
    call.check()
    call.check(workspace=False)


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,causal,window", [
    (F16, 128, 17, 1, 16, [1], [200], 1, 0),                   # a tile of 17 rows
    (BF16, 128, 31, 1, 64, [1, 1], [31, 32], 1, 0),
    (F16, 64, 32, 1, 16, [1, 1], [33, 0], 1, 0),
    (BF16, 64, 33, 1, 32, [1, 2, 3], [127, 128, 129], 1, 0),    # a second tile of one row
    (BF16, 128, 5, 1, 16, [7, 7], [300, 97], 1, 0),             # a token's heads in two tiles
    (F16, 128, 4, 2, 64, [20, 20], [1000, 20], 1, 0),
    (BF16, 64, 10, 2, 16, [13, 13], [400, 13], 1, 50),
    (F16, 128, 6, 1, 128, [40], [500], 0, 0),
    (F16, 64, 3, 3, 16, [97, 5], [97, 211], 1, 0),
    (BF16, 128, 4, 2, 16, [20], [5000], 1, 0),                  # keys in parts
    (F16, 64, 40, 2, 256, [5, 5, 5], [3000, 2999, 1], 1, 700)])
def test_tiles_of_32_rows(dev, elem, dim, heads, kv_heads, page, new, lengths, causal, window):
    call = Call(dev, elem, dim, heads, kv_heads, page, new, lengths, causal=causal, window=window)
    call.check()
    call.check(workspace=False)


# Sequences of more than 4,096 rows, which only the tiles of 256 take.
@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,causal,window", [
    (BF16, 128, 64, 1, 16, [65], [65], 1, 0),
    (F16, 64, 64, 1, 64, [65], [700], 1, 0),
    (F16, 128, 64, 1, 16, [70, 1, 0], [900, 300, 50], 1, 0),      # one line of keys
    (BF16, 128, 32, 1, 16, [140, 1, 9], [1200, 700, 300], 1, 0),  # both kinds of launch
    (F16, 64, 16, 1, 32, [300, 1, 40], [1500, 600, 40], 1, 0),
    (BF16, 64, 64, 1, 64, [70], [700], 0, 0),
    (F16, 128, 64, 1, 64, [70], [700], 1, 100),                   # a window
    (BF16, 128, 71, 1, 32, [60, 61], [60, 300], 1, 0),            # rows before any key, odd groups
    (F16, 128, 64, 1, 16, [80, 66], [70, 3], 1, 5)])
def test_tiles_of_256_rows(dev, elem, dim, heads, kv_heads, page, new, lengths, causal, window):
    call = Call(dev, elem, dim, heads, kv_heads, page, new, lengths, causal=causal, window=window)
    call.check()
    call.check(workspace=False)


@pytest.mark.parametrize("elem", [F16, BF16])
def test_masked_places_of_256_rows(dev, elem):
    """Pages that are none of the cache's, and a NaN key that the last three tokens see."""
    call = Call(dev, elem, 128, 64, 1, 16, [70, 66], [150, 66])
    call.table[0, 3] = -1
    call.table[1, 0] = call.cfg.pages
    call.check()
    at = 150 - 3
    slot = call.table[0, at // 16] * 16 + at % 16
    for part in (0, 1):
        call.plain.words[part, slot] = 0x7fff
        out, lse, out_tol, lse_tol = call.want()
        got, got_lse = call.run()
        P.within(np.delete(got, [67, 68, 69], 0), np.delete(out, [67, 68, 69], 0),
                 np.delete(out_tol, [67, 68, 69], 0))
        assert np.isnan(got[67:70]).all() and np.isnan(got_lse[67:70]).all()
        call.plain.words[part, slot] = 0


def test_many_sequences(dev):
    """More sequences than the tiles' line holds, among them prompts beside single tokens."""
    new = [1, 3, 0, 2] * 130 + [200]
    lengths = [5 + i % 23 for i in range(520)] + [260]
    for i in range(0, 520, 7):
        lengths[i] = new[i]
    Call(dev, F16, 64, 32, 1, 16, new, lengths).check()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,causal,window", [
    (F16, 128, 8, 2, 16, [300, 40, 1, 9], [2000, 40, 700, 1111], 1, 0),  # both kinds of launch
    (BF16, 128, 4, 1, 64, [513, 257], [600, 3001], 1, 0),                # tiles that end past 256 rows
    (F16, 64, 6, 3, 32, [100, 0, 100], [4500, 50, 99], 1, 2000),         # a window, rows before any key
    (BF16, 64, 2, 2, 16, [300], [3900], 0, 0)])
def test_long_rows_in_parts_and_in_one(dev, elem, dim, heads, kv_heads, page, new, lengths, causal, window):
    """Few long sequences, whose keys are divided."""
    call = Call(dev, elem, dim, heads, kv_heads, page, new, lengths, causal=causal, window=window)
    need = H.kv4_workspace_bytes(call.cfg, call.acfg, len(new), call.rows, max(new))
    assert need >= 2 * 2 * 256 * (dim + 2) * 4
    call.check()
    call.check(workspace=False)


def test_a_line_of_sequences_that_overlap(dev):
    """q_starts that name rows twice ask for more row tiles than the rows have: nothing is read or
    written out of bounds, and sequences whose tiles fit are right."""
    for heads in (8, 32):  # in tiles of 32 rows, and of 256 along one line
        call = Call(dev, F16, 128, heads, 1, 16, [200], [1500])
        out, lse, out_tol, lse_tol = call.want()
        call.new, call.lengths = [200] * 4, [1500] * 4
        call.table = np.repeat(call.table, 4, 0)
        call.rows = 200
        got, got_lse = call.run(max_q=200, starts=np.array([0, 200, 0, 200, 0]))
        P.within(got, out, out_tol)
        P.within(got_lse, lse, lse_tol)


def test_a_table_wider_than_the_sequences(dev):
    """Most parts of a call planned for the table's width have no keys."""
    Call(dev, F16, 128, 4, 2, 16, [1, 1, 2], [3, 0, 40], columns=4000).check()


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("heads", [3, 7, 13, 30])
def test_a_table_of_more_keys_than_the_caches_hold(dev, elem, heads):
    """Codes go past the caches then: by the table's width, not by the lengths."""
    call = Call(dev, elem, 128, heads, 1, 64, [1, 1], [1700, 33], columns=16384)
    call.check()
    call.check(workspace=False)


def test_entries_that_are_no_page_hide_their_keys(dev):
    call = Call(dev, BF16, 128, 4, 2, 16, [2, 1, 20], [100, 48, 200])
    call.table[0, 2] = -1
    call.table[0, 6] = call.cfg.pages
    call.table[1] = 2 ** 31 - 1
    call.table[2, 3:5] = -2 ** 31
    call.check()


def test_lengths_and_rows_outside_their_ranges_are_cut(dev):
    call = Call(dev, F16, 64, 2, 2, 16, [3, 2], [32, 32])
    call.check()
    want = call.run()[0]
    call.lengths = [2 ** 31 - 1, -5]  # cut to the table's two pages, and to none
    got, lse = call.run()
    assert np.array_equal(got[:3], want[:3])
    assert (got[3:] == 0).all() and (lse[3:] == -np.inf).all()
    call.lengths = [32, 32]
    got, _ = call.run(starts=np.array([-4, 3, 10 ** 9]))  # cut to [0, q_rows]: rows 0..2 and 3..4
    assert np.array_equal(got[3:], want[3:])


def test_rows_of_no_sequence_are_left(dev):
    call = Call(dev, BF16, 128, 6, 2, 32, [2, 0, 5], [33, 10, 64])
    out, lse, out_tol, lse_tol = call.want()
    got, got_lse = call.run(extra=9)  # nine rows behind the last sequence: checked in run
    P.within(got, out, out_tol)
    P.within(got_lse, lse, lse_tol)
    # a bound below a sequence's rows: the rows past it are left
    call = Call(dev, BF16, 128, 6, 2, 32, [5], [64])
    out, lse, out_tol, lse_tol = call.want()
    got, got_lse = call.run(max_q=3)
    P.within(got[:3], out[:3], out_tol[:3])
    assert (got[3:] == 5.0).all() and (got_lse[3:] == 9.0).all()


@pytest.mark.parametrize("new", [6, 200])
@pytest.mark.parametrize("elem", [F16, BF16])
def test_a_nan_key_reaches_only_the_rows_that_see_it(dev, elem, new):
    """The cache's masked places may hold anything: stale words (every test here), and keys behind a
    row's own position."""
    call = Call(dev, elem, 128, 4, 2, 16, [new], [new + 40])
    at = new + 40 - 3  # the third key from the end: the last three rows see it
    slot = call.table[0, at // 16] * 16 + at % 16
    for part in (0, 1):
        call.plain.words[part, slot] = 0x7fff
        out, lse, out_tol, lse_tol = call.want()
        got, got_lse = call.run()
        P.within(got[:-3], out[:-3], out_tol[:-3])
        P.within(got_lse[:-3], lse[:-3], lse_tol[:-3])
        assert np.isnan(got[-3:]).all()
        call.plain.words[part, slot] = 0


@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** 12])
@pytest.mark.parametrize("new,heads", [(1, 4), (100, 4), (70, 128)])
def test_values_far_from_one(dev, size, new, heads):
    """f16 values of any size weigh alike: the probabilities' 16-bit form is relative to the
    values' scale."""
    call = Call(dev, F16, 128, heads, 2, 16, [new], [new + 700])
    # The last keys' values a thousandfold smaller: f16 still holds them.
    j = np.arange(new + 700)
    slots = call.table[0, j // 16] * 16 + j % 16
    x = P.rows(call.rng, (len(j), 2, 128), F16).double() * size * 0.25
    x[-50:] /= 4
    call.plain.put(1, slots, x.to(torch.float16))
    out, lse, out_tol, lse_tol = call.want()
    got, _ = call.run()
    P.within(got, out, out_tol)


def test_scores_far_apart(dev):
    """One key's score far above the others', late and early, and scores of both signs past e^88."""
    for late, heads, new in ((False, 2, [1, 100]), (True, 2, [1, 100]), (True, 64, [1, 100])):
        call = Call(dev, F16, 128, heads, 1, 16, new, [900, 900])
        for b in (0, 1):
            at = 790 if late else 2
            slot = call.table[b, at // 16] * 16 + at % 16
            x = call.q[0 if b == 0 else 50, 0].double() * 12
            call.plain.put(0, np.array([slot]), x.to(torch.float16).reshape(1, 1, 128))
        call.check()


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_any_finite_scale(dev, scale):
    call = Call(dev, BF16, 64, 4, 2, 32, [1, 90], [333, 90])
    call.acfg.scale = scale
    call.check()


def test_a_call_repeats_bit_for_bit_and_on_another_stream(dev):
    call = Call(dev, F16, 128, 8, 2, 64, [1, 130, 4], [3000, 700, 4])
    first = call.run()
    again = call.run(stream=torch.cuda.Stream())
    assert all(np.array_equal(x, y) for x, y in zip(first, again))


def test_a_captured_step_follows_its_lengths(dev):
    """Write and attention in one graph, replayed as a decoding loop does: the slots, lengths and
    rows change between the replays, every replay equals the eager calls."""
    heads, kv_heads, dim, page, steps = 4, 2, 128, 16, 4
    call = Call(dev, F16, dim, heads, kv_heads, page, [1, 1], [542, 60], columns=40)
    spare = [p for p in range(call.cfg.pages) if p not in call.table]
    call.table[0, 34] = spare[0]  # the page that the first sequence grows into
    c, a = call.cfg, call.acfg
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    need = H.kv4_workspace_bytes(c, a, 2, 2, 1)
    state = []
    for _ in range(2):  # one set for the graph, one for the eager calls
        state.append({
            "cache": put(call.plain.bytes()), "table": put(call.table),
            "lengths": put(np.array(call.lengths, np.int32)),
            "starts": put(np.arange(3, dtype=np.int32)),
            "slots": torch.zeros(2, dtype=torch.int32, device=dev),
            "rows": torch.zeros(3, 2, kv_heads * dim, dtype=torch.float16, device=dev),
            "q": torch.zeros(2, heads * dim, dtype=torch.float16, device=dev),
            "out": torch.zeros(2, heads * dim, dtype=torch.float16, device=dev),
            "ws": torch.empty(need, dtype=torch.uint8, device=dev) if need else None})

    def step(s):
        H.kv4_write(c, 2, kv_heads * dim, kv_heads * dim, s["rows"][0], s["rows"][1], s["slots"],
                    s["cache"])
        H.attention_kv4(c, a, 2, 2, 1, s["q"], s["cache"], s["table"], s["lengths"], s["starts"],
                        s["out"], workspace=s["ws"])

    side = torch.cuda.Stream()
    state[0]["slots"].fill_(-1)
    with torch.cuda.stream(side):
        step(state[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(state[0])
    noise = torch.randn(1 << 18, device=dev)
    for i in range(steps):
        g = torch.Generator().manual_seed(i)
        rows = torch.randn(2, 2, kv_heads * dim, generator=g).to(torch.float16)
        q = torch.randn(2, heads * dim, generator=g).to(torch.float16)
        lengths = [542 + i + 1, 60 + i + 1]
        slots = [int(call.table[b, (n - 1) // page]) * page + (n - 1) % page
                 for b, n in enumerate(lengths)]
        for s in state:
            s["rows"][:2].copy_(rows)
            s["q"].copy_(q)
            s["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
            s["slots"].copy_(torch.tensor(slots, dtype=torch.int32))
            s["out"].zero_()
        noise.mul_(1.0001).add_(0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(state[1])
        torch.cuda.synchronize()
        for name in ("out", "cache"):
            assert torch.equal(state[0][name], state[1][name]), (i, name)
        assert state[0]["out"].abs().sum() > 0
    del graph


def test_offsets_past_32_bits(dev):
    """A cache of 4.6 GB whose used pages are its last."""
    cfg = H.Kv4Cfg(8, 128, 1024, 4200, F16)
    size = H.kv4_cache_bytes(cfg)
    assert size > 2 ** 32
    small = Call(dev, F16, 128, 16, 8, 1024, [1, 3], [1500, 20])
    cache = torch.empty(size, dtype=torch.uint8, device=dev)
    page_bytes = size // cfg.pages
    used = small.cfg.pages
    cache[-used * page_bytes:] = torch.from_numpy(small.plain.bytes()).to(dev)
    want, want_lse = small.run()
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    out = torch.zeros(4, 16 * 128, dtype=torch.float16, device=dev)
    args = (cfg, small.acfg, 2, 4, 3)
    table = np.where(small.table >= 0, small.table + cfg.pages - used, -1).astype(np.int32)
    H.attention_kv4(*args, small.q.reshape(4, -1).to(dev), cache, put(table),
                    put(np.array(small.lengths, np.int32)), put(np.array([0, 1, 4], np.int32)), out)
    got = out.cpu().double().numpy().reshape(want.shape)
    small_plain = small.run(workspace=False)[0]
    assert np.array_equal(got, small_plain)
    # rows written there and read back
    slot = torch.tensor([cfg.pages * 1024 - 1, 2 ** 22 + 5], dtype=torch.int32, device=dev)
    rows = torch.randn(2, 2, 8 * 128, device=dev).to(torch.float16)
    H.kv4_write(cfg, 2, 1024, 1024, rows[0], rows[1], slot, cache)
    back = torch.empty_like(rows)
    H.kv4_read(cfg, 2, 1024, 1024, slot, cache, back[0], back[1])
    step = (rows.float().view(2, 2, 8, 128).amax(-1) - rows.float().view(2, 2, 8, 128).amin(-1)) / 15
    off = (back.float() - rows.float()).view(2, 2, 8, 128).abs().amax(-1)
    assert (off <= step * 0.53 + 2.0 ** -9).all()


def test_a_decoder_layer_runs_on_the_cache(dev):
    """As a decoder uses them: the fused projection's rows through RMSNorm and RoPE, the prompt's keys
    and values into the cache, attention over it, then single tokens one after the other; every row
    against 64-bit attention over the cache's values, and the cache read back."""
    heads = kv_heads = 4
    dim, page, prompt, steps = 128, 32, 75, 3
    width, total = heads * dim, prompt + steps
    pages = -(-total // page)
    cfg = H.Kv4Cfg(kv_heads, dim, page, pages, F16)
    acfg = H.Kv4AttentionCfg(heads, width, width, pages, 1, 0, P.softmax_scale(dim))
    g = torch.Generator(device=dev).manual_seed(5)
    fused = torch.randn(total, 3 * width, generator=g, device=dev).to(torch.float16)
    ones = torch.ones(dim, device=dev)
    angle = torch.rand(total, 48, generator=g, device=dev) * 6 - 3
    cos, sin = angle.cos(), angle.sin()
    q, k = (torch.empty(total, width, dtype=torch.float16, device=dev) for _ in range(2))
    H.rope_qknorm_f16(H.RopeCfg(3 * width, heads, heads, width, 1e-5, 0, F16), total, fused, ones,
                      ones, cos, sin, q, k)
    table = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    at = torch.arange(total, device=dev)
    slots = (table[at // page] * page + at % page).to(torch.int32)
    cache = torch.zeros(H.kv4_cache_bytes(cfg), dtype=torch.uint8, device=dev)
    out = torch.zeros(total, width, dtype=torch.float16, device=dev)
    first = 0
    for n in [prompt] + [1] * steps:
        last = first + n
        v = fused[first:].view(-1)[2 * width:]  # the V columns, in place
        H.kv4_write(cfg, n, width, 3 * width, k[first:last], v, slots[first:last], cache)
        need = H.kv4_workspace_bytes(cfg, acfg, 1, n, n)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        H.attention_kv4(cfg, acfg, 1, n, n, q[first:last], cache, table[None].contiguous(),
                        torch.tensor([last], dtype=torch.int32, device=dev),
                        torch.tensor([0, n], dtype=torch.int32, device=dev), out[first:last],
                        workspace=ws)
        first = last
    torch.cuda.synchronize()
    plain = P.Cache(cfg)
    host = slots.cpu().numpy()
    rows = (k.cpu(), fused[:, 2 * width:].cpu())
    near = sum(plain.put(part, host, x.reshape(total, kv_heads, dim)).sum()
               for part, x in enumerate(rows))
    assert (cache.cpu().numpy() != plain.bytes()).sum() <= near
    want, _, tol, _ = P.attend(plain, acfg, q.cpu().reshape(total, heads, dim),
                               table.cpu().numpy()[None], [total], [total])
    P.within(out.cpu().double().numpy().reshape(want.shape), want, tol)
    back = torch.empty(2, total, width, dtype=torch.float16, device=dev)
    H.kv4_read(cfg, total, width, width, slots, cache, back[0], back[1])
    for part in (0, 1):
        value = plain.values(part, host).reshape(total, width)
        P.within(back[part].cpu().double().numpy(), value,
                 P.HALF_STEP[F16] * np.abs(value) * (1 + 2.0 ** -12) + 2.0 ** -25)
