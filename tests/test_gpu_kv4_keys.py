"""attention_kv4_sinks and attention_kv4_prefix on the GPU against 64-bit attention over what the cache stands
for (kv4_step_plain.py, which derives the bounds)."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
import kv4_step_plain as S
from test_gpu_kv4 import STALE, Call
from test_kv4_step_host import prefix_plan

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16


class Front(Call):
    """A call with first tokens (sinks) or behind a prefix of `prefix` keys, whose words past its end are stale."""

    def __init__(self, dev, elem, dim, heads, kv_heads, page, new, lengths, sinks=None, prefix=None,
                 prefix_columns=0, **more):
        self.sinks, self.prefix = sinks, prefix
        held = -(-prefix // page) if prefix else 0
        # The prefix's pages are one more sequence's, taken off again.
        super().__init__(dev, elem, dim, heads, kv_heads, page, list(new) + [0],
                         list(lengths) + [prefix or 0], **more)
        self.new, self.lengths = list(new), list(lengths)
        self.prefix_table = np.full(max(1, held, prefix_columns), -3, np.int32)
        self.prefix_table[:held] = self.table[-1, :held]
        self.table = np.ascontiguousarray(self.table[:-1, :max(1, *[-(-n // page) for n in lengths],
                                                               more.get("columns", 0))])
        self.acfg.table_stride = self.table.shape[1]
        self.prefix_length = prefix

    def need(self, rows, max_q):
        c, a, n = self.cfg, self.acfg, len(self.new)
        if self.sinks is not None:
            return H.kv4_sinks_workspace_bytes(c, a, self.sinks, n, rows, max_q)
        return H.kv4_prefix_workspace_bytes(c, a, len(self.prefix_table), n, rows, max_q)

    def run(self, workspace=True, max_q=None, stream=None, extra=0, starts=None):
        dev, a, c = self.dev, self.acfg, self.cfg
        rows = self.rows + extra
        q = torch.full((rows, a.q_stride), float("nan"), dtype=P.DTYPES[c.elem])
        q[:self.rows, :self.width] = self.q.reshape(self.rows, self.width)
        out = torch.full((rows + 1, a.out_stride), 5.0, dtype=P.DTYPES[c.elem], device=dev)
        lse = torch.full((rows + 1, a.heads), 9.0, dtype=torch.float32, device=dev)
        if starts is None:
            starts = np.concatenate([[0], np.cumsum(self.new)])
        max_q = max_q or max(1, *self.new)
        need = self.need(rows, max_q)
        ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=dev) if workspace else None
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
        sequences = (put(self.table), put(np.array(self.lengths, np.int32)), put(starts.astype(np.int32)))
        q, cache = q.to(dev), put(self.plain.bytes())
        torch.cuda.synchronize()
        if self.sinks is not None:
            H.attention_kv4_sinks(c, a, self.sinks, len(self.new), rows, max_q, q, cache, *sequences, out, lse,
                                  ws, stream)
        else:
            H.attention_kv4_prefix(c, a, len(self.prefix_table), len(self.new), rows, max_q, q, cache,
                                   put(self.prefix_table), put(np.array([self.prefix_length], np.int32)),
                                   *sequences, out, lse, ws, stream)
        torch.cuda.synchronize()
        if ws is not None:
            assert (ws[need:] == 0xFF).all()
        assert (out[self.rows:] == 5.0).all() and (out[:, self.width:] == 5.0).all()
        assert (lse[self.rows:] == 9.0).all()
        return (out[:self.rows, :self.width].cpu().double().numpy().reshape(self.rows, a.heads, -1),
                lse[:self.rows].cpu().double().numpy())

    def want(self):
        prefix = (self.prefix_table, self.prefix) if self.sinks is None else None
        return S.attend(self.plain, self.acfg, self.q, self.table, self.new, self.lengths,
                        sinks=self.sinks or 0, prefix=prefix)

    def both(self):
        """With a workspace and without."""
        self.check()
        self.check(workspace=False)


# ---------------------------------------------------------------- first tokens beside a window

LENGTHS = [0, 1, 2, 5, 16, 31, 33, 63, 64, 65, 66, 127, 129, 130, 193, 257, 300]


@pytest.mark.parametrize("elem,dim", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("window,sinks", [(1, 1), (1, 64), (33, 4), (64, 65), (100, 129), (7, 1000), (500, 3)])
def test_sinks_of_single_tokens(dev, elem, dim, page, window, sinks):
    Front(dev, elem, dim, 4, 2, page, [1] * len(LENGTHS), LENGTHS, sinks=sinks, window=window).check()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,window,sinks", [
    (F16, 128, 8, 1, 16, [1, 2], [900, 40], 100, 5),                  # 8 rows to a tile, and 16
    (BF16, 64, 7, 1, 32, [2, 1, 2], [901, 333, 2], 130, 31),
    (F16, 128, 4, 2, 64, [5, 3, 0, 9], [400, 3, 10, 5], 33, 70),      # 32; rows before the first key
    (BF16, 128, 5, 1, 16, [7, 7], [300, 97], 1, 1),
    (F16, 64, 40, 2, 256, [5, 5, 5], [3000, 2999, 1], 700, 300),
    (BF16, 64, 33, 1, 32, [1, 2, 3], [127, 128, 300], 64, 64),
    (F16, 128, 4, 1, 64, [70, 1], [2500, 900], 200, 90),
    (BF16, 128, 4, 1, 16, [300, 1, 40], [1500, 600, 40], 320, 17)])
def test_sinks_in_tiles(dev, elem, dim, heads, kv_heads, page, new, lengths, window, sinks):
    Front(dev, elem, dim, heads, kv_heads, page, new, lengths, sinks=sinks, window=window).both()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,window,sinks", [
    (BF16, 128, 64, 1, 16, [65], [700], 100, 1),
    (F16, 64, 64, 1, 64, [65, 66], [700, 66], 64, 64),
    (F16, 128, 64, 1, 16, [70, 1, 0], [900, 300, 50], 130, 65),
    (BF16, 64, 64, 1, 32, [80, 66], [70, 900], 5, 200),
    (F16, 128, 32, 1, 16, [140, 1, 9], [1200, 700, 300], 300, 129),
    (BF16, 128, 4, 2, 64, [1100], [1100], 150, 40),
    (F16, 64, 8, 1, 16, [600], [1500], 70, 333)])
def test_sinks_in_tiles_of_256_rows(dev, elem, dim, heads, kv_heads, page, new, lengths, window, sinks):
    Front(dev, elem, dim, heads, kv_heads, page, new, lengths, sinks=sinks, window=window).both()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,new", [
    (F16, 128, 4, 1, [1]), (BF16, 64, 16, 2, [2]), (F16, 64, 4, 1, [9])])
def test_sinks_behind_a_long_window_in_parts(dev, elem, dim, heads, kv_heads, new):
    call = Front(dev, elem, dim, heads, kv_heads, 64, new, [12000], sinks=777, window=9000)
    assert call.need(call.rows, max(new)) > 0
    call.both()


def test_pages_between_the_first_tokens_and_the_window_are_not_read(dev):
    for new, heads in (([1, 1], 4), ([9, 2], 4), ([70, 3], 64)):
        call = Front(dev, BF16, 128, heads, 1, 16, new, [1000, 500], sinks=20, window=100)
        got = call.run()
        first = [(n - m + 1 - 100) // 16 for n, m in zip(call.lengths, new)]
        for b, column in enumerate(first):
            for at in range(2 * 16, column * 16):  # what a recycled page would hold
                slot = call.table[b, at // 16] * 16 + at % 16
                call.plain.words[:, slot] = STALE
            call.table[b, 2:column] = -1
        again = call.run()
        assert all(np.array_equal(x, y) for x, y in zip(got, again))
        call.check()


def test_sinks_that_hold_no_number_reach_every_row(dev):
    call = Front(dev, F16, 128, 4, 2, 16, [3, 1], [400, 300], sinks=4, window=50)
    slot = call.table[0, 0] * 16 + 3
    call.plain.words[1, slot] = 0x7fff
    call.check()
    call.plain.words[1, slot] = 0
    slot = call.table[0, 0] * 16 + 4  # the token after them: no row's
    call.plain.words[:, slot] = 0x7fff
    call.check()


@pytest.mark.parametrize("window,sinks", [(0, 40), (77, 0)])
def test_without_sinks_or_window_it_is_the_plain_call(dev, window, sinks):
    call = Front(dev, F16, 64, 6, 2, 32, [1, 40, 3], [900, 300, 70], sinks=sinks, window=window)
    got = call.run()
    plain = Call.run(call)
    assert all(np.array_equal(x, y) for x, y in zip(got, plain))


# ---------------------------------------------------------------- a shared prefix

@pytest.mark.parametrize("elem,dim", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("prefix", [1, 15, 63, 64, 65, 250, 511])
def test_single_tokens_behind_a_prefix(dev, elem, dim, page, prefix):
    Front(dev, elem, dim, 4, 2, page, [1] * len(LENGTHS), LENGTHS, prefix=prefix).check()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,prefix,causal", [
    (F16, 128, 8, 1, 16, [1, 2], [90, 40], 900, 1),
    (BF16, 64, 7, 7, 32, [2, 1, 2], [201, 333, 2], 1111, 1),
    (F16, 128, 4, 2, 64, [5, 3, 0, 9], [400, 3, 10, 5], 77, 1),       # rows before their own first key
    (BF16, 128, 5, 1, 16, [7, 7], [300, 97], 2000, 1),
    (F16, 64, 40, 2, 128, [5, 5, 5], [300, 299, 1], 3001, 1),
    (BF16, 64, 33, 1, 32, [1, 2, 3], [127, 128, 300], 640, 0),
    (F16, 128, 4, 1, 64, [70, 1], [250, 900], 1000, 1),
    (BF16, 128, 4, 1, 16, [300, 1, 40], [500, 600, 40], 1500, 1),
    (F16, 64, 12, 12, 16, [1, 1, 1, 1], [20, 1, 40, 33], 4099, 1),
    (BF16, 128, 16, 1, 1024, [3] * 9, [5] * 9, 1500, 1)])
def test_tiles_behind_a_prefix(dev, elem, dim, heads, kv_heads, page, new, lengths, prefix, causal):
    Front(dev, elem, dim, heads, kv_heads, page, new, lengths, prefix=prefix, causal=causal).both()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,prefix", [
    (BF16, 128, 64, 1, 16, [65], [65], 700),
    (F16, 64, 64, 1, 64, [65, 66], [700, 66], 129),
    (F16, 128, 64, 1, 16, [70, 1, 0], [900, 300, 50], 333),
    (BF16, 64, 64, 1, 32, [80, 66], [70, 100], 2000),                 # rows before their own first key
    (F16, 128, 32, 1, 128, [140, 1, 9], [1200, 700, 300], 400),
    (BF16, 128, 4, 2, 64, [1100], [1100], 1300)])
def test_tiles_of_256_rows_behind_a_prefix(dev, elem, dim, heads, kv_heads, page, new, lengths, prefix):
    Front(dev, elem, dim, heads, kv_heads, page, new, lengths, prefix=prefix).both()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,batch,prefix,most", [
    (F16, 128, 4, 1, 130, 2100, 60),       # 520 rows of one cache head
    (BF16, 128, 8, 2, 64, 5000, 200),
    (F16, 64, 12, 12, 40, 3000, 90),
    (BF16, 64, 3, 1, 300, 700, 33),
    (F16, 128, 40, 1, 9, 9001, 20)])
def test_many_single_tokens_share_a_prefix(dev, elem, dim, heads, kv_heads, batch, prefix, most):
    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, most + 1, batch)]
    Front(dev, elem, dim, heads, kv_heads, 16, [1] * batch, lengths, prefix=prefix).both()


def test_drafted_tokens_share_a_prefix(dev):
    rng = np.random.default_rng(3)
    new = [int(n) for n in rng.integers(0, 7, 50)]
    lengths = [n + int(m) for n, m in zip(new, rng.integers(0, 150, 50))]
    Front(dev, BF16, 128, 8, 2, 64, new, lengths, prefix=3500).both()


def test_a_prefix_of_no_keys_is_the_plain_call(dev):
    for new in ([1, 1, 1], [1, 30, 3], [200, 1, 70]):
        lengths = [900, 300, 70]
        call = Front(dev, F16, 128, 4, 1, 32, new, [max(n, m) for n, m in zip(lengths, new)], prefix=0,
                     prefix_columns=7)
        call.check()


def test_the_prefix_length_is_cut_to_its_table(dev):
    call = Front(dev, F16, 64, 4, 2, 16, [1, 3], [40, 90], prefix=96)
    want = call.run()
    call.prefix_length = 2 ** 31 - 1
    assert all(np.array_equal(x, y) for x, y in zip(want, call.run()))
    call.prefix_length = -5
    call.prefix = 0
    call.check()


def test_a_prefix_shorter_than_its_table(dev):
    call = Front(dev, BF16, 128, 8, 2, 64, [1] * 20, [50] * 20, prefix=130, prefix_columns=500)
    call.check()


def test_places_of_a_prefix_that_are_no_page_or_no_number(dev):
    for batch in (2, 70):
        call = Front(dev, BF16, 128, 4, 1, 16, [1] * batch, [30] * batch, prefix=1500)
        call.prefix_table[3] = -1
        call.prefix_table[40] = call.cfg.pages
        call.table[1, 0] = 2 ** 31 - 1
        call.both()
        slot = call.prefix_table[7] * 16 + 5
        call.plain.words[0, slot] = 0x7fff  # a key that every row sees
        out, lse = call.run()
        assert np.isnan(out).all() and np.isnan(lse).all()
        call.plain.words[0, slot] = 0
        slot = call.table[0, 1] * 16 + 3  # and one that the first sequence sees
        call.plain.words[1, slot] = 0x7fff
        call.check()


def test_rows_of_no_sequence_are_left_behind_a_prefix(dev):
    for new in ([2, 0, 5], [1] * 70):
        call = Front(dev, BF16, 128, 6, 2, 32, new, [33 + n for n in new], prefix=900)
        out, lse, out_tol, lse_tol = call.want()
        got, got_lse = call.run(extra=9)  # their q is NaN
        P.within(got, out, out_tol)
        P.within(got_lse, lse, lse_tol)
    call = Front(dev, BF16, 128, 6, 2, 32, [5], [64], prefix=900)
    out, lse, out_tol, lse_tol = call.want()
    got, got_lse = call.run(max_q=3)
    P.within(got[:3], out[:3], out_tol[:3])
    assert (got[3:] == 5.0).all() and (got_lse[3:] == 9.0).all()


def test_prefix_values_far_from_the_sequences(dev):
    """f16 weights are held relative to the largest scale of V: the prefix's and the sequences' differ."""
    for factor in (2.0 ** -10, 2.0 ** 10):
        for batch in (3, 80):
            call = Front(dev, F16, 128, 4, 1, 16, [1] * batch, [40] * batch, prefix=1200)
            j = np.arange(1200)
            slots = call.prefix_table[j // 16] * 16 + j % 16
            x = P.rows(call.rng, (len(j), 1, 128), F16).double() * factor
            call.plain.put(1, slots, x.to(torch.float16))
            call.check()


def test_scores_of_the_prefix_far_from_the_sequences(dev):
    for batch in (3, 80):
        for where in ("prefix", "own"):
            call = Front(dev, F16, 128, 2, 1, 16, [1] * batch, [40] * batch, prefix=700)
            slot = call.prefix_table[9] * 16 + 3 if where == "prefix" else call.table[1, 1] * 16 + 3
            x = call.q[1, 0].double() * 12
            call.plain.put(0, np.array([slot]), x.to(torch.float16).reshape(1, 1, 128))
            call.check()


@pytest.mark.parametrize("kind", ["sinks", "prefix"])
def test_calls_repeat_bit_for_bit_and_on_another_stream(dev, kind):
    for new in ([1, 130, 4], [1] * 60):
        lengths = [300 + n for n in new]
        how = {"sinks": 70, "window": 120} if kind == "sinks" else {"prefix": 3000}
        call = Front(dev, F16, 128, 8, 2, 64, new, lengths, **how)
        first = call.run()
        again = call.run(stream=torch.cuda.Stream())
        assert all(np.array_equal(x, y) for x, y in zip(first, again))


# Calls that are cut in each way: all rows over the prefix in tiles of 32 beside the sequences' own tiles of 4 to 32
# rows, or along a line of tiles of 256.
@pytest.mark.parametrize("cut,elem,dim,heads,kv_heads,page,new,most,prefix", [
    (4, F16, 128, 8, 2, 16, [1] * 64, 200, 5003),
    (4, BF16, 64, 12, 4, 64, [1] * 60 + [0], 90, 9001),
    (8, BF16, 128, 14, 2, 32, [1] * 90, 150, 6000),
    (8, F16, 64, 8, 2, 16, [2, 1] * 20, 130, 7777),
    (16, F16, 128, 32, 2, 16, [1] * 60, 100, 7000),
    (16, BF16, 64, 8, 2, 128, [4, 3, 0, 1] * 9, 333, 5000),
    (32, BF16, 128, 20, 4, 64, [5] * 30, 150, 8000),
    (32, F16, 64, 4, 1, 16, [17, 30, 1, 20] * 5, 99, 12000),
    ("apart", F16, 128, 12, 3, 16, [1] * 500, 70, 2000),                  # a wave to a cache head
    ("apart", BF16, 64, 30, 6, 64, [1] * 300 + [0], 90, 1500),
    ("apart", F16, 64, 10, 5, 32, [3, 1, 0, 2] * 80, 130, 1200),
    ("apart", BF16, 64, 45, 5, 32, [1] * 200, 60, 2000),
    ("line", F16, 64, 4, 1, 16, [1] * 1100, 20, 3001),
    ("line", BF16, 128, 64, 2, 64, [65] * 6, 300, 5000),                  # own keys in tiles of 32
    ("line", F16, 128, 64, 2, 16, [66, 1, 1, 90] * 4, 250, 9000),         # of 32 and of 256
    ("line", BF16, 64, 64, 2, 32, [1] * 60 + [140], 120, 9000)])
def test_calls_behind_a_prefix_cut_in_every_way(dev, cut, elem, dim, heads, kv_heads, page, new, most, prefix):
    rng = np.random.default_rng(len(new) + prefix)
    lengths = [n + int(m) for n, m in zip(new, rng.integers(0, most, len(new)))]
    lengths[0] = max(0, new[0] - 1)  # its first row sees no key of its own
    call = Front(dev, elem, dim, heads, kv_heads, page, new, lengths, prefix=prefix)
    plan = prefix_plan(call.cfg, call.acfg, len(call.prefix_table), len(new), call.rows, max(new))
    assert plan.shared
    if cut == "line":
        assert plan.front_parts == 0
    else:
        assert plan.front_parts > 0 and (plan.heads_apart if cut == "apart" else plan.own.few.tile == cut)
    call.check()
    # replays of what the workspace held before do no harm, nor do a length and starts that changed
    call.lengths[1] = max(0, call.lengths[1] - 1)
    call.check()
    for length in (0, 1, prefix // 2):
        call.prefix = call.prefix_length = length
        call.check()
    if max(new) > 1:  # a bound below a sequence's rows: the rows past it are left
        out, lse, out_tol, lse_tol = call.want()
        got, got_lse = call.run(max_q=max(new) - 1)
        last = np.cumsum(new)[np.array(new) == max(new)] - 1
        some = np.setdiff1d(np.arange(call.rows), last)
        P.within(got[some], out[some], out_tol[some])
        P.within(got_lse[some], lse[some], lse_tol[some])
        assert (got[last] == 5.0).all() and (got_lse[last] == 9.0).all()
    call.prefix = call.prefix_length = prefix
    call.plain.words[1, call.prefix_table[0] * page + 9] = 0x7fff  # a key that every row sees
    out, lse = call.run()
    assert np.isnan(out).all() and np.isnan(lse).all()


@pytest.mark.parametrize("more", [{"prefix": 700}, {"sinks": 9, "window": 100}])
@pytest.mark.parametrize("kv_heads,batch", [(2, 20001), (20, 65535)])
def test_batches_of_which_few_sequences_have_rows(dev, more, kv_heads, batch):
    new, lengths = [0] * batch, [0] * batch
    for b, n, length in ((5, 1, 300), (4444, 2, 77), (batch - 1, 3, 120)):
        new[b], lengths[b] = n, length
    lengths[7] = 40  # keys and no rows
    Front(dev, F16, 64, kv_heads, kv_heads, 16, new, lengths, **more).both()
