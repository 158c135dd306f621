"""kv4_advance on the GPU against its restatement one sequence after the other: whole numbers, all equal."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_step_plain as S

pytestmark = pytest.mark.gpu


def put(x, dev):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)


def both(dev, cfg, columns, rows, asked, lengths, free, count, table, prefix=None, in_place=False):
    batch = len(asked)
    want = S.advance(cfg, columns, rows, asked, lengths, free, count, table, prefix or 0)
    guard = 7  # behind every output
    pad = lambda x: put(np.concatenate([np.asarray(x, np.int32).reshape(-1), np.full(3, guard)]), dev)  # noqa: E731
    d_free, d_table, d_lengths, d_count = pad(free), pad(table), pad(lengths), pad([count])
    out = d_lengths if in_place else pad(np.zeros(batch))
    count_out = d_count if in_place else pad([0])
    starts, slots, positions = pad(np.zeros(batch + 1)), pad(np.zeros(rows)), pad(np.zeros(rows))
    H.kv4_advance(cfg, batch, columns, rows, put(asked, dev), d_lengths, d_free, d_count, d_table, out,
                  count_out, starts, slots, positions, None if prefix is None else put([prefix], dev))
    torch.cuda.synchronize()
    got = (d_free, count_out, d_table, out, starts, slots, positions)
    names = ("free_pages", "free_count", "table", "lengths", "q_starts", "slots", "positions")
    for name, x, y in zip(names, got, want):
        x, y = x.cpu().numpy(), np.asarray(y, np.int32).reshape(-1)
        assert (x[-3:] == guard).all(), name
        assert np.array_equal(x[:-3], y), name
    if not in_place:
        assert np.array_equal(d_lengths.cpu().numpy()[:-3], np.asarray(lengths, np.int32))
    return want


def state(rng, batch, page, most, new, ended, free, columns=None):
    """(cfg, columns, asked, lengths, free, count, table) of sequences of up to `most` tokens."""
    lengths = rng.integers(0, most + 1, batch)
    asked = np.where(rng.random(batch) < ended, -rng.integers(1, 9, batch), rng.integers(0, new + 1, batch))
    held = -(-lengths // page)
    columns = columns or int(-(-(most + new) // page)) + 1
    pages = int(held.sum()) + free + 3
    order = rng.permutation(pages)
    table = np.full((batch, columns), -1, np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    stack = np.full(pages, -9, np.int32)
    stack[:free] = order[at:at + free]
    return H.Kv4Cfg(2, 64, page, pages, 0), columns, asked, lengths, stack, free, table


@pytest.mark.parametrize("batch,page,most,new,ended,free,rows", [
    (1, 16, 0, 1, 0.0, 1, 1),               # the first token of the first sequence
    (1, 16, 16, 16, 0.0, 0, 16),            # a page is needed and none is there
    (3, 16, 40, 1, 0.0, 5, 3),
    (7, 32, 100, 60, 0.3, 9, 200),
    (64, 64, 900, 1, 0.1, 20, 64),
    (65, 16, 300, 40, 0.2, 60, 900),        # short of pages
    (100, 16, 300, 40, 0.0, 400, 700),      # short of rows
    (300, 128, 1000, 300, 0.1, 500, 20000),
    (1023, 16, 60, 3, 0.2, 300, 1400),
    (1024, 16, 60, 3, 0.2, 300, 1400),
    (1025, 16, 60, 3, 0.2, 300, 1400),
    (2500, 16, 90, 5, 0.1, 900, 9001),
    (70, 1024, 5000, 3000, 0.1, 300, 131071)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_match_the_definition(dev, batch, page, most, new, ended, free, rows, in_place):
    rng = np.random.default_rng(batch * 31 + rows)
    for prefix in (None, 777):
        cfg, columns, asked, lengths, stack, count, table = state(rng, batch, page, most, new, ended, free)
        both(dev, cfg, columns, rows, asked, lengths, stack, count, table, prefix, in_place)


@pytest.mark.parametrize("new,rows", [(1, 2000), (1, 70000), (3, 60000)])
def test_the_largest_batch(dev, new, rows):
    rng = np.random.default_rng(rows)
    cfg, columns, asked, lengths, stack, count, table = state(rng, 65535, 16, 40, new, 0.3, 3000)
    if rows == 2000:
        asked[rng.random(len(asked)) < 0.95] = 0  # nearly all idle
    both(dev, cfg, columns, rows, asked, lengths, stack, count, table, 5, True)


def test_a_refused_sequence_keeps_what_it_has(dev):
    cfg = H.Kv4Cfg(1, 64, 16, 12, 0)
    table = np.array([[0, 1, -1], [2, -1, -1], [3, 4, 5], [6, -1, -1]], np.int32)
    stack = np.array([9, 8, 7] + [-1] * 9, np.int32)
    lengths = [32, 10, 48, 16]
    # pages: 0 asks for one, 1 for two more than there are, 2 is at its table's end, 3 asks for one of none left
    want = both(dev, cfg, 3, 100, [1, 38, 1, 1], lengths, stack, 2, table)
    assert list(want[4]) == [0, 1, 1, 1, 1] and want[1] == 1
    # 3 needs none and is granted
    want = both(dev, cfg, 3, 100, [1, 38, 1, 0], lengths, stack, 2, table)
    want = both(dev, cfg, 3, 100, [1, 38, 0, 1], [32, 10, 48, 15], stack, 2, table)
    assert list(want[4]) == [0, 1, 1, 1, 2]
    # and what ends makes room in the same step
    want = both(dev, cfg, 3, 100, [1, 38, -1, 1], lengths, stack, 2, table)
    assert list(want[4]) == [0, 1, 39, 39, 40]


def test_values_outside_their_ranges(dev):
    rng = np.random.default_rng(8)
    cfg, columns, asked, lengths, stack, count, table = state(rng, 20, 16, 100, 5, 0.2, 30)
    asked[:5] = [2 ** 31 - 1, -2 ** 31, 2 ** 24, 3, 0]
    lengths[4:9] = [2 ** 31 - 1, -7, 2 ** 20, 10 ** 6, 50]
    table[9] = 2 ** 31 - 1
    table[10] = -2 ** 31
    table[11, 0] = cfg.pages
    for free_count in (count, -3, 2 ** 31 - 1, cfg.pages):
        both(dev, cfg, columns, 60, asked, lengths, stack, free_count, table, prefix=-4)


def test_a_captured_step_follows_its_requests(dev):
    """The whole of a sequence's life in replays of one graph: admitted, grown over pages, ended, its pages
    another's."""
    rng = np.random.default_rng(4)
    batch, page, columns, rows = 5, 16, 9, 40
    cfg = H.Kv4Cfg(2, 64, page, 24, 0)
    stack, count = rng.permutation(24).astype(np.int32), 24
    table, lengths = np.full((batch, columns), -1, np.int32), np.zeros(batch, np.int32)
    asked_d, free_d, count_d = put(np.zeros(batch), dev), put(stack, dev), put([count], dev)
    table_d, lengths_d, starts = put(table, dev), put(lengths, dev), put(np.zeros(batch + 1), dev)
    slots, positions = put(np.zeros(rows), dev), put(np.zeros(rows), dev)

    def step():
        H.kv4_advance(cfg, batch, columns, rows, asked_d, lengths_d, free_d, count_d, table_d, lengths_d,
                      count_d, starts, slots, positions)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()  # of no rows: nothing changes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    noise = torch.randn(1 << 16, device=dev)
    for i in range(30):
        asked = np.where(rng.random(batch) < 0.15, -1, rng.integers(0, 15, batch)).astype(np.int32)
        asked_d.copy_(put(asked, dev))
        noise.mul_(1.001)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        stack, count, table, lengths, *rest = S.advance(cfg, columns, rows, asked, lengths, stack, count, table)
        for x, y in zip((free_d, count_d, table_d, lengths_d, starts, slots, positions),
                        (stack, [count], table, lengths, *rest)):
            assert np.array_equal(x.cpu().numpy(), np.asarray(y, np.int32)), i
        owned = np.concatenate([table[b, :-(-n // page)] for b, n in enumerate(lengths)] + [stack[:count]])
        assert sorted(owned) == list(range(24))  # every page is one's
    del graph
