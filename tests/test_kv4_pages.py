"""Pages that a program has taken back before their sequence ends (behind a window, -1 in their entries): every
page keeps one owner, and no row is granted without a slot. The restatement that the GPU tests compare with."""
import numpy as np

import h3attn as H
import kv4_step_plain as S


def behind_windows(rng, table, lengths, page, sinks, window):
    """Takes the pages that lie between the first tokens and the window of each sequence's next row off the table:
    their ids."""
    back = []
    for b, n in enumerate(lengths):
        for column in range(-(-sinks // page), max(0, int(n) + 1 - window) // page):
            if table[b, column] >= 0 and rng.random() < 0.8:
                back.append(int(table[b, column]))
                table[b, column] = -1
    return back


def test_an_ended_sequence_gives_back_the_pages_it_has():
    cfg = H.Kv4Cfg(1, 64, 16, 9, 0)
    table = np.array([[0, -1, -1, -1, 4, 5], [-1] * 6], np.int32)
    stack = np.array([7, 8] + [-9] * 7, np.int32)
    stack, count, table, lengths, starts, slots, _ = S.advance(cfg, 6, 80, [-1, 70], [90, 0], stack, 2, table)
    assert count == 0 and list(lengths) == [0, 70] and list(starts) == [0, 0, 70]
    assert list(table[1]) == [5, 4, 0, 8, 7, -1] and (slots[:70] >= 0).all()


def test_pages_taken_back_have_one_owner():
    rng = np.random.default_rng(5)
    cfg, page, sinks, window = H.Kv4Cfg(1, 64, 16, 40, 0), 16, 20, 40
    stack, count = rng.permutation(40).astype(np.int32), 40
    table, lengths = np.full((5, 14), -1, np.int32), np.zeros(5, np.int32)
    ended = taken = 0
    for _ in range(300):
        asked = np.where(rng.random(5) < 0.08, -1, rng.integers(0, 25, 5))
        ended += sum(-1 in table[b, :-(-n // page)] for b, n in enumerate(lengths) if asked[b] < 0)
        stack, count, table, lengths, starts, slots, _ = S.advance(cfg, 14, 90, asked, lengths, stack, count, table)
        assert (slots[:starts[-1]] >= 0).all()
        back = behind_windows(rng, table, lengths, page, sinks, window)
        stack[count:count + len(back)] = back
        count += len(back)
        taken += len(back)
        held = [table[b, :-(-n // page)] for b, n in enumerate(lengths)]
        owned = np.concatenate([h[h >= 0] for h in held] + [stack[:count]])
        assert sorted(owned) == list(range(40))
    assert ended > 10 and taken > 100
