"""kv4_advance where entries of an ended sequence's row are no page: a program has taken pages back from behind a
window, or the row holds anything else. Whole numbers, all equal to the restatement's."""
import numpy as np
import pytest
import torch

import h3attn as H
from test_gpu_kv4_advance import both, put, state
from test_gpu_kv4_step import Server
from test_kv4_pages import behind_windows

pytestmark = pytest.mark.gpu


def test_an_ended_sequence_gives_back_the_pages_it_has(dev):
    cfg = H.Kv4Cfg(1, 64, 16, 9, 0)
    table = np.array([[0, -1, 9, -1, 4, 5], [-1] * 6], np.int32)
    want = both(dev, cfg, 6, 80, [-1, 70], [90, 0], np.array([7, 8] + [-9] * 7, np.int32), 2, table)
    assert list(want[4]) == [0, 0, 70] and (want[5][:70] >= 0).all()


@pytest.mark.parametrize("batch,page,most,new,ended,free,rows", [
    (1, 16, 900, 1, 1.0, 5, 1), (5, 16, 3000, 40, 0.6, 9, 200), (64, 64, 9000, 1, 0.5, 20, 64),
    (70, 16, 6000, 9, 0.5, 60, 300),         # more entries than the workgroup's threads hold at a time
    (1023, 16, 60, 3, 0.3, 300, 1400), (2500, 16, 200, 5, 0.4, 900, 9001)])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.9, 1.0])
def test_entries_that_are_no_page(dev, batch, page, most, new, ended, free, rows, share):
    rng = np.random.default_rng(batch + most)
    cfg, columns, asked, lengths, stack, count, table = state(rng, batch, page, most, new, ended, free)
    none = (rng.random(table.shape) < share) & (asked < 0)[:, None]
    table[none] = rng.choice([-1, -2 ** 31, cfg.pages, 2 ** 31 - 1], none.sum())
    for free_count in (count, cfg.pages - 2):  # with room for all of them, and for two
        both(dev, cfg, columns, rows, asked, lengths, stack, free_count, table)


def test_a_windows_pages_serve_others(dev):
    """Replays of one captured step; between them the pages that have left the windows go back on the stack."""
    server = Server(dev, H.H3_ELEM_F16, "sinks", sinks=5, window=20, rows=30, max_q=9, seed=9)
    x = server.buffers()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        server.step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        server.step(x)
    taken = ended = 0
    noise = torch.randn(1 << 16, device=dev)
    for i in range(60):
        asked, fused = server.request()
        asked = np.where((server.lengths > 60) & (server.rng.random(6) < 0.3), -1, np.abs(asked)).astype(np.int32)
        ended += sum(-1 in server.table[b, :-(-int(server.lengths[b]) // 16)] for b in np.nonzero(asked < 0)[0])
        new, n, *rest = server.follow(asked, fused)
        x["asked"].copy_(torch.from_numpy(asked))
        x["fused"].copy_(fused)
        noise.mul_(1.001)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        server.check(x, new, n, *rest)
        back = behind_windows(server.rng, server.table, server.lengths, 16, 5, 20)
        server.stack[server.count:server.count + len(back)] = back
        server.count += len(back)
        taken += len(back)
        held = [server.table[b, :-(-int(m) // 16)] for b, m in enumerate(server.lengths)]
        owned = np.concatenate([h[h >= 0] for h in held] + [server.stack[:server.count]])
        assert sorted(owned) == list(range(server.pages)), i
        for name, value in (("table", server.table), ("free", server.stack), ("count", [server.count])):
            x[name].copy_(put(value, dev))
    assert taken > 10 and ended > 3
    del graph
