"""kv4_advance over places of which most ask for nothing, with rows enough for the launch that finds slots and positions
by itself: right, and in a time that the idle places do not set."""
import numpy as np
import pytest
import torch

import h3attn as H
from test_gpu_kv4_advance import both, put, state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [5, 300, 2047, 2048, 2049, 5000, 65535])
@pytest.mark.parametrize("where", ["first", "last", "middle", "few", "pairs"])
def test_idle_sequences_between_rows(dev, batch, where):
    rng = np.random.default_rng(batch)
    cfg, columns, asked, lengths, stack, count, table = state(rng, batch, 16, 40, 3, 0.0, 3000)
    at = np.arange(batch)
    active = {"first": at < 3, "last": at >= batch - 3, "middle": np.abs(at - batch // 2) < 2,
              "few": rng.random(batch) < 5 / batch, "pairs": at // 2 % max(1, batch // 40) == 0}[where]
    asked = np.where(active, rng.integers(1, 4, batch), np.where(rng.random(batch) < 0.1, -1, 0))
    both(dev, cfg, columns, 2049 + batch % 7, asked, lengths, stack, count, table, 5)


def test_idle_sequences_cost_no_time(dev):
    """One token of 65,535 places: the first's, behind whose row all the others are passed, and the last's. 180 us each;
    passing them one at a time took 8,300 for the first."""
    batch, rows = 65535, 4096
    cfg = H.Kv4Cfg(1, 64, 16, 10, 0)
    zeros = lambda n: put(np.zeros(n), dev)  # noqa: E731

    def least(asks):
        asked = np.zeros(batch, np.int32)
        asked[asks] = 1
        args = (put(asked, dev), zeros(batch), put(np.arange(10), dev), put([10], dev), zeros(batch), zeros(batch),
                zeros(1), zeros(batch + 1), zeros(rows), zeros(rows))
        times = []
        for _ in range(8):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            H.kv4_advance(cfg, batch, 1, rows, *args)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        assert int((args[-1] == 0).sum()) == 1 and int((args[-1] == -1).sum()) == rows - 1
        return min(times)

    assert least(0) < 8 * least(batch - 1)
