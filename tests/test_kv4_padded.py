"""How a call behind a prefix divides its line among the rows that there are, of as many as it has places for: the
arithmetic of attention_kv4_prefix.hip's FrontLine, for every number of rows."""
import numpy as np

import h3attn as H
from test_kv4_step_host import prefix_plan

TILE, STEP, LEAST, JOIN = 256, 64, 8, 64


def line(plan, places, rows, kv_heads, length):
    """(steps of a tile, tiles, range of a workgroup)"""
    each, groups = -(-rows // TILE), plan.front_groups
    steps = max(-(-length // STEP), 1)
    most = min(places // max(rows, 1), JOIN - 1)
    return steps, each * kv_heads, max(-(-steps * each * kv_heads // groups), -(-steps // (most - 1)), LEAST)


def test_every_number_of_rows_has_places_for_its_pieces():
    rng = np.random.default_rng(11)
    lines = 0
    for _ in range(4000):
        dim, page = int(rng.choice([64, 128])), 16 << int(rng.integers(0, 7))
        kv_heads = int(2 ** rng.uniform(0, 8))
        group = min(int(2 ** rng.uniform(0, 7)), 4096 // kv_heads)
        batch, max_q = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 9))
        q_rows = int(rng.integers(max_q, batch * max_q + 1))
        stride = max(1, int(2 ** rng.uniform(10, 20)) // page)
        cfg = H.Kv4Cfg(kv_heads, dim, page, 1000, 0)
        width = kv_heads * group * dim
        acfg = H.Kv4AttentionCfg(kv_heads * group, width, width, max(1, 300 // page), 1, 0, 0.1)
        p = prefix_plan(cfg, acfg, stride, batch, q_rows, max_q)
        if not p.shared or p.front_parts:
            continue
        lines += 1
        places = (p.parts - 1) * q_rows * group
        for tokens in {0, 1, q_rows // 7, q_rows // 2, q_rows - 1, q_rows}:
            for length in {0, 65, stride * page // 3, stride * page}:
                rows = tokens * group
                steps, tiles, each = line(p, places, rows, kv_heads, length)
                assert each * p.front_groups >= steps * tiles  # all of it is some workgroup's
                assert p.front_groups * each < 2 ** 31
                first = np.arange(tiles, dtype=np.int64) * steps
                pieces = (first + steps - 1) // each - first // each + 1
                most = pieces.max(initial=0)
                assert most <= JOIN - 1 and most * rows <= places
                if tokens == q_rows:  # no padding: as the plan counts them
                    assert each == max(LEAST, -(-steps * tiles // p.front_groups))
    assert lines > 300
