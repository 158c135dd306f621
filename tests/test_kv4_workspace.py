"""What attention over the 4-bit cache asks for as its workspace: a bound that every call stays under."""
import numpy as np

import h3attn as H

MOST = 66 << 20  # of head dim 128 on 256 compute units; the header's figure


def test_no_call_asks_for_more_than_the_stated_bound():
    rng = np.random.default_rng(11)
    seen = []
    for _ in range(20000):
        dim, page = int(rng.choice([64, 128])), 16 << int(rng.integers(0, 7))
        kv_heads = int(2 ** rng.uniform(0, 8))
        group = min(int(2 ** rng.uniform(0, 9)), 4096 // kv_heads)
        batch, max_q = int(2 ** rng.uniform(0, 15.9)), int(2 ** rng.uniform(0, 18))
        q_rows = min(2 ** 24, int(rng.integers(max_q, batch * max_q + 1)))
        columns = max(1, int(2 ** rng.uniform(0, 24)) // page)
        window = int(rng.integers(0, 2)) * int(2 ** rng.uniform(0, 20))
        width = kv_heads * group * dim
        if width > 2 ** 20 or max_q * group > 2 ** 30:
            continue
        cfg = H.Kv4Cfg(kv_heads, dim, page, 1000, 0)
        acfg = H.Kv4AttentionCfg(kv_heads * group, width, width, columns, 1, window, 0.1)
        seen.append(H.kv4_workspace_bytes(cfg, acfg, batch, q_rows, max_q))
    assert max(seen) <= MOST
    assert max(seen) > MOST // 2 and min(seen) == 0  # the sweep reaches both ends


def test_the_need_may_fall_where_the_batch_grows():
    """So a workspace that served one call may be too small for another of fewer sequences."""
    cfg = H.Kv4Cfg(8, 128, 64, 4096, H.H3_ELEM_F16)
    acfg = H.Kv4AttentionCfg(32, 4096, 4096, 2048, 1, 0, 0.1)
    need = [H.kv4_workspace_bytes(cfg, acfg, b, b, 1) for b in (1, 8, 1024)]
    assert need[0] > 0 and need[1] > 0 and need[2] == 0
