"""The numpy restatements of the step's operators against others: attention with nothing in front of it, the
rounding against torch's, pages against what must always hold."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
import kv4_step_plain as S


@pytest.mark.parametrize("elem", [H.H3_ELEM_F16, H.H3_ELEM_BF16])
def test_attention_with_nothing_in_front(elem):
    rng = np.random.default_rng(2)
    cfg = H.Kv4Cfg(2, 64, 16, 12, elem)
    cache = P.Cache(cfg)
    for part in (0, 1):
        cache.put(part, np.arange(192), P.rows(rng, (192, 2, 64), elem))
    table = rng.permutation(12).reshape(2, 6).astype(np.int32)
    q = P.rows(rng, (7, 4, 64), elem)
    for window in (0, 20):
        acfg = H.Kv4AttentionCfg(4, 256, 256, 6, 1, window, 0.125)
        a = P.attend(cache, acfg, q, table, [3, 4], [90, 4])
        b = S.attend(cache, acfg, q, table, [3, 4], [90, 4])
        for x, y in zip(a, b):
            assert np.allclose(x, y, rtol=1e-9, atol=1e-12)
    # a prefix and then the rest is the whole: the first 32 keys of sequence 0 as its prefix
    acfg = H.Kv4AttentionCfg(4, 256, 256, 6, 1, 0, 0.125)
    whole = S.attend(cache, acfg, q[:3], table[:1], [3], [90])
    split = S.attend(cache, acfg, q[:3], table[:1, 2:], [3], [58], prefix=(table[0, :2], 32))
    assert np.allclose(whole[0], split[0]) and np.allclose(whole[1], split[1])
    # sinks as long as the sequence make the window no matter
    acfg.window = 5
    assert np.allclose(S.attend(cache, acfg, q[:3], table[:1], [3], [90], sinks=90)[0], whole[0])


@pytest.mark.parametrize("elem", [H.H3_ELEM_F16, H.H3_ELEM_BF16])
def test_nearest_is_the_types_rounding(elem):
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.standard_normal(5000) * np.exp2(rng.integers(-30, 17, 5000)),
                        [0.0, -0.0, np.inf, -np.inf, np.nan, 65519.0, 65520.0, 2.0 ** -25, 2.0 ** -26]])
    x = x.astype(np.float32).astype(np.float64)  # torch rounds f32 values once
    want = torch.from_numpy(x).float().to(P.DTYPES[elem])
    got = S.nearest(x, elem)
    assert torch.equal(got.nan_to_num(3.0), want.nan_to_num(3.0))
    assert torch.equal(got.isnan(), want.isnan())


def test_pages_have_one_owner():
    rng = np.random.default_rng(0)
    cfg = H.Kv4Cfg(1, 64, 16, 40, 0)
    stack, count = rng.permutation(40).astype(np.int32), 40
    table, lengths = np.full((6, 8), -1, np.int32), np.zeros(6, np.int32)
    for _ in range(200):
        asked = np.where(rng.random(6) < 0.1, -1, rng.integers(0, 30, 6))
        before = lengths
        stack, count, table, lengths, starts, slots, positions = S.advance(cfg, 8, 90, asked, lengths, stack,
                                                                            count, table)
        owned = np.concatenate([table[b, :-(-n // 16)] for b, n in enumerate(lengths)] + [stack[:count]])
        assert sorted(owned) == list(range(40))
        n = starts[-1]
        assert (slots[:n] >= 0).all() and (slots[n:] == -1).all() and (positions[n:] == -1).all()
        assert len(set(slots[:n])) == n
        for b in range(6):
            if asked[b] >= 0:
                assert lengths[b] - before[b] == starts[b + 1] - starts[b] in (0, asked[b])
