"""The 4-bit cache's attention over whole matrices (kv4_plain.attend_all), which the kernels are held to, against
the row-by-row form; no GPU."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P


def cache_and_rows(elem, causal, window):
    rng = np.random.default_rng(3)
    cfg = H.Kv4Cfg(2, 64, 16, 12, elem)
    cache = P.Cache(cfg, rng)
    for part in (0, 1):
        cache.put(part, np.arange(192), P.rows(rng, (192, 2, 64), elem))
    table = np.concatenate([rng.permutation(12).reshape(3, 4), np.zeros((1, 4))]).astype(np.int32)
    table[1, 1] = -1
    new, lengths = [5, 3, 2, 0], [40, 33, 0, 7]
    acfg = H.Kv4AttentionCfg(6, 384, 384, 4, causal, window, P.softmax_scale(64))
    q = torch.from_numpy(rng.standard_normal((10, 6, 64))).to(P.DTYPES[elem])
    return cache, acfg, q, table, new, lengths


@pytest.mark.parametrize("elem", [H.H3_ELEM_F16, H.H3_ELEM_BF16])
@pytest.mark.parametrize("causal,window", [(1, 0), (0, 0), (1, 7)])
def test_attention_over_matrices_is_the_row_by_row_one(elem, causal, window):
    args = cache_and_rows(elem, causal, window)
    out, lse, _, lse_tol = P.attend(*args)
    for kernel in ("few", "rows"):
        got, got_lse, tol, got_tol = P.attend_all(*args, kernel)
        P.within(got, out, np.full(out.shape, 1e-12))
        P.within(got_lse, lse, np.full(lse.shape, 1e-12))
        assert np.allclose(got_tol, lse_tol, rtol=1e-9)
        assert (tol >= 0).all() and (tol[np.isneginf(lse)] == 0).all()


def test_a_nan_row_makes_the_rows_that_see_it_nan():
    cache, acfg, q, table, new, lengths = cache_and_rows(H.H3_ELEM_F16, 1, 0)
    for part in (0, 1):
        slot = table[0, 38 // 16] * 16 + 38 % 16
        kept = cache.words[part, slot, 1].copy()
        cache.words[part, slot, 1] = 0x7fff
        out, lse, _, _ = P.attend_all(cache, acfg, q, table, new, lengths, "rows")
        gone = np.zeros((10, 6), bool)
        gone[3:5, 3:] = True  # tokens at 38 and 39, the second cache head's three heads
        assert (np.isnan(lse) == gone).all() and (np.isnan(out).all(-1) == gone).all()
        cache.words[part, slot, 1] = kept
