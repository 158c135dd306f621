"""qk_norm_rope and qk_norm_rope_kv4 on rows of zeros, of the type's largest and smallest values, and with NaN and
infinities in them, against the definition in 64 bits channel by channel: which are NaN, which infinite, which neither.
With the norm a NaN makes its head's whole row NaN, an infinity (r = 0) its own channel and its pair's other, beside
zeros; without it both stay in their pair."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
from test_gpu_qk_rows import BF16, F16, Rows

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def extreme(dev, elem, norm, interleaved, rotary, eps=1e-5):
    rows = Rows(dev, elem, 128, 2, 2, 14, rotary, interleaved, norm, pad=8, skip=0)
    rows.cfg.eps = eps
    big = torch.finfo(P.DTYPES[elem]).max / (1 if norm else 2)  # without the norm a pair's length has to be one too
    tiny = 2.0 ** -24 if elem == F16 else 2.0 ** -133
    other = 3 if interleaved else 2 + rotary // 2
    for x in (rows.q, rows.k):
        x[0] = 0.0
        x[1] = big
        x[2, :, ::2] = -big
        x[3] = tiny
        x[4, :, 5:] = 0.0
        x[5, 0, 7] = NAN
        x[6, 1, 9] = INF
        x[7, 0, 100] = -INF
        x[8, 0, 2] = x[8, 0, other] = INF  # a pair's two
        x[9, 0, 127], x[9, 1, 0] = INF, NAN
        x[10] = 0.0
        x[10, :, 60] = tiny
        x[11] = -0.0
        x[12] = tiny
        x[12, 0, 3] = INF
    rows.fused[:, :rows.q_width + rows.width] = torch.cat([rows.q.flatten(1), rows.k.flatten(1)], 1)
    return rows


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("interleaved,rotary", [(0, 0), (0, 32), (0, 128), (1, 32), (1, 128)])
@pytest.mark.parametrize("norm,eps", [(0, 0.0), (1, 0.0), (1, 2.0 ** -149), (1, 2.0 ** -140), (1, 2.0 ** -126),
                                      (1, 1e-5), (1, 2.0 ** 127)])
def test_each_channel_of_extreme_rows(dev, elem, interleaved, rotary, norm, eps):
    rows = extreme(dev, elem, norm, interleaved, rotary, eps)
    with np.errstate(all="ignore"):
        rows.check(*rows.run(), least=2.0 ** -133)


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("norm", [0, 1])
def test_extreme_rows_into_the_cache(dev, elem, norm):
    rows = extreme(dev, elem, norm, 0, 128)
    kv = H.Kv4Cfg(2, 128, 16, 2, elem)
    size, tokens = H.kv4_cache_bytes(kv), rows.tokens
    cache, want = (torch.full((size,), 0xA5, dtype=torch.uint8, device=dev) for _ in range(2))
    flat = rows.fused.to(dev).view(-1)
    slots = torch.from_numpy(rows.rng.permutation(32)[:tokens].astype(np.int32)).to(dev)
    q_out = torch.full((tokens, rows.cfg.q_out_stride), 5.0, dtype=flat.dtype, device=dev)
    v = flat[rows.q_width + rows.width:]
    H.qk_norm_rope_kv4(rows.cfg, kv, tokens, flat, flat[rows.q_width:], v, *rows.args(), slots, q_out, cache)
    plain_q, plain_k = rows.run()
    bits = lambda x: x.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(q_out.cpu()[:, :rows.q_width].reshape(plain_q.shape)), bits(plain_q))
    H.kv4_write(kv, tokens, rows.width, rows.cfg.v_stride, plain_k.to(dev).flatten(1), v, slots, want)
    assert torch.equal(cache, want)
