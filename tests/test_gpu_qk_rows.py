"""qk_norm_rope and qk_norm_rope_kv4 on the GPU against their definition in 64 bits.

Queries: r is off by the roundings of dim squares' sum, of its mean, root and quotient ((dim / 16 + 16) 2^-24), a
product by a weight's factor is one rounding in the factor and one of its own, and a channel is the sum of two such
products, rounded, times r: 8 roundings of |a| + |b|, (dim / 16 + 24) 2^-24 (|a| + |b|) in all, and half a step.
Keys: the definition's value rounded once; only where that lies within 2^-40 of the middle of two may the other be
right."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
import kv4_step_plain as S

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16


class Rows:
    """Rows of [q | k | v] and what they are turned by."""

    def __init__(self, dev, elem, dim, heads, kv_heads, tokens, rotary, interleaved, norm, positions=300, pad=0,
                 skip=0.2, seed=0):
        rng = self.rng = np.random.default_rng(seed + tokens * 7 + heads)
        self.dev, self.tokens, self.dim = dev, tokens, dim
        self.q_width, self.width = heads * dim, kv_heads * dim
        pitch = self.q_width + 2 * self.width + pad
        self.cfg = H.QkCfg(heads, kv_heads, dim, rotary, interleaved, norm, positions, 1e-5, elem, pitch, pitch,
                           pitch, self.q_width + pad, self.width + 2 * pad)
        self.fused = torch.full((tokens, pitch), float("nan"), dtype=P.DTYPES[elem])
        parts = [P.rows(rng, (tokens, n, dim), elem) for n in (heads, kv_heads, kv_heads)]
        self.q, self.k, self.v = parts
        self.fused[:, :self.q_width + 2 * self.width] = torch.cat([x.flatten(1) for x in parts], 1)
        self.weights = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
        angle = rng.uniform(-3, 3, (positions, rotary // 2))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.positions = rng.integers(0, positions, tokens).astype(np.int32)
        self.positions[rng.random(tokens) < skip] = -1

    def args(self):
        put = lambda x: torch.from_numpy(x).to(self.dev)  # noqa: E731
        weights = [put(w) if self.cfg.norm else None for w in self.weights]
        turns = [put(t) if self.cfg.rotary else None for t in (self.cos, self.sin)]
        return (*weights, *turns, put(self.positions))

    def run(self):
        """(q_out, k_out) with their padding columns checked."""
        c = self.cfg
        flat = self.fused.to(self.dev).view(-1)
        q_out = torch.full((self.tokens + 1, c.q_out_stride), 5.0, dtype=flat.dtype, device=self.dev)
        k_out = torch.full((self.tokens + 1, c.k_out_stride), 6.0, dtype=flat.dtype, device=self.dev)
        H.qk_norm_rope(c, self.tokens, flat, flat[self.q_width:], *self.args(), q_out, k_out)
        q_out, k_out = q_out.cpu(), k_out.cpu()
        assert (q_out[-1] == 5.0).all() and (q_out[:, self.q_width:] == 5.0).all()
        assert (k_out[-1] == 6.0).all() and (k_out[:, self.width:] == 6.0).all()
        return (q_out[:-1, :self.q_width].reshape(self.q.shape),
                k_out[:-1, :self.width].reshape(self.k.shape))

    def live(self):
        return (self.positions >= 0) & (self.positions < self.cfg.positions)

    def check(self, q_out, k_out, least=0.0):
        c, live = self.cfg, self.live()
        q, k = (S.norm_rope(c, x, w, self.cos, self.sin, self.positions)
                for x, w in zip((self.q, self.k), self.weights))
        # |a| + |b| of each channel: the rotation of the magnitudes, with the tables' magnitudes
        both = H.QkCfg.from_buffer_copy(c)
        size = S.norm_rope(both, self.q.abs(), np.abs(self.weights[0]), np.abs(self.cos), -np.abs(self.sin),
                           self.positions)
        other = S.norm_rope(both, self.q.abs(), np.abs(self.weights[0]), np.abs(self.cos), np.abs(self.sin),
                            self.positions)
        size = np.maximum(np.abs(size), np.abs(other))
        half, tiny = P.HALF_STEP[c.elem], 2.0 ** -25 if c.elem == F16 else least
        tol = half * np.abs(q) * (1 + 2.0 ** -10) + (self.dim / 16 + 24) * P.F32 * size + tiny
        got = q_out.double().numpy()
        P.within(got[live], q[live], tol[live])
        assert (got[~live] == 5.0).all()
        want = S.nearest(k, c.elem).double().numpy()
        got = k_out.double().numpy()
        differ = (got != want) & ~(np.isnan(got) & np.isnan(want))
        differ[~live] = False
        # the middle of two neighbours, where the definition's value is on its border
        middle = (got + want) / 2
        assert (np.abs(middle - k)[differ] <= 2.0 ** -40 * np.abs(k)[differ]).all(), f"{differ.sum()} keys differ"
        assert (got[~live] == 6.0).all()


KINDS = [(0, 0), (0, 1), (1, 0), (1, 1)]


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim,rotary", [(64, 0), (64, 16), (64, 48), (64, 64), (128, 32), (128, 96), (128, 128)])
@pytest.mark.parametrize("interleaved,norm", KINDS)
def test_rows_match_the_definition(dev, elem, dim, rotary, interleaved, norm):
    rows = Rows(dev, elem, dim, 6, 2, 37, rotary, interleaved, norm, pad=8)
    rows.check(*rows.run())


@pytest.mark.parametrize("elem,dim,heads,kv_heads,tokens,pad", [
    (F16, 128, 1, 1, 1, 0), (BF16, 64, 1, 1, 1, 8), (F16, 128, 3, 5, 2, 16), (BF16, 128, 40, 8, 5, 0),
    (F16, 64, 71, 1, 9, 8), (BF16, 64, 12, 12, 1001, 0), (F16, 128, 32, 8, 2003, 24), (BF16, 128, 9, 3, 9001, 0)])
def test_heads_and_lengths(dev, elem, dim, heads, kv_heads, tokens, pad):
    rows = Rows(dev, elem, dim, heads, kv_heads, tokens, dim, 0, 1, pad=pad)
    rows.check(*rows.run())


def test_rows_in_place(dev):
    """q_out and k_out the rows themselves."""
    for interleaved in (0, 1):
        rows = Rows(dev, BF16, 128, 8, 2, 301, 128, interleaved, 1)
        want = rows.run()
        c, flat = rows.cfg, rows.fused.to(dev).view(-1)
        c.q_out_stride = c.k_out_stride = c.q_stride
        H.qk_norm_rope(c, rows.tokens, flat, flat[rows.q_width:], *rows.args(), flat, flat[rows.q_width:])
        got = flat.cpu().view(rows.tokens, -1)
        live = torch.from_numpy(rows.live())
        assert torch.equal(got[live, :rows.q_width], want[0].flatten(1)[live])
        assert torch.equal(got[live, rows.q_width:rows.q_width + rows.width], want[1].flatten(1)[live])
        assert torch.equal(got[~live], rows.fused[~live])  # padding rows, as they were
        assert torch.equal(got[:, -rows.width:], rows.fused[:, -rows.width:])  # and v


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("norm", [0, 1])
def test_rows_of_extreme_values(dev, elem, norm):
    """Zeros, the type's largest and smallest values, NaN, infinities."""
    rows = Rows(dev, elem, 128, 2, 2, 12, 128, 0, norm, skip=0)
    big = torch.finfo(P.DTYPES[elem]).max
    tiny = 2.0 ** -24 if elem == F16 else 2.0 ** -133
    for x in (rows.q, rows.k):
        x[0] = 0.0
        x[1] = big
        x[2, :, ::2] = -big
        x[3] = tiny
        x[4, :, 5:] = 0.0
        x[5, 0, 7] = float("nan")
        x[6, 1, 9] = float("inf")
        x[7, 0, 100] = -float("inf")
    rows.fused[:, :rows.q_width + rows.width] = torch.cat([rows.q.flatten(1), rows.k.flatten(1)], 1)
    if elem == BF16:  # f32's squares of these overflow in q; k is held in f64 to the end
        rows.q[1:3] = 1.0
        rows.fused[1:3, :rows.q_width] = 1.0
    q_out, k_out = rows.run()
    q, k = (S.norm_rope(rows.cfg, x, w, rows.cos, rows.sin, rows.positions)
            for x, w in zip((rows.q, rows.k), rows.weights))
    if norm:
        for got, want in ((q_out, q), (k_out, k)):
            for t, h in ((5, 0), (6, 1), (7, 0)):
                assert torch.isnan(got[t, h]).any() and not np.isfinite(want[t, h]).all()
                got[t, h] = 0
                want[t, h] = 0
        P.within(q_out.double().numpy(), q, P.HALF_STEP[elem] * np.abs(q) * 1.01 + 1e-4)
        want = S.nearest(k, elem)
        assert torch.equal(torch.nan_to_num(k_out, 1.5), torch.nan_to_num(want, 1.5))
    else:
        keep = np.array([0, 3, 4, 8, 9, 10, 11])
        want = S.nearest(k, elem)
        assert torch.equal(k_out[keep], want[keep])
        for t, h in ((5, 0), (6, 1), (7, 0)):
            assert not torch.isfinite(k_out[t, h]).all()


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -140, 1e-5, 2.0 ** 127])
@pytest.mark.parametrize("dim,interleaved", [(64, 0), (128, 1), (128, 0)])
def test_squares_outside_f32(dev, dim, interleaved, eps):
    """Rows whose squares f32 does not hold, beside rows whose squares it does."""
    rows = Rows(dev, BF16, dim, 5, 2, 41, dim, interleaved, 1, skip=0)
    rows.cfg.eps = eps
    scale = torch.exp2(torch.from_numpy(rows.rng.integers(-110, 120, (rows.tokens, 5, 1)).astype(np.float32)))
    scale[::3] = 1.0
    rows.q = (rows.q.float() * scale).bfloat16()
    rows.k = (rows.k.float() * scale[:, :2]).bfloat16()
    rows.fused[:, :rows.q_width + rows.width] = torch.cat([rows.q.flatten(1), rows.k.flatten(1)], 1)
    assert torch.isfinite(rows.q.float()).all()
    q_out, k_out = rows.run()
    if eps == 0:
        assert (q_out.float().abs().amax(-1) > 0.1).all() and torch.isfinite(q_out.float()).all()
    rows.check(q_out, k_out, least=2.0 ** -133)  # a step of bf16 below its normal range


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("rotary", [0, 32])
def test_no_number_stays_in_its_pair(dev, elem, interleaved, rotary):
    """Without a norm an infinity or a NaN reaches its own channel and its pair's other; the channels that are not
    rotated are copies, signs of zeros included."""
    rows = Rows(dev, elem, 64, 2, 2, 9, rotary, interleaved, 0, skip=0)
    for x in (rows.q, rows.k):
        x[0, 0, 40], x[1, 0, 41], x[2, 1, 63] = float("inf"), float("nan"), -float("inf")
        x[3, :, 33:50] = -0.0
        x[4, 1, 3] = float("inf")
        x[5, 0, 17] = float("nan")
    rows.fused[:, :rows.q_width + rows.width] = torch.cat([rows.q.flatten(1), rows.k.flatten(1)], 1)
    q_out, k_out = rows.run()
    for x, got in ((rows.q, q_out), (rows.k, k_out)):
        bits = [y[..., rotary:].contiguous().view(torch.int16) for y in (got, x)]
        assert torch.equal(*bits)
    if rotary:
        other = 2 if interleaved else 3 + 16
        pair17 = {17, 16 if interleaved else 1}
        for got in (q_out, k_out):
            bad = ~torch.isfinite(got[..., :rotary].float())
            assert set(bad[4, 1].nonzero().flatten().tolist()) == {3, other}
            assert set(bad[5, 0].nonzero().flatten().tolist()) == pair17
            bad[4, 1], bad[5, 0] = False, False
            assert not bad.any()


@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,tokens,interleaved,norm", [
    (F16, 128, 32, 8, 16, 1, 0, 1), (BF16, 128, 4, 2, 64, 37, 1, 1), (F16, 64, 6, 3, 32, 130, 0, 0),
    (BF16, 64, 5, 5, 256, 700, 0, 1), (F16, 128, 2, 1, 16, 4003, 1, 1), (BF16, 128, 32, 8, 64, 3001, 0, 1),
    (F16, 64, 1, 9, 128, 9000, 0, 1)])
def test_into_the_cache_is_the_write_of_the_rows(dev, elem, dim, heads, kv_heads, page, tokens, interleaved, norm):
    rows = Rows(dev, elem, dim, heads, kv_heads, tokens, dim, interleaved, norm)
    pages = tokens // page + 2
    kv = H.Kv4Cfg(kv_heads, dim, page, pages, elem)
    slots = rows.rng.permutation(pages * page)[:tokens].astype(np.int32)
    slots[rows.rng.random(tokens) < 0.1] = -1
    if tokens > 5:
        slots[4], slots[5] = pages * page, -2 ** 31
    size = H.kv4_cache_bytes(kv)
    cache, want = (torch.full((size + 64,), 0xA5, dtype=torch.uint8, device=dev) for _ in range(2))
    flat = rows.fused.to(dev).view(-1)
    d_slots = torch.from_numpy(slots).to(dev)
    q_out = torch.full((tokens, rows.cfg.q_out_stride), 5.0, dtype=flat.dtype, device=dev)
    k, v = flat[rows.q_width:], flat[rows.q_width + rows.width:]
    H.qk_norm_rope_kv4(rows.cfg, kv, tokens, flat, k, v, *rows.args(), d_slots, q_out, cache)
    plain_q, plain_k = rows.run()
    assert torch.equal(q_out.cpu()[:, :rows.q_width].reshape(plain_q.shape), plain_q)
    live = np.where(rows.live(), slots, -1).astype(np.int32)
    H.kv4_write(kv, tokens, rows.width, rows.cfg.v_stride, plain_k.to(dev).flatten(1), v,
                torch.from_numpy(live).to(dev), want)
    assert torch.equal(cache, want)


def test_rows_past_32_bits(dev):
    """Rows whose last element lies past 2^32 bytes."""
    stride, tokens = 2 ** 20, 2100
    rows = Rows(dev, F16, 64, 1, 1, tokens, 64, 0, 1, skip=0)
    c = rows.cfg
    want = rows.run()
    flat = torch.zeros((tokens - 1) * stride + 128, dtype=torch.float16, device=dev)
    at = torch.arange(tokens, device=dev)[:, None] * stride + torch.arange(128, device=dev)
    flat[at] = rows.fused[:, :128].to(dev)
    c.q_stride = c.k_stride = c.q_out_stride = c.k_out_stride = stride
    H.qk_norm_rope(c, tokens, flat, flat[64:], *rows.args(), flat, flat[64:])
    got = flat[at].cpu()
    assert torch.equal(got[:, :64], want[0][:, 0]) and torch.equal(got[:, 64:], want[1][:, 0])


def test_rows_on_another_stream_and_again(dev):
    rows = Rows(dev, BF16, 128, 8, 2, 500, 128, 0, 1)
    want = rows.run()
    stream = torch.cuda.Stream()
    flat, args = rows.fused.to(dev).view(-1), rows.args()
    out = [torch.empty(rows.tokens, s, dtype=flat.dtype, device=dev)
           for s in (rows.cfg.q_out_stride, rows.cfg.k_out_stride)]
    torch.cuda.synchronize()
    H.qk_norm_rope(rows.cfg, rows.tokens, flat, flat[rows.q_width:], *args, *out, stream=stream)
    stream.synchronize()
    live = torch.from_numpy(rows.live())
    assert torch.equal(out[0].cpu()[live], want[0].flatten(1)[live])
    assert torch.equal(out[1].cpu()[live], want[1].flatten(1)[live])
