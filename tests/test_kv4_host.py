"""What the 4-bit cache's entry points refuse, before any device work, and the numpy restatement's own
consistency. No kernel is launched here."""
import ctypes

import numpy as np
import pytest

import h3attn as H
import kv4_plain as P
from test_abi import fake
from test_rust_sys import header_struct_fields, rust_struct_fields


def cache_cfg(**change):
    cfg = H.Kv4Cfg(4, 128, 32, 10, H.H3_ELEM_BF16)
    for name, value in change.items():
        setattr(cfg, name, value)
    return cfg


def attention_cfg(**change):
    cfg = H.Kv4AttentionCfg(8, 1024, 1032, 5, 1, 0, 0.1)
    for name, value in change.items():
        setattr(cfg, name, value)
    return cfg


CACHE = 10 * 4 * 32 * 136


def test_cache_bytes():
    assert H.kv4_cache_bytes(cache_cfg()) == CACHE
    assert H.kv4_cache_bytes(cache_cfg(head_dim=64)) == 10 * 4 * 32 * 72
    assert H.kv4_cache_bytes(H.Kv4Cfg(256, 128, 1024, 2 ** 21 - 1, 0)) == (2 ** 21 - 1) * 2 ** 18 * 136
    assert H.kv4_cache_bytes(cache_cfg(head_dim=96)) == 0
    assert H.lib().h3_kv4_cache_bytes(None) == 0


BAD_CACHE = [("kv_heads", 0), ("kv_heads", 257), ("head_dim", 32), ("head_dim", 256),
             ("page_tokens", 8), ("page_tokens", 48), ("page_tokens", 2048), ("pages", 0),
             ("pages", 2 ** 26), ("elem", 2)]


def call_rows(name, cfg, tokens, ks, vs, views):
    return getattr(H.lib(), name)(ctypes.byref(cfg), tokens, ks, vs, *views, None)


def write_need(tokens, ks, vs):
    return [((tokens - 1) * ks + 512) * 2, ((tokens - 1) * vs + 512) * 2, tokens * 4, CACHE]


@pytest.mark.parametrize("name", ["h3_kv4_write", "h3_kv4_read"])
def test_rows_refuse_what_they_cannot_take(name):
    tokens, ks, vs = 7, 512, 1536
    need = write_need(tokens, ks, vs)
    align = [16, 16, 4, 16]
    if name == "h3_kv4_read":
        need, align = need[2:] + need[:2], align[2:] + align[:2]
    views = [fake(n) for n in need]
    assert call_rows(name, cache_cfg(), tokens, ks, vs, views) == H.H3_ERR_NO_DEVICE, H.last_error()
    for i in range(4):
        short = list(views)
        short[i] = fake(need[i] - 1)
        assert call_rows(name, cache_cfg(), tokens, ks, vs, short) == H.H3_ERR_BINDING
        assert H.last_error() == (f"{name[3:]}: binding {i} is {need[i] - 1} bytes, the kernel "
                                  f"addresses {need[i]}")
        moved = list(views)
        moved[i] = H.raw_view(0x1000 + align[i] // 2, need[i])
        assert call_rows(name, cache_cfg(), tokens, ks, vs, moved) == H.H3_ERR_ARGUMENT
        assert H.last_error() == f"{name[3:]}: binding {i} is not {align[i]}-byte aligned"
        null = list(views)
        null[i] = H.raw_view(None, need[i])
        assert call_rows(name, cache_cfg(), tokens, ks, vs, null) == H.H3_ERR_ARGUMENT
    for field, value in BAD_CACHE:
        assert call_rows(name, cache_cfg(**{field: value}), tokens, ks, vs,
                         [fake(1 << 50)] * 4) == H.H3_ERR_CONFIG, (field, value)
    for t, a, b in [(0, ks, vs), (2 ** 24 + 1, ks, vs), (tokens, 504, vs), (tokens, ks, 504),
                    (tokens, 516, vs), (tokens, ks, 2 ** 20 + 8)]:
        assert call_rows(name, cache_cfg(), t, a, b, [fake(1 << 50)] * 4) == H.H3_ERR_ARGUMENT
    assert getattr(H.lib(), name)(None, 1, 512, 512, *views, None) == H.H3_ERR_ARGUMENT


def call_attention(cfg, acfg, batch, q_rows, max_q, views):
    return H.lib().h3_attention_kv4(ctypes.byref(cfg), ctypes.byref(acfg), batch, q_rows, max_q,
                                    *views, None)


def test_attention_refuses_what_it_cannot_take():
    batch, rows, most = 3, 11, 5
    need = [(10 * 1024 + 1024) * 2, CACHE, 3 * 5 * 4, 3 * 4, 4 * 4, (10 * 1032 + 1024) * 2,
            rows * 8 * 4, H.kv4_workspace_bytes(cache_cfg(), attention_cfg(), batch, rows, most)]
    align = [16, 16, 4, 4, 4, 16, 4, 16]
    views = [fake(n) for n in need]
    empty = H.raw_view(None, 0)
    ask = lambda v: call_attention(cache_cfg(), attention_cfg(), batch, rows, most, v)  # noqa: E731
    assert ask(views) == H.H3_ERR_NO_DEVICE, H.last_error()
    assert ask(views[:6] + [empty, empty]) == H.H3_ERR_NO_DEVICE, H.last_error()
    for i in range(8):
        if need[i]:
            short = list(views)
            short[i] = fake(need[i] - 1)
            assert ask(short) == H.H3_ERR_BINDING and f"binding {i} is" in H.last_error()
        moved = list(views)
        moved[i] = H.raw_view(0x1000 + align[i] // 2, need[i])
        assert ask(moved) == H.H3_ERR_ARGUMENT and f"binding {i} is not" in H.last_error()
        if i < 6:
            null = list(views)
            null[i] = H.raw_view(None, need[i])
            assert ask(null) == H.H3_ERR_ARGUMENT
    big = [fake(1 << 50)] * 8
    for field, value in BAD_CACHE:
        assert call_attention(cache_cfg(**{field: value}), attention_cfg(), batch, rows, most,
                              big) == H.H3_ERR_CONFIG, (field, value)
    for field, value in [("heads", 0), ("heads", 6), ("heads", 4100), ("q_stride", 1016),
                         ("q_stride", 1028), ("out_stride", 1016), ("out_stride", 2 ** 20 + 8),
                         ("table_stride", 0), ("table_stride", 2 ** 19 + 1), ("causal", 2),
                         ("window", 2 ** 31), ("scale", float("nan")), ("scale", float("inf"))]:
        assert call_attention(cache_cfg(), attention_cfg(**{field: value}), batch, rows, most,
                              big) == H.H3_ERR_CONFIG, (field, value)
    assert call_attention(cache_cfg(), attention_cfg(causal=0, window=5), batch, rows, most,
                          big) == H.H3_ERR_CONFIG
    for b, r, m in [(0, rows, most), (65536, rows, most), (batch, 0, 1), (batch, 2 ** 24 + 1, 1),
                    (batch, rows, 0), (batch, rows, rows + 1)]:
        assert call_attention(cache_cfg(), attention_cfg(), b, r, m, big) == H.H3_ERR_ARGUMENT
        assert H.kv4_workspace_bytes(cache_cfg(), attention_cfg(), b, r, m) == 0
    many = H.Kv4AttentionCfg(4096, 2 ** 19, 2 ** 19, 5, 1, 0, 0.1)
    assert call_attention(cache_cfg(kv_heads=1), many, 1, 2 ** 24, 2 ** 18 + 1,
                          big) == H.H3_ERR_ARGUMENT and "2^30" in H.last_error()
    assert H.lib().h3_attention_kv4(ctypes.byref(cache_cfg()), None, 1, 1, 1, *big,
                                    None) == H.H3_ERR_ARGUMENT


def test_a_call_that_leaves_the_chip_idle_asks_for_a_workspace():
    one = H.Kv4Cfg(8, 128, 64, 4096, H.H3_ELEM_F16)
    long = H.Kv4AttentionCfg(32, 4096, 4096, 2048, 1, 0, 0.1)
    need = H.kv4_workspace_bytes(one, long, 1, 1, 1)
    assert need and need % (32 * 130 * 4) == 0 and need // (32 * 130 * 4) <= 128
    assert H.kv4_workspace_bytes(one, long, 1024, 1024, 1) == 0
    short = H.Kv4AttentionCfg(32, 4096, 4096, 1, 1, 0, 0.1)
    assert H.kv4_workspace_bytes(one, short, 1, 1, 1) == 0


class Launch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("tile", "tiles", "parts", "rows_from", "rows_to")]


class Plan(ctypes.Structure):
    _fields_ = [("many", Launch), ("few", Launch)]


def test_every_sequence_has_one_launch():
    """How calls are cut: every count of rows that a sequence can have belongs to one launch, whose tiles
    hold it; grids and workspaces stay inside their limits."""
    plan = H.lib()._ZN2h38kv4_planERK10h3_kv4_cfgRK20h3_kv4_attention_cfgjjjjb
    plan.restype = Plan
    plan.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_uint32] * 4 + [ctypes.c_bool]
    rng = np.random.default_rng(5)
    for _ in range(3000):
        dim, page = int(rng.choice([64, 128])), 16 << int(rng.integers(0, 7))
        kv_heads = int(2 ** rng.uniform(0, 8))
        group = min(int(2 ** rng.uniform(0, 7)), 4096 // kv_heads)
        batch, max_q = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 14))
        q_rows = min(2 ** 24, int(rng.integers(max_q, batch * max_q + 1)))
        columns = max(1, int(2 ** rng.uniform(0, 20)) // page)
        window = int(rng.integers(0, 2)) * int(2 ** rng.uniform(0, 14))
        cfg = H.Kv4Cfg(kv_heads, dim, page, 1000, 0)
        width = kv_heads * group * dim
        acfg = H.Kv4AttentionCfg(kv_heads * group, width, width, columns, 1, window, 0.1)
        for divide in (True, False):
            p = plan(ctypes.byref(cfg), ctypes.byref(acfg), batch, q_rows, max_q, 256, divide)
            taken = [0] * 4
            counts = [1, group, max_q * group, max(1, max_q // 2) * group]
            for launch in (p.many, p.few):
                if not launch.tiles:
                    continue
                assert launch.parts >= 1 and (divide or launch.parts == 1)
                for i, n in enumerate(counts):
                    if launch.rows_from <= n <= launch.rows_to:
                        taken[i] += 1
                        assert n <= launch.tile * launch.tiles
            assert taken == [1] * 4
            assert p.few.tiles == 0 or p.few.tile in (4, 8, 16, 32)
            assert p.few.tile == 32 or p.few.tiles <= 1
            assert p.few.tiles * kv_heads <= 65535 and p.few.parts <= 64
        need = H.kv4_workspace_bytes(cfg, acfg, batch, q_rows, max_q)
        assert need <= 2 ** 28


def test_rust_mirrors_have_the_header_fields():
    for c_name, rs_name, py in [("h3_kv4_cfg", "H3Kv4Cfg", H.Kv4Cfg),
                                ("h3_kv4_attention_cfg", "H3Kv4AttentionCfg", H.Kv4AttentionCfg)]:
        fields = header_struct_fields(c_name)
        assert fields == rust_struct_fields(rs_name) == [f for f, _ in py._fields_]


@pytest.mark.parametrize("elem", [H.H3_ELEM_F16, H.H3_ELEM_BF16])
def test_the_restatement_stays_inside_its_rows(elem):
    """m + s u lies in [min x, max x], within half a step of x but for the scale's rounding."""
    rng = np.random.default_rng(3)
    cfg = H.Kv4Cfg(3, 64, 16, 2, elem)
    x = P.rows(rng, (32, 3, 64), elem)
    cache = P.Cache(cfg)
    cache.put(0, np.arange(32), x)
    y, z = cache.values(0, np.arange(32)), x.double().numpy()
    assert (y >= z.min(-1, keepdims=True)).all() and (y <= z.max(-1, keepdims=True)).all()
    step = (z.max(-1) - z.min(-1))[..., None] / 15
    assert (np.abs(y - z) <= step * (0.5 + 30 * P.HALF_STEP[elem])).all()
    raw = cache.bytes()
    # the layout, spelt out for one place: page 1, head 2, token 5, channel 7 of K
    at = (1 * 3 + 2) * 16 * 72
    assert raw[at + 5 * 32 + 3] >> 4 == cache.codes[0, 21, 2, 7]
    word = raw[at + 16 * 64 + 5 * 4:at + 16 * 64 + 5 * 4 + 4]
    assert word.view(np.uint32)[0] == cache.words[0, 21, 2]
