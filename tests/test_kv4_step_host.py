"""What the operators of a serving step refuse, before any device work. No kernel is launched here."""
import ctypes

import numpy as np
import pytest

import h3attn as H
from test_abi import fake
from test_kv4_host import BAD_CACHE, CACHE, attention_cfg, cache_cfg
from test_rust_sys import header_struct_fields, rust_struct_fields

EMPTY = H.raw_view(None, 0)


def refuses(call, need, align, optional=()):
    """call(views) reaches the device with views of `need` bytes, and refuses each one short, moved or null."""
    views = [fake(n) for n in need]
    assert call(views) == H.H3_ERR_NO_DEVICE, H.last_error()
    for i, n in enumerate(need):
        if not n:
            continue
        short, moved, null = list(views), list(views), list(views)
        short[i] = fake(n - 1)
        assert call(short) == H.H3_ERR_BINDING
        assert f"binding {i} is {n - 1} bytes, the kernel addresses {n}" in H.last_error()
        moved[i] = H.raw_view(0x1000 + align[i] // 2, n)
        assert call(moved) == H.H3_ERR_ARGUMENT
        assert f"binding {i} is not {align[i]}-byte aligned" in H.last_error()
        null[i] = H.raw_view(None, n)
        assert call(null) == (H.H3_ERR_NO_DEVICE if i in optional else H.H3_ERR_ARGUMENT)


# ---------------------------------------------------------------- attention

def sinks_call(cfg, acfg, sinks, batch, q_rows, max_q, views):
    return H.lib().h3_attention_kv4_sinks(ctypes.byref(cfg), ctypes.byref(acfg), sinks, batch, q_rows, max_q,
                                          *views, None)


def prefix_call(cfg, acfg, stride, batch, q_rows, max_q, views):
    return H.lib().h3_attention_kv4_prefix(ctypes.byref(cfg), ctypes.byref(acfg), stride, batch, q_rows, max_q,
                                           *views, None)


BATCH, ROWS, MOST = 3, 11, 5
Q, OUT, LSE = (10 * 1024 + 1024) * 2, (10 * 1032 + 1024) * 2, ROWS * 8 * 4


@pytest.mark.parametrize("window", [0, 40])
def test_sinks_refuse_what_they_cannot_take(window):
    acfg = attention_cfg(window=window)
    ws = H.kv4_sinks_workspace_bytes(cache_cfg(), acfg, 4, BATCH, ROWS, MOST)
    refuses(lambda v: sinks_call(cache_cfg(), acfg, 4, BATCH, ROWS, MOST, v),
            [Q, CACHE, 3 * 5 * 4, 3 * 4, 4 * 4, OUT, LSE, ws], [16, 16, 4, 4, 4, 16, 4, 16], optional=(6,))


def test_a_prefix_refuses_what_it_cannot_take():
    ws = H.kv4_prefix_workspace_bytes(cache_cfg(), attention_cfg(), 7, BATCH, ROWS, MOST)
    refuses(lambda v: prefix_call(cache_cfg(), attention_cfg(), 7, BATCH, ROWS, MOST, v),
            [Q, CACHE, 7 * 4, 4, 3 * 5 * 4, 3 * 4, 4 * 4, OUT, LSE, ws],
            [16, 16, 4, 4, 4, 4, 4, 16, 4, 16], optional=(8,))


@pytest.mark.parametrize("call,n", [(sinks_call, 8), (prefix_call, 10)])
def test_attention_configs_outside_their_ranges(call, n):
    big = [fake(1 << 50)] * n
    for field, value in BAD_CACHE:
        assert call(cache_cfg(**{field: value}), attention_cfg(), 4, BATCH, ROWS, MOST, big) == H.H3_ERR_CONFIG
    for field, value in [("heads", 6), ("q_stride", 1016), ("table_stride", 0), ("causal", 2),
                         ("scale", float("nan"))]:
        assert call(cache_cfg(), attention_cfg(**{field: value}), 4, BATCH, ROWS, MOST, big) == H.H3_ERR_CONFIG
    for b, r, m in [(0, ROWS, MOST), (BATCH, 0, 1), (BATCH, ROWS, 0), (BATCH, ROWS, ROWS + 1)]:
        assert call(cache_cfg(), attention_cfg(), 4, b, r, m, big) == H.H3_ERR_ARGUMENT


def test_sinks_and_prefixes_outside_their_ranges():
    big = [fake(1 << 50)] * 10
    cfg, acfg = cache_cfg(), attention_cfg(window=9)
    assert sinks_call(cfg, acfg, 2 ** 24 + 1, BATCH, ROWS, MOST, big[:8]) == H.H3_ERR_ARGUMENT
    assert H.kv4_sinks_workspace_bytes(cfg, acfg, 2 ** 24 + 1, BATCH, ROWS, MOST) == 0
    assert sinks_call(cfg, acfg, 2 ** 24, BATCH, ROWS, MOST, big[:8]) == H.H3_ERR_NO_DEVICE
    assert prefix_call(cfg, acfg, 7, BATCH, ROWS, MOST, big) == H.H3_ERR_CONFIG and "window" in H.last_error()
    assert H.kv4_prefix_workspace_bytes(cfg, acfg, 7, BATCH, ROWS, MOST) == 0
    for stride in (0, 2 ** 19 - 4, 2 ** 32 - 1):
        assert prefix_call(cfg, attention_cfg(), stride, BATCH, ROWS, MOST, big) == H.H3_ERR_ARGUMENT
    assert prefix_call(cfg, attention_cfg(), 2 ** 19 - 5, BATCH, ROWS, MOST, big) == H.H3_ERR_NO_DEVICE


# ---------------------------------------------------------------- pages and slots

def advance_call(cfg, batch, stride, rows, views):
    return H.lib().h3_kv4_advance(ctypes.byref(cfg), batch, stride, rows, *views, None)


def test_advance_refuses_what_it_cannot_take():
    need = [12, 12, 40, 4, 60, 12, 4, 16, 28, 28, 4]
    refuses(lambda v: advance_call(cache_cfg(), 3, 5, 7, v), need, [4] * 11, optional=(10,))
    views = [fake(n) for n in need]
    assert advance_call(cache_cfg(), 3, 5, 7, views[:10] + [EMPTY]) == H.H3_ERR_NO_DEVICE
    for field, value in BAD_CACHE:
        assert advance_call(cache_cfg(**{field: value}), 3, 5, 7, [fake(1 << 50)] * 11) == H.H3_ERR_CONFIG
    for batch, stride, rows in [(0, 5, 7), (65536, 5, 7), (3, 0, 7), (3, 2 ** 19 + 1, 7), (3, 5, 0),
                                (3, 5, 2 ** 24 + 1)]:
        assert advance_call(cache_cfg(), batch, stride, rows, [fake(1 << 50)] * 11) == H.H3_ERR_ARGUMENT
    assert H.lib().h3_kv4_advance(None, 3, 5, 7, *views, None) == H.H3_ERR_ARGUMENT


# ---------------------------------------------------------------- norm and rotation

def qk_cfg(**change):
    cfg = H.QkCfg(8, 4, 128, 64, 0, 1, 50, 1e-5, H.H3_ELEM_BF16, 1536, 1544, 1552, 1032, 520)
    for name, value in change.items():
        setattr(cfg, name, value)
    return cfg


def rows_call(cfg, tokens, views):
    return H.lib().h3_qk_norm_rope(ctypes.byref(cfg), tokens, *views, None)


def cached_call(cfg, tokens, views, kv=None):
    return H.lib().h3_qk_norm_rope_kv4(ctypes.byref(cfg), ctypes.byref(kv or cache_cfg()), tokens, *views, None)


def test_rows_refuse_what_they_cannot_take():
    n, turns = 9, 50 * 32 * 4
    q, k, v = (8 * 1536 + 1024) * 2, (8 * 1544 + 512) * 2, (8 * 1552 + 512) * 2
    q_out, k_out = (8 * 1032 + 1024) * 2, (8 * 520 + 512) * 2
    refuses(lambda w: rows_call(qk_cfg(), n, w), [q, k, 512, 512, turns, turns, n * 4, q_out, k_out],
            [16] * 6 + [4, 16, 16])
    refuses(lambda w: cached_call(qk_cfg(), n, w),
            [q, k, v, 512, 512, turns, turns, n * 4, n * 4, q_out, CACHE], [16] * 7 + [4, 4, 16, 16])
    # neither weights nor tables are asked for where there is no norm and no rotation
    refuses(lambda w: rows_call(qk_cfg(norm=0, rotary=0), n, w), [q, k, 0, 0, 0, 0, n * 4, q_out, k_out],
            [16] * 6 + [4, 16, 16])
    # the stride that a form does not read may be anything
    assert rows_call(qk_cfg(v_stride=3), n, [fake(1 << 50)] * 9) == H.H3_ERR_NO_DEVICE
    assert cached_call(qk_cfg(k_out_stride=3), n, [fake(1 << 50)] * 11) == H.H3_ERR_NO_DEVICE


@pytest.mark.parametrize("call,views", [(rows_call, 9), (cached_call, 11)])
def test_row_configs_outside_their_ranges(call, views):
    big = [fake(1 << 50)] * views
    for field, value in [("heads", 0), ("heads", 4097), ("kv_heads", 0), ("kv_heads", 257), ("head_dim", 96),
                         ("rotary", 8), ("rotary", 144), ("rotary", 40), ("interleaved", 2), ("norm", 2),
                         ("positions", 0), ("positions", 2 ** 24 + 1), ("eps", -1e-9), ("eps", float("nan")),
                         ("eps", float("inf")), ("elem", 2), ("q_stride", 1016), ("q_stride", 1540),
                         ("k_stride", 504), ("q_out_stride", 1016), ("q_out_stride", 2 ** 20 + 8),
                         ("k_out_stride" if call is rows_call else "v_stride", 504)]:
        assert call(qk_cfg(**{field: value}), 9, big) == H.H3_ERR_CONFIG, (field, value)
    for tokens in (0, 2 ** 24 + 1):
        assert call(qk_cfg(), tokens, big) == H.H3_ERR_ARGUMENT
    assert H.lib().h3_qk_norm_rope(None, 9, *big[:9], None) == H.H3_ERR_ARGUMENT


def test_rows_and_their_cache_are_of_one_kind():
    big = [fake(1 << 50)] * 11
    for field, value in [("kv_heads", 8), ("head_dim", 64), ("elem", H.H3_ELEM_F16)] + BAD_CACHE:
        assert cached_call(qk_cfg(), 9, big, cache_cfg(**{field: value})) == H.H3_ERR_CONFIG, (field, value)
    assert H.lib().h3_qk_norm_rope_kv4(ctypes.byref(qk_cfg()), None, 9, *big, None) == H.H3_ERR_ARGUMENT


def test_rust_mirror_has_the_header_fields():
    fields = header_struct_fields("h3_qk_cfg")
    assert fields == rust_struct_fields("H3QkCfg") == [f for f, _ in H.QkCfg._fields_]


# ---------------------------------------------------------------- how a call behind a prefix is cut

class Launch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("tile", "tiles", "parts", "rows_from", "rows_to")]


class Plan(ctypes.Structure):
    _fields_ = [("many", Launch), ("few", Launch)]


class PrefixPlan(ctypes.Structure):
    _fields_ = [("shared", ctypes.c_bool), ("heads_apart", ctypes.c_bool), ("one", Plan), ("own", Plan),
                ("front_parts", ctypes.c_uint32),
                ("front_groups", ctypes.c_uint32), ("parts", ctypes.c_uint32)]


def prefix_plan(cfg, acfg, stride, batch, q_rows, max_q, divide=True):
    call = H.lib()._ZN2h315kv4_prefix_planERK10h3_kv4_cfgRK20h3_kv4_attention_cfgjjjjjb
    call.restype = PrefixPlan
    call.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_uint32] * 5 + [ctypes.c_bool]
    return call(ctypes.byref(cfg), ctypes.byref(acfg), stride, batch, q_rows, max_q, 256, divide)


def test_grids_of_the_largest_batches():
    """65,535 sequences, most of them without rows: the launch that holds them all in its first dimension is taken only
    where it stays below 2^32 threads there."""
    rng = np.random.default_rng(1)
    shared = past = 0
    for _ in range(3000):
        kv_heads, group = int(rng.choice([64, 128, 200, 255, 256])), int(rng.choice([1, 2, 4, 8, 16]))
        batch, q_rows = 65535, int(2 ** rng.uniform(0, 13))
        max_q, dim = max(1, min(q_rows, int(2 ** rng.uniform(0, 12)))), int(rng.choice([64, 128]))
        cfg = H.Kv4Cfg(kv_heads, dim, 16, 1000, 0)
        width = kv_heads * group * dim
        columns, causal = int(2 ** rng.uniform(0, 14)), int(rng.integers(0, 2))
        acfg = H.Kv4AttentionCfg(kv_heads * group, width, width, columns, causal, 0, 0.1)
        p = prefix_plan(cfg, acfg, int(2 ** rng.uniform(0, 18)), batch, q_rows, max_q)
        own = batch * (-(-kv_heads // 4) if p.heads_apart else kv_heads * p.own.few.tiles)
        past += (kv_heads * p.own.few.tiles * batch + 256) * 256 >= 2 ** 32
        if p.shared and p.front_parts:
            shared += 1
            assert (p.front_groups + own) * 256 < 2 ** 32, (kv_heads, group, q_rows, max_q)
    assert shared > 100 and past > 100


def test_every_row_behind_a_prefix_has_its_launches():
    """Every count of rows that a sequence can have belongs to one launch of its own keys; the parts fit the join's
    wave and the workspace, the pieces of a line the parts; grids stay inside their limits."""
    rng = np.random.default_rng(6)
    kinds = set()
    for _ in range(3000):
        dim, page = int(rng.choice([64, 128])), 16 << int(rng.integers(0, 7))
        kv_heads = int(2 ** rng.uniform(0, 8))
        group = min(int(2 ** rng.uniform(0, 7)), 4096 // kv_heads)
        batch, max_q = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 12))
        q_rows = min(2 ** 24, int(rng.integers(max_q, batch * max_q + 1)))
        columns = max(1, int(2 ** rng.uniform(0, 16)) // page)
        stride = max(1, int(2 ** rng.uniform(0, 20)) // page)
        cfg = H.Kv4Cfg(kv_heads, dim, page, 1000, 0)
        width = kv_heads * group * dim
        acfg = H.Kv4AttentionCfg(kv_heads * group, width, width, columns, 1, 0, 0.1)
        assert not prefix_plan(cfg, acfg, stride, batch, q_rows, max_q, False).shared
        p = prefix_plan(cfg, acfg, stride, batch, q_rows, max_q)
        need = H.kv4_prefix_workspace_bytes(cfg, acfg, stride, batch, q_rows, max_q)
        rows = q_rows * group
        if not p.shared:
            kinds.add("one")
            assert need <= 2 ** 28
            continue
        own = max(1, p.own.few.parts)
        assert own == 1 and p.parts <= 64 and need == p.parts * rows * kv_heads * (dim + 2) * 4 <= 200e6
        for n in (1, group, max_q * group, max(1, max_q // 2) * group):
            taken = [x for x in (p.own.many, p.own.few) if x.tiles and x.rows_from <= n <= x.rows_to]
            assert len(taken) == 1 and n <= taken[0].tile * taken[0].tiles
        if p.front_parts:
            kinds.add(("tiles of 32", p.own.few.tile))
            tiles = -(-rows // 32) * kv_heads
            assert p.own.many.tiles == 0 and p.parts == own + p.front_parts
            assert p.front_groups == tiles * p.front_parts
            assert p.front_groups + kv_heads * p.own.few.tiles * batch < 2 ** 31
            assert p.own.few.tile in (4, 8, 16, 32)
        else:
            kinds.add(("line", bool(p.own.many.tiles), bool(p.own.few.tiles)))
            tiles = -(-rows // 256) * kv_heads
            for length in {1, 64, stride * page // 2 + 1, stride * page}:
                steps = max(1, -(-length // 64))
                each = max(8, -(-steps * tiles // p.front_groups))
                assert steps * tiles < 2 ** 30 and each * p.front_groups >= steps * tiles
                first = np.arange(tiles, dtype=np.int64) * steps
                pieces = (first + steps - 1) // each - first // each + 1
                assert pieces.max() <= p.parts - own
    assert kinds >= {"one", ("tiles of 32", 4), ("tiles of 32", 8), ("tiles of 32", 16), ("tiles of 32", 32),
                     ("line", False, True), ("line", True, False), ("line", True, True)}, kinds
