"""attention_kv4 kernel by kernel: each test names the kernels that its calls run and asks the library's rule
for them, and holds the results to the bounds of those kernels (kv4_plain.attend_all)."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
from helpers import kv4_kernels
from test_gpu_kv4 import Call

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16

# heads, cache heads, each sequence's rows and keys, the table's columns of 16 tokens (0: as many as it needs),
# with a workspace or not: the kernels of such a call
CALLS = {
    "few4": (4, 1, [1, 1], [300, 33], 0, False, ["few4"]),
    "few4 in parts": (4, 1, [1, 1], [300, 33], 512, True, ["few4", "join"]),
    "few8": (4, 1, [2, 1], [300, 33], 0, False, ["few8"]),
    "few8 in parts": (14, 2, [1, 1], [300, 33], 512, True, ["few8", "join"]),
    "few16": (16, 2, [2, 1], [300, 33], 0, False, ["few16"]),
    "few16 in parts": (16, 2, [2, 1], [300, 33], 512, True, ["few16", "join"]),
    "mid": (4, 2, [20, 9], [700, 9], 0, False, ["mid"]),
    "mid in parts": (4, 2, [20, 9], [700, 9], 512, True, ["mid", "join"]),
    "rows": (128, 2, [70, 9], [700, 300], 0, False, ["rows"]),
    "line": (128, 2, [70, 9], [700, 300], 160, True, ["line", "rows_join"])}


def kernels_of(call, workspace):
    return kv4_kernels(call.cfg, call.acfg, len(call.new), call.rows, max(1, *call.new), workspace)


def make(dev, name, elem, dim, **more):
    heads, kv_heads, new, lengths, columns, workspace, kernels = CALLS[name]
    call = Call(dev, elem, dim, heads, kv_heads, 16, new, lengths, columns=columns, **more)
    assert kernels_of(call, workspace) == kernels
    return call, workspace


def check(call, workspace, kernels=None):
    kernels = kernels or kernels_of(call, workspace)
    large = any(k in ("rows", "line") for k in kernels)
    out, lse, out_tol, lse_tol = P.attend_all(call.plain, call.acfg, call.q, call.table, call.new, call.lengths,
                                              "rows" if large else "few")
    if large and len(kernels) > 1 and not kernels[-1] == "rows_join":  # beside single tokens' kernel
        small = P.attend_all(call.plain, call.acfg, call.q, call.table, call.new, call.lengths, "few")
        out_tol = np.maximum(out_tol, small[2])
    got, got_lse = call.run(workspace=workspace)
    P.within(got_lse, lse, lse_tol)
    P.within(got, out, out_tol)


def slots_of(call, b, keys):
    return call.table[b, keys // 16] * 16 + keys % 16


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", CALLS)
def test_every_kernel_to_its_roundings(dev, name, elem, dim):
    check(*make(dev, name, elem, dim))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", CALLS)
def test_single_values_at_the_end_of_the_range(dev, name, dim):
    """f16 rows of V whose midpoint m + 8 s lies between two f16 numbers and whose extreme is the type's: no
    value becomes infinite, and none reaches a row that does not see it."""
    call, workspace = make(dev, name, F16, dim)
    kv_heads = call.cfg.kv_heads
    for b, length in enumerate(call.lengths):
        keys = np.arange(1, length, 5)
        x = torch.empty(len(keys), kv_heads, dim, dtype=torch.float64)
        x[0::2, :, 0::2], x[0::2, :, 1::2] = 17264, 65504    # s = 3216, m + 8 s = 42992
        x[1::2, :, 0::2], x[1::2, :, 1::2] = -65504, -4212   # s = 4086, m + 8 s = -32816
        call.plain.put(1, slots_of(call, b, keys), x.to(torch.float16))
    check(call, workspace)


@pytest.mark.parametrize("high", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", CALLS)
def test_means_at_the_end_of_the_range(dev, name, dim, high):
    """f16 rows of V that hold the type's largest (lowest) value in every other channel: a mean of them is that
    value, and what the weights lose in rounding does not carry it past it."""
    call, workspace = make(dev, name, F16, dim)
    kv_heads = call.cfg.kv_heads
    # constant rows, and rows of the widest range whose ends are both held exactly (s = 8000), under weights of many
    # keys and of hardly more than one
    for other, size in (([-54496.0, 17264.0, 65504.0], 1), ([-54496.0], 6)):
        other = torch.tensor(other) * (1 if high else -1)
        for b, length in enumerate(call.lengths):
            x = other[torch.arange(length) % len(other)].view(-1, 1, 1).repeat(1, kv_heads, dim)
            x[:, :, ::2] = 65504 if high else -65504
            call.plain.put(1, slots_of(call, b, np.arange(length)), x.to(torch.float16))
        for _ in range(1 if call.rows > 40 else 8):
            call.q = torch.from_numpy(size * call.rng.standard_normal(tuple(call.q.shape))).to(torch.float16)
            check(call, workspace)


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("name", CALLS)
def test_a_nan_row_of_k_or_of_v_is_one_rule(dev, name, elem):
    """A key whose row of K or of V is no number makes out and lse NaN for the rows that see it, wherever it lies:
    in the middle of the keys that all rows see, and at their end, where some rows do not see it."""
    call, workspace = make(dev, name, elem, 128)
    for at in (70, call.lengths[0] - 2):
        for part in (0, 1):
            slot = slots_of(call, 0, np.array([at]))[0]
            kept = call.plain.words[part, slot].copy()
            call.plain.words[part, slot, 0] = 0x7fff
            check(call, workspace)
            call.plain.words[part, slot] = kept


@pytest.mark.parametrize("order", ["up", "down", "mixed"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", CALLS)
def test_values_whose_sizes_are_far_apart(dev, name, dim, order):
    """f16 rows of V from 2^-13 to 2^12 in size in one sequence, growing, shrinking and in any order: p s is held
    relative to the largest scale so far."""
    call, workspace = make(dev, name, F16, dim)
    for b, length in enumerate(call.lengths):
        size = call.rng.uniform(-13, 12, length)
        size = size if order == "mixed" else np.sort(size)[::1 if order == "up" else -1]
        x = P.rows(call.rng, (length, call.cfg.kv_heads, dim), F16).double() * torch.from_numpy(
            2.0 ** size).view(-1, 1, 1)
        call.plain.put(1, slots_of(call, b, np.arange(length)), x.to(torch.float16))
    check(call, workspace)


# Along one line of keys: ranges that cross cache heads, both joins (more than 64 tiles and cache heads: one wave a
# row), windows, no mask, odd groups, single tokens' launch beside it.
@pytest.mark.parametrize("elem,dim,heads,kv_heads,page,new,lengths,causal,window,columns,beside", [
    (F16, 128, 128, 2, 16, [70, 1, 30], [2500, 700, 300], 1, 0, 0, []),
    (BF16, 64, 128, 2, 32, [70, 1, 30], [2500, 700, 300], 1, 0, 0, []),
    (BF16, 128, 256, 4, 16, [70, 20], [700, 300], 1, 0, 160, []),
    (F16, 64, 256, 4, 64, [70, 0, 20], [700, 50, 300], 1, 0, 80, []),
    (BF16, 64, 128, 2, 16, [70, 1], [700, 300], 0, 0, 160, []),
    (F16, 128, 165, 5, 16, [130, 20], [700, 300], 0, 0, 160, []),
    (F16, 64, 128, 2, 16, [70, 1], [1700, 300], 1, 1200, 160, []),
    (BF16, 64, 165, 5, 16, [130, 20], [1700, 300], 1, 1400, 160, []),
    (F16, 128, 32, 2, 16, [270, 1, 30], [900, 300, 30], 1, 0, 512, ["few16", "join"]),
    (BF16, 64, 32, 2, 16, [270, 1, 30], [900, 300, 20], 1, 0, 256, ["few16", "join"])])
def test_one_line_of_keys(dev, elem, dim, heads, kv_heads, page, new, lengths, causal, window, columns, beside):
    call = Call(dev, elem, dim, heads, kv_heads, page, new, lengths, causal=causal, window=window, columns=columns)
    assert kernels_of(call, True) == ["line", "rows_join"] + beside
    assert kernels_of(call, False)[0] == "rows"
    check(call, True)
    check(call, False)


@pytest.mark.parametrize("causal", [1, 0])
@pytest.mark.parametrize("elem", [F16, BF16])
def test_masked_places_along_a_line(dev, elem, causal):
    """Pages that are none of the cache's, a sequence that sees no key, and a NaN row of K and of V."""
    call = Call(dev, elem, 128, 128, 2, 16, [70, 9, 5], [700, 300, 64], causal=causal, columns=160)
    assert kernels_of(call, True) == ["line", "rows_join"]
    call.table[0, 3] = -1
    call.table[0, 20:25] = call.cfg.pages
    call.table[1, 18] = 2 ** 31 - 1
    call.table[2] = -2 ** 31
    check(call, True)
    for part, at in ((0, 698), (1, 698), (0, 200), (1, 200)):
        slot = slots_of(call, 0, np.array([at]))[0]
        kept = call.plain.words[part, slot].copy()
        call.plain.words[part, slot, 1] = 0x7fff
        check(call, True)
        call.plain.words[part, slot] = kept


# Replays of a divided call: parts and ranges gain and lose their keys.
@pytest.mark.parametrize("elem,heads,kv_heads,max_q,columns,kernels", [
    (F16, 8, 2, 1, 4000, ["few4", "join"]),
    (BF16, 32, 2, 1, 512, ["few16", "join"]),
    (F16, 8, 2, 6, 512, ["mid", "join"]),
    (BF16, 128, 2, 70, 160, ["line", "rows_join"]),
    (F16, 32, 2, 260, 160, ["line", "rows_join", "few16", "join"])])
def test_captured_divided_calls_follow_their_lengths(dev, elem, heads, kv_heads, max_q, columns, kernels):
    """One graph with a workspace that is never cleared, replayed with lengths and rows that grow, shrink and
    vanish: every replay equals the eager call on a workspace of its own, bit for bit, and the definition."""
    steps = [([max_q, 1, min(2, max_q)], [900, 640, 70]), ([1, max_q, 0], [40, 900, 0]),
             ([max_q, max_q, max_q], [900, 890, 880]), ([1, 1, 1], [1, 0, 17]),
             ([0, 1, max_q], [900, 320, 500]), ([max_q, 1, 1], [899, 900, 900])]
    call = Call(dev, elem, 128, heads, kv_heads, 16, [max_q] * 3, [900] * 3, columns=columns)
    assert kernels_of(call, True) == kernels or max_q > 70  # that one is asked with fewer rows, below
    rows, width = 2 * max_q + 2 if max_q > 70 else 3 * max_q, call.width
    if max_q > 70:
        steps[2] = ([max_q, 1, max_q], [900, 890, 880])
    c, a = call.cfg, call.acfg
    assert kv4_kernels(c, a, 3, rows, max_q) == kernels
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    need = H.kv4_workspace_bytes(c, a, 3, rows, max_q)
    cache, table, q = put(call.plain.bytes()), put(call.table), call.q[:rows].reshape(rows, width).to(dev)

    def state():
        return {"lengths": torch.zeros(3, dtype=torch.int32, device=dev),
                "starts": torch.zeros(4, dtype=torch.int32, device=dev),
                "out": torch.zeros(rows, width, dtype=P.DTYPES[elem], device=dev),
                "lse": torch.zeros(rows, heads, dtype=torch.float32, device=dev),
                "ws": torch.full((need,), 0xFF, dtype=torch.uint8, device=dev)}

    def step(s):
        H.attention_kv4(c, a, 3, rows, max_q, q, cache, table, s["lengths"], s["starts"], s["out"], lse=s["lse"],
                        workspace=s["ws"])

    held = state()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(held)
    noise = torch.randn(1 << 18, device=dev)
    for i, (new, lengths) in enumerate(steps):
        fresh = state()
        for s in (held, fresh):
            s["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
            s["starts"].copy_(torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32))
            s["out"].fill_(3.0)
            s["lse"].fill_(3.0)
        noise.mul_(1.0001).add_(0.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(fresh)
        torch.cuda.synchronize()
        n = sum(new)
        for name in ("out", "lse"):
            assert torch.equal(held[name], fresh[name]), (i, name)
            assert (held[name][n:] == 3.0).all(), (i, name)
        wants = [P.attend_all(call.plain, a, call.q[:n], call.table, new, lengths, k) for k in ("rows", "few")]
        P.within(held["lse"][:n].double().cpu().numpy(), wants[0][1], wants[0][3])
        P.within(held["out"][:n].double().cpu().numpy().reshape(wants[0][0].shape), wants[0][0],
                 np.maximum(wants[0][2], wants[1][2]) if "rows_join" in kernels else wants[1][2])
    del graph


@pytest.mark.parametrize("elem", [F16, BF16])
@pytest.mark.parametrize("name", CALLS)
def test_every_kernel_repeats_bit_for_bit(dev, name, elem):
    call, workspace = make(dev, name, elem, 128)
    first = call.run(workspace=workspace)
    for _ in range(3):
        assert all(np.array_equal(x, y) for x, y in zip(first, call.run(workspace=workspace)))


@pytest.mark.parametrize("name", ["few4 in parts", "mid in parts", "line"])
def test_two_calls_at_once(dev, name):
    """On two streams over one cache, each with a workspace of its own: as one after the other."""
    call, _ = make(dev, name, F16, 128)
    c, a, batch, rows = call.cfg, call.acfg, len(call.new), call.rows
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    cache, table = put(call.plain.bytes()), put(call.table)
    lengths, starts = put(np.array(call.lengths, np.int32)), put(np.concatenate([[0], np.cumsum(call.new)])
                                                                 .astype(np.int32))
    need = H.kv4_workspace_bytes(c, a, batch, rows, max(call.new))
    assert need > 0
    q = [call.q.reshape(rows, -1).to(dev) * f for f in (1.0, -0.5)]
    streams, spaces = [torch.cuda.Stream() for _ in q], [torch.empty(need, dtype=torch.uint8, device=dev) for _ in q]
    outs = [[torch.zeros(rows, call.width, dtype=torch.float16, device=dev) for _ in range(12)] for _ in q]
    torch.cuda.synchronize()
    for i in range(12):
        for n, stream in enumerate(streams):
            H.attention_kv4(c, a, batch, rows, max(call.new), q[n], cache, table, lengths, starts, outs[n][i],
                            workspace=spaces[n], stream=stream)
    torch.cuda.synchronize()
    for n in (0, 1):
        want = torch.zeros_like(outs[n][0])
        H.attention_kv4(c, a, batch, rows, max(call.new), q[n], cache, table, lengths, starts, want,
                        workspace=spaces[0])
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs[n])
    assert not torch.equal(outs[0][0], outs[1][0])
