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
