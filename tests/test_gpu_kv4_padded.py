"""attention_kv4_prefix of a call with more rows than its sequences have, as a captured step's padding: rows of no
sequence are neither written nor multiplied with the prefix, whatever they hold, and those that there are keep their
places for every number of them."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
from test_gpu_kv4_keys import Front
from test_kv4_step_host import prefix_plan

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16


def kept(monkeypatch):
    """The workspaces of the calls from here on."""
    spaces, real = [], H.attention_kv4_prefix

    def call(*args):
        spaces.append(args[-2])
        real(*args)

    monkeypatch.setattr(H, "attention_kv4_prefix", call)
    return spaces


CUTS = [("tiles", F16, 128, 8, 2, 16, 1, 200, 5003, 64), ("tiles", BF16, 64, 8, 2, 128, 4, 333, 5000, 40),
        ("tiles", BF16, 128, 20, 4, 64, 5, 150, 8000, 30), ("tiles", F16, 64, 10, 5, 32, 1, 130, 1200, 320),
        ("line", F16, 64, 4, 1, 16, 1, 20, 3001, 1100), ("line", BF16, 128, 64, 2, 64, 65, 300, 5000, 6),
        ("line", BF16, 64, 64, 2, 32, 20, 120, 9000, 30)]


@pytest.mark.parametrize("cut,elem,dim,heads,kv_heads,page,each,most,prefix,places", CUTS)
def test_places_of_which_some_have_rows(dev, monkeypatch, cut, elem, dim, heads, kv_heads, page, each, most, prefix,
                                        places):
    rng = np.random.default_rng(places + prefix)
    budget, spaces = places * each, kept(monkeypatch)
    for live, length in [(1, prefix), (2, 0), (places // 9 + 1, prefix), (places // 2, prefix // 2),
                         (places - 1, 1), (places, prefix)]:
        new = [each] * live + [0] * (places - live)
        if live == places // 2:  # idle places between them
            new = [int(n) for n in rng.permutation(new)]
        lengths = [n + int(m) for n, m in zip(new, rng.integers(0, most, places))]
        call = Front(dev, elem, dim, heads, kv_heads, page, new, lengths, prefix=prefix,
                     columns=-(-(most + each) // page))
        plan = prefix_plan(call.cfg, call.acfg, len(call.prefix_table), places, budget, each)
        assert plan.shared and (plan.front_parts == 0) == (cut == "line")
        rows, call.prefix, call.prefix_length = call.rows, length, length
        out, lse, out_tol, lse_tol = call.want()
        got, got_lse = call.run(max_q=each, extra=budget - rows)  # the rows of none hold NaN
        P.within(got, out, out_tol)
        P.within(got_lse, lse, lse_tol)
        # The sums that the call left are those of rows that there are.
        need = call.need(budget, each)
        assert need == plan.parts * budget * heads * (dim + 2) * 4
        words = int((spaces[-1][:need].view(torch.int32) != -1).sum())
        assert words <= (plan.parts if plan.front_parts else 64) * rows * heads * (dim + 2)


@pytest.mark.parametrize("cut,elem,dim,heads,kv_heads,page,each,most,prefix,places", CUTS)
def test_starts_that_decrease_write_no_other_rows(dev, cut, elem, dim, heads, kv_heads, page, each, most, prefix, places):
    """Rows that q_starts names and then takes back are right or left."""
    new = [each] * places
    call = Front(dev, elem, dim, heads, kv_heads, page, new, [most] * places, prefix=prefix,
                 columns=-(-(most + each) // page))
    starts = np.concatenate([[0], np.cumsum(new)])
    starts[-1] = end = starts[-1] // 3
    out, lse, out_tol, lse_tol = call.want()
    got, got_lse = call.run(starts=starts)
    P.within(got[:end], out[:end], out_tol[:end])
    P.within(got_lse[:end], lse[:end], lse_tol[:end])
    left = (got[end:] == 5.0).all((1, 2)) & (got_lse[end:] == 9.0).all(1)
    right = ((np.abs(got - out) <= out_tol).all((1, 2)) & (np.abs(got_lse - lse) <= lse_tol).all(1))[end:]
    assert (left | right).all()


def test_a_captured_call_follows_its_rows(dev):
    """Replays of one graph with other numbers of rows: as the call made eagerly."""
    for _, elem, dim, heads, kv_heads, page, each, most, prefix, places in (CUTS[0], CUTS[4]):
        call = Front(dev, elem, dim, heads, kv_heads, page, [each] * places, [most] * places, prefix=prefix)
        c, a, budget = call.cfg, call.acfg, call.rows
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
        q = call.q.reshape(budget, -1).to(dev)
        q = torch.cat([q, q[:, :1].expand(budget, a.q_stride - q.shape[1])], 1).contiguous()
        starts = put(np.zeros(places + 1, np.int32))
        fixed = (put(call.plain.bytes()), put(call.prefix_table), put(np.array([prefix], np.int32)), put(call.table),
                 put(np.array(call.lengths, np.int32)))

        def buffers():
            return (torch.full((budget, a.out_stride), 5.0, dtype=q.dtype, device=dev),
                    torch.full((budget, heads), 9.0, device=dev),
                    torch.empty(call.need(budget, each), dtype=torch.uint8, device=dev))

        def run(out, lse, ws):
            H.attention_kv4_prefix(c, a, len(call.prefix_table), places, budget, each, q, *fixed, starts, out, lse, ws)

        graphed, side = buffers(), torch.cuda.Stream()
        with torch.cuda.stream(side):
            run(*graphed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(*graphed)
        noise = torch.randn(1 << 16, device=dev)
        for live in (places, 1, places // 2, 0, places - 3):
            starts.copy_(put(np.minimum(np.arange(places + 1), live).astype(np.int32) * each))
            eager = buffers()
            for x, y in zip(graphed[:2], eager):
                x.copy_(y)
            noise.mul_(1.001)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            run(*eager)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(graphed[:2], eager)), live
            assert (eager[0][live * each:] == 5.0).all() and not (eager[0][:live * each, :8] == 5.0).all(1).any()
        del graph
