"""The operators of a serving step together, as a program uses them: pages and slots from the rows asked for, queries
and keys normed, rotated and written, attention over the cache; captured once and replayed for steps of any
kind, every one of them against the same calls made eagerly and against 64-bit attention over what the cache
stands for."""
import numpy as np
import pytest
import torch

import h3attn as H
import kv4_plain as P
import kv4_step_plain as S

pytestmark = pytest.mark.gpu

F16, BF16 = H.H3_ELEM_F16, H.H3_ELEM_BF16


class Server:
    """The buffers of a serving loop of up to `batch` sequences and `rows` rows a step."""

    def __init__(self, dev, elem, kind, heads=8, kv_heads=2, dim=128, page=16, batch=6, rows=40, max_q=24, columns=12,
                 prefix=0, sinks=0, window=0, seed=0):
        rng = np.random.default_rng(seed)
        self.dev, self.kind, self.elem, self.sinks, self.prefix = dev, kind, elem, sinks, prefix
        self.batch, self.rows, self.max_q, self.columns, self.dim = batch, rows, max_q, columns, dim
        self.heads, self.kv_heads = heads, kv_heads
        held = -(-prefix // page)
        self.pages = batch * columns * 2 // 3 + held
        self.cfg = H.Kv4Cfg(kv_heads, dim, page, self.pages, elem)
        width, pitch = heads * dim, (heads + 2 * kv_heads) * dim
        limit = prefix + columns * page
        self.qk = H.QkCfg(heads, kv_heads, dim, dim, 0, 1, limit, 1e-6, elem, pitch, pitch, pitch, width, 0)
        self.att = H.Kv4AttentionCfg(heads, width, width, columns, 1, window, P.softmax_scale(dim))
        angle = np.arange(limit)[:, None] * 100.0 ** (-np.arange(dim // 2) / (dim // 2))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.weights = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2)]
        order = rng.permutation(self.pages).astype(np.int32)
        self.prefix_table = order[:max(held, 1)].copy()
        self.stack, self.count = np.full(self.pages, -1, np.int32), self.pages - held
        self.stack[:self.count] = order[held:]
        self.table = np.full((batch, columns), -1, np.int32)
        self.lengths = np.zeros(batch, np.int32)
        self.plain = P.Cache(self.cfg)
        at = np.arange(prefix)
        for part in (0, 1):
            self.plain.put(part, self.prefix_table[at // page] * page + at % page,
                           P.rows(rng, (prefix, kv_heads, dim), elem))
        self.rng = rng

    def buffers(self, workspace=None):
        put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(self.dev)  # noqa: E731
        ints = lambda n: torch.zeros(n, dtype=torch.int32, device=self.dev)  # noqa: E731
        dtype = P.DTYPES[self.elem]
        if workspace is None:
            need = (H.kv4_sinks_workspace_bytes(self.cfg, self.att, self.sinks, self.batch, self.rows, self.max_q)
                    if self.kind == "sinks" else
                    H.kv4_prefix_workspace_bytes(self.cfg, self.att, len(self.prefix_table), self.batch, self.rows,
                                                 self.max_q))
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=self.dev)
        return {"asked": ints(self.batch), "lengths": put(self.lengths), "free": put(self.stack),
                "count": put(np.array([self.count], np.int32)), "table": put(self.table),
                "starts": ints(self.batch + 1), "slots": ints(self.rows), "positions": ints(self.rows),
                "prefix_table": put(self.prefix_table), "prefix": put(np.array([self.prefix], np.int32)),
                "fused": torch.zeros(self.rows, self.qk.q_stride, dtype=dtype, device=self.dev),
                "weights": [put(w) for w in self.weights], "cos": put(self.cos), "sin": put(self.sin),
                "q": torch.zeros(self.rows, self.att.q_stride, dtype=dtype, device=self.dev),
                "out": torch.zeros(self.rows, self.att.out_stride, dtype=dtype, device=self.dev),
                "lse": torch.zeros(self.rows, self.heads, dtype=torch.float32, device=self.dev),
                "cache": put(self.plain.bytes()), "workspace": workspace}

    def step(self, x):
        """One step of a program: every argument a device buffer or a number that no step changes."""
        flat, width = x["fused"].view(-1), self.kv_heads * self.dim
        H.kv4_advance(self.cfg, self.batch, self.columns, self.rows, x["asked"], x["lengths"], x["free"], x["count"],
                      x["table"], x["lengths"], x["count"], x["starts"], x["slots"], x["positions"], x["prefix"])
        H.qk_norm_rope_kv4(self.qk, self.cfg, self.rows, flat, flat[self.att.q_stride:],
                           flat[self.att.q_stride + width:], *x["weights"], x["cos"], x["sin"], x["positions"],
                           x["slots"], x["q"], x["cache"])
        args = (self.batch, self.rows, self.max_q, x["q"], x["cache"])
        sequences = (x["table"], x["lengths"], x["starts"], x["out"], x["lse"], x["workspace"])
        if self.kind == "sinks":
            H.attention_kv4_sinks(self.cfg, self.att, self.sinks, *args, *sequences)
        else:
            H.attention_kv4_prefix(self.cfg, self.att, len(self.prefix_table), *args, x["prefix_table"], x["prefix"],
                                   *sequences)

    def request(self):
        """Rows asked for, and a projection's rows of them; NaN in the rows that nobody has."""
        asked = np.where(self.rng.random(self.batch) < 0.12, -1,
                         np.where(self.rng.random(self.batch) < 0.3, self.rng.integers(0, self.max_q, self.batch), 1))
        fused = P.rows(self.rng, (self.rows, self.heads + 2 * self.kv_heads, self.dim), self.elem)
        return asked.astype(np.int32), fused.reshape(self.rows, -1)

    def follow(self, asked, fused):
        """The restatement's step: (new rows, valid rows), with the tables and the cache advanced."""
        (self.stack, self.count, self.table, self.lengths, starts, slots, positions) = S.advance(
            self.cfg, self.columns, self.rows, asked, self.lengths, self.stack, self.count, self.table, self.prefix)
        n = starts[-1]
        rows = fused[:n].reshape(n, -1, self.dim)
        k = rows[:, self.heads:self.heads + self.kv_heads]
        k = S.nearest(S.norm_rope(self.qk, k, self.weights[1], self.cos, self.sin, positions[:n]), self.elem)
        near = self.plain.put(0, slots[:n], k).sum()
        near += self.plain.put(1, slots[:n], rows[:, self.heads + self.kv_heads:]).sum()
        return np.diff(starts), n, slots, positions, near

    def check(self, x, new, n, slots, positions, near):
        for name, want in (("table", self.table), ("lengths", self.lengths), ("free", self.stack),
                           ("slots", slots), ("positions", positions)):
            assert np.array_equal(x[name].cpu().numpy(), want), name
        assert int(x["count"]) == self.count
        assert (x["cache"].cpu().numpy() != self.plain.bytes()).sum() <= near
        q = x["q"][:n].cpu().reshape(n, self.heads, self.dim)
        prefix = (self.prefix_table, self.prefix) if self.kind == "prefix" else None
        out, lse, out_tol, lse_tol = S.attend(self.plain, self.att, q, self.table, new, self.lengths, self.sinks,
                                              prefix)
        P.within(x["out"][:n].cpu().double().numpy().reshape(out.shape), out, out_tol)
        P.within(x["lse"][:n].cpu().double().numpy(), lse, lse_tol)


@pytest.mark.parametrize("kind,elem,more", [
    ("prefix", BF16, {"prefix": 70}), ("prefix", F16, {"prefix": 900, "batch": 20, "rows": 60, "max_q": 5}),
    ("sinks", F16, {"sinks": 5, "window": 40}), ("sinks", BF16, {"sinks": 20, "window": 33, "dim": 64, "heads": 6})])
def test_a_captured_step_serves_a_generation(dev, kind, elem, more):
    server = Server(dev, elem, kind, **more)
    graphed, eager = server.buffers(), server.buffers()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        server.step(graphed)  # nobody asks for anything
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        server.step(graphed)
    noise = torch.randn(1 << 16, device=dev)
    for i in range(12):
        asked, fused = server.request()
        new, n, *rest = server.follow(asked, fused)
        fused[n:] = float("nan")  # padding rows hold anything
        for x in (graphed, eager):
            x["asked"].copy_(torch.from_numpy(asked))
            x["fused"].copy_(fused)
        noise.mul_(1.001)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        server.step(eager)
        torch.cuda.synchronize()
        for name in ("table", "lengths", "free", "count", "starts", "slots", "positions", "q", "cache", "out", "lse"):
            assert torch.equal(graphed[name], eager[name]), (i, name)
        server.check(graphed, new, n, *rest)
    assert server.lengths.max() > 0
    del graph


def test_two_captured_steps_share_a_workspace(dev):
    """Replayed one after the other: neither leaves anything for the other to find."""
    servers = [Server(dev, F16, "prefix", prefix=2500, batch=40, rows=44, max_q=3, columns=4, seed=1),
               Server(dev, F16, "sinks", sinks=9, window=4000, batch=2, rows=3, max_q=2, columns=600, seed=2)]
    for s in servers:
        s.lengths[:] = s.rng.integers(0, 30, s.batch) if s.kind == "prefix" else 4500
        at, count = 0, s.count
        for b in range(s.batch):
            held = -(-int(s.lengths[b]) // 16)
            s.table[b, :held] = s.stack[count - at - held:count - at]
            at += held
        s.count -= at
        s.plain.codes[:] = s.rng.integers(0, 16, s.plain.codes.shape)
        s.plain.words[:] = P.bits16(torch.tensor([-1.0, 0.13]).to(torch.float16)).view(np.uint32)[0]
    shared = torch.empty(1 << 24, dtype=torch.uint8, device=dev)
    buffers = [s.buffers(shared) for s in servers]
    assert all(s.buffers()["workspace"].numel() > 16 for s in servers)  # both divide their keys
    eager = [s.buffers() for s in servers]
    graphs = []
    for s, x in zip(servers, buffers):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            s.step(x)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            s.step(x)
    for i in range(4):
        for s, x, y in zip(servers, buffers, eager):
            asked, fused = s.request()
            asked = np.ones_like(asked)
            new, n, *rest = s.follow(asked, fused)
            for z in (x, y):
                z["asked"].copy_(torch.from_numpy(asked))
                z["fused"].copy_(fused)
        torch.cuda.synchronize()
        for g in graphs if i % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for s, x, y in zip(servers, buffers, eager):
            s.step(y)
            torch.cuda.synchronize()
            for name in ("q", "cache", "out", "lse"):
                assert torch.equal(x[name], y[name]), (i, s.kind, name)
    del graphs


def test_two_steps_at_once(dev):
    """On two streams, with buffers of their own."""
    servers = [Server(dev, BF16, "prefix", prefix=900, batch=20, rows=60, max_q=5, seed=3),
               Server(dev, BF16, "sinks", sinks=7, window=30, seed=4)]
    for _ in range(5):
        states = []
        for s in servers:
            s.plain = P.Cache(s.cfg, s.rng)
            s.plain.words[:] = P.bits16(torch.tensor([-1.0, 0.13]).to(torch.bfloat16)).view(np.uint32)[0]
            asked, fused = s.request()
            pair = [s.buffers(), s.buffers()]
            for x in pair:
                x["asked"].copy_(torch.from_numpy(asked))
                x["fused"].copy_(fused)
            states.append(pair)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in servers]
        for s, (x, _), stream in zip(servers, states, streams):
            with torch.cuda.stream(stream):
                s.step(x)
        torch.cuda.synchronize()
        for s, (x, y) in zip(servers, states):
            s.step(y)
            torch.cuda.synchronize()
            for name in ("table", "lengths", "slots", "q", "cache", "out", "lse"):
                assert torch.equal(x[name], y[name]), (s.kind, name)
