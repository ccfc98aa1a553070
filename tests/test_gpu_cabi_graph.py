"""Captured calls of the ctypes binding: each graph has workspaces of its own."""

from __future__ import annotations

import pytest
import torch
from pages_cases import SCALE, make_cache, make_rows
from trianglemix import cabi
from trianglemix import pages as TP

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Recorder:
    """The library, noting the workspace pointer of each attention call."""

    def __init__(self, lib):
        self.lib, self.pointers = lib, []

    def __getattr__(self, name):
        fn = getattr(self.lib, name)
        if name != "tm_selected_page_attention":
            return fn

        def call(*args):
            self.pointers.append(args[-3])
            return fn(*args)

        return call


def inputs(gpu):
    lens = [128 * 60]
    keys, values, table = (t.to(gpu) for t in make_cache(lens, 2, BF16, seed=71))
    lens_d = torch.tensor(lens, dtype=torch.int32, device=gpu)
    low, high = TP.page_bounds_like(keys)
    TP.update_page_bounds(keys, table, lens_d, 128 * 60, low, high)
    queries = [make_rows(rows, 8, BF16, 72 + rows).to(gpu) for rows in (1, 70)]
    chosen = [TP.select_pages(q, low, high, table, lens_d, 40) for q in queries]
    return keys, values, table, lens_d, queries, chosen


def attend(i, which, out):
    keys, values, table, lens, queries, chosen = i
    cabi.selected_page_attention(queries[which], keys, values, table, lens, chosen[which], out, scale=SCALE)
    return out


def test_a_captured_call_leaves_the_streams_buffer_alone(gpu, monkeypatch):
    """Nothing is replayed: where the captured call's workspace lies."""
    print("ctypes capture", flush=True)
    i = inputs(gpu)
    out = torch.zeros_like(i[4][0])
    recorder = Recorder(cabi.load_hip_library())
    monkeypatch.setattr(cabi, "load_hip_library", lambda: recorder)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(i, 0, out)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph, stream=side):
            attend(i, 0, out)
    with torch.cuda.stream(side):
        attend(i, 0, out)
    torch.cuda.synchronize()
    eager, first, second, again = recorder.pointers
    assert eager == again and len({eager, first, second}) == 3


def test_graphs_replayed_at_once_and_after_larger_eager_calls(gpu):
    print("ctypes graphs", flush=True)
    i = inputs(gpu)
    want = [attend(i, k, torch.zeros_like(q)) for k, q in enumerate(i[4])]
    outs = [torch.zeros_like(q) for q in i[4]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(i, 0, outs[0])
    torch.cuda.synchronize()
    graphs = []
    for k, out in enumerate(outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            attend(i, k, out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for out in outs:
            out.fill_(9.0)
        with torch.cuda.stream(side):
            eager = attend(i, 1, torch.zeros_like(i[4][1]))  # needs more than the first call on this stream
        torch.cuda.synchronize()
        others = [torch.full((1 << 20,), 7.0, device=gpu) for _ in range(8)]
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                for _ in range(10):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, want[1])
        assert all(torch.equal(out, w) for out, w in zip(outs, want))
        assert all(bool((x == 7.0).all()) for x in others)
