"""The ctypes binding with a stand-in for the library: what a call holds until its launch is enqueued, what it refuses."""

from __future__ import annotations

import weakref

import pytest
import torch
from trianglemix import cabi


class Library:
    """Launches ``during`` in the middle of the first call, as another host thread would."""

    def __init__(self, sizes, during):
        self.sizes, self.during = iter(sizes), [during]

    def __getattr__(self, name):
        if name.endswith("_workspace_size"):
            return lambda *geometry: next(self.sizes)

        def call(*args):
            if self.during:
                self.during.pop()()
            return cabi.TM_OK

        return call


def calls():
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    kv = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    cache = torch.zeros(3, 128, 2, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pages, offsets = torch.zeros(2, 1, 2, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    mask = torch.zeros(4, dtype=torch.int64)
    chunk = dict(query_start=0, seq_len=4, scale=1.0, stream=0)
    return {
        "sparse": lambda: cabi.triangle_paged_sparse_attention(q, cache, cache, table[:1], q, prompt_len=4, **chunk),
        "dense": lambda: cabi.dense_paged_causal_attention(q, cache, cache, table[:1], q, **chunk),
        "selected": lambda: cabi.selected_page_attention(q, cache, cache, table, lens, pages, q, scale=1.0, stream=0),
        "tree": lambda: cabi.tree_attention(q, kv, kv, cache, cache, table, lens, offsets, mask, q, scale=1.0, stream=0),
        "select": lambda: cabi.select_pages(q, cache[:, 0], cache[:, 0], table, lens, pages, stream=0),
    }


@pytest.mark.parametrize("kind", sorted(calls()))
def test_a_buffer_lives_until_its_call_has_launched(monkeypatch, kind):
    """A call of another thread that needs more replaces the stream's buffer, which the first call is about to use."""
    made, alive = [], []

    def buffer(query, need, stream):
        tensor = torch.empty(need, dtype=torch.uint8)
        made.append(weakref.ref(tensor))
        return tensor

    def another_thread():
        calls()["selected"]()
        alive.append(made[0]() is not None)

    library = Library([1024, 4096], another_thread)
    monkeypatch.setattr(cabi, "load_hip_library", lambda: library)
    monkeypatch.setattr(cabi, "_buffer", buffer)
    monkeypatch.setattr(cabi, "_WORKSPACES", {})
    calls()[kind]()
    assert len(made) == 2 and alive == [True]


@pytest.mark.parametrize("kind", ["selected", "select"])
@pytest.mark.parametrize("requests,rows", [(2, 3), (2, 5), (3, 4), (0, 4)])
def test_rows_that_do_not_divide_are_refused(monkeypatch, kind, requests, rows):
    """Not taken as fewer rows a request, the second one's beginning in the first one's."""
    launched = []
    monkeypatch.setattr(cabi, "load_hip_library", lambda: Library([1024], lambda: launched.append(kind)))
    monkeypatch.setattr(cabi, "_buffer", lambda query, need, stream: torch.empty(need, dtype=torch.uint8))
    monkeypatch.setattr(cabi, "_WORKSPACES", {})
    q = torch.zeros(rows, 8, 128, dtype=torch.bfloat16)
    cache = torch.zeros(3, 128, 2, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(requests, 3, dtype=torch.int32), torch.zeros(requests, dtype=torch.int32)
    pages = torch.zeros(requests, 1, 2, 4, dtype=torch.int32)
    with pytest.raises(cabi.TriangleMixError, match="same number of rows"):
        if kind == "select":
            cabi.select_pages(q, cache[:, 0], cache[:, 0], table, lens, pages, stream=0)
        else:
            cabi.selected_page_attention(q, cache, cache, table, lens, pages, q, scale=1.0, stream=0)
    assert not launched
