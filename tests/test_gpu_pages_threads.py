"""Paged serving operators called by several host threads on one stream: every call's result as if it were alone."""

from __future__ import annotations

import threading

import pytest
import torch
from pages_cases import SCALE, make_cache, make_rows
from trianglemix import cabi
from trianglemix import pages as TP

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def ints(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def test_selection_keeps_no_workspace(gpu):
    """The scores of a call lie in memory of its own, not in a buffer that the stream's other calls share."""
    print("select workspace", flush=True)
    cols, kv, heads = 8192, 8, 32
    low = torch.zeros(4, kv, 128, dtype=BF16, device=gpu)
    table = torch.zeros(16, cols, dtype=torch.int32, device=gpu)
    lens = ints([128 * cols] * 16, gpu)
    query = make_rows(16, heads, BF16, 1).to(gpu)
    stream = torch.cuda.Stream()  # no call has run on it
    stream.wait_stream(torch.cuda.current_stream())
    out = torch.empty(16, 1, kv, 4, dtype=torch.int32, device=gpu)
    with torch.cuda.stream(stream):
        before = torch.cuda.memory_allocated()
        TP.select_pages(query, low, low, table, lens, 4, out=out)
        assert torch.cuda.memory_allocated() <= before
        held = len(cabi._WORKSPACES)
        cabi.select_pages(query, low, low, table, lens, out)
        assert torch.cuda.memory_allocated() <= before and len(cabi._WORKSPACES) == held
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()


@pytest.mark.parametrize("binding", ["torch", "ctypes"])
def test_threads_on_one_stream(gpu, binding):
    """Three threads: a batch that decodes, a chunk (pooled queries and scores), and attention that splits its groups."""
    print(f"select threads {binding}", flush=True)
    lens = [128 * 200 - 3, 9000, 128 * 77]
    keys, values, table = (t.to(gpu) for t in make_cache(lens, 2, BF16, seed=61))
    lens_d = ints(lens, gpu)
    low, high = TP.page_bounds_like(keys)
    TP.update_page_bounds(keys, table, lens_d, 128 * 200, low, high)
    decode, chunk = make_rows(3, 8, BF16, 62).to(gpu), make_rows(300, 8, BF16, 63).to(gpu)
    stream = torch.cuda.current_stream()

    def select(query, rows, batch, count):
        if binding == "torch":
            return TP.select_pages(query, low, high, table[:batch], lens_d[:batch], count)
        out = torch.empty(batch, -(-rows // 32), 2, count, dtype=torch.int32, device=gpu)
        cabi.select_pages(query, low, high, table[:batch], lens_d[:batch], out)
        return out

    chosen = select(decode, 1, 3, 60)

    def attend():
        if binding == "torch":
            return TP.selected_page_attention(decode, keys, values, table, lens_d, chosen, SCALE)
        out = torch.zeros_like(decode)
        cabi.selected_page_attention(decode, keys, values, table, lens_d, chosen, out, scale=SCALE)
        return out

    calls = [lambda: select(decode, 1, 3, 60), lambda: select(chunk, 300, 1, 20), attend]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    failed = []

    def work(i):
        try:
            torch.cuda.set_device(gpu)
            with torch.cuda.stream(stream):
                for _ in range(150):
                    got[i].append(calls[i]())
        except Exception as error:  # noqa: BLE001  (reported by the test)
            failed.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for i, outs in enumerate(got):
        assert len(outs) == 150 and all(torch.equal(o, want[i]) for o in outs), i
