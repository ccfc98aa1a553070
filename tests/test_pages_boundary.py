"""The boundary of the paged serving operators on the CPU: C ABI, torch operators, mask words.

No kernel runs here: every call either is refused before any HIP call (fake, never-dereferenced pointers) or has no
work to enqueue.
"""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch
from test_boundary_abi import lib  # noqa: F401  (fixture)
from trianglemix import native, pages, tree

HEADER = Path(__file__).resolve().parents[1] / "include" / "trianglemix_pages.h"
BF16, FP16 = 0, 1
COUNTER_BYTES = 65536
# fake device addresses, 2^46 apart
A = [0x4000_0000_0000 * (i + 1) for i in range(16)]


def test_header_functions_are_exported_and_declared(lib):  # noqa: F811
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = set(re.findall(r"\b(tm_[a-z_]+)\s*\(", text))
    assert names == {"tm_update_page_bounds", "tm_select_pages", "tm_select_pages_workspace_size",
                     "tm_selected_page_attention", "tm_selected_page_attention_workspace_size", "tm_tree_attention",
                     "tm_tree_attention_workspace_size"}
    for name in names:
        declared = re.search(rf"\b{name}\s*\(([^)]*)\)", text).group(1)
        assert len(getattr(lib, name).argtypes) == len(declared.split(",")), name
    assert pages.SELECT_ROWS == int(re.search(r"#define TM_SELECT_ROWS (\d+)", HEADER.read_text()).group(1))
    assert re.search(r"#define TM_BF16 0\b", HEADER.read_text()) and re.search(r"#define TM_FP16 1\b", HEADER.read_text())


# ---- refusals: (changed arguments, status, text) ----

PAGE = 128 * 8 * 128  # elements of a page of eight KV heads
COMMON = dict(table=A[3], table_stride=64, lens=A[4], batch=4, cols=64, num_pages=300, kv=8, dtype=BF16)
BOUNDS = dict(COMMON, keys=A[0], key_stride=PAGE, tokens=1, low=A[1], high=A[2])
SELECT = dict(COMMON, query=A[0], query_stride=4096, low=A[1], high=A[2], out=A[5], rows=40, heads=32, count=8, sink=1,
              recent=1, ws=A[6], ws_bytes=1 << 30)
ATTEND = dict(COMMON, query=A[0], query_stride=4096, keys=A[1], key_stride=PAGE, values=A[2], value_stride=PAGE,
              pages=A[7], out=A[5], rows=40, heads=32, count=8, scale=0.088, ws=A[6], ws_bytes=1 << 30)
TREE = dict(COMMON, query=A[0], query_stride=4096, key=A[8], key_rows=1024, value=A[9], value_rows=1024, keys=A[1],
            key_stride=PAGE, values=A[2], value_stride=PAGE, offsets=A[10], mask=A[11], out=A[5], total=40, heads=32,
            scale=0.088, ws=A[6], ws_bytes=1 << 30)


def run(lib, kind, **over):  # noqa: F811
    a = dict({"bounds": BOUNDS, "select": SELECT, "attend": ATTEND, "tree": TREE}[kind], **over)
    assert set(over) <= set(a) and len(a) == len(set(a))
    g = a.__getitem__
    if kind == "bounds":
        return lib.tm_update_page_bounds(*map(g, ("keys", "key_stride", "table", "table_stride", "lens", "tokens", "low",
                                                  "high", "batch", "cols", "num_pages", "kv", "dtype")), None)
    if kind == "select":
        return lib.tm_select_pages(*map(g, ("query", "query_stride", "low", "high", "table", "table_stride", "lens", "out",
                                            "batch", "rows", "heads", "kv", "cols", "num_pages", "count", "sink",
                                            "recent", "dtype", "ws", "ws_bytes")), None)
    if kind == "attend":
        return lib.tm_selected_page_attention(*map(g, (
            "query", "query_stride", "keys", "key_stride", "values", "value_stride", "table", "table_stride", "lens",
            "pages", "out", "batch", "rows", "heads", "kv", "cols", "num_pages", "count", "scale", "dtype", "ws",
            "ws_bytes")), None)
    return lib.tm_tree_attention(*map(g, (
        "query", "query_stride", "key", "key_rows", "value", "value_rows", "keys", "key_stride", "values",
        "value_stride", "table", "table_stride", "lens", "offsets", "mask", "out", "total", "batch", "heads", "kv",
        "cols", "num_pages", "scale", "dtype", "ws", "ws_bytes")), None)


ALL = [
    (dict(dtype=2), 1, "TM_BF16 or TM_FP16"),
    (dict(dtype=-1), 1, "TM_BF16 or TM_FP16"),
    (dict(kv=0), 1, "positive multiple"),
    (dict(batch=-1), 1, "negative"),
    (dict(batch=1025, table_stride=64), 2, "limit is 1024"),
    (dict(cols=0), 1, "block_table"),
    (dict(table_stride=63), 1, "block_table"),
    (dict(cols=16385, table_stride=16385), 2, "limit is 16384"),
    (dict(num_pages=0), 1, "pages > 0"),
    (dict(num_pages=(1 << 22) + 1), 2, "limit is 4194304"),
    (dict(lens=None), 1, "non-null"),
    (dict(table=None), 1, "non-null"),
    (dict(table=A[3] + 2), 1, "aligned to their elements"),
    (dict(lens=A[4] + 1), 1, "aligned to their elements"),
]
CACHES = [
    (dict(key_stride=PAGE - 8), 1, "key_cache pages"),
    (dict(key_stride=PAGE + 4), 1, "key_cache pages"),
    (dict(keys=None), 1, "non-null"),
    (dict(keys=A[0] + 8), 1, "16-byte"),
]
VALUES = [(dict(value_stride=PAGE - 8), 1, "value_cache pages"), (dict(values=None), 1, "non-null")]
ROWS = [
    (dict(heads=33), 1, "positive multiple"),
    (dict(heads=0), 1, "positive multiple"),
    (dict(heads=264, kv=8, query_stride=264 * 128), 2, "limits are 256 heads and 32"),
    (dict(heads=33, kv=1, query_stride=33 * 128), 2, "limits are 256 heads and 32"),
    (dict(query=None), 1, "non-null"),
    (dict(query=A[0] + 2), 1, "16-byte"),
    (dict(query_stride=4095), 1, "query rows"),
    (dict(query_stride=4088), 1, "query rows"),
    (dict(query_stride=-8), 1, "query rows"),
    (dict(out=None), 1, "non-null"),
    (dict(out=A[0]), 1, "must not overlap"),
    (dict(out=A[3] + 64), 1, "out must not overlap block_table"),
    (dict(out=A[6]), 1, "must not overlap"),
    (dict(ws=None), 3, "inconsistent"),
    (dict(ws_bytes=-1), 3, "inconsistent"),
    (dict(ws_bytes=1024), 3, "smaller than"),
    (dict(ws=A[6] + 8), 3, "16-byte"),
    (dict(ws=A[0]), 1, "must not overlap"),
]
COUNTS = [(dict(count=0), 1, "at least one page"), (dict(count=1025), 2, "limit is 1024"),
          (dict(rows=-1), 1, "negative"), (dict(rows=1 << 20, batch=4), 2, "query rows")]
SCALES = [(dict(scale=s), 1, "scale") for s in (0.0, -1.0, float("nan"), float("inf"))]
OWN = {
    "bounds": [(dict(tokens=-1), 1, "negative"), (dict(low=A[2]), 1, "must not overlap"),
               (dict(high=A[0] + 4096), 1, "page_max must not overlap key_cache"), (dict(low=None), 1, "non-null"),
               (dict(kv=257), 2, "limits are 256")],
    "select": [(dict(sink=-1), 1, "sink_pages"), (dict(recent=-1), 1, "sink_pages"), (dict(sink=9), 1, "sink_pages"),
               (dict(sink=4, recent=4), 1, "sink_pages"), (dict(sink=(1 << 62), recent=(1 << 62)), 1, "sink_pages"),
               (dict(low=A[1] + 2), 1, "16-byte"), (dict(out=A[5] + 2), 1, "aligned to their elements")],
    "attend": [(dict(pages=None), 1, "non-null"), (dict(pages=A[5]), 1, "out must not overlap pages"),
               (dict(batch=1024, rows=2048, heads=256, query_stride=256 * 128, count=1024), 2, "limit is 1073741824")],
    "tree": [(dict(key=None), 1, "non-null"), (dict(key_rows=1020), 1, "key rows"), (dict(value_rows=0), 1, "value rows"),
             (dict(mask=A[11] + 4), 1, "aligned to their elements"), (dict(offsets=None), 1, "non-null"),
             (dict(out=A[11]), 1, "out must not overlap tree_mask"), (dict(total=-1), 1, "negative"),
             (dict(total=(1 << 21) + 1), 2, "query rows"),
             (dict(total=1 << 16, batch=1024, heads=256, kv=256, query_stride=256 * 128, key_rows=256 * 128,
                   value_rows=256 * 128, cols=16384, table_stride=16384, key_stride=32 * PAGE, value_stride=32 * PAGE),
              2, "limit is 1073741824")],
}


def _refusals():
    table = {"bounds": ALL + CACHES, "select": ALL + ROWS + COUNTS,
             "attend": ALL + CACHES + VALUES + ROWS + COUNTS + SCALES, "tree": ALL + CACHES + VALUES + ROWS + SCALES}
    for kind, cases in table.items():
        for over, status, text in cases + OWN[kind]:
            if kind != "bounds" and over == dict(keys=A[0] + 8):
                over = dict(keys=A[1] + 8)
            yield pytest.param(kind, over, status, text, id=f"{kind}-{'-'.join(over)}-{text[:12]}")


@pytest.mark.parametrize("kind,over,status,text", _refusals())
def test_refusals(lib, kind, over, status, text):  # noqa: F811
    assert run(lib, kind, **over) == status, lib.tm_last_error()
    assert text in lib.tm_last_error().decode()


@pytest.mark.parametrize("kind,over", [
    ("bounds", dict(batch=0)), ("bounds", dict(tokens=0)),
    ("select", dict(batch=0)), ("select", dict(rows=0)), ("attend", dict(batch=0)), ("attend", dict(rows=0)),
    ("tree", dict(batch=0)), ("tree", dict(total=0)),
])
def test_nothing_to_do_enqueues_nothing(lib, kind, over):  # noqa: F811
    """Without work null tensors and no workspace are fine, and an earlier error's text goes."""
    assert run(lib, kind, dtype=7) == 1
    none = {k: None for k in ("out", "query", "keys", "values", "table", "lens", "pages", "key", "value", "offsets", "mask",
                              "low", "high", "ws") if k in {"bounds": BOUNDS, "select": SELECT, "attend": ATTEND,
                                                            "tree": TREE}[kind]}
    if "ws" in none:
        none["ws_bytes"] = 0
    assert run(lib, kind, **none, **over) == 0
    assert lib.tm_last_error() == b""


def test_workspace_sizes(lib):  # noqa: F811
    select, attend, tree_size = (lib.tm_select_pages_workspace_size, lib.tm_selected_page_attention_workspace_size,
                                 lib.tm_tree_attention_workspace_size)
    for size in (select, attend):
        assert size(0, 1, 32, 8, 64) == size(4, 0, 32, 8, 64) == 0
        assert size(-1, 1, 32, 8, 64) == size(4, -1, 32, 8, 64) == size(4, 1, 33, 8, 64) == size(1025, 1, 32, 8, 64) == -1
    assert tree_size(0, 4, 32, 8, 64) == tree_size(9, 0, 32, 8, 64) == 0
    assert tree_size(9, 4, 32, 8, 0) == tree_size(-1, 4, 32, 8, 64) == tree_size(9, 4, 31, 8, 64) == -1
    assert select(4, 1, 32, 8, 16385) == select(4, 1, 32, 8, 0) == -1
    assert attend(4, 1, 32, 8, 0) == attend(4, 1, 32, 8, 1025) == -1
    # scores alone for single tokens, the pooled queries too for blocks; large calls go slab by slab
    assert select(4, 1, 32, 8, 64) == 4 * 8 * 64 * 8
    assert select(4, 33, 32, 8, 64) == 4 * 2 * (8 * 64 + 32 * 128) * 8
    for args in ((1, 1 << 20, 256, 8, 16384), (1024, 2048, 32, 8, 1024), (1024, 1, 256, 256, 16384), (1, 32, 256, 256, 16384)):
        assert 0 < select(*args) <= 40 << 20
    # arrival words, then two partial records a workgroup; never more than the GPU holds at once
    for size in (lambda *a: attend(*a[:4], 32), lambda b, r, h, k: tree_size(b * r, b, h, k, 64)):
        for b, r, h, k in ((1, 1, 32, 8), (64, 1, 32, 8), (8, 20, 32, 8), (1, 2048, 32, 8), (3, 64, 256, 8)):
            n = size(b, r, h, k)
            assert n > COUNTER_BYTES and n % 16 == 0 and n <= COUNTER_BYTES + 2 * 512 * 128 * 132 * 4


# ---- torch operators ----

@pytest.fixture(scope="module")
def ops(lib):  # noqa: F811
    native.load_triangle_mix_adapter()
    return torch.ops.trianglemix


def test_schemas(ops):
    assert str(ops.update_page_bounds.default._schema) == (
        "trianglemix::update_page_bounds(Tensor key_cache, Tensor block_table, Tensor seq_lens, int num_tokens, "
        "Tensor(a!) page_min, Tensor(b!) page_max) -> ()")
    assert str(ops.select_pages.out._schema) == (
        "trianglemix::select_pages.out(Tensor query, Tensor page_min, Tensor page_max, Tensor block_table, "
        "Tensor seq_lens, int count, int sink_pages, int recent_pages, *, Tensor(a!) out) -> Tensor(a!)")
    assert str(ops.selected_page_attention.out._schema) == (
        "trianglemix::selected_page_attention.out(Tensor query, Tensor key_cache, Tensor value_cache, "
        "Tensor block_table, Tensor seq_lens, Tensor pages, float scale, *, Tensor(a!) out) -> Tensor(a!)")
    assert str(ops.tree_attention.out._schema) == (
        "trianglemix::tree_attention.out(Tensor query, Tensor key, Tensor value, Tensor key_cache, Tensor value_cache, "
        "Tensor block_table, Tensor context_lens, Tensor tree_offsets, Tensor tree_mask, float scale, *, "
        "Tensor(a!) out) -> Tensor(a!)")


def test_meta_shapes_and_no_cpu_kernel(ops):
    def make(device):
        e = dict(device=device, dtype=torch.bfloat16)
        cache = torch.zeros(20, 128, 2, 128, **e)
        i = dict(device=device, dtype=torch.int32)
        return (torch.zeros(80, 8, 128, **e), torch.zeros(80, 2, 128, **e), cache, torch.zeros(2, 9, **i),
                torch.zeros(2, **i), torch.zeros(2, 2, 2, 4, **i), torch.zeros(3, **i),
                torch.zeros(80, device=device, dtype=torch.int64), *pages.page_bounds_like(cache))

    q, kv, cache, table, lens, chosen, offsets, mask, low, high = make("meta")
    assert low.shape == (20, 2, 128) and low.dtype == torch.bfloat16
    picked = pages.select_pages(q, low, high, table, lens, 4)
    assert picked.shape == (2, 2, 2, 4) and picked.dtype == torch.int32 and picked.device.type == "meta"
    out = torch.empty_like(q)
    assert pages.selected_page_attention(q, cache, cache, table, lens, chosen, 0.1).shape == q.shape
    assert pages.selected_page_attention(q, cache, cache, table, lens, chosen, 0.1, out=out) is out
    assert tree.tree_attention(q, kv, kv, cache, cache, table, lens, offsets, mask, 0.1).shape == q.shape
    assert tree.tree_attention(q, kv, kv, cache, cache, table, lens, offsets, mask, 0.1, out=out) is out

    q, kv, cache, table, lens, chosen, offsets, mask, low, high = make("cpu")
    for call in (lambda: pages.update_page_bounds(cache, table, lens, 1, low, high),
                 lambda: pages.select_pages(q, low, high, table, lens, 4),
                 lambda: pages.selected_page_attention(q, cache, cache, table, lens, chosen, 0.1),
                 lambda: tree.tree_attention(q, kv, kv, cache, cache, table, lens, offsets, mask, 0.1)):
        with pytest.raises(NotImplementedError):
            call()


# ---- mask words ----

def test_ancestor_masks():
    assert tree.ancestor_masks([]) == []
    assert tree.ancestor_masks([-1, 0, 0, -1, 2]) == [0b1, 0b11, 0b101, 0b1000, 0b10101]
    chain = tree.ancestor_masks(range(-1, 63))
    assert len(chain) == tree.MAX_TREE_NODES and chain[62] == (1 << 63) - 1 and chain[63] == -1
    assert torch.tensor(chain, dtype=torch.int64)[63] == -1
    star = tree.ancestor_masks([-1] * 64)
    assert star[63] == -(1 << 63) and star[62] == 1 << 62
    for parents in ([0], [-1, 1], [-1, -2], [-1] * 65):
        with pytest.raises(ValueError):
            tree.ancestor_masks(parents)
    assert ctypes.sizeof(ctypes.c_int64) * 8 == tree.MAX_TREE_NODES
