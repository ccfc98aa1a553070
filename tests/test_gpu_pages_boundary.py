"""The paged serving operators' boundary on the GPU: what the torch operators refuse, and the C ABI binding."""

from __future__ import annotations

import pytest
import torch
from pages_cases import SCALE, make_cache, make_rows
from trianglemix import cabi
from trianglemix import pages as TP
from trianglemix import tree as TT

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def ints(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


@pytest.fixture(scope="module")
def inputs(gpu):
    lens = [300, 41]
    keys, values, table = (t.to(gpu) for t in make_cache(lens, 2, BF16, seed=91))
    low, high = TP.page_bounds_like(keys)
    query = make_rows(80, 8, BF16, 92).to(gpu)
    draft = make_rows(80, 2, BF16, 93).to(gpu)
    return dict(query=query, key=draft, value=draft.flip(0), keys=keys, values=values, table=table,
                lens=ints(lens, gpu), low=low, high=high, pages=ints([[[[0, 1, 2, -1]] * 2] * 2] * 2, gpu),
                out=torch.zeros_like(query), offsets=ints([0, 40, 80], gpu),
                mask=torch.full((80,), -1, dtype=torch.int64, device=gpu),
                picked=torch.zeros(2, 2, 2, 4, dtype=torch.int32, device=gpu), tokens=40, count=4, scale=SCALE)


def call(kind, i):
    if kind == "bounds":
        return TP.update_page_bounds(i["keys"], i["table"], i["lens"], i["tokens"], i["low"], i["high"])
    if kind == "select":
        return TP.select_pages(i["query"], i["low"], i["high"], i["table"], i["lens"], i["count"], out=i["picked"])
    if kind == "attend":
        return TP.selected_page_attention(i["query"], i["keys"], i["values"], i["table"], i["lens"], i["pages"], i["scale"],
                                          out=i["out"])
    return TT.tree_attention(i["query"], i["key"], i["value"], i["keys"], i["values"], i["table"], i["lens"],
                             i["offsets"], i["mask"], i["scale"], out=i["out"])


def cpu(t):
    return t.cpu()


WRONG = [
    ("bounds select attend tree", "lens", lambda t: t.long(), "INT32"),
    ("bounds select attend tree", "lens", lambda t: t[:1], "one length per row"),
    ("bounds select attend tree", "lens", cpu, "GPU tensor"),
    ("bounds select attend tree", "table", lambda t: t.long(), "INT32"),
    ("bounds select attend tree", "table", lambda t: t.T.contiguous().T, "contiguous rows"),
    ("bounds select attend tree", "table", lambda t: t[:1].expand(2, -1), "do not overlap"),
    ("bounds attend tree", "keys", lambda t: t.half(), "type"),
    ("bounds attend tree", "keys", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "must be contiguous"),
    ("bounds attend tree", "keys", lambda t: t[:, :64], "128"),
    ("bounds", "keys", lambda t: t.float(), "BF16 or FP16"),
    ("bounds", "low", lambda t: t[1:], "page_min"),
    ("bounds", "high", lambda t: t[:, :1], "shape of page_min"),
    ("bounds", "tokens", lambda n: -1, "negative"),
    ("select attend tree", "query", lambda t: t.float(), "BF16 or FP16"),
    ("select attend tree", "query", lambda t: t.half(), "type"),
    ("select attend tree", "query", lambda t: t[..., :64], "heads, 128"),
    ("select attend tree", "query", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), "contiguous"),
    ("select attend tree", "query", lambda t: t[:, :7], "positive multiple|shape of query"),
    ("select attend", "query", lambda t: t[:79], "same number of rows"),
    ("select", "high", lambda t: t[:, :1], "shape of page_min"),
    ("select", "picked", lambda t: t[..., :3].contiguous(), "out must be"),
    ("select", "picked", lambda t: t.long(), "out must be"),
    ("select", "count", lambda n: 0, "out must be"),
    ("attend", "pages", lambda t: t.long(), "INT32"),
    ("attend", "pages", lambda t: t[:, :1].contiguous(), "pages must be"),
    ("attend", "pages", lambda t: t[..., :0].contiguous(), "at least one page"),
    ("attend tree", "values", lambda t: t[1:], "value_cache shape"),
    ("attend tree", "values", lambda t: t.half(), "type"),
    ("attend tree", "out", lambda t: t.half(), "type"),
    ("attend tree", "out", lambda t: t[:40], "shape of query"),
    ("attend tree", "out", lambda t: torch.zeros(80, 9, 128, dtype=t.dtype, device=t.device)[:, :8], "contiguous"),
    ("attend tree", "out", cpu, "GPU tensor"),
    ("attend tree", "scale", lambda s: 0.0, "scale"),
    ("attend tree", "scale", lambda s: 1e-60, "scale"),  # zero in 32 bits
    ("attend tree", "scale", lambda s: float("nan"), "scale"),
    ("tree", "key", lambda t: t[:40], "rows of query"),
    ("tree", "value", lambda t: t.half(), "type"),
    ("tree", "key", lambda t: t[:1].expand(80, -1, -1), "key rows"),
    ("tree", "offsets", lambda t: t[:2], "batch \\+ 1"),
    ("tree", "offsets", lambda t: t.long(), "INT32"),
    ("tree", "mask", lambda t: t.int(), "INT64"),
    ("tree", "mask", lambda t: t[:40], "INT64 \\[rows\\]"),
]


@pytest.mark.parametrize("kind,name,change,text", [
    pytest.param(kind, name, change, text, id=f"{kind}-{name}-{i}")
    for i, (kinds, name, change, text) in enumerate(WRONG) for kind in kinds.split()])
def test_torch_refusals(gpu, inputs, kind, name, change, text):
    before = inputs["out"].clone()
    with pytest.raises((RuntimeError, NotImplementedError), match=text):
        call(kind, dict(inputs, **{name: change(inputs[name])}))
    assert torch.equal(inputs["out"], before)


def test_outputs_over_inputs_are_refused(gpu, inputs):
    for kind in ("attend", "tree"):
        with pytest.raises(RuntimeError, match="overlap"):
            call(kind, dict(inputs, out=inputs["query"]))
    with pytest.raises(RuntimeError, match="overlap"):
        call("bounds", dict(inputs, high=inputs["low"]))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_c_binding_equals_the_operators(gpu, inputs, dtype):
    """On a stream of its own; split and unsplit work, workspaces by the binding and by the caller."""
    i = {k: v.to(dtype) if torch.is_tensor(v) and v.is_floating_point() else v for k, v in inputs.items()}
    side = torch.cuda.Stream()
    call("bounds", i)
    low, high = TP.page_bounds_like(i["keys"])
    want_pages, want = call("select", i).clone(), call("attend", i).clone()
    want_tree = call("tree", i).clone()
    out, picked = torch.zeros_like(want), torch.zeros_like(want_pages)
    out_tree = torch.zeros_like(want)
    own = torch.full((16 << 20,), 255, dtype=torch.uint8, device=gpu)
    side.wait_stream(torch.cuda.current_stream())
    s = side.cuda_stream
    for workspace in (None, own):
        out.zero_(), out_tree.zero_(), picked.zero_()
        torch.cuda.synchronize()
        cabi.update_page_bounds(i["keys"], i["table"], i["lens"], 40, low, high, stream=s)
        cabi.select_pages(i["query"], low, high, i["table"], i["lens"], picked, stream=s, workspace=workspace)
        cabi.selected_page_attention(i["query"], i["keys"], i["values"], i["table"], i["lens"], i["pages"], out,
                                     scale=SCALE, stream=s, workspace=workspace)
        cabi.tree_attention(i["query"], i["key"], i["value"], i["keys"], i["values"], i["table"], i["lens"], i["offsets"],
                            i["mask"], out_tree, scale=SCALE, stream=s, workspace=workspace)
        side.synchronize()
        assert torch.equal(low, i["low"]) and torch.equal(high, i["high"])
        assert torch.equal(picked, want_pages) and torch.equal(out, want) and torch.equal(out_tree, want_tree)
    with pytest.raises(cabi.TriangleMixError) as refused:
        cabi.selected_page_attention(i["query"], i["keys"], i["values"], i["table"], i["lens"], i["pages"], out,
                                     scale=SCALE, workspace=own[:1024])
    assert refused.value.status == cabi.TM_ERR_WORKSPACE
