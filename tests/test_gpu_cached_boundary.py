"""What the cached-attention torch operators refuse on the GPU, and calls that use streams and workspaces of their own."""

from __future__ import annotations

import pytest
import torch

from cached_cases import make_any_cache
from pages_cases import SCALE, make_rows
from trianglemix import cabi, cached, rotary

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def inputs(gpu):
    lens = [300, 41]
    keys, values, table, ks, vs = (t.to(gpu) for t in make_any_cache(lens, 2, BF16, "e4m3", seed=91))
    query, fresh = make_rows(80, 8, BF16, 92).to(gpu), make_rows(80, 2, BF16, 93).to(gpu)
    positions = torch.arange(80, device=gpu)
    return dict(x=query, query=query, key=fresh, value=fresh.flip(0), positions=positions, slots=positions.flip(0),
                freqs=rotary.frequencies(64).to(gpu), keys=keys, values=values, table=table,
                lens=torch.tensor(lens, dtype=torch.int32, device=gpu), ks=ks, vs=vs, out=torch.zeros_like(query), scale=SCALE,
                magnitude=1.0, window=-1, sinks=0)


def call(kind, i):
    if kind == "rotate":
        return rotary.rotate(i["x"], i["positions"], i["freqs"], magnitude=i["magnitude"], out=i["out"])
    if kind == "append":
        return rotary.rotate_and_cache(i["query"], i["key"], i["value"], i["positions"], i["slots"], i["freqs"], i["keys"],
                                       i["values"], magnitude=i["magnitude"], key_scale=i["ks"], value_scale=i["vs"],
                                       query_out=i["out"])
    return cached.cached_attention(i["query"], i["keys"], i["values"], i["table"], i["lens"], i["scale"], window=i["window"],
                                   sinks=i["sinks"], key_scale=i["ks"], value_scale=i["vs"], out=i["out"])


def cpu(t):
    return t.cpu()


WRONG = [
    ("rotate", "x", lambda t: t.float(), "BF16 or FP16"),
    ("rotate", "x", lambda t: t[..., :64], "heads, 128"),
    ("rotate", "x", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), "contiguous"),
    ("rotate", "x", lambda t: t[:40], "shape of x"),
    ("rotate append", "positions", lambda t: t.int(), "INT64"),
    ("rotate append", "positions", lambda t: t[:40], "INT64"),
    ("rotate append", "positions", lambda t: t.repeat(2)[::2], "INT64"),
    ("rotate append", "positions", cpu, "GPU tensor"),
    ("rotate append", "freqs", lambda t: t.float(), "FP64"),
    ("rotate append", "freqs", lambda t: t[:12], "multiple of 16"),
    ("rotate append", "freqs", lambda t: t.repeat(3), "multiple of 16"),
    ("rotate append", "freqs", lambda t: t[:0], "multiple of 16"),
    ("rotate append", "magnitude", lambda m: float("inf"), "magnitude"),
    ("rotate append", "magnitude", lambda m: 1e300, "magnitude"),  # infinite in 32 bits
    ("rotate append attend", "out", lambda t: t.half(), "type"),
    ("rotate append attend", "out", lambda t: t[:40], "shape of"),
    ("rotate append attend", "out", cpu, "GPU tensor"),
    ("append attend", "query", lambda t: t.half(), "type"),
    ("append attend", "query", lambda t: t[:, :7], "shape of"),
    ("append", "key", lambda t: t[:40], "rows of query"),
    ("append", "value", lambda t: t.half(), "type"),
    ("append", "key", lambda t: t[:1].expand(80, -1, -1), "key rows"),
    ("append", "slots", lambda t: t.int(), "INT64"),
    ("append", "slots", lambda t: t[:79], "INT64"),
    ("append attend", "keys", lambda t: t.to(BF16), "type of key_cache"),
    ("append attend", "keys", lambda t: t.view(torch.uint8)[:, :64].view(t.dtype), "128"),
    ("append attend", "values", lambda t: t[1:], "value_cache shape"),
    ("append attend", "ks", lambda t: None, "belong to FP8"),
    ("append attend", "vs", lambda t: None, "belong to FP8"),
    ("append attend", "ks", lambda t: t.double(), "FP32"),
    ("append attend", "ks", lambda t: t[:1], "FP32"),
    ("append attend", "vs", cpu, "GPU tensor"),
    ("attend", "out", lambda t: torch.zeros(80, 9, 128, dtype=t.dtype, device=t.device)[:, :8], "contiguous"),
    ("attend", "lens", lambda t: t.long(), "INT32"),
    ("attend", "lens", lambda t: t[:1], "one length per row"),
    ("attend", "table", lambda t: t.long(), "INT32"),
    ("attend", "table", lambda t: t[:1].expand(2, -1), "do not overlap"),
    ("attend", "table", lambda t: t.T.contiguous().T, "contiguous rows"),
    ("attend", "query", lambda t: t[:79], "same number of rows"),
    ("attend", "window", lambda w: -2, "window"),
    ("attend", "sinks", lambda s: 4, "window"),
    ("attend", "scale", lambda s: 0.0, "scale"),
    ("attend", "scale", lambda s: 1e-60, "scale"),  # zero in 32 bits
    ("attend", "scale", lambda s: float("nan"), "scale"),
]


@pytest.mark.parametrize("kind,name,change,text", [
    pytest.param(kind, name, change, text, id=f"{kind}-{name}-{i}")
    for i, (kinds, name, change, text) in enumerate(WRONG) for kind in kinds.split()])
def test_torch_refusals(gpu, inputs, kind, name, change, text):
    before = [inputs[k].clone() for k in ("out", "query")]
    cache = inputs["keys"].view(torch.uint8).clone()
    with pytest.raises((RuntimeError, NotImplementedError), match=text):
        call(kind, dict(inputs, **{name: change(inputs[name])}))
    assert torch.equal(inputs["out"], before[0]) and torch.equal(inputs["query"], before[1])
    assert torch.equal(inputs["keys"].view(torch.uint8), cache)


def test_16_bit_caches_of_another_type_and_with_scales_are_refused(gpu, inputs):
    keys = inputs["keys"].to(FP16)
    for more, text in ((dict(ks=None, vs=None), "type of query"), ({}, "belong to FP8")):
        for kind in ("append", "attend"):
            with pytest.raises(RuntimeError, match=text):
                cache = keys if more else keys.to(BF16)
                call(kind, dict(inputs, keys=cache, values=cache.clone(), **more))


def test_outputs_over_inputs_are_refused(gpu, inputs):
    with pytest.raises(RuntimeError, match="overlap"):
        call("attend", dict(inputs, out=inputs["query"]))
    with pytest.raises(RuntimeError, match="overlap"):
        call("append", dict(inputs, values=inputs["keys"]))
    wide = torch.zeros(81, 8, 128, dtype=BF16, device=gpu)
    with pytest.raises(RuntimeError, match="overlap"):
        call("rotate", dict(inputs, x=wide[1:], out=wide[:80]))
    fused = torch.zeros(80, 12, 128, dtype=BF16, device=gpu)
    with pytest.raises(RuntimeError, match="overlap"):
        call("append", dict(inputs, query=fused[:, :8], key=fused[:, 8:10], value=fused[:, 10:], out=fused[:, 1:9]))


@pytest.mark.parametrize("cache", ["e4m3", "same"])
def test_streams_and_workspaces(gpu, cache):
    """On a stream of its own, through both bindings, with the caller's workspace of any contents."""
    lens = [3000, 41]
    keys, values, table, ks, vs = make_any_cache(lens, 2, FP16, cache, seed=95)
    keys, values, table = keys.to(gpu), values.to(gpu), table.to(gpu)
    scales = {} if ks is None else {"key_scale": ks.to(gpu), "value_scale": vs.to(gpu)}
    query, n = make_rows(2, 8, FP16, 96).to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)
    want = cached.cached_attention(query, keys, values, table, n, SCALE, **scales)
    own = torch.full((16 << 20,), 255, dtype=torch.uint8, device=gpu)
    side = torch.cuda.Stream()
    for workspace in (None, own, own):
        out = torch.zeros_like(want)
        side.wait_stream(torch.cuda.current_stream())
        cabi.cached_attention(query, keys, values, table, n, out, scale=SCALE, stream=side.cuda_stream, workspace=workspace,
                              **scales)
        side.synchronize()
        assert torch.equal(out, want)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cached.cached_attention(query, keys, values, table, n, SCALE, **scales)
    side.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(cabi.TriangleMixError) as refused:
        cabi.cached_attention(query, keys, values, table, n, want, scale=SCALE, workspace=own[:1024], **scales)
    assert refused.value.status == cabi.TM_ERR_WORKSPACE
    with pytest.raises(cabi.TriangleMixError):
        cabi.cached_attention(query[:1], keys, values, table, n, want, scale=SCALE, **scales)


def test_empty_calls(gpu, inputs):
    assert call("rotate", dict(inputs, x=inputs["x"][:0], positions=inputs["positions"][:0], out=inputs["out"][:0])).shape == (0, 8, 128)
    none = dict(inputs, query=inputs["query"][:0], out=inputs["out"][:0])
    assert call("attend", none).shape == (0, 8, 128)
    assert call("attend", dict(none, table=inputs["table"][:0], lens=inputs["lens"][:0])).shape == (0, 8, 128)
    empty = {k: inputs[k][:0] for k in ("query", "key", "value", "positions", "slots", "out")}
    assert call("append", dict(inputs, **empty)).shape == (0, 8, 128)
