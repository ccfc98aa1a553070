"""The boundary of the cached-attention operators on the CPU: C ABI, torch operators, frequencies, scales.

No kernel runs here: every call either is refused before any HIP call (fake, never-dereferenced pointers) or has no
work to enqueue.
"""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch
from test_boundary_abi import lib  # noqa: F401  (fixture)
from trianglemix import cached, native, rotary

HEADER = Path(__file__).resolve().parents[1] / "include" / "trianglemix_cached.h"
BF16, FP16, E4M3 = 0, 1, 2
A = [0x4000_0000_0000 * (i + 1) for i in range(16)]  # fake device addresses, 2^46 apart


def test_header_functions_are_exported_and_declared(lib):  # noqa: F811
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = set(re.findall(r"\b(tm_[a-z_]+)\s*\(", text))
    assert names == {"tm_rotate_positions", "tm_rotate_and_cache", "tm_cached_attention",
                     "tm_cached_attention_workspace_size"}
    for name in names:
        declared = re.search(rf"\b{name}\s*\(([^)]*)\)", text).group(1)
        assert len(getattr(lib, name).argtypes) == len(declared.split(",")), name
    assert re.search(r"#define TM_E4M3 2\b", HEADER.read_text())


PAGE = 128 * 8 * 128  # numbers of a page of eight KV heads
TURN = dict(positions=A[3], freqs=A[4], rotary=128, interleaved=0, magnitude=1.0, dtype=BF16)
ROTATE = dict(TURN, x=A[0], x_stride=4096, out=A[1], out_stride=4096, rows=40, heads=32)
APPEND = dict(TURN, query=A[0], query_stride=4096, key=A[1], key_stride=1024, value=A[2], value_stride=1024, slots=A[5],
              out=A[6], out_stride=4096, keys=A[7], keys_stride=PAGE, values=A[8], values_stride=PAGE, key_scale=A[9],
              value_scale=A[10], rows=40, heads=32, kv=8, num_pages=300, cache=E4M3)
ATTEND = dict(query=A[0], query_stride=4096, keys=A[7], keys_stride=PAGE, values=A[8], values_stride=PAGE, key_scale=A[9],
              value_scale=A[10], table=A[3], table_stride=64, lens=A[4], out=A[6], batch=4, rows=5, heads=32, kv=8, cols=64,
              num_pages=300, window=-1, sinks=0, scale=0.088, dtype=BF16, cache=E4M3, ws=A[11], ws_bytes=1 << 30)
KINDS = {"rotate": ROTATE, "append": APPEND, "attend": ATTEND}


def run(lib, kind, **over):  # noqa: F811
    assert set(over) <= set(KINDS[kind])
    g = dict(KINDS[kind], **over).__getitem__
    if kind == "rotate":
        return lib.tm_rotate_positions(*map(g, ("x", "x_stride", "positions", "freqs", "out", "out_stride", "rows", "heads",
                                                "rotary", "interleaved", "magnitude", "dtype")), None)
    if kind == "append":
        return lib.tm_rotate_and_cache(*map(g, (
            "query", "query_stride", "key", "key_stride", "value", "value_stride", "positions", "slots", "freqs", "out",
            "out_stride", "keys", "keys_stride", "values", "values_stride", "key_scale", "value_scale", "rows", "heads", "kv",
            "num_pages", "rotary", "interleaved", "magnitude", "dtype", "cache")), None)
    return lib.tm_cached_attention(*map(g, (
        "query", "query_stride", "keys", "keys_stride", "values", "values_stride", "key_scale", "value_scale", "table",
        "table_stride", "lens", "out", "batch", "rows", "heads", "kv", "cols", "num_pages", "window", "sinks", "scale",
        "dtype", "cache", "ws", "ws_bytes")), None)


ALL = [
    (dict(dtype=2), 1, "TM_BF16 or TM_FP16"), (dict(dtype=-1), 1, "TM_BF16 or TM_FP16"),
    (dict(rows=-1), 1, "negative"), (dict(heads=0), 1, "positive multiple"), (dict(out=None), 1, "non-null"),
    (dict(out=A[6] + 8), 1, "16-byte"),
]
TURNS = [
    (dict(rows=(1 << 21) + 1), 2, "rows"), (dict(heads=264), 2, "limits are 256"),
    (dict(rotary=0), 2, "rotary_dim"), (dict(rotary=144), 2, "rotary_dim"), (dict(rotary=24), 2, "rotary_dim"),
    (dict(rotary=-16), 2, "rotary_dim"), (dict(magnitude=float("nan")), 1, "magnitude"),
    (dict(magnitude=float("inf")), 1, "magnitude"), (dict(positions=None), 1, "non-null"),
    (dict(positions=A[3] + 4), 1, "aligned to their elements"), (dict(freqs=None), 1, "non-null"),
    (dict(freqs=A[4] + 4), 1, "aligned to their elements"), (dict(out_stride=4095), 1, "rows"), (dict(out_stride=0), 1, "rows"),
    (dict(out=A[3]), 1, "must not overlap positions"), (dict(out=A[4] + 16), 1, "must not overlap frequencies"),
]
CACHES = [
    (dict(heads=33), 1, "positive multiple"), (dict(kv=0), 1, "positive multiple"),
    (dict(heads=33, kv=1), 2, "32 a KV head"),
    (dict(num_pages=0), 1, "pages > 0"), (dict(num_pages=(1 << 22) + 1), 2, "limit is 4194304"),
    (dict(keys_stride=PAGE - 16), 1, "key_cache pages"), (dict(keys_stride=PAGE + 8), 1, "multiple of 16"),
    (dict(values_stride=PAGE + 8), 1, "value_cache pages"), (dict(keys=None), 1, "non-null"),
    (dict(values=A[8] + 8), 1, "16-byte"), (dict(key_scale=None), 1, "non-null"), (dict(value_scale=None), 1, "non-null"),
    (dict(key_scale=A[9] + 2), 1, "aligned to their elements"), (dict(cache=FP16), 1, "rows' type"),
    (dict(cache=3), 1, "rows' type"), (dict(cache=-1), 1, "rows' type"), (dict(cache=BF16), 1, "have no scales"),
    (dict(cache=BF16, key_scale=None), 1, "have no scales"),
    (dict(cache=BF16, key_scale=None, value_scale=None, keys_stride=PAGE + 4), 1, "multiple of 8"),
    (dict(query=None), 1, "non-null"), (dict(query=A[0] + 2), 1, "16-byte"), (dict(query_stride=4088), 1, "query rows"),
    (dict(query_stride=4097), 1, "query rows"), (dict(out=A[7]), 1, "must not overlap"), (dict(out=A[9]), 1, "must not overlap"),
]
OWN = {
    "rotate": [
        (dict(x=None), 1, "non-null"), (dict(x=A[0] + 8), 1, "16-byte"), (dict(x_stride=4088), 1, "x rows"),
        (dict(out=A[0], out_stride=8192), 1, "must not overlap x"), (dict(out=A[0] + 256), 1, "must not overlap x"),
        (dict(x_stride=8192, out=A[0] + 4096 * 2 - 16, out_stride=8192), 1, "must not overlap x"),
        (dict(x_stride=8192, out=A[0] - 4096 * 2 + 16, out_stride=8192), 1, "must not overlap x"),
    ],
    "append": [
        (dict(key=None), 1, "non-null"), (dict(value=A[2] + 4), 1, "16-byte"), (dict(key_stride=1016), 1, "key rows"),
        (dict(value_stride=-8), 1, "value rows"), (dict(slots=None), 1, "non-null"),
        (dict(slots=A[5] + 4), 1, "aligned to their elements"), (dict(out=A[1]), 1, "must not overlap key"),
        (dict(out=A[2] + 1024), 1, "must not overlap value"), (dict(out=A[5]), 1, "must not overlap slot_mapping"),
        (dict(values=A[7]), 1, "must not overlap value_cache"), (dict(values=A[7] + PAGE), 1, "must not overlap value_cache"),
        (dict(keys=A[1]), 1, "key_cache must not overlap key"), (dict(values=A[0]), 1, "value_cache must not overlap query"),
        (dict(keys=A[3] - 4096), 1, "key_cache must not overlap positions"),
        (dict(out=A[0], out_stride=8192), 1, "must not overlap query"),
    ],
    "attend": [
        (dict(batch=-1), 1, "negative"), (dict(batch=1025), 2, "limit is 1024"), (dict(rows=1 << 20), 2, "query rows"),
        (dict(cols=0), 1, "block_table"), (dict(table_stride=63), 1, "block_table"),
        (dict(cols=16385, table_stride=16385), 2, "limit is 16384"), (dict(table=None), 1, "non-null"),
        (dict(lens=None), 1, "non-null"), (dict(table=A[3] + 2), 1, "aligned to their elements"),
        (dict(lens=A[4] + 1), 1, "aligned to their elements"), (dict(window=-2), 1, "window"), (dict(sinks=-1, window=4), 1, "window"),
        (dict(sinks=4), 1, "window"), (dict(ws=None), 3, "inconsistent"), (dict(ws_bytes=-1), 3, "inconsistent"),
        (dict(ws_bytes=1024), 3, "smaller than"), (dict(ws=A[11] + 8), 3, "16-byte"), (dict(ws=A[0]), 1, "must not overlap"),
        (dict(out=A[3] + 64), 1, "out must not overlap block_table"), (dict(out=A[11]), 1, "must not overlap"),
        (dict(batch=1024, rows=2048, heads=256, kv=256, query_stride=256 * 128, keys_stride=32 * PAGE,
              values_stride=32 * PAGE, cols=16384, table_stride=16384), 2, "limit is 1073741824"),
        *[(dict(scale=s), 1, "scale") for s in (0.0, -1.0, float("nan"), float("inf"))],
    ],
}


def _refusals():
    for kind, cases in {"rotate": ALL + TURNS, "append": ALL + TURNS + CACHES, "attend": ALL + CACHES}.items():
        for over, status, text in cases + OWN[kind]:
            if kind == "rotate" and over.get("out") == A[6] + 8:
                over = dict(out=A[1] + 8)
            yield pytest.param(kind, over, status, text, id=f"{kind}-{'-'.join(over)}-{text[:12]}")


@pytest.mark.parametrize("kind,over,status,text", _refusals())
def test_refusals(lib, kind, over, status, text):  # noqa: F811
    assert run(lib, kind, **over) == status, lib.tm_last_error()
    assert text in lib.tm_last_error().decode()


@pytest.mark.parametrize("kind,over", [("rotate", dict(rows=0)), ("append", dict(rows=0)), ("attend", dict(rows=0)),
                                       ("attend", dict(batch=0))])
def test_nothing_to_do_enqueues_nothing(lib, kind, over):  # noqa: F811
    """Without work null tensors and no workspace are fine, and an earlier error's text goes."""
    assert run(lib, kind, dtype=7) == 1
    none = {k: None for k, v in KINDS[kind].items() if v in A and not k.endswith("scale")}
    if "ws" in none:
        none["ws_bytes"] = 0
    assert run(lib, kind, **none, **over) == 0
    assert lib.tm_last_error() == b""


def test_workspace_sizes(lib):  # noqa: F811
    size = lib.tm_cached_attention_workspace_size
    assert size(0, 1, 32, 8, 64, -1, 0) == size(4, 0, 32, 8, 64, -1, 0) == 0
    for bad in ((-1, 1, 32, 8, 64, -1, 0), (4, -1, 32, 8, 64, -1, 0), (4, 1, 33, 8, 64, -1, 0), (1025, 1, 32, 8, 64, -1, 0),
                (4, 1, 32, 8, 0, -1, 0), (4, 1, 32, 8, 16385, -1, 0), (4, 1, 32, 8, 64, -2, 0), (4, 1, 32, 8, 64, -1, 1),
                (4, 1, 32, 8, 64, 5, -1), (1024, 2048, 256, 256, 16384, -1, 0)):
        assert size(*bad) == -1, bad
    # a window bounds the work, whatever the table holds, also at the largest numbers
    big = (1 << 63) - 1
    assert size(64, 1, 32, 8, 16384, 512, 8) > 0 and size(64, 1, 32, 8, 16384, big, 8) > 0
    assert size(1, 1, 32, 8, 64, 0, big) > 0
    for b, r, h, k in ((1, 1, 32, 8), (64, 1, 32, 8), (8, 20, 32, 8), (1, 2048, 32, 8), (3, 64, 256, 8)):
        n = size(b, r, h, k, 64, -1, 0)
        assert (n == 0 or n > 65536) and n % 16 == 0 and n <= 65536 + (64 << 20) + (2 << 20)


# ---- torch operators ----

@pytest.fixture(scope="module")
def ops(lib):  # noqa: F811
    native.load_triangle_mix_adapter()
    return torch.ops.trianglemix


def test_schemas(ops):
    assert str(ops.rotate_positions.out._schema) == (
        "trianglemix::rotate_positions.out(Tensor x, Tensor positions, Tensor frequencies, bool interleaved, "
        "float magnitude, *, Tensor(a!) out) -> Tensor(a!)")
    assert str(ops.rotate_and_cache.default._schema) == (
        "trianglemix::rotate_and_cache(Tensor query, Tensor key, Tensor value, Tensor positions, Tensor slot_mapping, "
        "Tensor frequencies, bool interleaved, float magnitude, Tensor(a!) query_out, Tensor(b!) key_cache, "
        "Tensor(c!) value_cache, Tensor? key_scale=None, Tensor? value_scale=None) -> ()")
    assert str(ops.cached_attention.out._schema) == (
        "trianglemix::cached_attention.out(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
        "Tensor seq_lens, float scale, int window=-1, int sinks=0, Tensor? key_scale=None, Tensor? value_scale=None, *, "
        "Tensor(a!) out) -> Tensor(a!)")


def test_meta_shapes_and_no_cpu_kernel(ops):
    def make(device):
        e = dict(device=device, dtype=torch.bfloat16)
        i = dict(device=device, dtype=torch.int64)
        keys, values = cached.new_cache(20, 2, device=device)
        assert keys.shape == (20, 128, 2, 128) and keys.dtype == torch.float8_e4m3fn
        scale = torch.ones(2, device=device)
        return (torch.zeros(80, 8, 128, **e), torch.zeros(80, 2, 128, **e), torch.zeros(80, **i), torch.zeros(80, **i),
                torch.zeros(64, device=device, dtype=torch.float64), keys, values, scale,
                torch.zeros(2, 9, device=device, dtype=torch.int32), torch.zeros(2, device=device, dtype=torch.int32))

    q, kv, pos, slots, f, keys, values, scale, table, lens = make("meta")
    out = torch.empty_like(q)
    assert rotary.rotate(q, pos, f).shape == q.shape and rotary.rotate(q, pos, f, out=out) is out
    assert rotary.rotate_and_cache(q, kv, kv, pos, slots, f, keys, values, key_scale=scale, value_scale=scale) is q
    assert rotary.rotate_and_cache(q, kv, kv, pos, slots, f, keys, values, key_scale=scale, value_scale=scale,
                                   query_out=out) is out
    args = (keys, values, table, lens, 0.1)
    assert cached.cached_attention(q, *args, key_scale=scale, value_scale=scale).shape == q.shape
    assert cached.cached_attention(q, *args, key_scale=scale, value_scale=scale, out=out) is out

    q, kv, pos, slots, f, keys, values, scale, table, lens = make("cpu")
    for call in (lambda: rotary.rotate(q, pos, f),
                 lambda: rotary.rotate_and_cache(q, kv, kv, pos, slots, f, keys, values, key_scale=scale, value_scale=scale),
                 lambda: cached.cached_attention(q, keys, values, table, lens, 0.1, key_scale=scale, value_scale=scale)):
        with pytest.raises(NotImplementedError):
            call()


# ---- frequencies and scales ----

def test_frequencies():
    f = rotary.frequencies(64, 500000.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1.0
    assert math.isclose(f[31].item(), 500000.0 ** (-62 / 64), rel_tol=1e-14)
    assert torch.equal(rotary.frequencies(64, 500000.0, stretch=1.0, method="parts"), f)
    assert torch.allclose(rotary.frequencies(64, 500000.0, stretch=4.0, method="positions"), f / 4, rtol=1e-15, atol=0)
    b = rotary.frequencies(64, 500000.0, stretch=4.0, method="base")
    assert b[0] == 1.0 and math.isclose(b[31].item(), f[31].item() / 4, rel_tol=1e-12) and (b[1:] < f[1:]).all()
    p = rotary.frequencies(64, 500000.0, stretch=4.0, trained_length=8192)
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and (turns >= 32).any()
    assert torch.allclose(p[turns <= 1], f[turns <= 1] / 4, rtol=1e-15, atol=0) and (turns <= 1).any()
    mid = (turns > 1) & (turns < 32)
    assert (p[mid] < f[mid]).all() and (p[mid] > f[mid] / 4).all()
    assert rotary.magnitude(1.0) == 1.0 and math.isclose(rotary.magnitude(8.0), 0.1 * math.log(8) + 1)
    for bad in (dict(rotary_dim=8), dict(rotary_dim=144), dict(rotary_dim=40), dict(rotary_dim=64, base=1.0),
                dict(rotary_dim=64, base=float("nan")), dict(rotary_dim=64, stretch=0.5),
                dict(rotary_dim=64, stretch=2.0), dict(rotary_dim=64, stretch=2.0, trained_length=0),
                dict(rotary_dim=64, stretch=2.0, trained_length=8, fast_turns=1.0), dict(rotary_dim=64, method="x")):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)


def test_head_scales():
    x = torch.zeros(5, 3, 128, dtype=torch.bfloat16)
    x[1, 0, 4], x[2, 1, 7] = -896.0, 2.0
    s = cached.head_scales(x)
    assert s.dtype == torch.float32 and torch.equal(s, torch.tensor([2.0, 2.0 / 448, 1.0]))
    assert torch.equal(cached.head_scales(x, margin=2.0), torch.tensor([4.0, 4.0 / 448, 1.0]))
    x[1, 0, 4], x[2, 1, 7] = 2.0 ** -120, 2.0 ** -117  # 2^-120 / 448 is no normal number of 32 bits
    assert torch.equal(cached.head_scales(x), torch.tensor([1.0, 2.0 ** -117 / 448, 1.0]))
    keys, values = cached.new_cache(3, 2, torch.float16)
    assert keys.shape == values.shape == (3, 128, 2, 128) and keys.dtype == torch.float16 and not keys.any()
