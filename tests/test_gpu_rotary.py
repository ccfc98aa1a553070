"""Position rotation and the rotated cache write against the 64-bit oracle."""

from __future__ import annotations

import pytest
import torch

from cached_cases import (E4M3, E4M3_MAX, bits, e4m3_tolerance, make_scales, quantised, rotation_tolerance,
                          side_by_side, turn_error)
from oracle import cached as OC
from pages_cases import make_rows
from trianglemix import cabi, cached, rotary

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def longs(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int64, device=device)


def some_positions(n: int, seed: int):
    """Near and far ones, the first position, and rows that are none."""
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, 1 << 21, (n,), generator=g)
    p[::5] = torch.randint(0, 300, (len(p[::5]),), generator=g)
    if n > 3:
        p[1], p[2], p[3] = 0, -1, 1 << 30
    if n > 8:
        p[7], p[8] = -(1 << 40), 131071
    return p


def check_rotated(got, x, want, positions, pairs, interleaved, magnitude, before):
    held = positions >= 0
    tol = rotation_tolerance(x[held], want[held], pairs, interleaved, magnitude, got.dtype)
    off = (got[held].double() - want[held]).abs() - tol
    assert off.max() <= 0 if off.numel() else True, off.max()
    assert torch.equal(got[held][..., 2 * pairs:], x[held][..., 2 * pairs:])  # copied bit by bit
    assert torch.equal(got[~held], before[~held])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,heads,rotary_dim,interleaved,magnitude", [
    (1, 1, 128, False, 1.0), (1, 40, 128, True, 1.2), (9, 7, 64, False, 1.0), (9, 9, 16, True, 1.0), (57, 8, 96, False, 1.1),
    (57, 33, 112, True, 1.0), (3, 256, 32, False, 1.0), (130, 12, 128, False, 0.5), (11, 3, 48, True, -1.0)])
def test_rotate(gpu, dtype, rows, heads, rotary_dim, interleaved, magnitude):
    print(f"rotate {rows} {heads} {rotary_dim} {interleaved} {dtype}", flush=True)
    x, positions = make_rows(rows, heads, dtype, rows + heads), some_positions(rows, rows)
    f = rotary.frequencies(rotary_dim, 500000.0, stretch=4.0, trained_length=8192)
    want = OC.rotate(x, positions, f, interleaved, magnitude)
    before = make_rows(rows, heads, dtype, 5)
    out = before.to(gpu)
    got = rotary.rotate(x.to(gpu), positions.to(gpu), f.to(gpu), interleaved=interleaved, magnitude=magnitude, out=out)
    assert got is out
    check_rotated(got.cpu(), x, want, positions, rotary_dim // 2, interleaved, magnitude, before)
    fresh = rotary.rotate(x.to(gpu), positions.to(gpu), f.to(gpu), interleaved=interleaved, magnitude=magnitude)
    held = positions >= 0
    assert torch.equal(fresh.cpu()[held], got.cpu()[held]) and not fresh.cpu()[~held].any()
    same = x.to(gpu)  # in place
    rotary.rotate(same, positions.to(gpu), f.to(gpu), interleaved=interleaved, magnitude=magnitude, out=same)
    assert torch.equal(same.cpu()[held], got.cpu()[held]) and torch.equal(same.cpu()[~held], x[~held])
    through_c = before.to(gpu)
    cabi.rotate_positions(x.to(gpu), positions.to(gpu), f.to(gpu), through_c, interleaved=interleaved, magnitude=magnitude)
    assert torch.equal(through_c, got)


def test_rotate_slices_of_a_fused_buffer_in_place(gpu):
    """Q and K side by side in rows of more; what lies between and behind them stays."""
    wide = make_rows(6, 30, BF16, 3)
    positions = longs([5, 9, -1, 70000, 0, 3])
    f = rotary.frequencies(128, 10000.0)
    buffer = wide.to(gpu)
    part = buffer[1:, 2:14]
    rotary.rotate(part, positions[1:].to(gpu), f.to(gpu), out=part)
    got = buffer.cpu()
    want = OC.rotate(wide[1:, 2:14], positions[1:], f, False, 1.0)
    check_rotated(got[1:, 2:14], wide[1:, 2:14], want, positions[1:], 64, False, 1.0, wide[1:, 2:14])
    assert torch.equal(got[0], wide[0]) and torch.equal(got[:, :2], wide[:, :2]) and torch.equal(got[:, 14:], wide[:, 14:])


def test_rotate_keeps_numbers_and_kinds(gpu):
    """What does not turn keeps its bits (NaN, signed zeros, infinities); NaN and infinities stay in their pairs."""
    x = torch.zeros(2, 3, 128, dtype=BF16)
    x[0, 0, 100], x[0, 0, 101], x[0, 0, 102] = float("nan"), -0.0, -float("inf")
    x[0, 1, 3], x[0, 2, 40] = float("nan"), float("inf")
    f = rotary.frequencies(64, 10000.0)
    got = rotary.rotate(x.to(gpu), longs([7, 0], gpu), f.to(gpu)).cpu()
    assert torch.equal(got[0, 0, 64:].view(torch.int16), x[0, 0, 64:].view(torch.int16))
    odd = ~got.float().isfinite()
    assert odd[0, 1].nonzero().flatten().tolist() == [3, 35] and odd[0, 2].nonzero().flatten().tolist() == [8, 40]
    assert torch.equal(got[1], x[1])


APPENDS = [
    # rows, heads, kv_heads, rotary_dim, interleaved
    (1, 32, 8, 128, False), (5, 4, 1, 64, True), (64, 8, 2, 128, False), (7, 9, 3, 96, False), (130, 12, 4, 128, True),
    (3, 32, 1, 16, False), (2, 64, 64, 128, False)]


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,heads,kv_heads,rotary_dim,interleaved", APPENDS)
def test_rotate_and_cache(gpu, dtype, cache, rows, heads, kv_heads, rotary_dim, interleaved):
    print(f"append {rows} {heads}/{kv_heads} {rotary_dim} {interleaved} {dtype} {cache}", flush=True)
    pages, m = 3, 1.1
    f = rotary.frequencies(rotary_dim, 10000.0)
    qkv = make_rows(rows, heads + 2 * kv_heads, dtype, rows * 3 + heads)
    positions = some_positions(rows, rows + 1)
    g = torch.Generator().manual_seed(rows)
    slots = torch.randperm(pages * 128, generator=g)[:rows]
    if rows > 4:
        slots[4] = -1       # padding of the cache alone: the query is a row
        slots[0] = pages * 128  # past the cache
    ks, vs = (make_scales(kv_heads, 1), make_scales(kv_heads, 2)) if cache == "e4m3" else (None, None)
    old = [make_rows(pages * 128, kv_heads, dtype, s).view(pages, 128, kv_heads, 128) for s in (8, 9)]
    if cache == "e4m3":
        old = [quantised(o, s) for o, s in zip(old, (ks, vs))]
    both = side_by_side(*old).to(gpu)
    before = make_rows(rows, heads, dtype, 5)
    q_out = before.to(gpu)
    buffer = qkv.to(gpu)
    q, k, v = buffer[:, :heads], buffer[:, heads:heads + kv_heads], buffer[:, heads + kv_heads:]
    scales = {} if ks is None else {"key_scale": ks.to(gpu), "value_scale": vs.to(gpu)}
    args = (positions.to(gpu), slots.to(gpu), f.to(gpu))
    rotary.rotate_and_cache(q, k, v, *args, both[:, 0], both[:, 1], interleaved=interleaved, magnitude=m, query_out=q_out,
                            **scales)
    assert torch.equal(buffer.cpu(), qkv)
    want_q = OC.rotate(qkv[:, :heads], positions, f, interleaved, m)
    check_rotated(q_out.cpu(), qkv[:, :heads], want_q, positions, rotary_dim // 2, interleaved, m, before)
    key, value = qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    turned = OC.rotate(key, positions, f, interleaved, m)
    held = (positions >= 0) & (slots >= 0) & (slots < pages * 128)
    new_k, new_v = (both[:, i].cpu().reshape(pages * 128, kv_heads, 128) for i in (0, 1))
    old_k, old_v = (o.reshape(pages * 128, kv_heads, 128) for o in old)
    at = slots[held]
    if cache == "same":
        tol = rotation_tolerance(key[held], turned[held], rotary_dim // 2, interleaved, m, dtype)
        assert ((new_k[at].double() - turned[held]).abs() <= tol).all()
        assert torch.equal(new_v[at], value[held])
    else:
        want = OC.quotient(turned, ks)[held]
        error = turn_error(key, rotary_dim // 2, interleaved, m)[held] / ks.double()[:, None]
        assert ((new_k.double()[at] - want).abs() <= e4m3_tolerance(want, error)).all()
        assert torch.equal(bits(new_v)[at], bits(quantised(value, vs))[held])
    rest = torch.ones(pages * 128, dtype=torch.bool)
    rest[at] = False
    for new, was in ((new_k, old_k), (new_v, old_v)):
        assert torch.equal(bits(new)[rest], bits(was)[rest])
    # in place and through the C ABI: the same numbers
    again = side_by_side(*old).to(gpu)
    assert rotary.rotate_and_cache(q, k, v, *args, again[:, 0], again[:, 1], interleaved=interleaved, magnitude=m,
                                   **scales).data_ptr() == q.data_ptr()
    ok = positions >= 0
    assert torch.equal(q.cpu()[ok], q_out.cpu()[ok]) and torch.equal(q.cpu()[~ok], qkv[:, :heads][~ok])
    assert torch.equal(again.view(torch.uint8), both.view(torch.uint8))
    third = side_by_side(*old).to(gpu)
    cabi.rotate_and_cache(qkv.to(gpu)[:, :heads], k, v, *args, q_out, third[:, 0], third[:, 1], interleaved=interleaved,
                          magnitude=m, **scales)
    assert torch.equal(third.view(torch.uint8), both.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_8_bit_numbers_of_every_kind(gpu, dtype):
    """Every 16-bit number as a value: nearest, ties to even, subnormals, the largest, infinities and NaN."""
    value = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype).view(512, 1, 128)
    slots = torch.arange(512, device=gpu)
    f = rotary.frequencies(128).to(gpu)
    zeros = torch.zeros(512, 1, 128, dtype=dtype, device=gpu)
    for scale in (1.0, 0.37, 2.0 ** -9, 900.0):
        s = torch.tensor([scale])
        keys, values = cached.new_cache(4, 1, device=gpu)
        rotary.rotate_and_cache(zeros, value.to(gpu), value.to(gpu), torch.zeros_like(slots), slots, f, keys, values,
                                key_scale=s.to(gpu), value_scale=s.to(gpu))
        got = values.view(-1, 1, 128).cpu()
        want = (value.float() / s).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        nan = value.isnan()
        assert torch.equal(got.float().isnan(), nan)
        assert torch.equal(bits(got)[~nan], bits(want)[~nan]), scale
        # position 0 turns nothing, but 0 * infinity is NaN: finite pairs alone
        k = keys.view(-1, 1, 128).cpu()
        fine = value.float().isfinite() & value.float().isfinite().roll(64, dims=-1)
        assert torch.equal(k.float()[fine], want.float()[fine]), scale


def test_slots_behind_2_31_bytes(gpu):
    """Slots far behind 2^31 bytes and numbers of the cache; everything else stays zero."""
    print("far slots", flush=True)
    pages, kv = 36000, 8
    keys, values = cached.new_cache(pages, kv, device=gpu)  # 4.7e9 bytes each
    ks, vs = make_scales(kv, 1), make_scales(kv, 2)
    qkv = make_rows(4, 32 + 2 * kv, BF16, 3)
    slots = longs([pages * 128 - 1, 17000 * 128 + 5, 33000 * 128, 3])
    b = qkv.to(gpu)
    rotary.rotate_and_cache(b[:, :32], b[:, 32:40], b[:, 40:], longs([0] * 4, gpu), slots.to(gpu),
                            rotary.frequencies(128).to(gpu), keys, values, key_scale=ks.to(gpu), value_scale=vs.to(gpu))
    for cache, part, s in ((keys, qkv[:, 32:40], ks), (values, qkv[:, 40:], vs)):
        flat = bits(cache).view(-1, kv, 128)
        assert torch.equal(flat[slots.to(gpu)].cpu(), bits(quantised(part, s)))
        flat[slots.to(gpu)] = 0
        assert not flat.any()


def test_graph_replays_with_other_positions(gpu):
    heads, kv, rows = 8, 2, 6
    f = rotary.frequencies(128, 10000.0)
    qkv = make_rows(rows, heads + 2 * kv, BF16, 31).to(gpu)
    keys, values = cached.new_cache(2, kv, torch.bfloat16, device=gpu)
    positions, slots = longs([0] * rows, gpu), longs([-1] * rows, gpu)
    q_out, x_out = torch.zeros_like(qkv[:, :heads]).contiguous(), torch.zeros_like(qkv)
    fd = f.to(gpu)

    def step():
        rotary.rotate_and_cache(qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], positions, slots, fd, keys,
                                values, query_out=q_out)
        rotary.rotate(qkv, positions, fd, interleaved=True, out=x_out)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        positions.copy_(longs([turn * 1000 + i if i != turn else -1 for i in range(rows)]))
        slots.copy_(longs([(turn * 50 + i * 7) % 256 for i in range(rows)]))
        for t in (q_out, x_out, keys, values):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q_out, x_out, keys, values)]
        for t in (q_out, x_out, keys, values):
            t.zero_()
        step()
        for a, b in zip(got, (q_out, x_out, keys, values)):
            assert torch.equal(a, b) and a.any()
