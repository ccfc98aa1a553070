"""Attention over draft trees against the 64-bit oracle, within the rounding of its type."""

from __future__ import annotations

import pytest
import torch

from oracle import pages as OP
from pages_cases import SCALE, make_cache, make_rows, to_gpu, tolerance
from trianglemix import tree as TT

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def make_trees(sizes, seed):
    """(offsets, masks): random trees, each node on one of the few before it."""
    g = torch.Generator().manual_seed(seed)
    offsets, masks = [0], []
    for n in sizes:
        back = torch.randint(1, 6, (max(n, 1),), generator=g).tolist()[:n]
        masks += TT.ancestor_masks([i - k if i >= k else -1 for i, k in enumerate(back)])
        offsets.append(offsets[-1] + n)
    return ints(offsets), torch.tensor(masks, dtype=torch.int64)


def check(gpu, qkv, heads, kv, keys, values, table, contexts, offsets, mask, longest):
    dtype, total = qkv.dtype, qkv.shape[0]
    query, key, value = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    out = make_rows(total, heads, dtype, 78)
    want, size, written = OP.tree_attention(query, key, value, keys, values, table, ints(contexts), offsets, mask, SCALE,
                                            out)
    qkv_d, out_d = qkv.to(gpu), out.to(gpu)
    TT.tree_attention(qkv_d[:, :heads], qkv_d[:, heads:heads + kv], qkv_d[:, heads + kv:], to_gpu(keys, gpu),
                      to_gpu(values, gpu), table.to(gpu), ints(contexts, gpu), offsets.to(gpu), mask.to(gpu), SCALE,
                      out=out_d)
    got = out_d.cpu()
    assert torch.equal(got[~written], out[~written])  # rows of no tree are left as they were
    finite = want.isfinite()
    assert torch.equal(got.isfinite()[written], finite[written])
    real = torch.cat([values[values.isfinite()], value[value.isfinite()]])
    tol = tolerance(want, size, real, longest + 64, dtype)
    off = (got.double() - want).abs()
    ok = (off <= tol) | ~finite
    assert bool(ok[written].all()), f"off by {(off / tol.clamp(min=1e-30))[written].nan_to_num(0).max():.2f} of the tolerance"
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("contexts,sizes,heads,kv_heads", [
    ([0], [1], 4, 1),
    ([1], [1], 4, 1),
    ([77], [7], 32, 8),
    ([128, 129, 127], [1, 1, 1], 8, 2),       # plain decoding
    ([500, 0, 1300], [4, 9, 2], 8, 2),
    ([300, 700], [33, 32], 4, 2),
    ([900], [64], 4, 1),
    ([260, 1000, 40], [64, 1, 17], 16, 2),    # larger trees than the average: several row parts
    ([640], [40], 7, 1),
    ([200], [64], 12, 1),                     # 768 rows: three row parts
    ([129] * 70, [1, 2, 3] * 23 + [5], 4, 2),  # many requests
])
def test_tree(gpu, dtype, contexts, sizes, heads, kv_heads):
    print(f"tree {contexts[:4]} {sizes[:4]} {heads}/{kv_heads} {dtype}", flush=True)
    keys, values, table = make_cache(contexts, kv_heads, dtype, seed=sum(sizes), stride_pages=len(sizes) == 2)
    offsets, mask = make_trees(sizes, 3)
    qkv = make_rows(int(offsets[-1]), heads + 2 * kv_heads, dtype, 4)
    check(gpu, qkv, heads, kv_heads, keys, values, table, contexts, offsets, mask, max(contexts))


def test_long_contexts_and_many_pages(gpu):
    """Contexts of more pages than one table block of 64, ending on either side of one."""
    contexts, sizes = [128 * 64, 128 * 64 + 1, 128 * 129 - 3], [3, 1, 2]
    keys, values, table = make_cache(contexts, 1, BF16, seed=13)
    offsets, mask = make_trees(sizes, 14)
    qkv = make_rows(6, 6, BF16, 15)
    check(gpu, qkv, 4, 1, keys, values, table, contexts, offsets, mask, max(contexts))
    # few workgroups and many pages each: contexts of one request far longer than the others'
    contexts, sizes = [30] * 6 + [128 * 150], [1] * 7
    keys, values, table = make_cache(contexts, 4, BF16, seed=16)
    offsets, mask = make_trees(sizes, 17)
    check(gpu, make_rows(7, 24, BF16, 18), 16, 4, keys, values, table, contexts, offsets, mask, max(contexts))


def test_masks_that_leave_nothing_and_values_nobody_attends(gpu):
    contexts, sizes = [0, 200, 0], [5, 6, 3]
    keys, values, table = make_cache(contexts, 2, BF16, seed=23)
    offsets, mask = make_trees(sizes, 24)
    mask[1] = 0                       # no context, no node: zeros
    mask[12] = -(1 << 63)             # only a bit past its tree's nodes: zeros
    mask[5] = mask[6] = 0             # the context alone
    mask[7:11] &= ~(1 << 3)
    qkv = make_rows(14, 12, BF16, 25)
    qkv[5 + 3, 8:] = float("nan")     # node 3 of request 1: nobody attends it
    qkv[5 + 4, 10:, 3] = float("inf")  # V of node 4 of request 1: those that attend it alone
    keys[table[1, 1].item(), 200 - 128:] = float("nan")
    values[table[1, 1].item(), 200 - 128:] = float("nan")
    got = check(gpu, qkv, 8, 2, keys, values, table, contexts, offsets, mask, 200)
    assert (got[1] == 0).all() and (got[12] == 0).all()


def test_padded_batches_and_bad_tables(gpu):
    """Requests without nodes, rows behind the last request, contexts past the table, pages that are none."""
    contexts, sizes = [300, 129, 5000, 400], [3, 0, 2, 4]
    keys, values, table = make_cache([300, 129, 256, 400], 2, FP16, seed=33)
    table[3, 1], table[3, 2] = -1, keys.shape[0]
    table[2, 2:] = -5
    offsets, mask = make_trees(sizes, 34)
    total = int(offsets[-1]) + 6
    mask = torch.cat([mask, torch.full((6,), -1, dtype=torch.int64)])
    qkv = make_rows(total, 8, FP16, 35)
    check(gpu, qkv, 4, 2, keys, values, table, contexts, offsets, mask, 700)
    # a tree of more than 64 nodes: the rows past them are left alone
    offsets = ints([0, 70])
    keys, values, table = make_cache([100], 2, FP16, seed=36)
    mask = torch.full((70,), -1, dtype=torch.int64)
    check(gpu, make_rows(70, 8, FP16, 37), 4, 2, keys, values, table, [100], offsets, mask, 200)


def test_a_tree_of_a_chain_is_a_causal_chunk(gpu):
    """A chain of drafts, then its accepted part written into the cache and decoded on: as the dense companion."""
    from trianglemix import cache, kernel

    print("tree then cache", flush=True)
    seq, nodes, heads, kv = 500, 9, 32, 8
    keys, values, table = make_cache([seq + 200], kv, BF16, seed=43)
    keys, values, table = keys.to(gpu), values.to(gpu), table.to(gpu)
    offsets, mask = ints([0, nodes], gpu), torch.tensor(TT.ancestor_masks(list(range(-1, nodes - 1))), device=gpu)
    qkv = make_rows(nodes, heads + 2 * kv, BF16, 44).to(gpu)
    got = TT.tree_attention(qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], keys, values, table,
                            ints([seq], gpu), offsets, mask, SCALE)
    slots = cache.chunk_slot_mapping(table, seq, nodes)
    slots[5:] = -1  # five drafts accepted
    cache.reshape_and_cache(qkv[:, heads:heads + kv], qkv[:, heads + kv:], keys, values, slots)
    dense = torch.empty(5, heads, 128, dtype=BF16, device=gpu)
    kernel.dense_paged_causal_attention(query=qkv[:5, :heads].contiguous(), key_cache=keys, value_cache=values,
                                        block_table=table, seq_len=seq + 5, output=dense, softmax_scale=SCALE)
    # both round the weights to bf16 and the result once: 4 half steps of values of up to 4 in all
    assert (got[:5].float() - dense.float()).abs().max() <= 4 * 2.0 ** -8 * 4


def test_captured_and_replayed_with_other_trees(gpu):
    print("tree graph", flush=True)
    kv, heads = 2, 8
    keys, values, table = make_cache([1400, 1300, 900], kv, BF16, seed=53)
    keys, values, table = keys.to(gpu), values.to(gpu), table.to(gpu)
    qkv = make_rows(24, heads + 2 * kv, BF16, 54).to(gpu)
    contexts, offsets = ints([1, 2, 3], gpu), ints([0, 1, 2, 3], gpu)
    mask = torch.zeros(24, dtype=torch.int64, device=gpu)
    out = torch.zeros(24, heads, 128, dtype=BF16, device=gpu)
    args = (qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], keys, values, table, contexts, offsets, mask,
            SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        TT.tree_attention(*args, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    pool = torch.cuda.graph_pool_handle()
    for graph in graphs:  # of one pool: their workspaces may lie in the same memory
        with torch.cuda.graph(graph, pool=pool):
            TT.tree_attention(*args, out=out)
    for n, (lens, sizes) in enumerate([([1400, 1300, 900], [8, 8, 8]), ([5, 1200, 0], [1, 20, 3]),
                                       ([0, 0, 900], [0, 0, 4]), ([1400, 1300, 900], [8, 8, 8])]):
        o, m = make_trees(sizes, 60 + n)
        contexts.copy_(ints(lens))
        offsets.copy_(o)
        mask.zero_()
        mask[:len(m)] = m.to(gpu)
        for graph in graphs:
            out.fill_(3.0)
            graph.replay()
            torch.cuda.synchronize()
            eager = torch.full_like(out, 3.0)
            TT.tree_attention(*args, out=eager)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), (n, lens)
            assert (out[sum(sizes):] == 3.0).all()
