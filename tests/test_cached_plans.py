"""The launch plans of attention over a cache, on the CPU, by the workspaces that they ask for."""

from __future__ import annotations

import itertools

import pytest
from test_boundary_abi import lib  # noqa: F401  (fixture)


@pytest.mark.parametrize("batch,rows,heads,kv_heads,cols", [
    (1, 4096, 12, 3, 64), (2, 8192, 3, 3, 256), (3, 3000, 6, 3, 1024), (1, 2048, 28, 7, 64), (1, 1024, 48, 12, 64),
    (2, 4096, 6, 3, 16)])
def test_a_round_of_the_gpu_counts_whatever_the_kv_heads(lib, batch, rows, heads, kv_heads, cols):  # noqa: F811
    """Chunks whose parts of 256 rows fit one round of 256 workgroups: halves of them take a round and a rest.

    The halves' first round is one where the KV heads divide no 256 too: the parts are taken, unshared.
    """
    tokens = 256 // (heads // kv_heads)
    assert batch * -(-rows // tokens) * kv_heads <= 256 < batch * -(-rows // (tokens // 2)) * kv_heads
    assert lib.tm_cached_attention_workspace_size(batch, rows, heads, kv_heads, cols, -1, 0) == 0


def test_no_workspace_is_larger_than_stated(lib):  # noqa: F811
    """64 MiB of records and 64 KiB of arrival words, at batches around the largest that is shared out too."""
    size = lib.tm_cached_attention_workspace_size
    most = (64 << 20) + 65536
    assert 0 <= size(315, 30, 12, 12, 64, -1, 0) <= most and 0 <= size(945, 30, 4, 4, 1, -1, 0) <= most
    largest = 0
    for rows, (heads, kv_heads), cols in itertools.product(
            (1, 2, 5, 8, 13, 16, 17, 30, 32, 33, 64), ((4, 4), (8, 2), (12, 12), (32, 8), (20, 5), (64, 64), (28, 7), (32, 1)),
            (1, 4, 64, 16384)):
        for batch in range(1, 1025, 3):
            largest = max(largest, size(batch, rows, heads, kv_heads, cols, -1, 0))
    assert largest <= most
    assert largest > most * 0.99  # the range reaches it
