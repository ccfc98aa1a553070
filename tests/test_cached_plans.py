"""The launch plans of attention over a cache, on the CPU, by the workspaces that they ask for."""

from __future__ import annotations

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
