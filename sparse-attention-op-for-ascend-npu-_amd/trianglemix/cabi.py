"""ctypes binding of the C ABI in ``include/trianglemix.h`` and ``include/trianglemix_pages.h``.

For callers that do not go through ``torch.ops`` (and for the parity tests,
which exercise the C boundary directly).  Tensors are only used for their
device pointers; the launch goes on the given stream (default: torch's
current stream of the query's device).
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext

from .native import load_hip_library

TM_OK = 0
TM_ERR_INVALID_ARGUMENT = 1
TM_ERR_UNSUPPORTED = 2
TM_ERR_WORKSPACE = 3
TM_ERR_LAUNCH = 4


class TriangleMixError(RuntimeError):
    def __init__(self, status: int, message: str) -> None:
        super().__init__(f"{message} (status {status})")
        self.status = status


def _check(status: int) -> None:
    if status != TM_OK:
        lib = load_hip_library()
        raise TriangleMixError(status, lib.tm_last_error().decode() or lib.tm_status_string(status).decode())


def _stream(query, stream):
    if stream is not None:
        return int(stream)
    import torch

    return torch.cuda.current_stream(query.device).cuda_stream


def workspace_size(query_tokens: int, query_start: int, seq_len: int, prompt_len: int | None) -> int:
    lib = load_hip_library()
    if prompt_len is None:
        n = lib.tm_dense_paged_causal_attention_workspace_size(query_tokens, query_start, seq_len)
    else:
        n = lib.tm_triangle_paged_sparse_attention_workspace_size(query_tokens, query_start, seq_len, prompt_len)
    if n < 0:
        raise TriangleMixError(TM_ERR_INVALID_ARGUMENT, lib.tm_last_error().decode())
    return int(n)


def chunk_plan(query_tokens: int, query_start: int, seq_len: int, prompt_len: int | None) -> tuple[int, int, int]:
    """(KV parts, tiles per work item, work items per KV head) the launch uses for this chunk geometry;
    ``prompt_len`` None plans the dense companion."""
    lib = load_hip_library()
    parts, tiles, items = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int64()
    dense = prompt_len is None
    status = lib.tm_chunk_plan(int(dense), query_tokens, query_start, seq_len, 0 if dense else prompt_len,
                               ctypes.byref(parts), ctypes.byref(tiles), ctypes.byref(items))
    _check(status)
    return parts.value, tiles.value, items.value


# Split-KV workspace per (device, stream), at most MAX_WORKSPACE_BYTES (the
# paged serving operators' may be 2.1 MiB larger).  Its
# contents before a call do not matter (the library tags every arrival word
# for its workspace), so a buffer is never cleared.  One buffer is kept per
# (device, stream), allocated on that stream; a call that needs more replaces
# it, and PyTorch's caching allocator hands the old buffer's memory out again
# only in that stream's order, after the work queued on it.  Under stream
# capture every call takes a buffer of its own from the graph's pool, so no
# graph depends on a buffer that is replaced here or shares it with another.
WORKSPACE_COUNTER_BYTES = 65536
MAX_WORKSPACE_BYTES = 64 << 20
_WORKSPACES: dict = {}


def _workspace(query, query_start, seq_len, prompt_len, workspace, stream):
    return _workspace_of(query, workspace_size(query.shape[0], query_start, seq_len, prompt_len), workspace, stream)


def _workspace_of(query, need, workspace, stream):
    """(buffer, pointer, bytes).  The caller keeps the buffer until its launch is enqueued: another thread's call
    may replace the one that is kept for the stream meanwhile, and its memory would go to whoever asks next."""
    if need == 0:
        return None, None, 0
    if workspace is None and _capturing(query, stream):
        workspace = _buffer(query, need, stream)  # from the graph's own pool, which it keeps for its replays
    if workspace is None:
        key = (query.device.index, int(stream))
        held = _WORKSPACES.get(key)
        if held is None or held.numel() < need:
            _WORKSPACES.pop(key, None)
            held = _WORKSPACES[key] = _buffer(query, need, stream)
        workspace = held
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _on(query, stream):
    """Makes the stream of the query's device torch's current one, if it is not."""
    import torch

    if query.device.index == torch.cuda.current_device() and int(stream) == torch.cuda.current_stream().cuda_stream:
        return nullcontext()
    return torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=query.device))


def _capturing(query, stream) -> bool:
    if not query.is_cuda:
        return False
    status = ctypes.c_int()
    # of the HIP runtime that the library is linked to; asking through torch takes several microseconds more
    if load_hip_library().hipStreamIsCapturing(ctypes.c_void_p(int(stream)), ctypes.byref(status)) != 0:
        raise TriangleMixError(TM_ERR_LAUNCH, "hipStreamIsCapturing failed")
    return status.value != 0


def _buffer(query, need, stream):
    """Memory of the caching allocator that is handed out again in this stream's order."""
    import torch

    with _on(query, stream):
        return torch.empty(need, dtype=torch.uint8, device=query.device)


def triangle_paged_sparse_attention(query, key_cache, value_cache, block_table, out, *, query_start: int,
                                    seq_len: int, prompt_len: int, scale: float, stream=None,
                                    workspace=None) -> None:
    lib = load_hip_library()
    st = _stream(query, stream)
    _held, ws_ptr, ws_bytes = _workspace(query, query_start, seq_len, prompt_len, workspace, st)
    _check(lib.tm_triangle_paged_sparse_attention(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr(), out.data_ptr(),
        query.shape[0], key_cache.shape[0], block_table.shape[-1], query_start, seq_len, prompt_len,
        float(scale), ws_ptr, ws_bytes, st))


def triangle_paged_sparse_attention_noalloc(query, key_cache, value_cache, block_table, out, *, query_start: int,
                                            seq_len: int, prompt_len: int, scale: float, stream=None) -> None:
    """The no-allocation entry point: split-KV scratch from the library's static per-GPU array."""
    lib = load_hip_library()
    st = _stream(query, stream)
    _check(lib.tm_triangle_paged_sparse_attention_noalloc(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr(), out.data_ptr(),
        query.shape[0], key_cache.shape[0], block_table.shape[-1], query_start, seq_len, prompt_len,
        float(scale), st))


def dense_paged_causal_attention(query, key_cache, value_cache, block_table, out, *, query_start: int,
                                 seq_len: int, scale: float, stream=None, workspace=None) -> None:
    lib = load_hip_library()
    st = _stream(query, stream)
    _held, ws_ptr, ws_bytes = _workspace(query, query_start, seq_len, None, workspace, st)
    _check(lib.tm_dense_paged_causal_attention(
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr(), out.data_ptr(),
        query.shape[0], key_cache.shape[0], block_table.shape[-1], query_start, seq_len,
        float(scale), ws_ptr, ws_bytes, st))


def reshape_and_cache(key, value, key_cache, value_cache, slot_mapping, *, stream=None) -> None:
    """Scatter key / value rows ``[T, 8, 128]`` (row-strided views allowed) into cache slots.

    Token ``i`` goes to page ``slot_mapping[i] // 128``, offset ``slot_mapping[i] % 128``
    (int64); negative slots are padding and are skipped.
    """
    lib = load_hip_library()
    st = _stream(key, stream)
    _check(lib.tm_reshape_and_cache(
        key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.data_ptr(),
        key.shape[0], key.stride(0), value.stride(0), key_cache.shape[0], st))


def _dtype(tensor) -> int:
    import torch

    return {torch.bfloat16: 0, torch.float16: 1}.get(tensor.dtype, -1)  # TM_BF16, TM_FP16


def _need(size, *geometry) -> int:
    n = size(*geometry)
    if n < 0:
        raise TriangleMixError(TM_ERR_INVALID_ARGUMENT, load_hip_library().tm_last_error().decode())
    return int(n)


def _rows_per_request(query, batch: int) -> int:
    if query.shape[0] % max(batch, 1) or (batch == 0 and query.shape[0]):
        raise TriangleMixError(TM_ERR_INVALID_ARGUMENT, "query must hold the same number of rows for each request")
    return query.shape[0] // max(batch, 1)


def update_page_bounds(key_cache, block_table, seq_lens, num_tokens: int, page_min, page_max, *, stream=None) -> None:
    """``pages.update_page_bounds`` through the C ABI."""
    lib = load_hip_library()
    _check(lib.tm_update_page_bounds(
        key_cache.data_ptr(), key_cache.stride(0), block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(),
        num_tokens, page_min.data_ptr(), page_max.data_ptr(), block_table.shape[0], block_table.shape[1],
        key_cache.shape[0], key_cache.shape[2], _dtype(key_cache), _stream(key_cache, stream)))


def select_pages(query, page_min, page_max, block_table, seq_lens, out, *, sink_pages: int = 1, recent_pages: int = 1,
                 stream=None, workspace=None) -> None:
    """``pages.select_pages`` through the C ABI; ``out`` holds the count."""
    lib = load_hip_library()
    st = _stream(query, stream)
    (batch, cols), heads, kv = block_table.shape, query.shape[1], page_min.shape[1]
    rows = _rows_per_request(query, batch)
    need = _need(lib.tm_select_pages_workspace_size, batch, rows, heads, kv, cols)
    if workspace is None and need > 0:
        import torch

        # scores that one launch of the call leaves for the next: out of reach of other threads' calls on the stream
        workspace = _buffer(query, need, st) if stream is not None else query.new_empty(need, dtype=torch.uint8)
    _held, ws_ptr, ws_bytes = _workspace_of(query, need, workspace, st)
    _check(lib.tm_select_pages(
        query.data_ptr(), query.stride(0), page_min.data_ptr(), page_max.data_ptr(), block_table.data_ptr(),
        block_table.stride(0), seq_lens.data_ptr(), out.data_ptr(), batch, rows, heads, kv, cols, page_min.shape[0],
        out.shape[-1], sink_pages, recent_pages, _dtype(query), ws_ptr, ws_bytes, st))


def selected_page_attention(query, key_cache, value_cache, block_table, seq_lens, pages, out, *, scale: float,
                            stream=None, workspace=None) -> None:
    """``pages.selected_page_attention`` through the C ABI."""
    lib = load_hip_library()
    st = _stream(query, stream)
    (batch, cols), heads, kv, count = block_table.shape, query.shape[1], key_cache.shape[2], pages.shape[-1]
    rows = _rows_per_request(query, batch)
    need = _need(lib.tm_selected_page_attention_workspace_size, batch, rows, heads, kv, count)
    _held, ws_ptr, ws_bytes = _workspace_of(query, need, workspace, st)
    _check(lib.tm_selected_page_attention(
        query.data_ptr(), query.stride(0), key_cache.data_ptr(), key_cache.stride(0), value_cache.data_ptr(),
        value_cache.stride(0), block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(), pages.data_ptr(),
        out.data_ptr(), batch, rows, heads, kv, cols, key_cache.shape[0], count, float(scale), _dtype(query), ws_ptr,
        ws_bytes, st))


def tree_attention(query, key, value, key_cache, value_cache, block_table, context_lens, tree_offsets, tree_mask, out, *,
                   scale: float, stream=None, workspace=None) -> None:
    """``tree.tree_attention`` through the C ABI."""
    lib = load_hip_library()
    st = _stream(query, stream)
    (batch, cols), (total, heads), kv = block_table.shape, query.shape[:2], key_cache.shape[2]
    need = _need(lib.tm_tree_attention_workspace_size, total, batch, heads, kv, cols)
    _held, ws_ptr, ws_bytes = _workspace_of(query, need, workspace, st)
    _check(lib.tm_tree_attention(
        query.data_ptr(), query.stride(0), key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0),
        key_cache.data_ptr(), key_cache.stride(0), value_cache.data_ptr(), value_cache.stride(0),
        block_table.data_ptr(), block_table.stride(0), context_lens.data_ptr(), tree_offsets.data_ptr(),
        tree_mask.data_ptr(), out.data_ptr(), total, batch, heads, kv, cols, key_cache.shape[0], float(scale),
        _dtype(query), ws_ptr, ws_bytes, st))
