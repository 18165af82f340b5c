"""Host-side API over libqkv.so for torch device tensors.

Mirrors the reference's append and attention launches (src/model.cuh call
sites) with torch tensors as the device-memory container.  Every function
calls the gfx950 HIP kernels through the C ABI; there is no CPU path.

Cache tensors are uint8 tensors whose last dimension is the block size
(52 bytes per TQ3 block, 36 bytes per Q8 block); fp16 tensors are
torch.float16.  Calls are ordered on the current torch stream.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import bench_lib, check, lib

TQ3_BLOCK_BYTES = 52
Q8_BLOCK_BYTES = 36


def _stream(stream=None) -> int:
    """The raw stream of `stream`, or of the current stream of the current device
    (looked up as an integer: a torch.cuda.Stream object costs 2.7 us of a call's
    host time, as much as a kernel launch)."""
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


# fp16 arguments: torch.float16, or 16-bit integer tensors holding fp16 bit
# patterns (the C ABI takes uint16_t)
FP16 = (torch.float16, torch.uint16, torch.int16)


def _need(t, nbytes: int, what: str, dtype=None) -> None:
    """Raise ValueError (before any launch) when `t` is not of `dtype` or
    holds fewer than `nbytes` bytes: the kernels trust the sizes implied by
    the shape arguments, so an undersized buffer would be read or written
    out of bounds on the device."""
    if t is None:
        raise ValueError(f"{what} is required")
    allowed = dtype if isinstance(dtype, tuple) else (dtype,)
    if dtype is not None and t.dtype not in allowed:
        raise ValueError(f"{what} must be {' or '.join(str(d) for d in allowed)}, got {t.dtype}")
    have = t.numel() * t.element_size()
    if have < nbytes:
        raise ValueError(f"{what} holds {have} bytes, the call needs {int(nbytes)}")


def _dev_ptr(t: torch.Tensor, what: str) -> int:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr()


def _scratch(n_bytes, device, stream) -> torch.Tensor:
    """Scratch of a call on `stream` (the current one when None), out of that stream's memory: a block of
    another stream's may still be written by work under way there."""
    n = max(1, n_bytes // 4)
    if stream is None:
        return torch.empty(n, dtype=torch.int32, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(n, dtype=torch.int32, device=device)


def _result(n, device, stream) -> torch.Tensor:
    """n fp16 numbers that a call on `stream` writes and its caller uses on the current stream: out of the
    memory of the former, and kept until the latter is done with them."""
    if stream is None:
        return torch.empty(n, dtype=torch.float16, device=device)
    with torch.cuda.stream(stream):
        t = torch.empty(n, dtype=torch.float16, device=device)
    t.record_stream(torch.cuda.current_stream(device))
    return t


def tq3_blocks(n_blocks: int, device) -> torch.Tensor:
    """Zero-initialised TQ3 block storage [n_blocks, 52] (model.cuh:1914-1920)."""
    return torch.zeros((n_blocks, TQ3_BLOCK_BYTES), dtype=torch.uint8, device=device)


def q8_blocks(n_blocks: int, device) -> torch.Tensor:
    return torch.zeros((n_blocks, Q8_BLOCK_BYTES), dtype=torch.uint8, device=device)


def tq3_init(device: int = 0) -> None:
    check(lib().qkv_tq3_init(device), "qkv_tq3_init")


def tq3_append(x: torch.Tensor, out: torch.Tensor, stream=None) -> None:
    """turboquant.cuh:112-165.  x: fp16 [..., 128*k]; out: uint8 blocks [n, 52]."""
    assert x.dtype == torch.float16
    n = x.numel() // 128
    assert x.numel() == n * 128 and out.numel() >= n * TQ3_BLOCK_BYTES
    check(lib().qkv_tq3_append(_dev_ptr(x, "x"), _dev_ptr(out, "out"), n, _stream(stream)),
          "qkv_tq3_append")


def tq3_append_kv(k: torch.Tensor, v: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor,
                  stream=None) -> None:
    assert k.dtype == torch.float16 and v.dtype == torch.float16 and k.numel() == v.numel()
    n = k.numel() // 128
    check(lib().qkv_tq3_append_kv(_dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(k_out, "k_out"),
                                  _dev_ptr(v_out, "v_out"), n, _stream(stream)),
          "qkv_tq3_append_kv")


def tq3_dequant(blocks: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """turboquant.cuh:169-200.  Returns fp16 [n_blocks*128]."""
    n = blocks.numel() // TQ3_BLOCK_BYTES
    if out is None:
        out = _result(n * 128, blocks.device, stream)
    check(lib().qkv_tq3_dequant(_dev_ptr(blocks, "blocks"), _dev_ptr(out, "out"), n,
                                _stream(stream)), "qkv_tq3_dequant")
    return out


def q8_append(x: torch.Tensor, out: torch.Tensor, stream=None) -> None:
    """attention.cuh:2587-2609.  x: fp16 [..., 32*k]; out: uint8 blocks [n, 36]."""
    assert x.dtype == torch.float16
    n = x.numel() // 32
    assert x.numel() == n * 32 and out.numel() >= n * Q8_BLOCK_BYTES
    check(lib().qkv_q8_append(_dev_ptr(x, "x"), _dev_ptr(out, "out"), n, _stream(stream)),
          "qkv_q8_append")


def q8_append_kv(k: torch.Tensor, v: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor,
                 stream=None) -> None:
    """K and V in one launch (the two quantize_kv_q8_0_kern launches of
    model.cuh:2316-2333)."""
    assert k.dtype == torch.float16 and v.dtype == torch.float16 and k.numel() == v.numel()
    n = k.numel() // 32
    assert k.numel() == n * 32
    assert k_out.numel() >= n * Q8_BLOCK_BYTES and v_out.numel() >= n * Q8_BLOCK_BYTES
    check(lib().qkv_q8_append_kv(_dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(k_out, "k_out"),
                                 _dev_ptr(v_out, "v_out"), n, _stream(stream)),
          "qkv_q8_append_kv")


def q8_dequant(blocks: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """attention.cuh:2614-2626."""
    n = blocks.numel() // Q8_BLOCK_BYTES
    if out is None:
        out = _result(n * 32, blocks.device, stream)
    check(lib().qkv_q8_dequant(_dev_ptr(blocks, "blocks"), _dev_ptr(out, "out"), n,
                               _stream(stream)), "qkv_q8_dequant")
    return out


def kv_move_tokens(k: torch.Tensor, v: torch.Tensor, moves, *, k_row_bytes: int,
                   v_row_bytes: int, slot_row0: int = 0, slot_rows: int | None = None,
                   stream=None) -> None:
    """kv_move_token (model.cuh:7430-7471) for a list of (from_pos, to_pos)
    moves of one layer, applied in list order, in one launch."""
    import ctypes
    moves = list(moves)
    if slot_rows is None:
        slot_rows = k.numel() // k_row_bytes - slot_row0
    flat = (ctypes.c_int32 * max(1, 2 * len(moves)))(*[int(x) for m in moves for x in m])
    check(lib().qkv_kv_move_tokens(_dev_ptr(k, "k"), _dev_ptr(v, "v"), k_row_bytes, v_row_bytes,
                                   slot_row0, slot_rows, ctypes.cast(flat, ctypes.c_void_p),
                                   len(moves), _stream(stream)), "qkv_kv_move_tokens")


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _pool_rows(k_pool, v_pool, k_row_bytes, v_row_bytes):
    rows = k_pool.numel() * k_pool.element_size() // k_row_bytes
    if v_pool is not None:
        rows = min(rows, v_pool.numel() * v_pool.element_size() // v_row_bytes)
    return rows


def _flat_sizes(k_flat, v_flat, v_pool, n_rows, k_row_bytes, v_row_bytes, block_table,
                block_tokens) -> None:
    """The flat buffers hold n_rows rows and the table covers them."""
    _need(k_flat, n_rows * k_row_bytes, "k_flat")
    if v_pool is not None or v_flat is not None:
        _need(v_flat, n_rows * v_row_bytes, "v_flat")
    if block_tokens > 0:
        _need(block_table, -(-n_rows // block_tokens) * 4, "block_table", torch.int32)


def kv_gather_rows(k_pool, v_pool, k_flat, v_flat, block_table, *, n_rows, block_tokens,
                   k_row_bytes, v_row_bytes=0, stream=None) -> None:
    """Slot snapshot over a paged pool: logical rows 0 .. n_rows-1 of the slot
    whose block-table row is `block_table` (int32 device tensor) into the flat
    buffers [n_rows][row_bytes] (model.cuh:3394-3417 for the contiguous
    layout).  v_pool / v_flat may be None (keys only)."""
    _flat_sizes(k_flat, v_flat, v_pool, n_rows, k_row_bytes, v_row_bytes, block_table, block_tokens)
    pool_rows = _pool_rows(k_pool, v_pool, k_row_bytes, v_row_bytes)
    check(lib().qkv_kv_gather_rows(
        _dev_ptr(k_pool, "k_pool"), _opt_ptr(v_pool), _dev_ptr(k_flat, "k_flat"),
        _opt_ptr(v_flat), k_row_bytes, v_row_bytes, pool_rows,
        _i32(block_table, "block_table"), block_table.numel(),
        block_tokens, n_rows, _stream(stream)), "qkv_kv_gather_rows")


def kv_scatter_rows(k_pool, v_pool, k_flat, v_flat, block_table, *, n_rows, block_tokens,
                    k_row_bytes, v_row_bytes=0, stream=None) -> None:
    """Slot restore over a paged pool: the inverse of kv_gather_rows
    (model.cuh:3314-3335 for the contiguous layout)."""
    _flat_sizes(k_flat, v_flat, v_pool, n_rows, k_row_bytes, v_row_bytes, block_table, block_tokens)
    pool_rows = _pool_rows(k_pool, v_pool, k_row_bytes, v_row_bytes)
    check(lib().qkv_kv_scatter_rows(
        _dev_ptr(k_pool, "k_pool"), _opt_ptr(v_pool), _dev_ptr(k_flat, "k_flat"),
        _opt_ptr(v_flat), k_row_bytes, v_row_bytes, pool_rows,
        _i32(block_table, "block_table"), block_table.numel(),
        block_tokens, n_rows, _stream(stream)), "qkv_kv_scatter_rows")


def dfk2_dequant(q, scales, out, *, kv_dim, stream=None) -> None:
    """dfki2_dequant_kernel (model.cuh:149-159): int8 plane rows with
    group-128 fp16 scales to fp16."""
    check(lib().qkv_dfk2_dequant(_dev_ptr(q, "q"), _dev_ptr(scales, "scales"),
                                 _dev_ptr(out, "out"), q.numel(), kv_dim, _stream(stream)),
          "qkv_dfk2_dequant")


def tq3_append_dfk2(q, scales, out, stream=None) -> None:
    """KV-inject re-quantization into TQ3 (model.cuh:3189-3192 + 3218-3226 in
    one launch): block i from q[128 i ..] with scale scales[i]."""
    check(lib().qkv_tq3_append_dfk2(_dev_ptr(q, "q"), _dev_ptr(scales, "scales"),
                                    _dev_ptr(out, "out"), q.numel() // 128, _stream(stream)),
          "qkv_tq3_append_dfk2")


def q8_append_dfk2(q, scales, out, stream=None) -> None:
    """KV-inject re-quantization into Q8_0 (model.cuh:3189-3192 + 3227-3233):
    32-element block i with scale scales[i // 4]."""
    check(lib().qkv_q8_append_dfk2(_dev_ptr(q, "q"), _dev_ptr(scales, "scales"),
                                   _dev_ptr(out, "out"), q.numel() // 32, _stream(stream)),
          "qkv_q8_append_dfk2")


def hbm_read_bench(buf, sink, stream=None) -> None:
    """One streaming read of the whole tensor `buf` (bandwidth measurement;
    libqkv_bench.so, not the product library)."""
    check(bench_lib().qkv_hbm_read_bench(_dev_ptr(buf, "buf"), buf.numel() * buf.element_size(),
                                   _dev_ptr(sink, "sink"), _stream(stream)), "qkv_hbm_read_bench")


def mfma_rate_bench(workgroups, iters, sink, stream=None) -> None:
    """One launch of the MFMA-rate loop (workgroups x 8 waves x 16 * iters
    32x32x16 fp16 MFMAs on data-like operands; libqkv_bench.so)."""
    check(bench_lib().qkv_mfma_rate_bench(int(workgroups), int(iters), _dev_ptr(sink, "sink"),
                                          _stream(stream)), "qkv_mfma_rate_bench")


def _opt_ptr(t):
    return 0 if t is None else _dev_ptr(t, "tensor")


def attn_split_tq3(q, k, v, part_m, part_l, part_o, *, num_q, num_kv, start_pos, sub_n,
                   sub_n_max, active_end_max, scale, k_splits, sink_tok=0, window_tok=0,
                   tree_mask=None, head_dim=256, stream=None) -> None:
    """attention.cuh:1905-2177: unnormalised split partials, reference layout."""
    check(lib().qkv_attn_split_tq3(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(part_m, "part_m"),
        _dev_ptr(part_l, "part_l"), _dev_ptr(part_o, "part_o"), num_q, num_kv, head_dim,
        start_pos, sub_n, sub_n_max, active_end_max, float(scale), k_splits, sink_tok,
        window_tok, _opt_ptr(tree_mask), _stream(stream)), "qkv_attn_split_tq3")


def attn_split_q8(q, k, v, part_m, part_l, part_o, *, num_q, num_kv, start_pos, sub_n,
                  sub_n_max, active_end_max, scale, k_splits, head_dim=256, stream=None) -> None:
    """attention.cuh:2633-2801: unnormalised split partials over the Q8_0 cache."""
    check(lib().qkv_attn_split_q8(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(part_m, "part_m"),
        _dev_ptr(part_l, "part_l"), _dev_ptr(part_o, "part_o"), num_q, num_kv, head_dim,
        start_pos, sub_n, sub_n_max, active_end_max, float(scale), k_splits, _stream(stream)),
        "qkv_attn_split_q8")


def attn_split_merge(part_m, part_l, part_o, out, *, num_q, num_kv, sub_n, sub_n_max, k_splits,
                     head_dim=256, stream=None) -> None:
    """attention.cuh:1837-1891."""
    check(lib().qkv_attn_split_merge(
        _dev_ptr(part_m, "part_m"), _dev_ptr(part_l, "part_l"), _dev_ptr(part_o, "part_o"),
        _dev_ptr(out, "out"), num_q, num_kv, head_dim, sub_n, sub_n_max, k_splits,
        _stream(stream)), "qkv_attn_split_merge")


def tq3_kpool_update(k_cache, k_pool, k_pool_max, *, num_kv, total_kv, blk_lo, block_size_n=64,
                     head_dim=256, stream=None) -> None:
    """Block signatures of the TQ3 keys (attention.cuh:2445-2533): pools are
    fp16 tensors [num_kv][n_blocks_stride][256]; blocks blk_lo ..
    ceil(total_kv / block_size_n) - 1 are rebuilt."""
    check(lib().qkv_tq3_kpool_update(
        _dev_ptr(k_cache, "k_cache"), _dev_ptr(k_pool, "k_pool"), _dev_ptr(k_pool_max, "k_pool_max"),
        num_kv, head_dim, total_kv, blk_lo, k_pool.shape[1], block_size_n, _stream(stream)),
        "qkv_tq3_kpool_update")


def block_index_ms(q, k_pool, k_pool_max, block_index, *, num_q, num_kv, sub_n, start_pos,
                   top_k, n_blocks, block_size_n=64, beta=0.5, head_dim=256, workspace=None,
                   stream=None) -> None:
    """Top-k block selection (sparse_attn/sparse_index.cuh:214-330) into the
    int32 tensor block_index [num_kv][sub_n_max][top_k]; the block scores pass
    through `workspace` (allocated here when None)."""
    if workspace is None:
        n = int(lib().qkv_block_index_ms_workspace_bytes(num_kv, sub_n, n_blocks))
        workspace = _scratch(max(n, 256), block_index.device, stream)
    check(lib().qkv_block_index_ms(
        _dev_ptr(q, "q"), _dev_ptr(k_pool, "k_pool"), _dev_ptr(k_pool_max, "k_pool_max"),
        _i32(block_index, "block_index"), num_q, num_kv, head_dim, sub_n, block_index.shape[1],
        start_pos, top_k, block_size_n, n_blocks, k_pool.shape[1], float(beta),
        _dev_ptr(workspace, "workspace"), workspace.numel() * workspace.element_size(),
        _stream(stream)), "qkv_block_index_ms")


def attn_block_sparse_split_tq3(q, k, v, block_index, part_m, part_l, part_o, *, num_q, num_kv,
                                start_pos, sub_n, sub_n_max, scale, top_k, k_splits,
                                block_size_n=64, tree_mask=None, head_dim=256,
                                stream=None) -> None:
    """attention.cuh:2193-2433: split partials over each query's selected blocks."""
    check(lib().qkv_attn_block_sparse_split_tq3(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _i32(block_index, "block_index"),
        _dev_ptr(part_m, "part_m"), _dev_ptr(part_l, "part_l"), _dev_ptr(part_o, "part_o"),
        num_q, num_kv, head_dim, start_pos, sub_n, sub_n_max, float(scale), top_k, block_size_n,
        k_splits, _opt_ptr(tree_mask), _stream(stream)), "qkv_attn_block_sparse_split_tq3")


# bytes per token row and kv head of one cache (head_dim 256): TQ3 two 52-byte
# blocks, Q8_0 eight 36-byte blocks
TQ3_ROW = 2 * TQ3_BLOCK_BYTES
Q8_ROW = 8 * Q8_BLOCK_BYTES


def _attn_sizes(q, k, v, out, num_q, num_kv, n_keys, sub_n, head_dim, k_row, v_row) -> None:
    """q / out hold sub_n x num_q fp16 rows; k / v hold n_keys token rows."""
    _need(q, sub_n * num_q * head_dim * 2, "q", FP16)
    _need(out, sub_n * num_q * head_dim * 2, "out", FP16)
    _need(k, n_keys * num_kv * k_row, "k")
    _need(v, n_keys * num_kv * v_row, "v")


def decode_attn_tq3_workspace_bytes(num_q, num_kv, sub_n, n_keys) -> int:
    return int(lib().qkv_decode_attn_tq3_workspace_bytes(num_q, num_kv, sub_n, n_keys))


def decode_attn_tq3_workspace(num_q, num_kv, sub_n, n_keys, device) -> torch.Tensor:
    """Zero-filled workspace for decode_attn_tq3 (the kernel keeps it zeroed)."""
    n = decode_attn_tq3_workspace_bytes(num_q, num_kv, sub_n, n_keys)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def decode_attn_tq3(q, k, v, out, workspace, *, num_q, num_kv, start_pos, sub_n, scale,
                    sink_tok=0, window_tok=0, tree_mask=None, head_dim=256, stream=None) -> None:
    """Fast path: split-K decode and its merge in one call."""
    _attn_sizes(q, k, v, out, num_q, num_kv, start_pos + sub_n, sub_n, head_dim, TQ3_ROW, TQ3_ROW)
    check(lib().qkv_decode_attn_tq3(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(out, "out"), num_q,
        num_kv, head_dim, start_pos, sub_n, float(scale), sink_tok, window_tok,
        _opt_ptr(tree_mask), _dev_ptr(workspace, "workspace"),
        workspace.numel() * workspace.element_size(), _stream(stream)), "qkv_decode_attn_tq3")


def decode_attn_tq3_append(q, k_new, v_new, k, v, out, workspace, *, num_q, num_kv, start_pos,
                           sub_n, scale, sink_tok=0, window_tok=0, tree_mask=None, head_dim=256,
                           stream=None) -> None:
    """decode_attn_tq3 of a block of sub_n new tokens whose K / V rows (fp16
    [sub_n][num_kv][256]) are appended in the same call: encoded into rows
    start_pos .. start_pos + sub_n - 1 of k / v (inside the decode launch for one
    query, and with more than 16 query-head columns).  k and v must hold those rows."""
    _attn_sizes(q, k, v, out, num_q, num_kv, start_pos + sub_n, sub_n, head_dim, TQ3_ROW, TQ3_ROW)
    _need(k_new, sub_n * num_kv * head_dim * 2, "k_new", FP16)
    _need(v_new, sub_n * num_kv * head_dim * 2, "v_new", FP16)
    check(lib().qkv_decode_attn_tq3_append(
        _dev_ptr(q, "q"), _dev_ptr(k_new, "k_new"), _dev_ptr(v_new, "v_new"), _dev_ptr(k, "k"),
        _dev_ptr(v, "v"), _dev_ptr(out, "out"), num_q, num_kv, head_dim, start_pos, sub_n,
        float(scale), sink_tok, window_tok, _opt_ptr(tree_mask), _dev_ptr(workspace, "workspace"),
        workspace.numel() * workspace.element_size(), _stream(stream)), "qkv_decode_attn_tq3_append")


def decode_attn_tq3_noalloc(q, k, v, out, *, num_q, num_kv, start_pos, sub_n, scale,
                            sink_tok=0, window_tok=0, tree_mask=None, head_dim=256,
                            stream=None) -> None:
    """decode_attn_tq3 without a workspace argument: the library's fixed
    per-GPU scratch serves as the workspace (no allocation in the call)."""
    _attn_sizes(q, k, v, out, num_q, num_kv, start_pos + sub_n, sub_n, head_dim, TQ3_ROW, TQ3_ROW)
    check(lib().qkv_decode_attn_tq3_noalloc(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(out, "out"), num_q,
        num_kv, head_dim, start_pos, sub_n, float(scale), sink_tok, window_tok,
        _opt_ptr(tree_mask), _stream(stream)), "qkv_decode_attn_tq3_noalloc")


def decode_attn_q8_workspace(num_q, num_kv, sub_n, n_keys, device) -> torch.Tensor:
    """Zero-filled workspace for decode_attn_q8."""
    n = int(lib().qkv_decode_attn_q8_workspace_bytes(num_q, num_kv, sub_n, n_keys))
    return torch.zeros(n, dtype=torch.uint8, device=device)


def decode_attn_q8(q, k, v, out, workspace, *, num_q, num_kv, start_pos, sub_n, scale,
                   head_dim=256, stream=None) -> None:
    """Fast path over the Q8_0 cache: split-K decode with the merge inside the
    same launch."""
    _attn_sizes(q, k, v, out, num_q, num_kv, start_pos + sub_n, sub_n, head_dim, Q8_ROW, Q8_ROW)
    check(lib().qkv_decode_attn_q8(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(out, "out"), num_q,
        num_kv, head_dim, start_pos, sub_n, float(scale), _dev_ptr(workspace, "workspace"),
        workspace.numel() * workspace.element_size(), _stream(stream)), "qkv_decode_attn_q8")


def decode_attn_q8_append(q, k_new, v_new, k, v, out, workspace, *, num_q, num_kv, start_pos,
                          scale, head_dim=256, stream=None) -> None:
    """One launch for a decode step over the Q8_0 cache: k_new / v_new (fp16
    [num_kv][256]) are quantized into row start_pos of k / v and attended as
    key start_pos by the one query q (keys 0..start_pos).  k and v must hold
    row start_pos (the kernel writes it)."""
    _attn_sizes(q, k, v, out, num_q, num_kv, start_pos + 1, 1, head_dim, Q8_ROW, Q8_ROW)
    _need(k_new, num_kv * head_dim * 2, "k_new", FP16)
    _need(v_new, num_kv * head_dim * 2, "v_new", FP16)
    check(lib().qkv_decode_attn_q8_append(
        _dev_ptr(q, "q"), _dev_ptr(k_new, "k_new"), _dev_ptr(v_new, "v_new"), _dev_ptr(k, "k"),
        _dev_ptr(v, "v"), _dev_ptr(out, "out"), num_q, num_kv, head_dim, start_pos, float(scale),
        _dev_ptr(workspace, "workspace"), workspace.numel() * workspace.element_size(),
        _stream(stream)), "qkv_decode_attn_q8_append")


def decode_attn_q8k_tq3v_workspace(num_q, num_kv, sub_n, n_keys, device) -> torch.Tensor:
    """Zero-filled workspace for decode_attn_q8k_tq3v."""
    n = int(lib().qkv_decode_attn_q8k_tq3v_workspace_bytes(num_q, num_kv, sub_n, n_keys))
    return torch.zeros(n, dtype=torch.uint8, device=device)


def decode_attn_q8k_tq3v(q, k, v, out, workspace, *, num_q, num_kv, start_pos, sub_n, scale,
                         head_dim=256, stream=None) -> None:
    """V-only TurboQuant (reference TQ_KEYS_Q8 mode): keys in Q8_0 blocks, values
    in TQ3 blocks; one fused decode launch with the merge inside it."""
    _attn_sizes(q, k, v, out, num_q, num_kv, start_pos + sub_n, sub_n, head_dim, Q8_ROW, TQ3_ROW)
    check(lib().qkv_decode_attn_q8k_tq3v(
        _dev_ptr(q, "q"), _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(out, "out"), num_q,
        num_kv, head_dim, start_pos, sub_n, float(scale), _dev_ptr(workspace, "workspace"),
        workspace.numel() * workspace.element_size(), _stream(stream)), "qkv_decode_attn_q8k_tq3v")


def decode_workspace_status(workspace, stream=None) -> int:
    """Synchronises the stream and returns QKV_OK (0) or QKV_ERR_TIMEOUT (-8): an
    in-kernel merge on this workspace ran out of polls and its rows were NaN."""
    return int(lib().qkv_decode_workspace_status(_dev_ptr(workspace, "workspace"),
                                                 _stream(stream)))


def decode_workspace_status_async(workspace, status, stream=None) -> None:
    """Enqueue the health check without synchronising: once the stream gets
    there, status[0] (an int32 device tensor) holds QKV_OK (0) or
    QKV_ERR_TIMEOUT (-8).  Capturable in a HIP graph."""
    _need(status, 4, "status", dtype=(torch.int32,))
    check(lib().qkv_decode_workspace_status_async(_dev_ptr(workspace, "workspace"),
                                                  _dev_ptr(status, "status"), _stream(stream)),
          "qkv_decode_workspace_status_async")


def decode_workspace_reset(workspace, stream=None) -> None:
    """Zero-fill a fast-path decode workspace (clears a sticky merge error)."""
    check(lib().qkv_decode_workspace_reset(_dev_ptr(workspace, "workspace"),
                                           workspace.numel() * workspace.element_size(),
                                           _stream(stream)), "qkv_decode_workspace_reset")


def decode_noalloc_status(device: int = 0, stream=None) -> int:
    """decode_workspace_status for the allocation-free decode's scratch of
    `device`: synchronises the stream, returns QKV_OK (0) or QKV_ERR_TIMEOUT (-8)."""
    return int(lib().qkv_decode_noalloc_status(int(device), _stream(stream)))


def decode_noalloc_status_async(status, device: int = 0, stream=None) -> None:
    """decode_workspace_status_async for the allocation-free decode's scratch
    of `device`."""
    _need(status, 4, "status", dtype=(torch.int32,))
    check(lib().qkv_decode_noalloc_status_async(int(device), _dev_ptr(status, "status"),
                                                _stream(stream)), "qkv_decode_noalloc_status_async")


def decode_noalloc_reset(device: int = 0, stream=None) -> None:
    """Zero-fill the allocation-free decode's scratch of `device` (clears a
    sticky merge error)."""
    check(lib().qkv_decode_noalloc_reset(int(device), _stream(stream)), "qkv_decode_noalloc_reset")


def debug_set_merge_spin_limit(limit: int) -> None:
    """Test hook: merger poll limit of later fast-path launches (negative = default)."""
    check(lib().qkv_debug_set_merge_spin_limit(int(limit)), "qkv_debug_set_merge_spin_limit")


# ---------------------------------------------------------------------------
# paged caches (per-slot int32 block tables)
# ---------------------------------------------------------------------------

def _i32(t, what):
    if t.dtype != torch.int32:
        raise ValueError(f"{what} must be int32")
    return _dev_ptr(t, what)


def tq3_append_kv_paged(k, v, k_pool, v_pool, block_tables, positions, *, block_tokens,
                        head_dim=256, stream=None) -> None:
    """Paged append: k, v fp16 [n_slots][n_tok][num_kv][256]; token t of slot s
    goes to position positions[s] + t through block_tables [n_slots][max_blocks]."""
    assert k.dtype == torch.float16 and v.dtype == torch.float16 and k.shape == v.shape
    n_slots, n_tok, num_kv = k.shape[0], k.shape[1], k.shape[2]
    pool_rows = k_pool.numel() // (TQ3_BLOCK_BYTES * num_kv * head_dim // 128)
    check(lib().qkv_tq3_append_kv_paged(
        _dev_ptr(k, "k"), _dev_ptr(v, "v"), _dev_ptr(k_pool, "k_pool"), _dev_ptr(v_pool, "v_pool"),
        n_slots, n_tok, num_kv, head_dim, _i32(block_tables, "block_tables"),
        block_tables.shape[1], block_tokens, pool_rows, _i32(positions, "positions"),
        _stream(stream)), "qkv_tq3_append_kv_paged")


def decode_attn_tq3_paged_workspace(num_q, num_kv, n_slots, max_ctx, device) -> torch.Tensor:
    n = int(lib().qkv_decode_attn_tq3_paged_workspace_bytes(num_q, num_kv, n_slots, max_ctx))
    return torch.zeros(n, dtype=torch.uint8, device=device)


def decode_attn_tq3_paged(q, k_pool, v_pool, out, workspace, block_tables, ctx_lens, *, num_q,
                          num_kv, max_ctx, block_tokens, scale, head_dim=256,
                          stream=None) -> None:
    """One decode query per slot over per-slot block tables (ragged contexts)."""
    pool_rows = k_pool.numel() // (TQ3_BLOCK_BYTES * num_kv * head_dim // 128)
    check(lib().qkv_decode_attn_tq3_paged(
        _dev_ptr(q, "q"), _dev_ptr(k_pool, "k_pool"), _dev_ptr(v_pool, "v_pool"),
        _dev_ptr(out, "out"), num_q, num_kv, head_dim, q.shape[0],
        _i32(block_tables, "block_tables"), block_tables.shape[1], block_tokens, pool_rows,
        _i32(ctx_lens, "ctx_lens"), max_ctx, float(scale), _dev_ptr(workspace, "workspace"),
        workspace.numel() * workspace.element_size(), _stream(stream)),
        "qkv_decode_attn_tq3_paged")


# ---------------------------------------------------------------------------
# chunked prefill over the TQ3 cache
# ---------------------------------------------------------------------------

def prefill_attn_tq3_workspace(num_q, num_kv, n_tok, start_pos, device) -> torch.Tensor:
    n = int(lib().qkv_prefill_attn_tq3_workspace_bytes(num_q, num_kv, n_tok, start_pos))
    return torch.empty(n, dtype=torch.uint8, device=device)


def prefill_attn_tq3(q, k_cache, v_cache, k_chunk, v_chunk, out, workspace, *, num_q, num_kv,
                     start_pos, scale, head_dim=256, stream=None) -> None:
    """Causal attention of a chunk (q [n_tok][num_q][256]) over the cache
    history rows 0..start_pos-1 (TQ3) and the chunk's own fp16 k/v; with
    k_chunk = v_chunk = None (verify) every key comes from the cache rows
    0..start_pos+n_tok-1."""
    n_tok = q.shape[0]
    from_cache = k_chunk is None
    kc = _dev_ptr(k_cache, "k_cache") if (start_pos > 0 or from_cache) else 0
    vc = _dev_ptr(v_cache, "v_cache") if (start_pos > 0 or from_cache) else 0
    check(lib().qkv_prefill_attn_tq3(
        _dev_ptr(q, "q"), kc, vc, _opt_ptr(k_chunk), _opt_ptr(v_chunk),
        _dev_ptr(out, "out"), num_q, num_kv, head_dim, start_pos, n_tok, float(scale),
        _dev_ptr(workspace, "workspace"), workspace.numel() * workspace.element_size(),
        _stream(stream)), "qkv_prefill_attn_tq3")


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

_ROPE_SCALING = {"linear": 1, "ntk": 2, "yarn": 3}
_ROPE_LAYOUT = {"half": 0, "interleaved": 1}


class RopeTable:
    """Frequencies for `rope`: `turns`, an int64 device tensor [rot_dim / 2] of 64-bit
    fractions of a turn a position (f / 2 pi * 2^64), and the amplitude of the scaling.  Made by
    `rope_table`, or by hand for frequencies or an amplitude that it does not offer."""

    def __init__(self, turns, amplitude, rot_dim):
        if turns.dtype is not torch.int64 or 2 * turns.numel() != rot_dim:
            raise ValueError(f"turns must hold {rot_dim // 2} numbers of torch.int64")
        self.turns, self.amplitude, self.rot_dim = turns, amplitude, rot_dim


def rope_table(rot_dim: int, *, base: float = 10000.0, scaling=None, device="cuda") -> RopeTable:
    """Frequencies base^(-2i/rot_dim).  scaling: None, ("linear", factor), ("ntk", factor) or
    ("yarn", factor, original_ctx[, beta_fast=32, beta_slow=1]), whose ramp between the betas is
    linear in a pair's turns over the original context, not in its index."""
    kind, args = 0, ()
    if scaling is not None:
        if scaling[0] not in _ROPE_SCALING:
            raise ValueError(f"unknown rope scaling {scaling[0]!r}")
        kind, args = _ROPE_SCALING[scaling[0]], tuple(float(x) for x in scaling[1:])
        if not (len(args) == 1 if kind < 3 else 2 <= len(args) <= 4):
            raise ValueError(f"rope scaling {scaling[0]!r} with {len(args)} numbers")
    factor, ctx, fast, slow = (args + (1.0, 1.0, 32.0, 1.0)[len(args):])[:4]
    turns = (ctypes.c_uint64 * max(1, rot_dim // 2))()
    amp = ctypes.c_float()
    check(lib().qkv_rope_table(rot_dim, float(base), kind, factor, ctx, fast, slow, ctypes.addressof(turns),
                               ctypes.addressof(amp)), "qkv_rope_table")
    host = torch.frombuffer(turns, dtype=torch.int64).clone()
    return RopeTable(host.to(device), float(amp.value), rot_dim)


def _run_device(stream, t) -> int:
    """The device that the call launches on, that of `stream` or the current one: tensor t's."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError("every tensor must be a device tensor")
    if dev != (torch._C._cuda_getDevice() if stream is None else stream.device.index):
        raise ValueError(f"the tensors are on {t.device}, the call runs on another device")
    return dev


def _on_device(dev, *tensors) -> None:
    """Every tensor contiguous and on device `dev`."""
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError(f"every tensor must be on cuda:{dev}, where the call runs; got {t.device}")
        if not t.is_contiguous():
            raise ValueError("every tensor but q, k and v must be contiguous")


def _raw_stream(stream, dev) -> int:
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream


_INT32, _UINT8 = torch.int32, torch.uint8


def _need_i32(n, what, t) -> None:
    if t.dtype is not _INT32 or t.numel() < n:
        raise ValueError(f"{what} must hold {n} numbers of torch.int32")


def _rows3(t, what, dev, shape):
    """Pointer and token stride (elements) of a tensor [tokens][heads][head_dim], a token's heads
    contiguous."""
    if t.shape != shape:
        raise ValueError(f"{what} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype not in FP16:
        raise ValueError(f"{what} must be {' or '.join(str(d) for d in FP16)}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{what} must be on cuda:{dev}, where the call runs; got {t.device}")
    n, heads, hd = shape
    s0, s1, s2 = t.stride()
    if (s2 != 1 and hd > 1) or (s1 != hd and heads > 1):
        raise ValueError(f"{what}: the heads of a token must be contiguous")
    return t.data_ptr(), s0 if n > 1 else heads * hd


def _rope_layout(layout) -> int:
    if layout not in _ROPE_LAYOUT:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    return _ROPE_LAYOUT[layout]


def rope(q, k, positions, table: RopeTable, *, layout="half", inverse=False, q_out=None, k_out=None,
         stream=None) -> None:
    """Rotates q and k (fp16 [tokens][heads][head_dim], views into a fused projection
    buffer among them; either may be None) by int32 `positions` [tokens], into q_out / k_out,
    or in place where these are None.  `inverse` turns back; it is also the gradient."""
    one = q if q is not None else k
    if one is None:
        raise ValueError("q or k is required")
    if (q is None and q_out is not None) or (k is None and k_out is not None):
        raise ValueError("an output without its input")
    n_tok, nq, hd = one.shape
    nk, dev = 0, _run_device(stream, one)
    qp = kp = (0, 0, 0, 0)
    if q is not None:
        shape = q.shape
        qp = _rows3(q, "q", dev, shape)
        qp += _rows3(q_out, "q_out", dev, shape) if q_out is not None else qp
    else:
        nq = 0
    if k is not None:
        shape = k.shape
        if shape[0] != n_tok or shape[2] != hd:
            raise ValueError(f"k must be [{n_tok}][heads][{hd}]")
        nk = shape[1]
        kp = _rows3(k, "k", dev, shape)
        kp += _rows3(k_out, "k_out", dev, shape) if k_out is not None else kp
    _need_i32(n_tok, "positions", positions)
    turns = table.turns
    _on_device(dev, positions, turns)
    check(lib().qkv_rope(*qp, *kp, positions.data_ptr(), turns.data_ptr(), table.amplitude, n_tok, nq, nk, hd,
                         table.rot_dim, _rope_layout(layout), 1 if inverse else 0, _raw_stream(stream, dev)),
          "qkv_rope")


# ---------------------------------------------------------------------------
# norms of heads with the rotation
# ---------------------------------------------------------------------------

_FP32 = torch.float32


def _head_weight(w, hd, what, dev) -> int:
    """Pointer of a weight (or of its gradient) of a head's elements; None: 0."""
    if w is None:
        return 0
    if w.dtype is not _FP32 or w.numel() != hd:
        raise ValueError(f"{what} must hold {hd} numbers of torch.float32")
    _on_device(dev, w)
    return w.data_ptr()


def _turning(table, positions, n_tok, dev):
    """Pointers of positions and turns, the amplitude and the turned elements (table None: no rotation)."""
    if table is None:
        return 0, 0, 1.0, 0
    if positions is None:
        raise ValueError("positions are required with a table")
    _need_i32(n_tok, "positions", positions)
    _on_device(dev, positions, table.turns)
    return positions.data_ptr(), table.turns.data_ptr(), table.amplitude, table.rot_dim


def _sides(q, k):
    """Tokens and head size of the rows of a call, either of which may be None."""
    one = q if q is not None else k
    if one is None:
        raise ValueError("q or k is required")
    if one.dim() != 3 or (k is not None and k.dim() != 3):
        raise ValueError("q and k must be [tokens][heads][head_dim]")
    n_tok, _, hd = one.shape
    if k is not None and (k.shape[0] != n_tok or k.shape[2] != hd):
        raise ValueError(f"k must be [{n_tok}][heads][{hd}]")
    return one, n_tok, hd


def norm_rope(q, k, q_weight, k_weight, positions, table: RopeTable | None, *, eps=1e-6, layout="half", q_out=None,
              k_out=None, stream=None) -> None:
    """Norms of the heads of q and k (fp16 [tokens][heads][head_dim], views into a fused projection buffer among
    them; either may be None), x * weight / sqrt(mean(x^2) + eps) with fp32 weights [head_dim] (None: ones), then
    the rotation by `positions` (table None: none), into q_out / k_out, or in place where these are None."""
    if (q is None and q_out is not None) or (k is None and k_out is not None):
        raise ValueError("an output without its input")
    one, n_tok, hd = _sides(q, k)
    dev = _run_device(stream, one)
    sides, heads = [], []
    for x, out, w, what in ((q, q_out, q_weight, "q"), (k, k_out, k_weight, "k")):
        if x is None:
            sides += [0, 0, 0, 0, 0]
            heads.append(0)
            continue
        at = _rows3(x, what, dev, x.shape)
        sides += [*at, *(_rows3(out, what + "_out", dev, x.shape) if out is not None else at),
                  _head_weight(w, hd, what + "_weight", dev)]
        heads.append(x.shape[1])
    pos, turns, amp, rot = _turning(table, positions, n_tok, dev)
    check(lib().qkv_norm_rope(*sides, float(eps), pos, turns, amp, n_tok, *heads, hd, rot, _rope_layout(layout),
                              _raw_stream(stream, dev)), "qkv_norm_rope")


def norm_rope_grad_workspace(n_tok, num_q, num_k, head_dim, device) -> torch.Tensor:
    """Workspace of norm_rope_grad for up to these numbers."""
    n = int(lib().qkv_norm_rope_grad_workspace_bytes(n_tok, num_q, num_k, head_dim))
    if n == 0:
        raise ValueError(f"no call of these numbers: n_tok {n_tok}, num_q {num_q}, num_k {num_k}, head_dim {head_dim}")
    return torch.empty(n, dtype=torch.uint8, device=device)


def norm_rope_grad(q, k, dq, dk, q_weight, k_weight, positions, table: RopeTable | None, q_weight_grad=None,
                   k_weight_grad=None, *, eps=1e-6, layout="half", q_grad=None, k_grad=None, workspace=None,
                   stream=None) -> None:
    """The gradient of norm_rope at its inputs q and k: dq and dk, the gradients of its outputs, become those of
    its inputs, in q_grad / k_grad or in place, and q_weight_grad / k_weight_grad (fp32 [head_dim], None: not
    wanted) those of the weights.  workspace: norm_rope_grad_workspace's (allocated here when None)."""
    one, n_tok, hd = _sides(q, k)
    dev = _run_device(stream, one)
    sides, heads = [], []
    for x, dy, dx, w, dw, what in ((q, dq, q_grad, q_weight, q_weight_grad, "q"), (k, dk, k_grad, k_weight, k_weight_grad, "k")):
        if x is None:
            if dy is not None or dx is not None or dw is not None:
                raise ValueError(f"a gradient of {what} without {what}")
            sides += [0] * 8
            heads.append(0)
            continue
        if dy is None:
            raise ValueError(f"d{what} is required")
        at = _rows3(dy, "d" + what, dev, x.shape)
        sides += [*_rows3(x, what, dev, x.shape), *at,
                  *(_rows3(dx, what + "_grad", dev, x.shape) if dx is not None else at),
                  _head_weight(w, hd, what + "_weight", dev), _head_weight(dw, hd, what + "_weight_grad", dev)]
        heads.append(x.shape[1])
    pos, turns, amp, rot = _turning(table, positions, n_tok, dev)
    L = lib()
    if workspace is None:
        workspace = _scratch(int(L.qkv_norm_rope_grad_workspace_bytes(n_tok, *heads, hd)), one.device, stream)
    _on_device(dev, workspace)
    check(L.qkv_norm_rope_grad(*sides, float(eps), pos, turns, amp, n_tok, *heads, hd, rot, _rope_layout(layout),
                               workspace.data_ptr(), workspace.nbytes, _raw_stream(stream, dev)), "qkv_norm_rope_grad")


# ---------------------------------------------------------------------------
# paged 8-bit cache: e4m3 codes, an exponent per page and kv head
# ---------------------------------------------------------------------------

def f8_pool(n_pages: int, block_tokens: int, num_kv: int, head_dim: int, device):
    """Zeroed codes uint8 [n_pages][block_tokens][num_kv][head_dim] and exponents uint8
    [n_pages][num_kv] of one tensor (keys or values) of a paged 8-bit cache."""
    return (torch.zeros((n_pages, block_tokens, num_kv, head_dim), dtype=torch.uint8, device=device),
            torch.zeros((n_pages, num_kv), dtype=torch.uint8, device=device))


def _f8_batch(dev, k_pool, v_pool, k_exp, v_exp, block_tables, starts, positions):
    """Checks of a paged 8-bit batch.  Returns (n_pages, block_tokens, num_kv, head_dim, n_slots,
    max_blocks)."""
    n_pages, bt, kv, hd = shape = k_pool.shape
    if v_pool.shape != shape:
        raise ValueError("k_pool and v_pool must be [n_pages][block_tokens][num_kv][head_dim]")
    if k_exp.shape != (n_pages, kv) or v_exp.shape != (n_pages, kv):
        raise ValueError(f"k_exp and v_exp must be [{n_pages}][{kv}]")
    if not (k_pool.dtype is v_pool.dtype is k_exp.dtype is v_exp.dtype is _UINT8):
        raise ValueError("the pools and their exponents must be torch.uint8")
    if not (block_tables.dtype is starts.dtype is positions.dtype is _INT32):
        raise ValueError("block_tables, starts and positions must be torch.int32")
    n_slots, mb = block_tables.shape
    if starts.numel() != n_slots + 1 or positions.numel() != n_slots:
        raise ValueError(f"starts must hold {n_slots + 1} numbers and positions {n_slots}")
    _on_device(dev, k_pool, v_pool, k_exp, v_exp, block_tables, starts, positions)
    return n_pages, bt, kv, hd, n_slots, mb


def f8_append_kv_paged(k, v, k_pool, v_pool, k_exp, v_exp, block_tables, starts, positions, *, max_tok, q=None,
                       q_out=None, rope: RopeTable | None = None, layout="half", stream=None) -> None:
    """Ragged append: rows starts[s] .. starts[s+1]-1 of k and v (fp16 [rows][num_kv][head_dim])
    go to positions positions[s] .. of slot s.  With `rope` k is rotated first, and q (into
    q_out, or in place), in the same launch."""
    dev = _run_device(stream, k_pool)
    n_pages, bt, kv, hd, n_slots, mb = _f8_batch(dev, k_pool, v_pool, k_exp, v_exp, block_tables, starts, positions)
    rows = k.shape[0]
    shape = (rows, kv, hd)
    qp, nq, tp, amp, rot = (0, 0, 0, 0), 0, 0, 1.0, 0
    if rope is not None:
        _on_device(dev, rope.turns)
        tp, amp, rot = rope.turns.data_ptr(), rope.amplitude, rope.rot_dim
    if q is not None:
        if rope is None:
            raise ValueError("q without rope")
        nq = q.shape[1]
        qs = (rows, nq, hd)
        qp = _rows3(q, "q", dev, qs)
        qp += _rows3(q_out, "q_out", dev, qs) if q_out is not None else qp
    elif q_out is not None:
        raise ValueError("q_out without q")
    check(lib().qkv_f8_append_kv_paged(
        *_rows3(k, "k", dev, shape), *_rows3(v, "v", dev, shape), k_pool.data_ptr(), v_pool.data_ptr(),
        k_exp.data_ptr(), v_exp.data_ptr(), rows, n_slots, max_tok, kv, hd, block_tables.data_ptr(), mb, bt, n_pages,
        starts.data_ptr(), positions.data_ptr(), *qp, nq, tp, amp, rot, _rope_layout(layout),
        _raw_stream(stream, dev)), "qkv_f8_append_kv_paged")


def attn_f8_paged_workspace(num_q, num_kv, n_slots, n_rows, max_tok, max_ctx, device, *, head_dim=256) -> torch.Tensor:
    """Zero-filled workspace of attn_f8_paged for these numbers (calls leave it ready for the next)."""
    n = int(lib().qkv_attn_f8_paged_workspace_bytes(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx))
    if n == 0 and min(n_slots, n_rows, max_tok) > 0:   # (a batch without rows needs none)
        raise ValueError(f"no call of these numbers: num_q {num_q}, num_kv {num_kv}, head_dim {head_dim}, n_slots {n_slots}, "
                         f"n_rows {n_rows}, max_tok {max_tok}, max_ctx {max_ctx}")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def attn_f8_paged(q, k_pool, v_pool, k_exp, v_exp, out, workspace, block_tables, starts, positions, *, max_tok,
                  max_ctx, scale, window=0, sink=0, stream=None) -> None:
    """Causal attention of ragged query rows (fp16 [rows][num_q][head_dim]; slot s owns rows
    starts[s] .. starts[s+1]-1 at positions positions[s] ..) over the paged 8-bit cache:
    decode steps, verify blocks and prompts.  window > 0 limits a query to the last `window`
    keys and the first `sink`.  Rows past starts[-1] are left alone; out may be q."""
    dev = _run_device(stream, k_pool)
    n_pages, bt, kv, hd, n_slots, mb = _f8_batch(dev, k_pool, v_pool, k_exp, v_exp, block_tables, starts, positions)
    rows, nq, qd = shape = q.shape
    if qd != hd or out.shape != shape:
        raise ValueError(f"q and out must be [rows][num_q][{hd}]")
    if q.dtype not in FP16 or out.dtype not in FP16:
        raise ValueError(f"q and out must be fp16, got {q.dtype} and {out.dtype}")
    _on_device(dev, q, out, workspace)
    check(lib().qkv_attn_f8_paged(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), out.data_ptr(), rows,
        nq, kv, hd, n_slots, max_tok, max_ctx, block_tables.data_ptr(), mb, bt, n_pages, starts.data_ptr(),
        positions.data_ptr(), float(scale), window, sink, workspace.data_ptr(), workspace.nbytes,
        _raw_stream(stream, dev)), "qkv_attn_f8_paged")


# ---------------------------------------------------------------------------
# eviction from the paged 8-bit cache by accumulated attention weight
# ---------------------------------------------------------------------------

def f8_weights(n_pages: int, block_tokens: int, num_kv: int, device) -> torch.Tensor:
    """Zeroed weights fp32 [n_pages][num_kv][block_tokens] of the keys of a paged 8-bit cache (a plane of the page
    calls beside its pools)."""
    return torch.zeros((n_pages, num_kv, block_tokens), dtype=torch.float32, device=device)


def _need_weights(weights, k_pool) -> None:
    n_pages, bt, kv, _ = k_pool.shape
    if weights.dtype is not _FP32 or weights.shape != (n_pages, kv, bt):
        raise ValueError(f"weights must be torch.float32 [{n_pages}][{kv}][{bt}]")


def weigh_f8_paged_workspace(num_q, num_kv, n_slots, n_rows, max_tok, max_ctx, device, *, head_dim=256) -> torch.Tensor:
    """Workspace of weigh_f8_paged for up to these numbers."""
    n = int(lib().qkv_weigh_f8_paged_workspace_bytes(num_q, num_kv, head_dim, n_slots, n_rows, max_tok, max_ctx))
    if n == 0 and min(n_slots, n_rows, max_tok) > 0:
        raise ValueError(f"no call of these numbers: num_q {num_q}, num_kv {num_kv}, head_dim {head_dim}, n_slots {n_slots}, "
                         f"n_rows {n_rows}, max_tok {max_tok}, max_ctx {max_ctx}")
    return torch.empty(n, dtype=torch.uint8, device=device)


def weigh_f8_paged(q, k_pool, k_exp, weights, workspace, block_tables, starts, positions, *, max_tok, max_ctx, scale,
                   decay=1.0, weighed=None, window=0, sink=0, stream=None) -> None:
    """Adds to weights (fp32 [n_pages][num_kv][block_tokens]) what the ragged query rows (as for attn_f8_paged) give each
    key: softmax weights summed over rows and the heads of a KV group, after decay times what stood for the first
    weighed[s] keys of each slot (int32 [n_slots], None: positions) and from zero for the others.  Of slots that share a page
    only one may have rows in a call."""
    dev = _run_device(stream, k_pool)
    n_pages, bt, kv, hd = k_pool.shape
    if k_exp.shape != (n_pages, kv):
        raise ValueError(f"k_exp must be [{n_pages}][{kv}]")
    if not (k_pool.dtype is k_exp.dtype is _UINT8):
        raise ValueError("the pool and its exponents must be torch.uint8")
    _need_weights(weights, k_pool)
    if not (block_tables.dtype is starts.dtype is positions.dtype is _INT32):
        raise ValueError("block_tables, starts and positions must be torch.int32")
    n_slots, mb = block_tables.shape
    if starts.numel() != n_slots + 1 or positions.numel() != n_slots:
        raise ValueError(f"starts must hold {n_slots + 1} numbers and positions {n_slots}")
    rows, nq, qd = q.shape
    if qd != hd or q.dtype not in FP16:
        raise ValueError(f"q must be fp16 [rows][num_q][{hd}]")
    wp = 0
    if weighed is not None:
        if weighed.dtype is not _INT32 or weighed.numel() != n_slots:
            raise ValueError(f"weighed must hold {n_slots} numbers of torch.int32")
        _on_device(dev, weighed)
        wp = weighed.data_ptr()
    _on_device(dev, q, k_pool, k_exp, weights, workspace, block_tables, starts, positions)
    check(lib().qkv_weigh_f8_paged(
        q.data_ptr(), k_pool.data_ptr(), k_exp.data_ptr(), weights.data_ptr(), rows, nq, kv, hd, n_slots, max_tok, max_ctx,
        block_tables.data_ptr(), mb, bt, n_pages, starts.data_ptr(), positions.data_ptr(), wp, float(decay), float(scale),
        window, sink, workspace.data_ptr(), workspace.nbytes, _raw_stream(stream, dev)), "qkv_weigh_f8_paged")


def evict_f8_paged_workspace(n_slots, num_kv, block_tokens, max_ctx, max_keep, device) -> torch.Tensor:
    """Workspace of evict_f8_paged for up to these numbers."""
    n = int(lib().qkv_evict_f8_paged_workspace_bytes(n_slots, num_kv, block_tokens, max_ctx, max_keep))
    if n == 0 and n_slots > 0:
        raise ValueError(f"no call of these numbers: n_slots {n_slots}, num_kv {num_kv}, block_tokens {block_tokens}, "
                         f"max_ctx {max_ctx}, max_keep {max_keep}")
    return torch.empty(n, dtype=torch.uint8, device=device)


def evict_f8_paged(k_pool, v_pool, k_exp, v_exp, weights, block_tables, lens, keep, kept, workspace, *, max_ctx, sink=0,
                   recent=0, stream=None) -> None:
    """Of the lens[s] rows of each slot keep[s] stay in every KV head: the last `recent`, the first `sink` and those of
    the largest weights (fp32 [n_pages][num_kv][block_tokens]), moved in order to the slot's first rows, in the pools
    and in weights.  kept: int32 [n_slots][num_kv][max_keep], their former rows (-1 past the last).  The slot's length
    is then min(lens[s], keep[s]); rows are no longer positions."""
    dev = _run_device(stream, k_pool)
    n_pages, bt, kv, hd = shape = k_pool.shape
    if v_pool.shape != shape:
        raise ValueError("k_pool and v_pool must be [n_pages][block_tokens][num_kv][head_dim]")
    if k_exp.shape != (n_pages, kv) or v_exp.shape != (n_pages, kv):
        raise ValueError(f"k_exp and v_exp must be [{n_pages}][{kv}]")
    if not (k_pool.dtype is v_pool.dtype is k_exp.dtype is v_exp.dtype is _UINT8):
        raise ValueError("the pools and their exponents must be torch.uint8")
    _need_weights(weights, k_pool)
    if not (block_tables.dtype is lens.dtype is keep.dtype is kept.dtype is _INT32):
        raise ValueError("block_tables, lens, keep and kept must be torch.int32")
    n_slots, mb = block_tables.shape
    if lens.numel() != n_slots or keep.numel() != n_slots:
        raise ValueError(f"lens and keep must hold {n_slots} numbers")
    if kept.dim() != 3 or kept.shape[:2] != (n_slots, kv):
        raise ValueError(f"kept must be [{n_slots}][{kv}][max_keep]")
    _on_device(dev, k_pool, v_pool, k_exp, v_exp, weights, block_tables, lens, keep, kept, workspace)
    check(lib().qkv_evict_f8_paged(
        k_pool.data_ptr(), v_pool.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), weights.data_ptr(), n_slots, kv, hd,
        max_ctx, kept.shape[2], block_tables.data_ptr(), mb, bt, n_pages, lens.data_ptr(), keep.data_ptr(), sink, recent,
        kept.data_ptr(), workspace.data_ptr(), workspace.nbytes, _raw_stream(stream, dev)), "qkv_evict_f8_paged")


# ---------------------------------------------------------------------------
# pages: sharing, reserving, giving back, compacting
# ---------------------------------------------------------------------------

class _Plane(ctypes.Structure):
    _fields_ = [("base", ctypes.c_void_p), ("page_bytes", ctypes.c_size_t)]


class PagePlanes:
    """The pools that page calls copy: contiguous device tensors [n_pages, ...] of any type
    (keys, values and exponents of every layer).  Kept with the tensors."""

    def __init__(self, tensors):
        self.tensors = list(tensors)
        self.n = len(self.tensors)
        self.n_pages = min((t.shape[0] for t in self.tensors), default=0)
        self.device = self.tensors[0].get_device() if self.tensors else -1
        self.array = (_Plane * max(1, self.n))()
        for i, t in enumerate(self.tensors):
            if t.get_device() != self.device:
                raise ValueError("the planes must be on one device")
            self.array[i] = _Plane(_dev_ptr(t, f"plane {i}"), t.numel() * t.element_size() // max(1, t.shape[0]))
        self.ptr = ctypes.addressof(self.array)


def page_planes(tensors) -> PagePlanes:
    """The planes of pages_reserve, pages_compact and pages_copy."""
    return PagePlanes(tensors)


def _page_state(dev, block_tables, ref_counts):
    """Checks of the tables and counts; returns the leading arguments of the page calls."""
    if not (block_tables.dtype is ref_counts.dtype is _INT32):
        raise ValueError("block_tables and ref_counts must be torch.int32")
    n_slots, mb = block_tables.shape
    _on_device(dev, block_tables, ref_counts)
    return block_tables.data_ptr(), n_slots, mb, ref_counts.data_ptr(), ref_counts.numel()


def _page_lists(dev, status, *lists):
    """Checks of the int32 lists of a page call; returns their length and the status pointer."""
    n = lists[0].numel()
    for t in lists:
        if t.dtype is not _INT32 or t.numel() != n:
            raise ValueError(f"the lists must be torch.int32 of one length, {n}")
    _on_device(dev, *lists)
    if status is None:
        return n, 0
    _need_i32(n, "status", status)
    _on_device(dev, status)
    return n, status.data_ptr()


def _planes_of(planes, n_pages, dev):
    if planes is None:
        return 0, 0
    if planes.n:
        if planes.n_pages < n_pages:
            raise ValueError(f"the planes hold {planes.n_pages} pages, ref_counts {n_pages}")
        if planes.device != dev:
            raise ValueError(f"the planes must be on cuda:{dev}, where the call runs")
    return planes.ptr, planes.n


def pages_fork(block_tables, ref_counts, parents, children, n_tokens, status=None, *, block_tokens,
               stream=None) -> None:
    """children[i] shares the pages of the first n_tokens[i] tokens of parents[i] (device int32
    lists; block_tables int32 [n_slots][max_blocks], ref_counts int32 [n_pages])."""
    dev = _run_device(stream, block_tables)
    t, n_slots, mb, r, n_pages = _page_state(dev, block_tables, ref_counts)
    n, st = _page_lists(dev, status, parents, children, n_tokens)
    check(lib().qkv_pages_fork(t, n_slots, mb, block_tokens, r, n_pages, parents.data_ptr(), children.data_ptr(),
                               n_tokens.data_ptr(), n, st, _raw_stream(stream, dev)), "qkv_pages_fork")


def pages_release(block_tables, ref_counts, slots, keep_tokens, status=None, *, block_tokens, stream=None) -> None:
    """Gives back the pages of slots[i] past its first keep_tokens[i] tokens."""
    dev = _run_device(stream, block_tables)
    t, n_slots, mb, r, n_pages = _page_state(dev, block_tables, ref_counts)
    n, st = _page_lists(dev, status, slots, keep_tokens)
    check(lib().qkv_pages_release(t, n_slots, mb, block_tokens, r, n_pages, slots.data_ptr(), keep_tokens.data_ptr(),
                                  n, st, _raw_stream(stream, dev)), "qkv_pages_release")


def pages_reserve(block_tables, ref_counts, slots, positions, n_new, status=None, planes=None, *, block_tokens,
                  max_new, scratch=None, stream=None) -> None:
    """Pages of its own for tokens positions[i] .. positions[i] + n_new[i] - 1 of slots[i]: missing ones are
    taken, shared ones replaced (copied in `planes` where they hold earlier rows).  scratch: an int32
    tensor (allocated here when None) whose first 2n numbers are afterwards the copied pairs."""
    dev = _run_device(stream, block_tables)
    t, n_slots, mb, r, n_pages = _page_state(dev, block_tables, ref_counts)
    n, st = _page_lists(dev, status, slots, positions, n_new)
    L = lib()
    if scratch is None:
        scratch = _scratch(int(L.qkv_pages_reserve_scratch_bytes(n, max_new, block_tokens)), block_tables.device,
                           stream)
    _need_i32(0, "scratch", scratch)
    _on_device(dev, scratch)
    check(L.qkv_pages_reserve(t, n_slots, mb, block_tokens, r, n_pages, slots.data_ptr(), positions.data_ptr(),
                              n_new.data_ptr(), n, max_new, st, *_planes_of(planes, n_pages, dev), scratch.data_ptr(),
                              scratch.nbytes, _raw_stream(stream, dev)), "qkv_pages_reserve")


def pages_reorder(block_tables, ref_counts, slots, parents, n_tokens, status=None, states: PagePlanes | None = None, *,
                  block_tokens, stream=None) -> None:
    """slots[i] takes over what parents[i] held at the call (device int32 lists): the pages of its first n_tokens[i]
    tokens, and its row of every tensor of `states` (page_planes of tensors [n_slots, ...]).  Any permutation, with
    one parent for many slots: a beam search step's."""
    dev = _run_device(stream, block_tables)
    t, n_slots, mb, r, n_pages = _page_state(dev, block_tables, ref_counts)
    n, st = _page_lists(dev, status, slots, parents, n_tokens)
    sp, ns = 0, 0
    if states is not None and states.n:
        if states.n_pages < n_slots:
            raise ValueError(f"the states hold {states.n_pages} rows, block_tables {n_slots}")
        if states.device != dev:
            raise ValueError(f"the states must be on cuda:{dev}, where the call runs")
        sp, ns = states.ptr, states.n
    check(lib().qkv_pages_reorder(t, n_slots, mb, block_tokens, r, n_pages, slots.data_ptr(), parents.data_ptr(),
                                  n_tokens.data_ptr(), n, st, sp, ns, _raw_stream(stream, dev)), "qkv_pages_reorder")


def pages_copy(planes: PagePlanes, pairs, *, stream=None) -> None:
    """Page pairs[i][0] to page pairs[i][1] in every plane (device int32 [n][2])."""
    dev = _run_device(stream, pairs)
    if pairs.dim() != 2 or pairs.shape[1] != 2 or pairs.dtype is not _INT32:
        raise ValueError("pairs must be torch.int32 [n][2]")
    _on_device(dev, pairs)
    check(lib().qkv_pages_copy(*_planes_of(planes, 0, dev), planes.n_pages, pairs.data_ptr(), pairs.shape[0],
                               _raw_stream(stream, dev)), "qkv_pages_copy")


def pages_compact(block_tables, ref_counts, moved, n_used, planes=None, *, scratch=None, stream=None) -> None:
    """Moves the pages in use to indices 0 .. n_used[0]-1, in planes, tables and counts; moved[p] (int32
    [n_pages]) is where page p went, -1 if it was free."""
    dev = _run_device(stream, block_tables)
    t, n_slots, mb, r, n_pages = _page_state(dev, block_tables, ref_counts)
    _need_i32(n_pages, "moved", moved)
    _need_i32(1, "n_used", n_used)
    if scratch is None:
        scratch = _scratch((n_pages + 2) * 4, block_tables.device, stream)
    _need_i32(0, "scratch", scratch)
    _on_device(dev, moved, n_used, scratch)
    check(lib().qkv_pages_compact(t, n_slots, mb, r, n_pages, moved.data_ptr(), n_used.data_ptr(),
                                  *_planes_of(planes, n_pages, dev), scratch.data_ptr(), scratch.nbytes,
                                  _raw_stream(stream, dev)), "qkv_pages_compact")


# ---------------------------------------------------------------------------
# beam search
# ---------------------------------------------------------------------------

_LOGITS = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}


def beam_select_workspace(n, beams, vocab, take, device) -> torch.Tensor:
    """Workspace of beam_select for up to these numbers."""
    b = int(lib().qkv_beam_select_workspace_bytes(n, beams, vocab, take))
    if b == 0 and n > 0:
        raise ValueError(f"no call of these numbers: n {n}, beams {beams}, vocab {vocab}, take {take}")
    return torch.empty(b, dtype=torch.uint8, device=device)


def beam_select(logits, scores, parents, tokens, top_scores, workspace, *, done=None, end_token=0, stream=None) -> None:
    """The best continuations of every request: logits fp16, bf16 or fp32 [n * beams][vocab] (rows may be apart),
    scores fp32 [n][beams] (-inf: no beam), done int32 [n][beams] or None (ended beams offer end_token at their own
    score); into parents int32, tokens int32 and top_scores fp32 [n][take]: logits row, token, score + log
    probability, best first, -1, -1 and -inf where there are none."""
    dev = _run_device(stream, logits)
    if logits.dim() != 2 or logits.dtype not in _LOGITS:
        raise ValueError("logits must be torch.float16, torch.bfloat16 or torch.float32 [n * beams][vocab]")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits: a row must be contiguous")
    if scores.dim() != 2 or scores.dtype is not _FP32 or scores.numel() != rows:
        raise ValueError(f"scores must be torch.float32 [n][beams], {rows} in all")
    n, beams = scores.shape
    if parents.dim() != 2 or parents.shape[0] != n or tokens.shape != parents.shape or top_scores.shape != parents.shape:
        raise ValueError(f"parents, tokens and top_scores must be [{n}][take]")
    take = parents.shape[1]
    if not (parents.dtype is tokens.dtype is _INT32) or top_scores.dtype is not _FP32:
        raise ValueError("parents and tokens must be torch.int32, top_scores torch.float32")
    dp = 0
    if done is not None:
        if done.dtype is not _INT32 or done.numel() != rows:
            raise ValueError(f"done must hold {rows} numbers of torch.int32")
        _on_device(dev, done)
        dp = done.data_ptr()
    _on_device(dev, scores, parents, tokens, top_scores, workspace)
    check(lib().qkv_beam_select(
        logits.data_ptr(), _LOGITS[logits.dtype], logits.stride(0) if rows > 1 else vocab, scores.data_ptr(), dp, end_token,
        n, beams, vocab, take, parents.data_ptr(), tokens.data_ptr(), top_scores.data_ptr(), workspace.data_ptr(),
        workspace.nbytes, _raw_stream(stream, dev)), "qkv_beam_select")
