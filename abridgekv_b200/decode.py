"""Paged decode attention over per-quota-group page tables (host side).

Mirrors the reference's decode entry points:

* ``attend_decode_batched`` takes the arguments of
  ``PackedKVSidecar._attend_decode_batched``
  (third_party/vllm_overlay/vllm/v1/worker/compresslm_packed_kv.py:564-616):
  one query row per active request, the layer's paged ``kv_cache``
  ``[num_blocks, 2, page, H_kv, D]``, the KV-cache group's ``block_table``
  ``[R, max_pages]`` and physical ``seq_lens`` ``[R]``; it writes
  ``output[:n]`` in place.
* ``paged_decode`` runs many layers in one launch: layer ``l`` brings its own
  query, cache tensor, block table and seq_lens (its quota group's physical
  layout, gpu_model_runner.py:1672-1681, 2184-2204).

Both go through ``abkv_decode`` in libabkv.so.  There is no fallback: a
missing library or a non-CUDA tensor raises.
"""
from __future__ import annotations

import functools
import math
from typing import Sequence

import torch

from . import _lib
from .workspace import Workspace, call_scope, call_workspace, default_workspace

def _check_cuda(name: str, t: torch.Tensor, dtype: torch.dtype | None = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (libabkv has no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _validate(queries, kv_caches, block_tables, seq_lens, outputs, out_shape=None, alloc=True):
    """Check the per-layer arguments; -> (B, Hq, Hkv, D, page, outputs) (no outputs
    are allocated when `outputs` is None and `alloc` is False)."""
    L = len(queries)
    if not (L == len(kv_caches) == len(block_tables) == len(seq_lens)) or L == 0:
        raise ValueError("per-layer argument lists must be non-empty and of equal length")
    q0, kv0 = queries[0], kv_caches[0]
    B, Hq, D = q0.shape
    _, two, page, Hkv, D2 = kv0.shape
    if two != 2 or D2 != D:
        raise ValueError(f"kv cache must be [num_blocks, 2, page, Hkv, {D}], got {tuple(kv0.shape)}")
    device = q0.device
    out_shape = (B, Hq, D) if out_shape is None else tuple(out_shape)
    outs = []
    for l in range(L):
        q, kv, bt, sl = queries[l], kv_caches[l], block_tables[l], seq_lens[l]
        _check_cuda("query", q, torch.bfloat16)
        _check_cuda("kv_cache", kv, torch.bfloat16)
        _check_cuda("block_table", bt, torch.int32)
        _check_cuda("seq_lens", sl, torch.int32)
        if tuple(q.shape) != (B, Hq, D) or not q.is_contiguous():
            raise ValueError("every query must be a contiguous [B, Hq, D] tensor")
        if tuple(kv.shape[1:]) != (2, page, Hkv, D) or not kv.is_contiguous():
            raise ValueError("every kv cache must be a contiguous [num_blocks, 2, page, Hkv, D] tensor")
        if bt.dim() != 2 or bt.shape[0] < B or not bt.is_contiguous():
            raise ValueError("block_table must be a contiguous [>=B, max_pages] tensor")
        if sl.dim() != 1 or sl.shape[0] < B or not sl.is_contiguous():
            raise ValueError("seq_lens must be a contiguous [>=B] tensor")
        if outputs is not None:
            o = outputs[l]
            _check_cuda("output", o, torch.bfloat16)
            if tuple(o.shape) != out_shape or not o.is_contiguous():
                raise ValueError(f"every output must be a contiguous {list(out_shape)} tensor")
        elif alloc:
            o = torch.empty(out_shape, dtype=torch.bfloat16, device=device)
        else:
            continue
        outs.append(o)
    return B, Hq, Hkv, D, page, outs


def paged_decode(
    queries: Sequence[torch.Tensor],
    kv_caches: Sequence[torch.Tensor],
    block_tables: Sequence[torch.Tensor],
    seq_lens: Sequence[torch.Tensor],
    *,
    scale: float | None = None,
    outputs: Sequence[torch.Tensor] | None = None,
    max_pages_per_seq: int | None = None,
    chunk_tokens: int = 0,
    workspace: Workspace | None = None,
    stream: torch.cuda.Stream | None = None,
) -> list[torch.Tensor]:
    """Decode attention for ``len(queries)`` layers in one launch.

    queries[l]: [B, Hq, D] bf16; kv_caches[l]: [num_blocks, 2, page, Hkv, D] bf16;
    block_tables[l]: [B, max_pages_l] int32; seq_lens[l]: [B] int32.
    Returns outputs[l]: [B, Hq, D] bf16.
    """
    L = len(queries)
    B, Hq, Hkv, D, page, outs = _validate(queries, kv_caches, block_tables, seq_lens, outputs)
    device = queries[0].device
    if max_pages_per_seq is None:
        max_pages_per_seq = max(int(bt.shape[1]) for bt in block_tables)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    lib = _lib.lib()
    need = lib.abkv_decode_workspace_size(L, B, Hq, D, page, max_pages_per_seq, chunk_tokens)
    if need == 0:
        raise _lib.AbkvError("abkv_decode_workspace_size", 3,
                             f"unsupported shape (B={B}, Hq={Hq}, D={D}, page={page})")
    ws = (workspace or default_workspace(device)).ensure(need)
    s = torch.cuda.current_stream(device) if stream is None else stream
    with torch.cuda.device(device):
        st = _call_decode(lib, queries, kv_caches, block_tables, seq_lens, outs, L, B, Hq, Hkv, D, page,
                          max_pages_per_seq, scale, chunk_tokens, ws, s)
    _lib.check("abkv_decode", st)
    return outs


def _call_decode(lib, queries, kv_caches, block_tables, seq_lens, outs, L, B, Hq, Hkv, D, page,
                 max_pages_per_seq, scale, chunk_tokens, ws, s):
    return lib.abkv_decode(
        _lib.ptr_array([q.data_ptr() for q in queries]),
        _lib.ptr_array([kv.data_ptr() for kv in kv_caches]),
        _lib.ptr_array([bt.data_ptr() for bt in block_tables]),
        _lib.i64_array([bt.stride(0) for bt in block_tables]),
        _lib.ptr_array([sl.data_ptr() for sl in seq_lens]),
        _lib.i64_array([kv.shape[0] for kv in kv_caches]),
        _lib.ptr_array([o.data_ptr() for o in outs]),
        L, B, Hq, Hkv, D, page, max_pages_per_seq, float(scale), chunk_tokens,
        ws.ptr(), ws.nbytes, s.cuda_stream,
    )


def _per_layer(name: str, value, L: int) -> tuple[int, ...]:
    """An int (or None) for every layer, or one entry per layer; None counts as 0."""
    if value is None or isinstance(value, int):
        out = (value or 0,) * L
    else:
        out = tuple(0 if v is None else int(v) for v in value)
        if len(out) != L:
            raise ValueError(f"{name} must be one number or one per layer ({L})")
    if min(out) < 0 or max(out) > 0x7FFFFFFF:
        raise ValueError(f"{name} must lie in [0, 2^31), got {out}")
    return out


@functools.lru_cache(maxsize=256)
def _window_plan(L, B, Hq, Hkv, D, page, max_pages, chunk_tokens, windows, sinks, weighted):
    """(workspace bytes, windows array, sinks array) of a shape."""
    win, snk = _lib.i32_array(windows), _lib.i32_array(sinks)
    return _lib.lib().abkv_decode_window_workspace_size(L, B, Hq, Hkv, D, page, max_pages, chunk_tokens, win, snk,
                                                        weighted), win, snk


def _refuse(name: str, t, want: str) -> None:
    kind = TypeError if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in (
        torch.bfloat16, torch.int32) else ValueError
    raise kind(f"{name} must be {want}" + (
        f", got {t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else ""))


def _check_weights(weights, L, B, Hkv, device) -> tuple[int, int]:
    """-> (units, rows)"""
    if len(weights) != L:
        raise ValueError("weights must hold one accumulator tensor per layer")
    for w in weights:
        _check_cuda("weights", w, torch.float32)
    units, rows = (int(weights[0].shape[1]), int(weights[0].shape[2])) if weights[0].dim() == 3 else (0, 0)
    for w in weights:
        if w.dim() != 3 or w.shape[0] < B or w.shape[1] != units or w.shape[2] != rows or w.stride(2) != 1 or rows == 0:
            raise ValueError(f"every weights tensor must be [>=B, Hkv or 1, rows] with contiguous rows, got {tuple(w.shape)}")
        if (B > 1 and w.stride(0) < rows) or (units > 1 and w.stride(1) < rows):
            raise ValueError("the rows of weights must not overlap")
        if w.device != device:
            raise ValueError("every tensor of the call must be on the queries' device")
    if units not in (1, Hkv):
        raise ValueError(f"weights must hold one row per KV head ({Hkv}) or one per sequence, got {units}")
    if L > 1 and len({w.data_ptr() for w in weights}) != L:
        raise ValueError("every layer needs its own weights tensor")
    return units, rows


def _decode_window(queries, kv_caches, block_tables, seq_lens, weights, window, num_sinks, scale, outputs,
                   max_pages_per_seq, chunk_tokens, workspace, stream):
    L = len(queries)
    if not (L == len(kv_caches) == len(block_tables) == len(seq_lens)) or L == 0 or (
            outputs is not None and len(outputs) != L):
        raise ValueError("per-layer argument lists must be non-empty and of equal length")
    q0, kv0 = queries[0], kv_caches[0]
    _check_cuda("query", q0, torch.bfloat16)
    _check_cuda("kv_cache", kv0, torch.bfloat16)
    if q0.dim() != 3 or kv0.dim() != 5:
        raise ValueError("query must be [B, Hq, D] and kv_cache [num_blocks, 2, page, Hkv, D]")
    q_shape, kv_shape, device = q0.shape, kv0.shape, q0.device
    (B, Hq, D), (_, two, page, Hkv, D2) = q_shape, kv_shape
    if two != 2 or D2 != D:
        raise ValueError(f"kv cache must be [num_blocks, 2, page, Hkv, {D}], got {tuple(kv_shape)}")
    bf16, i32 = torch.bfloat16, torch.int32
    for l in range(L):
        q, kv, bt, sl = queries[l], kv_caches[l], block_tables[l], seq_lens[l]
        if not (q.dtype is bf16 and q.device == device and q.shape == q_shape and q.is_contiguous()):
            _refuse("query", q, f"a contiguous bf16 [{B}, {Hq}, {D}] tensor on {device}")
        if not (kv.dtype is bf16 and kv.device == device and kv.shape[1:] == kv_shape[1:] and kv.is_contiguous()):
            _refuse("kv_cache", kv, f"a contiguous bf16 [num_blocks, 2, {page}, {Hkv}, {D}] tensor on {device}")
        if not (bt.dtype is i32 and bt.device == device and bt.dim() == 2 and bt.shape[0] >= B and bt.is_contiguous()):
            _refuse("block_table", bt, f"a contiguous int32 [>={B}, max_pages] tensor on {device}")
        if not (sl.dtype is i32 and sl.device == device and sl.dim() == 1 and sl.shape[0] >= B and sl.is_contiguous()):
            _refuse("seq_lens", sl, f"a contiguous int32 [>={B}] tensor on {device}")
        if outputs is not None:
            o = outputs[l]
            if not (o.dtype is bf16 and o.device == device and o.shape == q_shape and o.is_contiguous()):
                _refuse("output", o, f"a contiguous bf16 [{B}, {Hq}, {D}] tensor on {device}")
    windows, sinks = _per_layer("window", window, L), _per_layer("num_sinks", num_sinks, L)
    if max_pages_per_seq is None:
        max_pages_per_seq = max([bt.shape[1] for bt in block_tables])
    units, rows = (1, 0) if weights is None else _check_weights(weights, L, B, Hkv, device)
    with call_scope(device, stream):
        outs = list(outputs) if outputs is not None else [torch.empty_like(q) for q in queries]
        if B == 0:
            return outs
        need, win, snk = _window_plan(L, B, Hq, Hkv, D, page, max_pages_per_seq, chunk_tokens, windows, sinks,
                                      0 if weights is None else units)
        if need == 0:
            raise _lib.AbkvError("abkv_decode_window_workspace_size", 3,
                                 f"unsupported shape (B={B}, Hq={Hq}, Hkv={Hkv}, D={D}, page={page}, "
                                 f"max_pages_per_seq={max_pages_per_seq}, chunk_tokens={chunk_tokens})")
        ws, raw = call_workspace(device, need, workspace)
        ptrs = _lib.data_ptrs
        st = _lib.lib().abkv_decode_window(
            ptrs(queries), ptrs(kv_caches), ptrs(block_tables), _lib.i64(*[bt.shape[1] for bt in block_tables]),
            ptrs(seq_lens), _lib.i64(*[kv.shape[0] for kv in kv_caches]), ptrs(outs), L, B, Hq, Hkv, D, page,
            max_pages_per_seq, 1.0 / math.sqrt(D) if scale is None else scale, chunk_tokens, win, snk,
            None if weights is None else ptrs(weights),
            None if weights is None else _lib.i64(*[x for w in weights for x in w.stride()[:2]]), rows, units,
            ws.ptr(), ws.nbytes, raw)
    if st:
        _lib.check("abkv_decode_window", st)
    return outs


def paged_decode_window(
    queries: Sequence[torch.Tensor],
    kv_caches: Sequence[torch.Tensor],
    block_tables: Sequence[torch.Tensor],
    seq_lens: Sequence[torch.Tensor],
    *,
    window: int | None | Sequence[int | None],
    num_sinks: int | Sequence[int] = 0,
    scale: float | None = None,
    outputs: Sequence[torch.Tensor] | None = None,
    max_pages_per_seq: int | None = None,
    chunk_tokens: int = 0,
    workspace: Workspace | None = None,
    stream: torch.cuda.Stream | None = None,
) -> list[torch.Tensor]:
    """``paged_decode`` under a sliding window with sinks (``abkv_decode_window``): the query of a
    sequence of n rows sees its last ``window`` rows (its own among them) and its first
    ``num_sinks`` rows.  ``window`` and ``num_sinks`` are one number, or one per layer; a window of
    None or 0 shows every row, so layers with and without a window share a launch.  Pages that hold
    no visible row are never read, and their block-table entries may be stale (freed pages).

    The launch is laid out for the most rows that a sequence can show: the window and the sinks, or without a window
    ``max_pages_per_seq`` pages (None: the block tables' width).  Where the tables are much wider than the
    longest sequence, pass that sequence's pages (a longer one would be cut): the work is then split for
    them, and a weighted call's scores take 4 x sequences x query heads x those rows bytes of workspace a layer
    instead of the table's."""
    return _decode_window(queries, kv_caches, block_tables, seq_lens, None, window, num_sinks, scale, outputs,
                          max_pages_per_seq, chunk_tokens, workspace, stream)


def paged_decode_weighted(
    queries: Sequence[torch.Tensor],
    kv_caches: Sequence[torch.Tensor],
    block_tables: Sequence[torch.Tensor],
    seq_lens: Sequence[torch.Tensor],
    weights: Sequence[torch.Tensor],
    *,
    window: int | None | Sequence[int | None] = None,
    num_sinks: int | Sequence[int] = 0,
    scale: float | None = None,
    outputs: Sequence[torch.Tensor] | None = None,
    max_pages_per_seq: int | None = None,
    chunk_tokens: int = 0,
    workspace: Workspace | None = None,
    stream: torch.cuda.Stream | None = None,
) -> list[torch.Tensor]:
    """``paged_decode_window`` that also adds every visible row's attention weight to ``weights``.

    weights[l]: fp32 [>=B, units, rows], rows contiguous and at least as many as the longest
    sequence (a longer sequence sets the workspace's SEQ_OOB bit and is cut): with units = Hkv,
    unit u collects KV head u's query heads; with units = 1, all query heads.  The sums are taken in
    head order, so repeated calls give the same bits.  ``compaction.evict_by_weight`` reads them.
    ``max_pages_per_seq``: see ``paged_decode_window``; it matters most here."""
    return _decode_window(queries, kv_caches, block_tables, seq_lens, list(weights), window, num_sinks, scale,
                          outputs, max_pages_per_seq, chunk_tokens, workspace, stream)


def attend_decode_batched(
    *,
    query: torch.Tensor,
    kv_cache: torch.Tensor,
    output: torch.Tensor,
    seq_lens: torch.Tensor,
    block_table: torch.Tensor,
    num_kv_heads: int,
    groups: int,
    scale: float,
    num_requests: int | None = None,
    workspace: Workspace | None = None,
) -> None:
    """Drop-in for ``PackedKVSidecar._attend_decode_batched`` (no sidecar pages).

    query: [>=n, Hq, D] (or [>=n, Hq*D]); output: same shape, written for the
    first n rows in place.  ``seq_lens`` may live on the host (vLLM's
    ``_seq_lens_cpu``); it is copied to the device when needed.
    """
    n = int(num_requests if num_requests is not None else block_table.shape[0])
    D = kv_cache.shape[-1]
    Hq = num_kv_heads * groups
    q = query[:n].reshape(n, Hq, D)
    if not q.is_contiguous():
        q = q.contiguous()
    sl = seq_lens[:n]
    if not sl.is_cuda:
        sl = sl.to(kv_cache.device, non_blocking=True)
    sl = sl.to(torch.int32).contiguous()
    bt = block_table[:n]
    if bt.dtype != torch.int32 or not bt.is_contiguous():
        bt = bt.to(torch.int32).contiguous()
    out_view = output[:n].reshape(n, Hq, D)
    direct = out_view.is_contiguous() and out_view.dtype == torch.bfloat16
    o = out_view if direct else torch.empty((n, Hq, D), dtype=torch.bfloat16, device=kv_cache.device)
    paged_decode([q], [kv_cache], [bt], [sl], scale=scale, outputs=[o], workspace=workspace)
    if not direct:
        out_view.copy_(o)


def forward_decode(
    query: torch.Tensor,
    kv_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    scale: float,
    output: torch.Tensor | None = None,
    workspace: Workspace | None = None,
) -> torch.Tensor:
    """vLLM ``AttentionImpl.forward``-shaped decode for one layer:
    query [T, Hq, D] (T = one decode row per request), output [T, Hq*D]."""
    T, Hq, D = query.shape
    if output is None:
        output = torch.empty((T, Hq * D), dtype=query.dtype, device=query.device)
    Hkv = kv_cache.shape[3]
    attend_decode_batched(query=query, kv_cache=kv_cache, output=output, seq_lens=seq_lens,
                          block_table=block_table, num_kv_heads=Hkv, groups=Hq // Hkv,
                          scale=scale, num_requests=T, workspace=workspace)
    return output
