"""Pause-token prefill attention with the compressed-cache mask (host side).

``prefill_masked`` runs ``abkv_prefill_masked`` (tcgen05 tensor cores) on
q [B, H, S, D], k/v [B, Hkv, S, D] bf16 CUDA tensors (last dim contiguous,
other strides free), evaluating CompressLM._arith_mask_mod
(abridgekv/compress_forward.py:695-727) arithmetically per tile from
(C, K_layout, per-query-head quotas, per-sequence raw-prompt lengths) instead of
materialising a BlockMask.

``abkv_attention_forward`` has the signature of transformers'
``flex_attention_forward`` (the attention function CompressLM forces with
``_attn_implementation = "flex_attention"``, compress_forward.py:248) and is
registered under the name ``"abkv_sm100"``.  It expects ``attention_mask`` to
be a :class:`CompressMask` descriptor (or a :class:`WindowMask` for a layer
under a causal sliding window with sinks, ``window_attention``): CompressLM's per-layer dispatch hook
(compress_forward.py:557-564) can hand each layer its own descriptor exactly as
it hands each layer its own BlockMask today.
"""
from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import Sequence

import torch

from . import _lib
from .workspace import Workspace, call_scope, call_workspace, default_workspace

TILE = 128


@dataclass(frozen=True)
class CompressMask:
    """The arithmetic mask of one layer: block layout [C content | K_layout codes],
    per-query-head code quotas (None = all K_layout slots) and optional raw
    prompt lengths [B] (int32 CUDA tensor)."""

    C: int
    K_layout: int
    quota_per_head: tuple[int, ...] | None = None
    prompt_len: torch.Tensor | None = None


def _check(name: str, t: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be a bf16 CUDA tensor (libabkv has no CPU path)")
    if t.dim() != 4 or t.stride(3) != 1:
        raise ValueError(f"{name} must be 4-D with a contiguous last dimension")


def prefill_masked(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, C: int, K_layout: int,
                   quota_per_head: Sequence[int] | None = None, prompt_len: torch.Tensor | None = None,
                   scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False,
                   workspace: Workspace | None = None, stream: torch.cuda.Stream | None = None):
    _check("query", q)
    _check("key", k)
    _check("value", v)
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    if tuple(k.shape) != (B, Hkv, S, D) or tuple(v.shape) != (B, Hkv, S, D):
        raise ValueError("key/value must be [B, Hkv, S, D] matching the query")
    if out is None:
        out = torch.empty((B, S, H, D), dtype=torch.bfloat16, device=q.device).transpose(1, 2)
    _check("out", out)
    if tuple(out.shape) != (B, H, S, D):
        raise ValueError("out must be [B, H, S, D] (any strides, last dim contiguous)")
    lse = torch.empty((B, H, S), dtype=torch.float32, device=q.device) if return_lse else None
    pl = None
    if prompt_len is not None:
        pl = prompt_len.to(device=q.device, dtype=torch.int32).contiguous()
        if pl.numel() != B:
            raise ValueError("prompt_len must hold one length per sequence")
    if quota_per_head is not None and len(quota_per_head) != H:
        raise ValueError("quota_per_head must hold one quota per query head")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    ws = workspace or default_workspace(q.device)
    s = torch.cuda.current_stream(q.device) if stream is None else stream
    strides = lambda t: _lib.i64_array([t.stride(0), t.stride(1), t.stride(2)])  # noqa: E731
    quota = _lib.i32_array(quota_per_head) if quota_per_head is not None else None
    with torch.cuda.device(q.device):
        st = _lib.lib().abkv_prefill_masked(
            q.data_ptr(), strides(q), k.data_ptr(), strides(k), v.data_ptr(), strides(v), out.data_ptr(),
            strides(out), lse.data_ptr() if lse is not None else None, quota,
            pl.data_ptr() if pl is not None else None, B, H, Hkv, S, D, C, K_layout, scale, ws.ptr(),
            ws.nbytes, s.cuda_stream)
    _lib.check("abkv_prefill_masked", st)
    return (out, lse) if return_lse else out


def prefill_masked_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                            dout: torch.Tensor, lse: torch.Tensor, *, C: int, K_layout: int,
                            quota_per_head: Sequence[int] | None = None, prompt_len: torch.Tensor | None = None,
                            scale: float | None = None, workspace: Workspace | None = None,
                            stream: torch.cuda.Stream | None = None):
    """Gradients (dq, dk, dv) of ``prefill_masked`` for the upstream gradient ``dout``, from the
    forward's output and log-sum-exp (abkv_prefill_masked_backward)."""
    for name, t in (("query", q), ("key", k), ("value", v), ("out", out), ("dout", dout)):
        _check(name, t)
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    if tuple(out.shape) != (B, H, S, D) or tuple(dout.shape) != (B, H, S, D):
        raise ValueError("out and dout must be [B, H, S, D] like the query")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, S) or not lse.is_contiguous():
        raise ValueError("lse must be the forward's contiguous float32 [B, H, S] log-sum-exp")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for name, t in (("query", q), ("key", k), ("value", v), ("out", out), ("dout", dout), ("dq", dq), ("dk", dk),
                    ("dv", dv)):
        if t.data_ptr() % 16:
            raise ValueError(f"{name} must start on a 16-byte boundary")
    for name, t in (("out", out), ("dout", dout), ("dq", dq), ("dk", dk), ("dv", dv)):
        if any(t.stride(i) % 8 for i in range(3)):
            raise ValueError(f"{name} strides must be multiples of 8 elements, got {tuple(t.stride())}")
    pl = None
    if prompt_len is not None:
        pl = prompt_len.to(device=q.device, dtype=torch.int32).contiguous()
    if quota_per_head is not None and len(quota_per_head) != H:
        raise ValueError("quota_per_head must hold one quota per query head")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    lib = _lib.lib()
    need = lib.abkv_prefill_masked_backward_workspace_size(B, H, S, D)
    if need == 0:
        raise _lib.AbkvError("abkv_prefill_masked_backward_workspace_size", 3, f"unsupported shape D={D}")
    ws = (workspace or default_workspace(q.device)).ensure(need)
    s = torch.cuda.current_stream(q.device) if stream is None else stream
    strides = lambda t: _lib.i64_array([t.stride(0), t.stride(1), t.stride(2)])  # noqa: E731
    quota = _lib.i32_array(quota_per_head) if quota_per_head is not None else None
    with torch.cuda.device(q.device):
        st = lib.abkv_prefill_masked_backward(
            q.data_ptr(), strides(q), k.data_ptr(), strides(k), v.data_ptr(), strides(v), out.data_ptr(),
            strides(out), dout.data_ptr(), strides(dout), lse.data_ptr(), dq.data_ptr(), strides(dq), dk.data_ptr(),
            strides(dk), dv.data_ptr(), strides(dv), quota, pl.data_ptr() if pl is not None else None, B, H, Hkv,
            S, D, C, K_layout, scale, ws.ptr(), ws.nbytes, s.cuda_stream)
    _lib.check("abkv_prefill_masked_backward", st,
               f"B={B} H={H} Hkv={Hkv} S={S} D={D} C={C} K_layout={K_layout} scale={scale} "
               f"quota={None if quota_per_head is None else list(quota_per_head)} "
               f"strides q{tuple(q.stride())} k{tuple(k.stride())} out{tuple(out.stride())} "
               f"dout{tuple(dout.stride())} dq{tuple(dq.stride())} dk{tuple(dk.stride())}")
    return dq, dk, dv


class PrefillMaskedAttention(torch.autograd.Function):
    """prefill_masked with its backward: the forward keeps its output and log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, C, K_layout, quota_per_head, prompt_len, scale):
        out, lse = prefill_masked(q, k, v, C=C, K_layout=K_layout, quota_per_head=quota_per_head,
                                  prompt_len=prompt_len, scale=scale, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.args = (C, K_layout, quota_per_head, prompt_len, scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        C, K_layout, quota, pl, scale = ctx.args
        if dout.stride(-1) != 1:
            dout = dout.contiguous()
        dq, dk, dv = prefill_masked_backward(q, k, v, out, dout, lse, C=C, K_layout=K_layout, quota_per_head=quota,
                                             prompt_len=pl, scale=scale)
        return dq, dk, dv, None, None, None, None, None


def prefill_masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, C: int, K_layout: int,
                             quota_per_head: Sequence[int] | None = None, prompt_len: torch.Tensor | None = None,
                             scale: float | None = None) -> torch.Tensor:
    """Differentiable ``prefill_masked`` (forward and backward on the tcgen05 kernels)."""
    return PrefillMaskedAttention.apply(q, k, v, C, K_layout, quota_per_head, prompt_len, scale)


@dataclass(frozen=True)
class WindowMask:
    """A causal sliding window with sinks: row i sees keys j <= i with j > i - window or j < num_sinks."""

    window: int
    num_sinks: int = 0


def _window_args(q, k, v, window, num_sinks, scale):
    for name, t in (("query", q), ("key", k), ("value", v)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or not t.is_cuda:
            raise TypeError(f"{name} must be a bf16 CUDA tensor (libabkv has no CPU path)")
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D")
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (B, Hkv, S, D) or v.shape != k.shape:
        raise ValueError("key/value must be [B, Hkv, S, D] matching the query")
    if Hkv == 0 or H % Hkv:
        raise ValueError("the KV heads must divide the query heads")
    if k.device != q.device or v.device != q.device:
        raise ValueError("key and value must be on the query's device")
    window, num_sinks = int(window), int(num_sinks)
    if not (1 <= window <= 0x7FFFFFFF and 0 <= num_sinks <= 0x7FFFFFFF):
        raise ValueError(f"window must be at least 1 and num_sinks at least 0, got {window} and {num_sinks}")
    return window, num_sinks, 1.0 / math.sqrt(D) if scale is None else float(scale)


def _tma_ready(t: torch.Tensor) -> tuple[torch.Tensor, "_lib.C.Array"]:
    """t and its element strides (batch, head, seq), where the copy engine can address it (16-byte rows and
    base, no broadcast dimension); else a contiguous copy and its strides."""
    a, b, c, d = t.stride()
    if d != 1 or (a | b | c) % 8 or not a * b * c or t.data_ptr() % 16:
        n = t.shape
        ok = d == 1 and t.data_ptr() % 16 == 0 and all(
            n[i] == 1 or (x > 0 and x % 8 == 0) for i, x in enumerate((a, b, c)))
        if not ok:
            t = t.clone(memory_format=torch.contiguous_format)
            a, b, c, _ = t.stride()
        # the stride of a dimension of one element addresses nothing: any legal one will do
        a, b, c = (n[1] * n[2] * n[3] if n[i] == 1 else x for i, x in enumerate((a, b, c)))
    return t, _lib.i64(a, b, c)


def window_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int, num_sinks: int = 0,
                   scale: float | None = None, return_lse: bool = False, return_low: bool = False,
                   workspace: Workspace | None = None, stream: torch.cuda.Stream | None = None):
    """Causal attention under a sliding window with sinks (``abkv_window_attention``): row i sees keys
    j <= i with j > i - window or j < num_sinks.  q [B, H, S, D], k/v [B, Hkv, S, D] bf16 (any strides;
    what the copy engine cannot address is copied first), D 64 or 128, any S up to 131072, finite values.
    Returns out [B, H, S, D] (stored as [B, S, H, D]), then lse [B, H, S] fp32 with ``return_lse``, then with
    ``return_low`` the output's next eight mantissa bits ([B, H, S, D] int8, for ``window_backward``)."""
    window, num_sinks, scale = _window_args(q, k, v, window, num_sinks, scale)
    B, H, S, D = q.shape
    device = q.device
    with call_scope(device, stream):
        out = q.new_empty((B, S, H, D)).transpose(1, 2)
        lse = q.new_empty((B, H, S), dtype=torch.float32) if return_lse else None
        low = q.new_empty((B, H, S, D), dtype=torch.int8) if return_low else None
        if B * H * S:
            (q, qs), (k, ks), (v, vs) = _tma_ready(q), _tma_ready(k), _tma_ready(v)
            os = _lib.i64(S * H * D, D, H * D)
            ws, raw = call_workspace(device, 256, workspace)
            st = _lib.lib().abkv_window_attention(
                q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(), os,
                low.data_ptr() if return_low else None, lse.data_ptr() if return_lse else None, B, H, k.shape[1], S, D,
                scale, window, num_sinks, ws.ptr(), ws.nbytes, raw)
            if st:
                _lib.check("abkv_window_attention", st)
    extra = tuple(t for t in (lse, low) if t is not None)
    return (out, *extra) if extra else out


def window_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, dout: torch.Tensor,
                    lse: torch.Tensor, *, window: int, num_sinks: int = 0, scale: float | None = None,
                    low: torch.Tensor | None = None, workspace: Workspace | None = None,
                    stream: torch.cuda.Stream | None = None):
    """Gradients (dq, dk, dv) of ``window_forward`` for the upstream gradient ``dout``, from the forward's
    output, log-sum-exp and (optionally) the output's low bits (``abkv_window_attention_backward``).  Repeated
    calls give the same bits."""
    window, num_sinks, scale = _window_args(q, k, v, window, num_sinks, scale)
    shape, device = q.shape, q.device
    for name, t in (("out", out), ("dout", dout)):
        if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be a bf16 tensor on the query's device")
        if t.shape != shape:
            raise ValueError("out and dout must be [B, H, S, D] like the query")
    if lse.dtype != torch.float32 or lse.shape != shape[:3] or not lse.is_contiguous() or lse.device != device:
        raise ValueError("lse must be the forward's contiguous float32 [B, H, S] log-sum-exp")
    if low is not None and (low.dtype != torch.int8 or low.shape != shape or not low.is_contiguous() or
                            low.device != device):
        raise ValueError("low must be the forward's contiguous int8 [B, H, S, D] low bits")
    with call_scope(device, stream):
        return _window_backward(q, k, v, out, dout, lse, low, window, num_sinks, scale, workspace)


@functools.lru_cache(maxsize=256)
def _window_backward_bytes(B: int, H: int, S: int, D: int) -> int:
    need = _lib.lib().abkv_window_attention_backward_workspace_size(B, H, S, D)
    if need == 0:
        raise _lib.AbkvError("abkv_window_attention_backward_workspace_size", 3, f"unsupported shape D={D}")
    return need


def _window_backward(q, k, v, out, dout, lse, low, window, num_sinks, scale, workspace=None):
    """The launch, on checked arguments and the current stream."""
    B, H, S, D = q.shape
    (q, qs), (k, ks), (v, vs) = _tma_ready(q), _tma_ready(k), _tma_ready(v)
    (out, os), (dout, ds) = _tma_ready(out), _tma_ready(dout)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    if B * H * S == 0:
        return dq, dk, dv
    ws, raw = call_workspace(q.device, _window_backward_bytes(B, H, S, D), workspace)
    # empty_like keeps the strides of a dense tensor; of others it makes its own
    dqs = qs if dq.stride() == q.stride() else _tma_ready(dq)[1]
    dks = ks if dk.stride() == k.stride() else _tma_ready(dk)[1]
    dvs = vs if dv.stride() == v.stride() else _tma_ready(dv)[1]
    st = _lib.lib().abkv_window_attention_backward(
        q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(), os,
        low.data_ptr() if low is not None else None, dout.data_ptr(), ds, lse.data_ptr(), dq.data_ptr(), dqs,
        dk.data_ptr(), dks, dv.data_ptr(), dvs, B, H, k.shape[1], S, D, scale, window, num_sinks, ws.ptr(), ws.nbytes,
        raw)
    if st:
        _lib.check("abkv_window_attention_backward", st)
    return dq, dk, dv


class WindowAttention(torch.autograd.Function):
    """window_forward with its backward: the forward keeps its output and log-sum-exp."""

    @staticmethod
    def forward(ctx, q, k, v, window, num_sinks, scale):
        out, lse, low = window_forward(q, k, v, window=window, num_sinks=num_sinks, scale=scale, return_lse=True,
                                       return_low=True)
        ctx.save_for_backward(q, k, v, out, lse, low)
        ctx.args = (int(window), int(num_sinks), 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale))
        return out

    def _gradients(ctx, dout):
        q, k, v, out, lse, low = ctx.saved_tensors
        with call_scope(q.device, None):
            return (*_window_backward(q, k, v, out, dout, lse, low, *ctx.args), None, None, None)

    _once = staticmethod(torch.autograd.function.once_differentiable(_gradients))

    @staticmethod
    def backward(ctx, dout):
        # what marks the gradients as not differentiable again is only needed under create_graph
        return WindowAttention._once(ctx, dout) if torch.is_grad_enabled() else WindowAttention._gradients(ctx, dout)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int, num_sinks: int = 0,
                     scale: float | None = None) -> torch.Tensor:
    """Differentiable ``window_forward`` (forward and backward on the tcgen05 kernels).  To capture forward
    and backward into a CUDA graph, release any eager autograd graph of the same leaf tensors first (torch
    ends the capture otherwise, as for every operator)."""
    return WindowAttention.apply(q, k, v, window, num_sinks, scale)


def abkv_attention_forward(module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                           attention_mask, scaling: float | None = None, dropout: float = 0.0,
                           softcap: float | None = None, s_aux=None, **kwargs):
    """transformers AttentionInterface function: (attn_output [B, S, H, D], None)."""
    if not isinstance(attention_mask, (CompressMask, WindowMask)):
        raise TypeError("abkv_sm100 attention needs a CompressMask (or WindowMask) descriptor as attention_mask")
    if dropout != 0.0 or softcap is not None or s_aux is not None:
        raise ValueError("abkv_sm100 attention supports no dropout, softcap or learned sink logits")
    if isinstance(attention_mask, WindowMask):
        kw = dict(window=attention_mask.window, num_sinks=attention_mask.num_sinks, scale=scaling)
        train = torch.is_grad_enabled() and any(t.requires_grad for t in (query, key, value))
        out = (window_attention if train else window_forward)(query, key, value, **kw)
        return out.transpose(1, 2), None
    kw = dict(C=attention_mask.C, K_layout=attention_mask.K_layout,
              quota_per_head=attention_mask.quota_per_head, prompt_len=attention_mask.prompt_len, scale=scaling)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (query, key, value)):
        out = prefill_masked_attention(query, key, value, **kw)  # training: gradients through the backward kernel
    else:
        out = prefill_masked(query, key, value, **kw)
    return out.transpose(1, 2), None


def register(name: str = "abkv_sm100") -> str:
    """Register abkv_attention_forward with transformers' AttentionInterface."""
    from transformers import AttentionInterface

    AttentionInterface.register(name, abkv_attention_forward)
    return name
