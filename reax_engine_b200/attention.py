"""Attention over packed sequences of different lengths, and over a prefix that a whole batch shares.

* :func:`prompt_attention`: causal attention with grouped heads and an optional sliding window over packed prompts, as
  ``Gemma4Attention.forward`` runs it (``vllm/model_executor/models/gemma4.py:505-539``); one query row per sequence (the last
  rows of a decision forward, a step of generation) is the same call.
* :func:`shared_prefix_attention`: the same for a batch whose sequences all continue one prefix, whose keys and values are
  stored, read and multiplied once for all of them.

Both run in ``libreaxmoe.so`` (``reaxmoe_attention``); there is no CPU or eager fallback. They take no part in autograd.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L
from .moe import _ptr, _require_cuda, _stream

_DTYPES = {torch.bfloat16: L.BF16, torch.float16: L.FP16}


def _heads(t: torch.Tensor) -> torch.Tensor:
    """t [tokens, heads, dim] as the kernels can read it: rows of contiguous elements that start on 16 bytes and do not
    overlap (a view of a fused projection is); anything else is copied."""
    n, h, d = t.shape
    ok = (t.stride(2) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0
          and (h <= 1 or t.stride(1) >= d) and (n <= 1 or t.stride(0) >= d))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _lengths(cu: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if cu.ndim != 1 or cu.numel() < 1 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 [sequences + 1]")
    if cu.device != device:
        raise ValueError(f"{name} is on {cu.device}, q on {device}")
    return cu.to(torch.int32).contiguous()


def _attention(q, k, v, prefix_k, prefix_v, cu_seqlens, cu_seqlens_k, scale, causal, window, return_lse, out, workspace, status):
    ts = [("q", q), ("k", k), ("v", v)] + ([] if prefix_k is None else [("prefix_k", prefix_k), ("prefix_v", prefix_v)])
    _require_cuda(*[t for _, t in ts], cu_seqlens, cu_seqlens_k, out, workspace, status)
    if q.dtype not in _DTYPES:
        raise ValueError(f"q must be bf16 or fp16, not {q.dtype}")
    for n, t in ts:
        if t.ndim != 3:
            raise ValueError(f"{n} must be [tokens, heads, head_dim]")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{n} must have the dtype and device of q")
        if t.shape[2] != q.shape[2] or (n != "q" and t.shape[1] != k.shape[1]):
            raise ValueError(f"{n} {tuple(t.shape)} does not go with q {tuple(q.shape)} and k {tuple(k.shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{n} requires grad: this attention has no backward")
    if k.shape[0] != v.shape[0] or (prefix_k is not None and prefix_k.shape[0] != prefix_v.shape[0]):
        raise ValueError("keys and values must have the same number of tokens")
    d = q.shape[2]
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if window is not None and (not causal or int(window) < 1):
        raise ValueError("window must be at least 1, with causal=True")
    cu_q = _lengths(cu_seqlens, "cu_seqlens", q.device)
    cu_k = cu_q if cu_seqlens_k is None else _lengths(cu_seqlens_k, "cu_seqlens_k", q.device)
    if cu_k.numel() != cu_q.numel():
        raise ValueError("cu_seqlens and cu_seqlens_k must have the same length")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError("out must have the shape, dtype and device of q")
        if any(out.untyped_storage().data_ptr() == t.untyped_storage().data_ptr() for _, t in ts):
            raise ValueError("out must not share its storage with an input")
    if status is not None and (status.dtype != torch.int32 or status.device != q.device or status.numel() < 1):
        raise ValueError("status must be an int32 tensor on the device of q")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    q_, k_, v_ = _heads(q), _heads(k), _heads(v)
    pk = None if prefix_k is None else _heads(prefix_k)
    pv = None if prefix_v is None else _heads(prefix_v)
    ok = out.stride(2) == 1 and out.data_ptr() % 16 == 0 and out.stride(0) % 8 == 0 and out.stride(1) % 8 == 0
    dst = out if ok else out.clone(memory_format=torch.contiguous_format)
    strides = [x for t in (q_, k_, v_, pk, pv, dst) for x in ((0, 0) if t is None else (t.stride(0), t.stride(1)))]
    args = L.AttentionArgs(_ptr(q_), _ptr(k_), _ptr(v_), _ptr(pk), _ptr(pv), _ptr(cu_q), _ptr(cu_k), _ptr(dst), _ptr(lse),
                           _ptr(status), *strides, q.shape[0], k.shape[0], 0 if pk is None else pk.shape[0],
                           cu_q.numel() - 1, q.shape[1], k.shape[1], d, _DTYPES[q.dtype], int(bool(causal)),
                           0 if window is None else min(int(window), 0x7FFFFFFF), scale)
    with torch.cuda.device(q.device):
        need = L.lib().reaxmoe_attention_workspace_size(ctypes.byref(args))
        if need == 0:
            raise L.ReaxMoEError(L.ERR_BAD_SHAPE, L.last_error())
        if workspace is None:
            # of this call alone: ordered with the stream, and private to a graph that is being captured
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif workspace.device != q.device or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous and on the device of q")
        L.check(L.lib().reaxmoe_attention(ctypes.byref(args), workspace.data_ptr(),
                                          workspace.numel() * workspace.element_size(), _stream(q.device)))
    if dst is not out:
        out.copy_(dst)
    return (out, lse) if return_lse else out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, *, scale: float | None = None, causal: bool = True,
                     window: int | None = None, return_lse: bool = False, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """Attention of packed sequences: q [tokens, heads, d], k / v [key tokens, kv_heads, d], bf16 or fp16, d 64, 128 or 256,
    heads a multiple (at most 128) of kv_heads (query head h reads KV head h // (heads / kv_heads)). Sequence b holds query rows
    [cu_seqlens[b], cu_seqlens[b + 1]) and keys [cu_seqlens_k[b], cu_seqlens_k[b + 1]) (default: the same); the cumulative
    lengths are int32 on the device, and nothing is read back from it.

    The mask is aligned to the end of the keys: with m query rows and n keys, row i sees keys j <= n - m + i (``causal``), of
    those the last ``window`` ones; a row that sees none (m > n) gets 0 and lse -inf. Keys that a row does not see do not
    change it, whatever they hold. ``scale`` defaults to d ** -0.5. Returns o like q, written into ``out`` where given
    (rows at and behind cu_seqlens[-1] are left as they were; without ``out`` their values are undefined), and with
    ``return_lse`` the natural logarithm of the softmax's sum [tokens, heads] fp32 too.

    ``workspace``: a uint8 buffer of at least ``reaxmoe_attention_workspace_size`` bytes, used by one call at a time (default:
    one from torch's allocator for this call). ``status``: an optional int32 device tensor that receives a device-timeout code.
    """
    return _attention(q, k, v, None, None, cu_seqlens, cu_seqlens_k, scale, causal, window, return_lse, out, workspace, status)


def shared_prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor,
                            prefix_v: torch.Tensor, cu_seqlens: torch.Tensor, cu_seqlens_k: torch.Tensor | None = None, *,
                            scale: float | None = None, causal: bool = True, window: int | None = None,
                            return_lse: bool = False, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """:func:`prompt_attention` of a batch whose sequences all continue one prefix: prefix_k / prefix_v [prefix, kv_heads, d]
    stand before every sequence's own keys, so that with n own keys and m query rows, row i stands at position
    prefix + n - m + i and sees prefix and own keys up to there (the last ``window`` of them). The prefix is stored once, and
    its keys are read once for a whole tile of query rows, whichever sequences these are of."""
    return _attention(q, k, v, prefix_k, prefix_v, cu_seqlens, cu_seqlens_k, scale, causal, window, return_lse, out, workspace,
                      status)
