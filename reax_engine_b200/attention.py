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
import struct

import torch
from torch.autograd import forward_ad

from . import _lib as L
from .moe import _require_cuda

_DTYPES = {torch.bfloat16: L.BF16, torch.float16: L.FP16}

# What the checks of a call found for one set of shapes, strides, types and options (of tensors that need no copy): the argument
# block behind its pointers and the workspace's size. Emptied when the SM budget changes, on which the size depends.
_checked: dict = {}
_unused: dict = {}        # device number -> the workspace of calls that use none
_CHECKED_MAX = 4096
_status: dict = {}        # device number -> the status word of calls that are given none, and its address
_POINTERS = struct.Struct("10Q")     # q, k, v, prefix_k, prefix_v, cu_q, cu_k, out, lse, status: the first of AttentionArgs
_UNUSED = 16             # a workspace of this size is never touched (reaxmoe_attention_workspace_size)


def forget_checked() -> None:
    _checked.clear()


def attention_status(device: torch.device | str | int | None = None, clear: bool = True) -> int:
    """Synchronise the current stream of ``device`` (default: the current one) and return the status word of the attention calls
    there that were given none: 0, or the code of a bounded wait that ran out in one of them, whose output is then not whole."""
    device = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError("attention runs on CUDA devices")
    word, _ = _status.get(torch.cuda.current_device() if device.index is None else device.index, (None, 0))
    if word is None:
        return 0
    code = int(word)
    if clear and code:
        word.zero_()
    return code


def _default_status(device: torch.device) -> int:
    """The address of the device's status word: none before the first call of a process that is not being captured (which could
    not zero it)."""
    if torch.cuda.is_current_stream_capturing():
        return 0
    word = torch.zeros(1, dtype=torch.int32, device=device)
    _status[device.index] = word, word.data_ptr()
    return word.data_ptr()


def _readable(t: torch.Tensor) -> bool:
    """t [tokens, heads, dim] as the kernels can address it: rows of contiguous elements that start on 16 bytes and do not
    overlap (a view of a fused projection is)."""
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    return (s2 == 1 and t.data_ptr() % 16 == 0 and s0 % 8 == 0 and s1 % 8 == 0 and (h <= 1 or s1 >= d)
            and (n <= 1 or s0 >= d))


def _heads(t: torch.Tensor) -> torch.Tensor:
    return t if _readable(t) else t.clone(memory_format=torch.contiguous_format)


def _lengths(cu: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if cu.dtype is torch.int32 and cu.ndim == 1 and cu.device == device and cu.is_contiguous() and cu.numel() > 0:
        return cu
    if cu.ndim != 1 or cu.numel() < 1 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 [sequences + 1]")
    if cu.device != device:
        raise ValueError(f"{name} is on {cu.device}, q on {device}")
    return cu.to(torch.int32).contiguous()


def _output(out: torch.Tensor, q: torch.Tensor, inputs) -> torch.Tensor:
    """What the kernels write for the caller's `out`: itself, or a copy where its rows cannot be addressed."""
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have the shape, dtype and device of q")
    if out.numel() and any(out.untyped_storage().data_ptr() == t.untyped_storage().data_ptr() for t in inputs):   # (none: 0)
        raise ValueError("out must not share its storage with an input")
    if out.ndim != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    s0, s1, s2 = out.stride()
    ok = s2 == 1 and out.data_ptr() % 16 == 0 and s0 % 8 == 0 and s1 % 8 == 0
    return out if ok else out.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, prefix_k, prefix_v, seqs, seqs_k, dst, scale, causal, window):
    """The argument block of these tensors behind its pointers, and the workspace's size."""
    ts = [("q", q), ("k", k), ("v", v)] + ([] if prefix_k is None else [("prefix_k", prefix_k), ("prefix_v", prefix_v)])
    if q.dtype not in _DTYPES:
        raise ValueError(f"q must be bf16 or fp16, not {q.dtype}")
    for n, t in ts:
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{n} must have the dtype and device of q")
        if t.shape[2] != q.shape[2] or (n != "q" and t.shape[1] != k.shape[1]):
            raise ValueError(f"{n} {tuple(t.shape)} does not go with q {tuple(q.shape)} and k {tuple(k.shape)}")
    if k.shape[0] != v.shape[0] or (prefix_k is not None and prefix_k.shape[0] != prefix_v.shape[0]):
        raise ValueError("keys and values must have the same number of tokens")
    d = q.shape[2]
    scale = d ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if window is not None and (not causal or window < 1):
        raise ValueError("window must be at least 1, with causal=True")
    if seqs_k != seqs:
        raise ValueError("cu_seqlens and cu_seqlens_k must have the same length")
    strides = [x for t in (q, k, v, prefix_k, prefix_v, dst) for x in ((0, 0) if t is None else t.stride()[:2])]
    args = L.AttentionArgs(*([None] * 10), *strides, q.shape[0], k.shape[0], 0 if prefix_k is None else prefix_k.shape[0],
                           seqs - 1, q.shape[1], k.shape[1], d, _DTYPES[q.dtype], int(causal),
                           0 if window is None else min(window, 0x7FFFFFFF), scale)
    need = L.lib().reaxmoe_attention_workspace_size(ctypes.byref(args))
    if need == 0:
        raise L.ReaxMoEError(L.ERR_BAD_SHAPE, L.last_error())
    return bytes(args)[_POINTERS.size:], need


def _no_gradients(ts) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t.requires_grad:
                raise ValueError("this attention has no backward: detach its inputs or call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ValueError("this attention has no forward-mode derivative: unpack its inputs")


def _aligned(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0


def _attention(q, k, v, prefix_k, prefix_v, cu_seqlens, cu_seqlens_k, scale, causal, window, return_lse, out, workspace, status):
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError("prefix_k and prefix_v go together")
    device = q.device
    if device.type != "cuda":
        _require_cuda(q)
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _attention(q, k, v, prefix_k, prefix_v, cu_seqlens, cu_seqlens_k, scale, causal, window, return_lse, out,
                              workspace, status)
    index = device.index
    ts = (q, k, v) if prefix_k is None else (q, k, v, prefix_k, prefix_v)
    if q.requires_grad or k.requires_grad or v.requires_grad or prefix_k is not None or forward_ad._current_level >= 0:
        _no_gradients(ts)
    cu_q = _lengths(cu_seqlens, "cu_seqlens", device)
    cu_k = cu_q if cu_seqlens_k is None else _lengths(cu_seqlens_k, "cu_seqlens_k", device)
    shape = q.shape
    if out is None:
        if len(shape) != 3:
            raise ValueError("q must be [tokens, heads, head_dim]")
        dst = torch.empty_strided(shape, (shape[1] * shape[2], shape[2], 1), dtype=q.dtype, device=device)
    else:
        dst = _output(out, q, ts)
    if status is None:
        found = _status.get(index)
        status_at = _default_status(device) if found is None else found[1]
    elif status.dtype != torch.int32 or status.device != device or status.numel() < 1:
        raise ValueError("status must be an int32 tensor on the device of q")
    else:
        status_at = status.data_ptr()
    if scale is not None:
        scale = float(scale)
    if window is not None:
        window = int(window)
    causal = bool(causal)           # values, not what held them: they are part of the key below
    key = (device, shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device,
           dst.stride(), cu_q.shape, cu_k.shape, scale, causal, window)
    aligned = _aligned(q) and _aligned(k) and _aligned(v)
    if prefix_k is not None:
        key += (prefix_k.shape, prefix_k.stride(), prefix_k.dtype, prefix_k.device, prefix_v.shape, prefix_v.stride(),
                prefix_v.dtype, prefix_v.device)
        aligned = aligned and _aligned(prefix_k) and _aligned(prefix_v)
    found = _checked.get(key) if aligned else None
    if found is None:
        for t in ts:
            _require_cuda(t)
            if t.ndim != 3:
                raise ValueError("q, k, v and the prefix must be [tokens, heads, head_dim]")
        as_they_are = all(map(_readable, ts))
        q, k, v = _heads(q), _heads(k), _heads(v)
        if prefix_k is not None:
            prefix_k, prefix_v = _heads(prefix_k), _heads(prefix_v)
        found = _check(q, k, v, prefix_k, prefix_v, cu_q.numel(), cu_k.numel(), dst, scale, causal, window)
        if as_they_are:
            if len(_checked) >= _CHECKED_MAX:
                _checked.clear()
            _checked[key] = found
    block, need = found
    lse = torch.empty_strided(shape[:2], (shape[1], 1), dtype=torch.float32, device=device) if return_lse else None
    if workspace is None:
        if need <= _UNUSED:
            workspace = _unused.get(index)
            if workspace is None:
                workspace = _unused[index] = torch.empty(_UNUSED, dtype=torch.uint8, device=device)
        else:
            # of this call alone: ordered with the stream, and private to a graph that is being captured
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        nbytes = need
    else:
        if workspace.device != device or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous and on the device of q")
        nbytes = workspace.numel() * workspace.element_size()
    args = L.AttentionArgs.from_buffer_copy(_POINTERS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if prefix_k is None else prefix_k.data_ptr(),
        0 if prefix_k is None else prefix_v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), dst.data_ptr(),
        0 if lse is None else lse.data_ptr(), status_at) + block)
    rc = L.lib().reaxmoe_attention(ctypes.byref(args), workspace.data_ptr(), nbytes, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        L.check(rc)
    if out is None:
        out = dst
    elif dst is not out:
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
    change it, whatever they hold (but infinities and NaN beside its keys make it slow: it is done again). ``scale`` defaults
    to d ** -0.5. Returns o like q, written into ``out`` where given (of a storage of its own; rows at and behind cu_seqlens[-1]
    are left as they were; without ``out`` their values are undefined), and with ``return_lse`` the natural logarithm of the
    softmax's sum [tokens, heads] fp32 too.

    ``workspace``: a uint8 buffer of at least ``reaxmoe_attention_workspace_size`` bytes, used by one call at a time (default:
    one from torch's allocator for this call). ``status``: an int32 device tensor that receives a device-timeout code if a bounded
    wait of the kernel runs out, in which case rows of the output are missing (default: a word per device,
    :func:`attention_status`; none where a process's first call is captured).
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
