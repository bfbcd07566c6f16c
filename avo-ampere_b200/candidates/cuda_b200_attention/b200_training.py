"""The training side of attention: shared key/value heads and the gradient.

Host side of the entry points of include/avo_b200_attn.h that the forward contract does not
cover, in the manner of b200_attention.py (argument checks that raise ``RuntimeError``, the
current CUDA stream of the tensors' device, the device's status word, no fallback):

* ``grouped_attention``: the forward with H query heads over Hkv key/value heads and
  seq_q != seq_kv, differentiable through torch's autograd;
* ``attention_backward``: its gradient as a plain call.

Scratch is allocated per call by torch's caching allocator on the current stream, so calls
on several streams, and several captured graphs, share nothing but the status word.
"""

from __future__ import annotations

import contextlib
import ctypes
import importlib.util
import math
import sys
from pathlib import Path
from typing import Any

_BINDING = "avo_b200_attention_binding"


def _binding():
    module = sys.modules.get(_BINDING)
    if module is None:
        spec = importlib.util.spec_from_file_location(_BINDING, Path(__file__).resolve().parent / "b200_attention.py")
        module = importlib.util.module_from_spec(spec)
        sys.modules[_BINDING] = module
        spec.loader.exec_module(module)
    return module


b = _binding()
HEAD_DIM = b.HEAD_DIM


def _torch():
    import torch

    return torch


def _on(index: int):
    """Makes device ``index`` current for a call, if it is not."""
    cuda = _torch().cuda
    return contextlib.nullcontext() if index == cuda.current_device() else cuda.device(index)


def _check_tensors(named, dtype, device=None) -> None:
    """CUDA, contiguous, of ``dtype``, and all on one device."""
    for name, t in named:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
    for name, t in named:
        if t.dtype != dtype:
            raise RuntimeError(f"{name} must be {str(dtype).replace('torch.', '').replace('bfloat16', 'bf16')}")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    device = named[0][1].device if device is None else device
    for name, t in named:
        if t.device != device:
            raise RuntimeError(f"{name} must be on {device}")


def _attention_shape(q, k, v) -> tuple[int, int, int, int, int]:
    """(batch, heads, kv_heads, seq_q, seq_kv) of checked q, k, v."""
    _check_tensors((("q", q), ("k", k), ("v", v)), _torch().bfloat16)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise RuntimeError("q, k, and v must have shape (batch, heads, seq, dim)")
    if k.shape != v.shape:
        raise RuntimeError("k and v must have the same shape")
    if q.shape[3] != HEAD_DIM or k.shape[3] != HEAD_DIM:
        raise RuntimeError(f"head_dim must be {HEAD_DIM}")
    if q.shape[0] != k.shape[0]:
        raise RuntimeError("q and k must have the same batch")
    heads, kv_heads = q.shape[1], k.shape[1]
    if kv_heads == 0 or heads % kv_heads != 0:
        raise RuntimeError("the query heads must be a multiple of the key/value heads")
    return q.shape[0], heads, kv_heads, q.shape[2], k.shape[2]


def _scale(softmax_scale) -> float:
    scale = b.default_scale() if softmax_scale is None else float(softmax_scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise RuntimeError("softmax_scale must be positive and finite")
    return scale


def _forward(q, k, v, causal: bool, scale: float):
    torch = _torch()
    batch, heads, kv_heads, seq_q, seq_kv = _attention_shape(q, k, v)
    out = torch.empty_like(q)
    lse = torch.empty((batch, heads, seq_q), dtype=torch.float32, device=q.device)
    if out.numel() == 0:
        return out, lse
    if seq_kv == 0:
        return out.zero_(), lse.fill_(-math.inf)
    lib = b.load_library()
    index = q.get_device()
    with _on(index):
        code = lib.avo_b200_attn_fwd_grouped(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), batch, heads, kv_heads, seq_q,
            seq_kv, HEAD_DIM, 1 if causal else 0, scale, b.status_word(index).data_ptr(), b._raw_stream(index))
    b._check(code, "avo_b200_attn_fwd_grouped")
    return out, lse


def _refuse_capture(what: str) -> None:
    # Autograd runs each leaf's gradient accumulation on the stream on which the leaf was
    # first used.  Captured while an eager graph of the same leaves lives, that leaves the
    # capture, which ends the process; the plain calls have no such state.
    if _torch().cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} of inputs that require gradients cannot be captured in a CUDA graph; "
                           "capture the call under torch.no_grad() and its *_backward call")


_autograd_functions: dict[str, Any] = {}


def _attention_function():
    fn = _autograd_functions.get("attention")
    if fn is not None:
        return fn
    torch = _torch()

    class GroupedAttention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, causal, scale):
            out, lse = _forward(q, k, v, causal, scale)
            ctx.save_for_backward(q, k, v, out, lse)
            ctx.causal, ctx.scale = causal, scale
            ctx.mark_non_differentiable(lse)
            ctx.set_materialize_grads(False)
            return out, lse

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dout, _dlse):
            if dout is None:
                return None, None, None, None, None
            q, k, v, out, lse = ctx.saved_tensors
            with _on(q.get_device()):
                _refuse_capture("the backward of grouped_attention")
            grads = attention_backward(dout.contiguous(), q, k, v, out, lse, ctx.causal, softmax_scale=ctx.scale)
            return (*grads, None, None)

    _autograd_functions["attention"] = GroupedAttention
    return GroupedAttention


def grouped_attention(q, k, v, causal: bool, *, softmax_scale: float | None = None):
    """(out, lse) of attention with shared key/value heads and separate lengths.

    q is bf16 [B, H, seq_q, 128], k and v [B, Hkv, seq_kv, 128] with H a multiple of Hkv
    (query head h reads head h // (H // Hkv)), all contiguous; out is like q, lse fp32
    [B, H, seq_q] (natural log).  ``causal`` aligns the sequences at their ends: query i sees
    keys j <= i + seq_kv - seq_q; a query that sees no key gets out 0 and lse -inf.

    With gradients enabled and an input that requires them, out is differentiable in q, k
    and v (once; lse is not).  Such a call cannot be captured in a CUDA graph: capture the
    call under ``torch.no_grad()`` and ``attention_backward``."""
    torch = _torch()
    scale = _scale(softmax_scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        _attention_shape(q, k, v)
        with _on(q.get_device()):
            _refuse_capture("grouped_attention")
        return _attention_function().apply(q, k, v, bool(causal), scale)
    return _forward(q, k, v, causal, scale)


def attention_backward(dout, q, k, v, out, lse, causal: bool, *, softmax_scale: float | None = None, dq=None,
                       dk=None, dv=None):
    """(dq, dk, dv), bf16, of ``out = attention(q, k, v)`` for the gradient ``dout`` of out.

    ``out`` and ``lse`` are what the forward (``grouped_attention``, or
    ``attention_with_lse`` for equal shapes) returned for the same inputs and scale.  dk and
    dv sum over the query heads that share a key/value head.  All tensors are contiguous;
    the results go to ``dq``, ``dk``, ``dv`` where given.  The result does not depend on the
    order in which the GPU runs the work: equal inputs give equal bits."""
    torch = _torch()
    batch, heads, kv_heads, seq_q, seq_kv = _attention_shape(q, k, v)
    scale = _scale(softmax_scale)
    _check_tensors((("dout", dout), ("out", out)), torch.bfloat16, q.device)
    _check_tensors((("lse", lse),), torch.float32, q.device)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape:
            raise RuntimeError(f"{name} must have the shape of q")
    if tuple(lse.shape) != (batch, heads, seq_q):
        raise RuntimeError("lse must have shape (batch, heads, seq)")
    grads = []
    for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
        if t is None:
            t = torch.empty_like(like)
        else:
            _check_tensors(((name, t),), torch.bfloat16, q.device)
            if t.shape != like.shape:
                raise RuntimeError(f"{name} must have the shape of {name[1:]}")
        grads.append(t)
    lib = b.load_library()
    size = ctypes.c_size_t(0)
    b._check(lib.avo_b200_attn_bwd_workspace_size(batch, heads, kv_heads, seq_q, seq_kv, ctypes.byref(size)),
             "avo_b200_attn_bwd_workspace_size")
    index = q.get_device()
    with _on(index):
        scratch = torch.empty(size.value, dtype=torch.uint8, device=q.device)
        code = lib.avo_b200_attn_bwd(
            dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            *(t.data_ptr() for t in grads), batch, heads, kv_heads, seq_q, seq_kv, HEAD_DIM, 1 if causal else 0,
            scale, scratch.data_ptr(), size.value, b.status_word(index).data_ptr(), b._raw_stream(index))
    b._check(code, "avo_b200_attn_bwd")
    return tuple(grads)
