"""The training side of attention: its input stage, shared key/value heads and the gradients.

Host side of the entry points of include/avo_b200_attn.h that the forward contract does not
cover, in the manner of b200_attention.py (argument checks that raise ``RuntimeError``, the
current CUDA stream of the tensors' device, the device's status word, no fallback):

* ``grouped_attention``: the forward with H query heads over Hkv key/value heads and
  seq_q != seq_kv, differentiable through torch's autograd;
* ``attention_backward``: its gradient as a plain call;
* ``qkv_norm_rope``: from a fused projection to attention's q, k, v (norms of queries and
  keys, rotary positions on one or several axes, heads in front of tokens), differentiable;
* ``qkv_norm_rope_backward``: its gradient as a plain call.

Scratch is allocated per call by torch's caching allocator on the current stream, so calls
on several streams, and several captured graphs, share nothing but the status word.  The plain
calls can be captured in a CUDA graph, after one call on the device (which creates that word).
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
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


@functools.cache
def _torch():
    import torch

    return torch


_here = contextlib.nullcontext()


def _on(index: int):
    """Makes device ``index`` current for a call, if it is not."""
    torch = _torch()
    return _here if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _plain(t, dtype, index: int) -> bool:
    """A contiguous tensor of ``dtype`` on CUDA device ``index``."""
    return t.is_cuda and t.dtype is dtype and t.get_device() == index and t.is_contiguous()


def _check_tensors(named, dtype, device=None) -> None:
    """Raises what is wrong with the first tensor that is not CUDA, of ``dtype``, contiguous
    and on ``device`` (or that of the first)."""
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


def _overlap(a, b) -> bool:
    """Whether two contiguous tensors share memory."""
    at, by = a.data_ptr(), b.data_ptr()
    return at < by + b.numel() * b.element_size() and by < at + a.numel() * a.element_size()


def _attention_shape(q, k, v) -> tuple[int, int, int, int, int]:
    """(batch, heads, kv_heads, seq_q, seq_kv) of checked q, k, v."""
    bf16 = _torch().bfloat16
    index = q.get_device()
    if not (_plain(q, bf16, index) and _plain(k, bf16, index) and _plain(v, bf16, index)):
        _check_tensors((("q", q), ("k", k), ("v", v)), bf16)
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != 4 or len(ks) != 4 or len(vs) != 4:
        raise RuntimeError("q, k, and v must have shape (batch, heads, seq, dim)")
    if ks != vs:
        raise RuntimeError("k and v must have the same shape")
    batch, heads, seq_q, dim = qs
    kv_batch, kv_heads, seq_kv, kv_dim = ks
    if dim != HEAD_DIM or kv_dim != HEAD_DIM:
        raise RuntimeError(f"head_dim must be {HEAD_DIM}")
    if batch != kv_batch:
        raise RuntimeError("q and k must have the same batch")
    if kv_heads == 0 or heads % kv_heads != 0:
        raise RuntimeError("the query heads must be a multiple of the key/value heads")
    return batch, heads, kv_heads, seq_q, seq_kv


def _scale(softmax_scale) -> float:
    scale = b.default_scale() if softmax_scale is None else float(softmax_scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise RuntimeError("softmax_scale must be positive and finite")
    return scale


@functools.lru_cache(maxsize=256)
def _forward_scratch_bytes(index: int, batch: int, heads: int, kv_heads: int, seq_q: int, seq_kv: int,
                           causal: bool) -> int:
    """Scratch of the forward for these sizes on device ``index``, the current one: what a plan that
    splits items between CTAs needs, 0 for the others (causal work is never split)."""
    if causal and seq_q > 1:
        return 0
    sms = _torch().cuda.get_device_properties(index).multi_processor_count
    if b.grouped_plan(batch, heads, kv_heads, seq_q, seq_kv, causal, sm_count=sms)[0] != b.PLAN_SPLIT:
        return 0
    size = ctypes.c_size_t(0)
    b._check(b.load_library().avo_b200_attn_workspace_size(ctypes.byref(size)), "avo_b200_attn_workspace_size")
    return size.value


def _forward(q, k, v, causal: bool, scale: float):
    torch = _torch()
    batch, heads, kv_heads, seq_q, seq_kv = _attention_shape(q, k, v)
    out = torch.empty_like(q)
    lse = q.new_empty((batch, heads, seq_q), dtype=torch.float32)
    if out.numel() == 0:
        return out, lse
    if seq_kv == 0:
        return out.zero_(), lse.fill_(-math.inf)
    b.load_library()
    index = q.get_device()
    with _on(index):
        size = _forward_scratch_bytes(index, batch, heads, kv_heads, seq_q, seq_kv, bool(causal))
        scratch = q.new_empty(size, dtype=torch.uint8) if size else None
        code = b.call_entry(
            0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), batch, heads, kv_heads, seq_q,
            seq_kv, HEAD_DIM, 1 if causal else 0, scale, None if scratch is None else scratch.data_ptr(), size,
            b.status_address(index), b._raw_stream(index))
    b._check(code, "avo_b200_attn_fwd_grouped")
    return out, lse


def _refuse_capture(what: str) -> None:
    # Autograd runs each leaf's gradient accumulation on the stream on which the leaf was
    # first used.  Captured while an eager graph of the same leaves lives, that leaves the
    # capture, which ends the process; the plain calls have no such state.
    if _torch().cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} of inputs that require gradients cannot be captured in a CUDA graph; "
                           "capture the call under torch.no_grad() and its *_backward call")


@functools.cache
def _forward_ad():
    import torch.autograd.forward_ad as forward_ad

    return forward_ad


def _refuse_tangents(what: str, *tensors) -> None:
    """Raises if one of the tensors carries a tangent of forward-mode differentiation, which the
    operators do not propagate (such a tensor need not require gradients)."""
    forward_ad = _forward_ad()
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")


def _incoming(grad):
    """A gradient as autograd hands it over, contiguous and on the kernels' 16-byte grid: a slice of
    a larger gradient (torch.cat's) can be contiguous and off it."""
    grad = grad.contiguous()
    return grad if grad.data_ptr() % 16 == 0 else grad.clone()


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
            grads = attention_backward(_incoming(dout), q, k, v, out, lse, ctx.causal, softmax_scale=ctx.scale)
            return (*grads, None, None)

    _autograd_functions["attention"] = GroupedAttention
    return GroupedAttention


def grouped_attention(q, k, v, causal: bool, *, softmax_scale: float | None = None):
    """(out, lse) of attention with shared key/value heads and separate lengths.

    q is bf16 [B, H, seq_q, 128], k and v [B, Hkv, seq_kv, 128] with H a multiple of Hkv
    (query head h reads head h // (H // Hkv)), all contiguous; out is like q, lse fp32
    [B, H, seq_q] (natural log).  ``causal`` aligns the sequences at their ends: query i sees
    keys j <= i + seq_kv - seq_q; a query that sees no key gets out 0 and lse -inf, one that
    sees a NaN score or a score of +infinity gets NaN in both.

    With gradients enabled and an input that requires them, out is differentiable in q, k
    and v (in reverse mode, once).  lse is not: what a loss computes from it adds nothing to
    the gradients.  Such a call cannot be captured in a CUDA graph: capture the
    call under ``torch.no_grad()`` and ``attention_backward``."""
    torch = _torch()
    scale = _scale(softmax_scale)
    _refuse_tangents("grouped_attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        _attention_shape(q, k, v)
        with _on(q.get_device()):
            _refuse_capture("grouped_attention")
        return _attention_function().apply(q, k, v, bool(causal), scale)
    return _forward(q, k, v, causal, scale)


@functools.lru_cache(maxsize=256)
def _backward_scratch_bytes(batch: int, heads: int, kv_heads: int, seq_q: int, seq_kv: int, causal: bool) -> int:
    """Scratch of the backward for these sizes."""
    size = ctypes.c_size_t(0)
    b._check(b.load_library().avo_b200_attn_bwd_workspace_size(batch, heads, kv_heads, seq_q, seq_kv, int(causal),
                                                               ctypes.byref(size)),
             "avo_b200_attn_bwd_workspace_size")
    return size.value


def attention_backward(dout, q, k, v, out, lse, causal: bool, *, softmax_scale: float | None = None, dq=None,
                       dk=None, dv=None):
    """(dq, dk, dv), bf16, of ``out = attention(q, k, v)`` for the gradient ``dout`` of out.

    ``out`` and ``lse`` are what the forward (``grouped_attention``, or
    ``attention_with_lse`` for equal shapes) returned for the same inputs and scale.  dk and
    dv sum over the query heads that share a key/value head.  All tensors are contiguous;
    the results go to ``dq``, ``dk``, ``dv`` where given (which overlap no other tensor of the
    call) and carry no gradient themselves.  The result does not depend on the
    order in which the GPU runs the work: equal inputs give equal bits."""
    torch = _torch()
    _refuse_tangents("attention_backward", dout, q, k, v, out, lse)
    batch, heads, kv_heads, seq_q, seq_kv = _attention_shape(q, k, v)
    scale = _scale(softmax_scale)
    index = q.get_device()
    if not (_plain(dout, torch.bfloat16, index) and _plain(out, torch.bfloat16, index)):
        _check_tensors((("dout", dout), ("out", out)), torch.bfloat16, q.device)
    if not _plain(lse, torch.float32, index):
        _check_tensors((("lse", lse),), torch.float32, q.device)
    shape = (batch, heads, seq_q, HEAD_DIM)
    if dout.shape != shape or out.shape != shape:
        raise RuntimeError(f"{'out' if dout.shape == shape else 'dout'} must have the shape of q")
    if lse.shape != shape[:3]:
        raise RuntimeError("lse must have shape (batch, heads, seq)")
    if dq is not None or dk is not None or dv is not None:
        given = [(name, t, like) for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)) if t is not None]
        for i, (name, t, like) in enumerate(given):
            _check_tensors(((name, t),), torch.bfloat16, q.device)
            if t.shape != like.shape:
                raise RuntimeError(f"{name} must have the shape of {name[1:]}")
            if any(_overlap(t, other) for other in (dout, q, k, v, out, lse, *(g[1] for g in given[:i]))):
                raise RuntimeError(f"{name} must not overlap another tensor of the call")
    grads = (torch.empty_like(q) if dq is None else dq, torch.empty_like(k) if dk is None else dk,
             torch.empty_like(v) if dv is None else dv)
    with _on(index):
        size = _backward_scratch_bytes(batch, heads, kv_heads, seq_q, seq_kv, bool(causal))
        scratch = q.new_empty(size, dtype=torch.uint8)
        code = b.call_entry(
            1, dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(), batch, heads, kv_heads, seq_q, seq_kv,
            HEAD_DIM, 1 if causal else 0, scale, scratch.data_ptr(), size, b.status_address(index),
            b._raw_stream(index))
    b._check(code, "avo_b200_attn_bwd")
    return grads


# ---------------------------------------------------------------- QKV norm + rotation
MAX_AXES = 4


@functools.lru_cache(maxsize=64)
def _section_array(counts: tuple[int, ...], pairs: int):
    """(axes, the C array) of checked section counts."""
    if not 1 <= len(counts) <= MAX_AXES or any(n < 0 for n in counts) or sum(counts) != pairs:
        raise RuntimeError(f"sections must be 1 to {MAX_AXES} counts that sum to rotary_dim / 2")
    return len(counts), (ctypes.c_int * len(counts))(*counts)


def _rope_args(qkv, heads: int, kv_heads: int, cos, sin, q_weight, k_weight, positions, sections, eps, interleaved):
    """Checks the arguments both directions share; (batch, seq, the C calls' arguments for qkv,
    those from `batch` to `eps`, what they point to)."""
    torch = _torch()
    if not qkv.is_cuda:
        raise RuntimeError("qkv must be a CUDA tensor")
    if qkv.dtype != torch.bfloat16:
        raise RuntimeError("qkv must be bf16")
    if heads < 0 or kv_heads < 0:
        raise RuntimeError("the numbers of heads must not be negative")
    shape = qkv.shape
    if len(shape) != 4 or shape[2] != heads + 2 * kv_heads or shape[3] != HEAD_DIM:
        raise RuntimeError(f"qkv must have shape (batch, seq, heads + 2 * kv_heads, {HEAD_DIM})")
    batch, seq, all_heads, _ = shape
    batch_stride, token_stride, head_stride, last_stride = qkv.stride()
    if (last_stride != 1 or (all_heads > 1 and head_stride != HEAD_DIM)) and qkv.numel():
        raise RuntimeError("the heads of a token of qkv must be contiguous")
    # (A dimension of one element has no stride to speak of.)
    place = (qkv.data_ptr(), batch_stride if batch > 1 else 0, token_stride if seq > 1 else 0)
    index = qkv.get_device()
    if not (_plain(cos, torch.float32, index) and _plain(sin, torch.float32, index)):
        _check_tensors((("cos", cos), ("sin", sin)), torch.float32, qkv.device)
    table = cos.shape
    if len(table) != 2 or table != sin.shape:
        raise RuntimeError("cos and sin must have the same shape (positions, rotary_dim / 2)")
    table_rows, pairs = table
    rotary = 2 * pairs
    if rotary == 0 or rotary > HEAD_DIM or rotary % 16 != 0:
        raise RuntimeError(f"rotary_dim must be a multiple of 16 up to {HEAD_DIM}")
    if (q_weight is None) != (k_weight is None):
        raise RuntimeError("q_weight and k_weight must be given together")
    weights_at, weights_bf16 = (None, None), 0
    if q_weight is not None:
        dtype = q_weight.dtype
        if dtype is not torch.float32 and dtype is not torch.bfloat16:
            raise RuntimeError("q_weight must be fp32 or bf16")
        if not (_plain(q_weight, dtype, index) and _plain(k_weight, dtype, index)):
            _check_tensors((("q_weight", q_weight), ("k_weight", k_weight)), dtype, qkv.device)
        if q_weight.shape != (HEAD_DIM,) or k_weight.shape != (HEAD_DIM,):
            raise RuntimeError(f"q_weight and k_weight must have shape ({HEAD_DIM},)")
        weights_at, weights_bf16 = (q_weight.data_ptr(), k_weight.data_ptr()), int(dtype is torch.bfloat16)
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise RuntimeError("eps must not be negative")
    axes, section_array, sections_at, strides, positions_at, wide = 1, None, None, (0, 0, 0), None, 0
    if sections is not None:
        axes, section_array = _section_array(tuple(map(int, sections)), pairs)
        if positions is None:
            raise RuntimeError("sections need positions")
        sections_at = ctypes.addressof(section_array)
    if positions is None:
        if seq > table_rows:
            raise RuntimeError("cos and sin have fewer rows than the sequence has tokens")
    else:
        if not positions.is_cuda or positions.get_device() != index:
            raise RuntimeError("positions must be on the device of qkv")
        wide = int(positions.dtype is torch.int64)
        if not wide and positions.dtype is not torch.int32:
            raise RuntimeError("positions must be int32 or int64")
        shape = positions.shape
        lead_ok = sections is None or shape[:1] == (axes,)
        if sections is not None:
            shape = shape[1:]
        if shape != (batch, seq) and shape != (seq,) or not lead_ok:
            lead = "" if sections is None else "axes, "
            raise RuntimeError(f"positions must have shape ({lead}seq) or ({lead}batch, seq)")
        if table_rows == 0 and positions.numel():
            raise RuntimeError("cos and sin have no rows")
        at = positions.stride()
        strides = (at[0] if sections is not None else 0, at[-2] if len(shape) == 2 else 0, at[-1])
        positions_at = positions.data_ptr()
    args = (batch, seq, heads, kv_heads, HEAD_DIM, *weights_at, weights_bf16, cos.data_ptr(), sin.data_ptr(),
            table_rows, rotary, 1 if interleaved else 0, positions_at, wide, *strides, axes, sections_at, eps)
    return batch, seq, place, args, section_array


def _norm_rope(qkv, heads, kv_heads, cos, sin, q_weight, k_weight, positions, sections, eps, interleaved):
    torch = _torch()
    batch, seq, place, args, keep = _rope_args(qkv, heads, kv_heads, cos, sin, q_weight, k_weight, positions, sections,
                                               eps, interleaved)
    q = qkv.new_empty((batch, heads, seq, HEAD_DIM))
    k = qkv.new_empty((batch, kv_heads, seq, HEAD_DIM))
    v = torch.empty_like(k)
    if qkv.numel() == 0:
        return q, k, v
    b.load_library()
    index = qkv.get_device()
    with _on(index):
        code = b.call_entry(2, *place, q.data_ptr(), k.data_ptr(), v.data_ptr(), *args,
                            b.status_address(index), b._raw_stream(index))
    del keep
    b._check(code, "avo_b200_qkv_norm_rope")
    return q, k, v


def qkv_norm_rope_backward(dq, dk, dv, qkv, cos, sin, *, q_weight=None, k_weight=None, positions=None, sections=None,
                           eps: float = 1e-6, interleaved: bool = False):
    """(dqkv, dq_weight, dk_weight) of ``qkv_norm_rope`` for the gradients of its outputs.

    dq is bf16 [B, H, S, 128], dk and dv [B, Hkv, S, 128], contiguous; qkv and the other
    arguments are the forward's.  dqkv is a new contiguous tensor of qkv's shape, the weight
    gradients are fp32 [128] (None without weights).  They carry no gradient themselves.
    Equal inputs give equal bits."""
    torch = _torch()
    _refuse_tangents("qkv_norm_rope_backward", dq, dk, dv, qkv, cos, sin, q_weight, k_weight)
    index = qkv.get_device()
    if not (_plain(dq, torch.bfloat16, index) and _plain(dk, torch.bfloat16, index)
            and _plain(dv, torch.bfloat16, index)):
        _check_tensors((("dq", dq), ("dk", dk), ("dv", dv)), torch.bfloat16, qkv.device)
    dq_shape, dk_shape = dq.shape, dk.shape
    if len(dq_shape) != 4 or len(dk_shape) != 4 or dk_shape != dv.shape:
        raise RuntimeError("dq, dk and dv must have shape (batch, heads, seq, dim), dk and dv the same")
    heads, kv_heads = dq_shape[1], dk_shape[1]
    batch, seq, place, args, keep = _rope_args(qkv, heads, kv_heads, cos, sin, q_weight, k_weight, positions, sections,
                                               eps, interleaved)
    if dq_shape != (batch, heads, seq, HEAD_DIM) or dk_shape != (batch, kv_heads, seq, HEAD_DIM):
        raise RuntimeError("dq, dk and dv must match qkv's batch and sequence")
    dqkv = qkv.new_empty(qkv.shape)
    b.load_library()
    with _on(index):
        weights, scratch, more = (None, None), None, (None, 0)
        weights_at = weights
        if q_weight is not None:
            weights = cos.new_empty((2, HEAD_DIM)).unbind()
            weights_at = (weights[0].data_ptr(), weights[1].data_ptr())
            size = _rope_scratch_bytes(index)
            scratch = qkv.new_empty(size, dtype=torch.uint8)
            more = (scratch.data_ptr(), size)
        code = b.call_entry(3, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *place, dqkv.data_ptr(), *weights_at, *args,
                            *more, b.status_address(index), b._raw_stream(index))
    del keep
    b._check(code, "avo_b200_qkv_norm_rope_bwd")
    return (dqkv, *weights)


_rope_scratch: dict[int, int] = {}


def _rope_scratch_bytes(index: int) -> int:
    """Scratch of the backward on device ``index`` (a function of the device alone)."""
    if index not in _rope_scratch:
        size = ctypes.c_size_t(0)
        b._check(b.load_library().avo_b200_qkv_norm_rope_bwd_workspace_size(ctypes.byref(size)),
                 "avo_b200_qkv_norm_rope_bwd_workspace_size")
        _rope_scratch[index] = size.value
    return _rope_scratch[index]


def _norm_rope_function():
    fn = _autograd_functions.get("norm_rope")
    if fn is not None:
        return fn
    torch = _torch()

    class QkvNormRope(torch.autograd.Function):
        @staticmethod
        def forward(ctx, qkv, q_weight, k_weight, cos, sin, positions, heads, kv_heads, sections, eps, interleaved):
            ctx.save_for_backward(qkv, q_weight, k_weight, cos, sin, positions)
            ctx.how = (sections, eps, interleaved)
            return _norm_rope(qkv, heads, kv_heads, cos, sin, q_weight, k_weight, positions, sections, eps, interleaved)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dq, dk, dv):
            qkv, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
            sections, eps, interleaved = ctx.how
            with _on(qkv.get_device()):
                _refuse_capture("the backward of qkv_norm_rope")
            dqkv, dqw, dkw = qkv_norm_rope_backward(
                _incoming(dq), _incoming(dk), _incoming(dv), qkv, cos, sin, q_weight=q_weight,
                k_weight=k_weight, positions=positions, sections=sections, eps=eps, interleaved=interleaved)
            if dqw is not None:
                dqw, dkw = dqw.to(q_weight.dtype), dkw.to(k_weight.dtype)
            return (dqkv, dqw, dkw, *([None] * 8))

    _autograd_functions["norm_rope"] = QkvNormRope
    return QkvNormRope


def qkv_norm_rope(qkv, num_heads: int, num_kv_heads: int, cos, sin, *, q_weight=None, k_weight=None, positions=None,
                  sections=None, eps: float = 1e-6, interleaved: bool = False):
    """(q, k, v) for attention from a fused projection, in one pass.

    qkv is bf16 [B, S, H + 2 Hkv, 128]: query, key and value heads of each token (batch and
    token strides are free).  Query and key heads are divided by their root mean square
    (with ``eps``) and multiplied by ``q_weight`` / ``k_weight`` ([128], fp32 or bf16; both
    None: no norm), then their first R values are rotated by the fp32 tables ``cos`` and
    ``sin`` [P, R / 2]: pair f is (f, f + R / 2), or (2 f, 2 f + 1) when ``interleaved``.
    q is bf16 [B, H, S, 128], k and v [B, Hkv, S, 128], contiguous.

    ``positions`` (int32 or int64) are the table rows: [S] or [B, S]; None is 0..S-1.  With
    ``sections`` (how many consecutive pairs each axis turns, up to 4 axes), positions are
    [axes, S] or [axes, B, S]; those of an axis that turns no pairs are not looked at.  A
    position outside the table makes the token's rotated values NaN and is reported by
    ``check_status()``.

    With gradients enabled and an input that requires them, the result is differentiable in
    qkv and the weights (in reverse mode, once), not in the tables, which must not require gradients then.
    Such a call cannot be captured in a CUDA graph: capture the call under
    ``torch.no_grad()`` and ``qkv_norm_rope_backward``."""
    torch = _torch()
    sections = None if sections is None else tuple(map(int, sections))
    heads, kv_heads, interleaved = int(num_heads), int(num_kv_heads), bool(interleaved)
    _refuse_tangents("qkv_norm_rope", qkv, cos, sin, q_weight, k_weight)
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise RuntimeError("qkv_norm_rope has no gradient for cos and sin: detach them")
    if torch.is_grad_enabled() and (qkv.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        _rope_args(qkv, heads, kv_heads, cos, sin, q_weight, k_weight, positions, sections, eps, interleaved)
        with _on(qkv.get_device()):
            _refuse_capture("qkv_norm_rope")
        return _norm_rope_function().apply(qkv, q_weight, k_weight, cos, sin, positions, heads, kv_heads, sections,
                                           float(eps), interleaved)
    return _norm_rope(qkv, heads, kv_heads, cos, sin, q_weight, k_weight, positions, sections, eps, interleaved)
