"""AVO candidate: B200-native (sm_100a) BF16 attention forward, head_dim 128.

Obeys the candidate contract of the AVO scorer: a module-level callable
``attention(q, k, v, causal) -> Tensor[B, H, S, D]`` (reference: loader
avo/benchmark.py:406-418; the SDPA seed candidates/torch_sdpa_seed.py:6-7).  Inputs are
contiguous CUDA bf16 ``[B, H, S, 128]``; the output is a new tensor of the same shape
and dtype, as ``torch::empty_like`` gives in the reference seeds
(candidates/cuda_mma_attention/attention_kernel.cu:188).

Additive export ``attention_with_lse(q, k, v, causal) -> (O, LSE)`` returns the fp32
natural-log LSE ``[B, H, S]`` as well.

For training, ``grouped_attention(q, k, v, causal) -> (O, LSE)`` is the forward with shared
key/value heads and separate query and key lengths, differentiable by autograd, and
``attention_backward(dO, q, k, v, O, LSE, causal) -> (dq, dk, dv)`` its gradient as a plain
call; ``qkv_norm_rope(qkv, H, Hkv, cos, sin, ...) -> (q, k, v)`` makes attention's inputs from
a fused projection (norms of queries and keys, rotary positions, layout) and
``qkv_norm_rope_backward`` is its gradient.

The kernel lives in the companion directory ``cuda_b200_attention/`` (TMA +
tcgen05/TMEM, warp-specialised, built ahead of time by nvcc for sm_100a and called
through a C ABI).  There is no CPU or eager fallback.
"""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

_DIR = Path(__file__).resolve().parent / "cuda_b200_attention"
_BINDING = "avo_b200_attention_binding"
_TRAINING = "avo_b200_training_binding"

AVO_SOURCE_FILES = (
    "cuda_b200_attention/sm100_ptx.cuh",
    "cuda_b200_attention/schedule.cuh",
    "cuda_b200_attention/attn_fwd.cuh",
    "cuda_b200_attention/attn_bwd.cuh",
    "cuda_b200_attention/qkv_norm_rope.cuh",
    "cuda_b200_attention/host_common.h",
    "cuda_b200_attention/attn_abi.cu",
    "cuda_b200_attention/attn_bwd.cu",
    "cuda_b200_attention/qkv_norm_rope.cu",
    "cuda_b200_attention/fast_call.c",
    "cuda_b200_attention/b200_attention.py",
    "cuda_b200_attention/b200_training.py",
    "cuda_b200_attention/build.py",
)


def _load(name: str, file: str):
    module = sys.modules.get(name)
    if module is None:
        spec = importlib.util.spec_from_file_location(name, _DIR / file)
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return module


def _binding():
    return _load(_BINDING, "b200_attention.py")


def _training():
    return _load(_TRAINING, "b200_training.py")


def attention(q, k, v, causal: bool):
    out, _ = _binding().attention_forward(q, k, v, causal, need_lse=False)
    return out


def attention_with_lse(q, k, v, causal: bool):
    return _binding().attention_forward(q, k, v, causal, need_lse=True)


def grouped_attention(q, k, v, causal: bool, *, softmax_scale: float | None = None):
    return _training().grouped_attention(q, k, v, causal, softmax_scale=softmax_scale)


def attention_backward(dout, q, k, v, out, lse, causal: bool, *, softmax_scale: float | None = None, dq=None,
                       dk=None, dv=None):
    return _training().attention_backward(dout, q, k, v, out, lse, causal, softmax_scale=softmax_scale, dq=dq,
                                          dk=dk, dv=dv)


def qkv_norm_rope(qkv, num_heads: int, num_kv_heads: int, cos, sin, *, q_weight=None, k_weight=None, positions=None,
                  sections=None, eps: float = 1e-6, interleaved: bool = False):
    return _training().qkv_norm_rope(qkv, num_heads, num_kv_heads, cos, sin, q_weight=q_weight, k_weight=k_weight,
                                     positions=positions, sections=sections, eps=eps, interleaved=interleaved)


def qkv_norm_rope_backward(dq, dk, dv, qkv, cos, sin, *, q_weight=None, k_weight=None, positions=None, sections=None,
                           eps: float = 1e-6, interleaved: bool = False):
    return _training().qkv_norm_rope_backward(dq, dk, dv, qkv, cos, sin, q_weight=q_weight, k_weight=k_weight,
                                              positions=positions, sections=sections, eps=eps,
                                              interleaved=interleaved)
