"""What the training entry points answer to forward-mode differentiation: a refusal, never a result
without its tangent.  The refusal comes before anything else is looked at, so it needs no GPU."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture(scope="module")
def seed():
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention_seed.py"
    spec = importlib.util.spec_from_file_location("avo_candidate_b200_seed_derivatives", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def calls(seed):
    """Each entry point with the tensors that a tangent can come in on, by name."""
    q, k = zeros(1, 4, 8, 128), zeros(1, 2, 8, 128)
    qkv, table, weight = zeros(1, 8, 8, 128), zeros(8, 64, dtype=torch.float32), zeros(128, dtype=torch.float32)
    rope = dict(cos=table, sin=table, q_weight=weight, k_weight=weight)
    return [
        (lambda q, k, v: seed.grouped_attention(q, k, v, True), dict(q=q, k=k, v=k)),
        (lambda dout, q, k, v, out, lse: seed.attention_backward(dout, q, k, v, out, lse, True),
         dict(dout=q, q=q, k=k, v=k, out=q, lse=zeros(1, 4, 8, dtype=torch.float32))),
        (lambda qkv, cos, sin, **w: seed.qkv_norm_rope(qkv, 4, 2, cos, sin, **w), dict(qkv=qkv, **rope)),
        (lambda dq, dk, dv, qkv, cos, sin, **w: seed.qkv_norm_rope_backward(dq, dk, dv, qkv, cos, sin, **w),
         dict(dq=q, dk=k, dv=k, qkv=qkv, **rope)),
    ]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(seed, which, grad):
    call, tensors = calls(seed)[which]
    for name, t in tensors.items():
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(**{**tensors, name: forward_ad.make_dual(t, torch.ones_like(t))})


@pytest.mark.parametrize("which", range(4))
def test_without_tangents_the_other_checks_answer(seed, which):
    call, tensors = calls(seed)[which]
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        call(**tensors)
    with forward_ad.dual_level():  # a level alone changes nothing
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call(**tensors)


def test_function_transforms_are_refused(seed):
    call, tensors = calls(seed)[0]
    ones = {name: torch.ones_like(t) for name, t in tensors.items()}
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda q, k, v: call(q, k, v)[0], tuple(tensors.values()), tuple(ones.values()))
