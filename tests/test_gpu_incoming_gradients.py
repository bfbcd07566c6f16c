"""Gradients as autograd hands them to the training operators, on a B200."""

from __future__ import annotations

import pytest

from test_gpu_qkv_norm_rope import make, seed  # noqa: F401 (seed is a fixture)

pytestmark = pytest.mark.gpu


def behind(*tensors):
    """The tensors in one vector behind three other values: their gradients are contiguous slices
    that start off the 16-byte grid."""
    import torch

    lead = torch.zeros(3, dtype=tensors[0].dtype, device=tensors[0].device)
    return torch.cat((lead, *(t.flatten() for t in tensors)))


def test_gradients_off_the_16_byte_grid(b200, seed):  # noqa: F811
    import torch

    case = (2, 70, 4, 2, 128, False, "fp32", "int64", None)
    qkv, cos, sin, how, grads = make(case, 41)
    leaves = [qkv.clone().requires_grad_(), *(how[n].clone().requires_grad_() for n in ("q_weight", "k_weight"))]
    named = {**how, "q_weight": leaves[1], "k_weight": leaves[2]}
    outs = seed.qkv_norm_rope(leaves[0], 4, 2, cos, sin, **named)
    behind(*outs).backward(behind(*grads))
    want = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, want))

    q, k, v = (t.detach().requires_grad_() for t in outs)
    out, lse = seed.grouped_attention(q, k, v, True)
    behind(out).backward(behind(grads[0]))
    want = seed.attention_backward(grads[0], q, k, v, out, lse, True)
    torch.cuda.synchronize()
    b200.check_status(qkv.device)
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip((q, k, v), want))


def test_a_loss_on_out_and_lse_gives_the_gradients_of_out(b200, seed):  # noqa: F811
    # lse is not differentiable: alone it gives no gradient to ask for, beside out it adds nothing.
    import torch

    qkv, cos, sin, how, grads = make((1, 90, 4, 2, 128, False, "fp32", None, None), 42)
    q, k, v = (t.requires_grad_() for t in seed.qkv_norm_rope(qkv, 4, 2, cos, sin, **how))
    out, lse = seed.grouped_attention(q, k, v, True)
    with pytest.raises(RuntimeError, match="does not require grad"):
        lse.sum().backward()
    ((out * grads[0]).sum().float() + lse.square().sum()).backward()
    want = seed.attention_backward(grads[0], q, k, v, out, lse, True)
    torch.cuda.synchronize()
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip((q, k, v), want))
