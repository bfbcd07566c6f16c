"""The norm weights' gradients over many tokens, on a B200, against sums in 64 bits.

A thread adds the terms of all its rows one after the other in fp32, then two half-warps, four
warps and the blocks (4 per multiprocessor, 128 threads to a column, their rows in order) are
added.  With n additions in a row and G = |dy cos| + |p(dy) sin|, where each term G |x_hat| has
fewer than 64 roundings of its own, the sum is within (64 + n) 2^-24 sum G |x_hat|.
"""

from __future__ import annotations

import pytest

from test_gpu_qkv_norm_rope import E, rotate, rotate_abs, seed  # noqa: F401 (seed is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,interleaved", [(16, 4, False), (5, 3, True)])
def test_weight_gradients_of_many_tokens(b200, seed, heads, kv_heads, interleaved):  # noqa: F811
    import torch

    batch, tokens, step = 2, 180_001, 20_000
    gen = torch.Generator(device="cuda").manual_seed(51)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16)

    qkv = randn(batch, tokens, heads + 2 * kv_heads, 128)
    grads = [randn(batch, n, tokens, 128) for n in (heads, kv_heads, kv_heads)]
    angle = torch.rand((1000, 64), device="cuda", generator=gen) * 6
    cos, sin = angle.cos(), angle.sin()
    positions = torch.arange(tokens, device="cuda") % 1000
    weight = 1 + torch.rand(128, device="cuda", generator=gen)
    _, *got = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, q_weight=weight, k_weight=weight, positions=positions,
                                          interleaved=interleaved)
    torch.cuda.synchronize()
    b200.check_status(qkv.device)

    case = (batch, tokens, heads, kv_heads, 128, interleaved)
    warps = 4 * 4 * torch.cuda.get_device_properties(0).multi_processor_count
    rows = {n: -(-((batch * tokens + 1) // 2) * -(-n // 16) // warps) * min(n, 16) for n in (heads, kv_heads)}
    first = 0
    for n, dy, mine in zip((heads, kv_heads), grads, got):
        want = torch.zeros(128, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(want)
        for at in range(0, tokens, step):
            cut = slice(at, min(tokens, at + step))
            x = qkv[:, cut, first:first + n].double()
            xh = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            d = dy[:, :, cut].double().transpose(1, 2)
            c, s = (t.double()[positions[cut]][:, None] for t in (cos, sin))
            want += (rotate(d, c, -s, case) * xh).sum((0, 1, 2))
            size += (rotate_abs(d, c, s, case) * xh.abs()).sum((0, 1, 2))
        first += n
        additions = rows[n] + 1 + 4 + warps // 4 // 128 + 1 + 12
        assert bool(((mine.double() - want).abs() <= (64 + additions) * E * size).all())
