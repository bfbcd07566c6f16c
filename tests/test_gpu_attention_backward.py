"""grouped_attention and attention_backward on a B200 against a plain implementation in 64 bits.

Tolerances are computed per element from the formulas, before any run: with u = 2^-8 (half a
bf16 step) the kernel rounds P and dS to bf16 once, receives out rounded to bf16, and rounds
each gradient once, so

    |dV err| <= sum_i P (u + e) |dO| + u |dV|
    |dS err| <= |dS| (u + e) + P (u sum_d |dO O| + f sum_d |dO V|),   |dQ err| <= scale sum_j |dS err| |K| + u |dQ|

(dK like dQ), where e bounds the relative error of P in fp32 (the score's dot product,
128 * 2^-24 * scale * sum_d |q k|, the exponential's 7.5e-5 and the roundings of the exponent)
and f = 128 * 2^-24 the dot product dP; the fp32 accumulation adds n * 2^-24 of the sum of
absolute terms.
"""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-8
EPS32 = 2.0**-24

CASES = [
    # batch, heads, kv_heads, seq_q, seq_kv, causal
    (1, 1, 1, 1, 1, False),
    (1, 2, 1, 1, 5, True),
    (1, 1, 1, 5, 1, True),        # four rows that see no key
    (2, 4, 2, 127, 128, False),
    (1, 2, 2, 129, 257, True),
    (1, 4, 1, 300, 170, True),    # the first 130 rows, more than a tile of them, see no key
    (1, 2, 2, 170, 300, False),
    (1, 1, 1, 64, 700, True),
    (1, 8, 2, 777, 1003, True),
    (1, 12, 12, 640, 640, True),
    (2, 16, 16, 1280, 1280, False),  # more items than multiprocessors
    (2, 16, 8, 1300, 1300, True),
    (1, 6, 1, 1024, 129, False),
]


@pytest.fixture(scope="module")
def training(b200):
    import importlib.util
    import sys

    name = "avo_b200_training_binding"
    if name not in sys.modules:
        path = b200.HERE / "b200_training.py"
        spec = importlib.util.spec_from_file_location(name, path)
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name]


def make(case, seed=0, std_do=1.0):
    import torch

    batch, heads, kv_heads, seq_q, seq_kv, causal = case
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(h, s, std=1.0):
        return (torch.randn((batch, h, s, 128), device="cuda", generator=gen) * std).bfloat16()

    return randn(heads, seq_q), randn(kv_heads, seq_kv), randn(kv_heads, seq_kv), randn(heads, seq_q, std_do)


def plain(q, k, v, do, causal, scale):
    """out, lse, dq, dk, dv in fp64 and the bounds of the gradients' errors."""
    import torch

    batch, heads, seq_q, _ = q.shape
    kv_heads, seq_kv = k.shape[1], k.shape[2]
    group = heads // kv_heads
    q, k, v, do = (t.double() for t in (q, k, v, do))
    kx, vx = (t.repeat_interleave(group, 1) for t in (k, v))
    s = scale * (q @ kx.transpose(-1, -2))
    if causal:
        i = torch.arange(seq_q, device=q.device)[:, None] + seq_kv - seq_q
        s = s.masked_fill(torch.arange(seq_kv, device=q.device)[None, :] > i, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse[..., None] == -math.inf, torch.zeros_like(s), torch.exp(s - lse[..., None]))
    out = p @ vx
    dp = do @ vx.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)

    def share(t):
        return t.unflatten(1, (kv_heads, group)).sum(2)

    dq, dk, dv = scale * (ds @ kx), share(scale * (ds.transpose(-1, -2) @ q)), share(p.transpose(-1, -2) @ do)
    e = 1e-4 + 128 * EPS32 * scale * (q.abs() @ kx.abs().transpose(-1, -2)) + 4 * EPS32 * s.abs().clamp(max=200)
    e_ds = ds.abs() * (U + e) + p * (U * (do * out).abs().sum(-1, keepdim=True)
                                     + 128 * EPS32 * (do.abs() @ vx.abs().transpose(-1, -2)))
    e_ds = e_ds + ds.abs() * (seq_q * group + seq_kv) * EPS32
    e_p = p * (U + e + seq_q * group * EPS32)
    bounds = (scale * (e_ds @ kx.abs()) + U * dq.abs(),
              share(scale * (e_ds.transpose(-1, -2) @ q.abs())) + U * dk.abs(),
              share(e_p.transpose(-1, -2) @ do.abs()) + U * dv.abs())
    return out, lse, (dq, dk, dv), bounds


def assert_within(got, want, bound, what):
    err = (got.double() - want).abs()
    over = err > bound * 1.001 + 1e-30
    assert not bool(over.any()), (what, int(over.sum()), float((err / (bound + 1e-30)).max()))


@pytest.mark.parametrize("case", CASES)
def test_backward_matches_fp64(b200, training, case):
    import torch

    q, k, v, do = make(case, seed=1)
    scale = 0.11 if case[4] % 2 else b200.default_scale()
    out, lse, grads, bounds = plain(q, k, v, do, case[5], scale)
    got = training.attention_backward(do, q, k, v, out.bfloat16(), lse.float(), case[5], softmax_scale=scale)
    torch.cuda.synchronize()
    b200.check_status(q.device)
    for name, g, w, bound in zip(("dq", "dk", "dv"), got, grads, bounds):
        assert g.dtype == torch.bfloat16 and g.shape == w.shape
        assert_within(g, w, bound, name)
