"""The degree-5 exponential of sm100_ptx.cuh at its lower end, evaluated in fp32 on the CPU.

The forward that saves its LSE clamps exponents at -127: a hidden key's P then is the smallest
subnormal, which is 0 as bf16, and nothing between the clamp and the normal range is negative or
off by more than 2^-127."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np


def exp2_poly5(x):
    """exp2_poly5_x2, one fp32 operation at a time."""
    here = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention"
    found = re.findall(r"d(\d) = f2_pack\(([-0-9.e]+)f,", (here / "sm100_ptx.cuh").read_text())
    d = {int(i): np.float32(value) for i, value in found}
    magic = np.float32(12582912.0)
    t = x + magic
    f = (x.astype(np.float64) - (t - magic)).astype(np.float32)
    p = np.full_like(x, d[5])
    for i in (4, 3, 2, 1, 0):
        p = (p.astype(np.float64) * f + d[i]).astype(np.float32)
    return (p.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))).view(np.float32)


def test_the_floor_is_zero_as_bf16_and_nothing_wraps():
    import torch

    x = np.concatenate(([-127.0, np.nextafter(np.float32(-127), np.float32(0))],
                        np.linspace(-127, -124, 1_000_001))).astype(np.float32)
    y = exp2_poly5(x)
    want = np.exp2(x.astype(np.float64))
    assert float(torch.from_numpy(y[:1]).bfloat16()) == 0.0 and 0.0 <= y[0] <= 2.0**-149
    assert (y >= 0).all()
    low = x < -126
    assert np.abs(y[low] - want[low]).max() <= 2.0**-127
    assert np.abs(y[~low] / want[~low] - 1).max() < 2.2e-7


