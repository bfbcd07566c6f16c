"""The error for an unexpected register allocation names what either kernel needs."""

from __future__ import annotations

import re
from pathlib import Path


def test_the_message_names_the_allocations_of_both_kernels(b200):
    here = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention"
    message = b200.strerror(b200.EREGS)
    for file, name in (("attn_fwd.cuh", "kRegsLaunch"), ("attn_bwd.cuh", "kBwdRegsLaunch")):
        (count,) = re.findall(rf"constexpr uint32_t {name} = (\d+);", (here / file).read_text())
        assert re.search(rf"\b{count}\b", message), (file, message)
