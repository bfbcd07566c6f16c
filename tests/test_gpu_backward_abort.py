"""The attention gradient's own watchdog path: a wait that runs out ends in a reported abort.

As for the forward kernel, a child process sets AVO_B200_TEST_SKIP_LOAD=n, so every CTA's
producer leaves out its (n + 1)th streamed copy, and a 20 ms watchdog.  The wait for that copy
runs out, the CTA aborts in the middle of an item, at an item's start or in a later item, and
every role must leave its pipeline cleanly (the model in test_bwd_protocol.py runs the same
schedules on the CPU).  The launches must return and set the watchdog bit, never the drain
bit.  The context stays usable: a problem whose CTAs have fewer copies than n + 1 gives the
same bits after the aborts as before.  Nothing faults, traps or hangs: a copy that is never
issued only makes a bounded wait give up.
"""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
TRAINING = ROOT / "avo-ampere_b200" / "candidates" / "cuda_b200_attention" / "b200_training.py"

CHILD = r"""
import importlib.util, sys, torch
spec = importlib.util.spec_from_file_location("avo_b200_training_binding", sys.argv[1])
t = importlib.util.module_from_spec(spec)
sys.modules[spec.name] = t
spec.loader.exec_module(t)
gen = torch.Generator(device="cuda").manual_seed(0)

def make(heads, kv_heads, seq):
    def randn(h):
        return torch.randn((1, h, seq, 128), device="cuda", generator=gen).bfloat16()
    return randn(heads), randn(heads), randn(kv_heads), randn(kv_heads), randn(heads)

def run(do, q, k, v, out, causal):
    lse = torch.full(q.shape[:3], 6.0, device="cuda")
    got = t.attention_backward(do, q, k, v, out, lse, causal)
    torch.cuda.synchronize()
    word = t.b.status_word(q.device)
    status = int(word.item())
    word.zero_()
    return got, status

small = make(2, 2, 128)
before, status = run(*small, False)
print("SMALL", status, flush=True)
big = make(*(int(x) for x in sys.argv[2].split(",")))
for causal in (False, True):
    print("STATUS", run(*big, causal)[1], flush=True)
after, status = run(*small, False)
print("SMALL", status, flush=True)
print("SAME", all(torch.equal(x, y) for x, y in zip(before, after)), flush=True)
"""


@pytest.mark.parametrize(
    "shape,skip",
    [
        ("8,8,2048", 5),     # 128 items of 16 tiles for each pass: abort in the first item
        ("8,2,2048", 5),     # shared heads: fewer items than CTAs, both passes side by side
        ("300,300,256", 5),  # 600 items of two tiles: abort in a later item of each CTA
    ],
)
def test_watchdog_abort_returns_and_reports(shape, skip):
    env = dict(os.environ)
    env["AVO_B200_TEST_SKIP_LOAD"] = str(skip)
    env["AVO_B200_WATCHDOG_MS"] = "20"
    proc = subprocess.run([sys.executable, "-c", CHILD, str(TRAINING), shape], env=env, capture_output=True,
                          text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-2000:]
    lines = proc.stdout.splitlines()
    watchdog_bit, drain_bit = 1, 2
    assert [line for line in lines if line.startswith("SMALL")] == ["SMALL 0", "SMALL 0"], lines
    statuses = [int(line.split()[1]) for line in lines if line.startswith("STATUS")]
    assert len(statuses) == 2
    assert all(s & watchdog_bit for s in statuses), statuses
    assert not any(s & drain_bit for s in statuses), statuses
    assert "SAME True" in lines, lines
