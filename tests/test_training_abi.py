"""Host-side refusals of the training entry points (no GPU: they answer before any device call)."""

from __future__ import annotations

import ctypes

INVALID, NODEV = 1, 2
FAKE = 0x10000


def _bwd(lib, **over):
    a = dict(dout=FAKE, q=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, batch=1, heads=4,
             kv_heads=2, seq_q=64, seq_kv=64, head_dim=128, causal=0, scale=0.088, ws=FAKE, ws_bytes=1 << 24)
    assert set(over) <= set(a)
    a.update(over)
    return lib.avo_b200_attn_bwd(*a.values(), None, None)


def test_attention_backward_refusals(b200):
    lib = b200.load_library()
    for name in ("dout", "q", "k", "v", "o", "lse", "dq", "dk", "dv", "ws"):
        assert _bwd(lib, **{name: None}) == INVALID, name
    for name in ("dout", "q", "k", "v", "o"):
        assert _bwd(lib, **{name: FAKE + 8}) == INVALID, name
    for name in ("dq", "dk", "dv"):
        assert _bwd(lib, **{name: FAKE + 16}) == INVALID, name
    for over in (dict(head_dim=64), dict(heads=5), dict(kv_heads=0), dict(batch=-1), dict(seq_q=-1), dict(seq_kv=-4),
                 dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(ws=FAKE + 16),
                 dict(ws_bytes=1023), dict(seq_q=2**31 - 1), dict(batch=2**31 - 1, heads=2)):
        assert _bwd(lib, **over) == INVALID, over


def test_attention_backward_workspace_size(b200):
    lib = b200.load_library()
    size = ctypes.c_size_t(0)
    ask = lib.avo_b200_attn_bwd_workspace_size
    assert ask(1, 4, 2, 64, 64, 0, None) == INVALID
    assert ask(1, 4, 3, 64, 64, 1, ctypes.byref(size)) == INVALID
    for batch, heads, seq in ((1, 4, 1), (2, 8, 128), (1, 3, 129), (3, 2, 1000)):
        for causal in (0, 1):
            assert ask(batch, heads, 1, seq, 77, causal, ctypes.byref(size)) == 0
            assert size.value >= batch * -(-heads * seq // 128) * 1024
    # A long sequence of one head is split along itself: partial sums in fp32.
    assert ask(1, 1, 1, 4096, 4096, 0, ctypes.byref(size)) == 0
    assert size.value > 2 * 4096 * 128 * 4
    # The largest sizes are answered without a loop over them.
    assert ask(1, 1, 1, 2**31 - 1000, 2**31 - 1000, 1, ctypes.byref(size)) == 0


def test_grouped_forward_refusals(b200):
    lib = b200.load_library()

    def call(q=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=None, batch=1, heads=4, kv_heads=2, sq=64, skv=64, d=128, causal=0,
             scale=0.088, ws=None, ws_bytes=0):
        return lib.avo_b200_attn_fwd_grouped(q, k, v, o, lse, batch, heads, kv_heads, sq, skv, d, causal, scale, ws,
                                             ws_bytes, None, None)

    for over in (dict(q=None), dict(k=None), dict(o=FAKE + 8), dict(heads=3), dict(kv_heads=0), dict(d=64),
                 dict(scale=-1.0), dict(batch=-1), dict(sq=-1), dict(skv=-1), dict(batch=2**30, heads=4),
                 dict(lse=FAKE + 2), dict(ws=FAKE + 8, ws_bytes=1 << 30)):
        assert call(**over) == INVALID, over
    assert call(batch=0) == 0 and call(sq=0) == 0


def _rope(lib, backward=False, **over):
    a = dict(qkv=FAKE, sb=1 << 20, ss=1024, q=FAKE, k=FAKE, v=FAKE)
    if backward:
        a = dict(q=FAKE, k=FAKE, v=FAKE, qkv=FAKE, sb=1 << 20, ss=1024, dqkv=FAKE, dqw=FAKE, dkw=FAKE)
    a.update(batch=1, seq=4, heads=4, kv_heads=2, d=128, qw=FAKE, kw=FAKE, bf16=0, cos=FAKE, sin=FAKE, rows=16,
             rot=128, inter=0, pos=None, pos64=0, pa=0, pb=0, ps=1, axes=1, sections=None, eps=1e-6)
    if backward:
        a.update(ws=FAKE, ws_bytes=1 << 24)
    assert set(over) <= set(a)
    a.update(over)
    fn = lib.avo_b200_qkv_norm_rope_bwd if backward else lib.avo_b200_qkv_norm_rope
    return fn(*a.values(), None, None)


def test_qkv_norm_rope_refusals(b200):
    lib = b200.load_library()
    three = (ctypes.c_int * 3)(16, 24, 24)
    wrong = (ctypes.c_int * 3)(16, 24, 25)
    negative = (ctypes.c_int * 3)(-8, 36, 36)
    for backward in (False, True):
        for over in (dict(qkv=None), dict(qkv=FAKE + 8), dict(sb=4), dict(ss=1028), dict(q=None), dict(v=None),
                     dict(k=FAKE + 4), dict(batch=-1), dict(seq=-1), dict(heads=-1), dict(kv_heads=-2), dict(d=64),
                     dict(kw=None), dict(qw=FAKE + 4), dict(cos=None), dict(sin=FAKE + 4), dict(rows=0),
                     dict(seq=17), dict(rot=0), dict(rot=24), dict(rot=144), dict(axes=0), dict(axes=5),
                     dict(axes=3, sections=ctypes.addressof(three)), dict(axes=3, pos=FAKE),
                     dict(axes=3, pos=FAKE, sections=ctypes.addressof(wrong)),
                     dict(axes=3, pos=FAKE, sections=ctypes.addressof(negative)), dict(pos=FAKE + 2),
                     dict(pos=FAKE + 4, pos64=1), dict(eps=-1.0), dict(eps=float("nan")),
                     dict(batch=2**20, seq=2**12, pos=FAKE)):
            assert _rope(lib, backward, **over) == INVALID, (backward, over)
    assert _rope(lib, batch=0) == 0 and _rope(lib, heads=0, kv_heads=0) == 0
    assert _rope(lib, True, dqkv=None) == INVALID and _rope(lib, True, dqw=None) == INVALID
    # The backward's workspace is checked against the device's CTA count, so after the device.
    import torch

    if not torch.cuda.is_available():
        assert _rope(lib) == NODEV and _rope(lib, True) == NODEV and _bwd(lib) == NODEV


def test_python_checks_without_a_gpu():
    import importlib.util
    from pathlib import Path

    import pytest
    import torch

    path = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention_seed.py"
    spec = importlib.util.spec_from_file_location("avo_candidate_b200_seed_training", path)
    seed = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(seed)
    q = torch.zeros((1, 2, 8, 128), dtype=torch.bfloat16)
    lse = torch.zeros((1, 2, 8))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        seed.grouped_attention(q, q, q, False)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        seed.attention_backward(q, q, q, q, q, lse, False)
    with pytest.raises(RuntimeError, match="qkv must be a CUDA tensor"):
        seed.qkv_norm_rope(q, 2, 3, lse, lse)
    with pytest.raises(RuntimeError, match="dq must be a CUDA tensor"):
        seed.qkv_norm_rope_backward(q, q, q, q, lse, lse)


def test_degree_five_exponential_is_the_fitted_polynomial():
    """The constants of exp2_poly5_x2 are what exp2_poly.py derives, within the stated error."""
    import importlib.util
    import re
    from pathlib import Path

    import numpy as np

    here = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention"
    spec = importlib.util.spec_from_file_location("avo_b200_exp2_fit_5", here / "exp2_poly.py")
    fit = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(fit)
    found = dict(re.findall(r"d(\d) = f2_pack\(([-0-9.e]+)f,", (here / "sm100_ptx.cuh").read_text()))
    header = np.float32([float(found[str(i)]) for i in range(6)])
    assert np.array_equal(header, np.float32(fit.float32_coefficients(5)[0]))
    f = np.linspace(-0.5, 0.5, 400_001).astype(np.float32)
    p = np.full_like(f, header[5])
    for c in header[4::-1]:
        p = (p.astype(np.float64) * f + c).astype(np.float32)  # an fp32 FMA
    assert np.abs(p / np.exp2(f.astype(np.float64)) - 1).max() < 2.2e-7
