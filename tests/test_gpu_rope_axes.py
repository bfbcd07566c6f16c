"""Positions outside the table where several axes turn the pairs, on a B200."""

from __future__ import annotations

import pytest

from test_gpu_qkv_norm_rope import assert_within, make, plain, seed  # noqa: F401 (seed is a fixture)

pytestmark = pytest.mark.gpu

SECTIONS = [(0, 12, 20), (12, 0, 20), (12, 20, 0), (0, 0, 32), (0, 32), (32, 0, 0, 0)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", SECTIONS)
def test_an_axis_without_pairs_may_hold_any_position(b200, seed, sections, interleaved):  # noqa: F811
    import torch

    case = (2, 20, 3, 2, 64, interleaved, "fp32", "int64", sections)
    qkv, cos, sin, how, grads = make(case, 21)
    outs, out_bounds, dqkv, dqkv_bound, dws, dw_bounds = plain(case, qkv, cos, sin, how, grads)
    for at, pairs in enumerate(sections):
        if pairs == 0:
            how["positions"][at] = torch.tensor([-1, 2**40], device="cuda").repeat(10)
    got = seed.qkv_norm_rope(qkv, 3, 2, cos, sin, **how)
    back = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    assert b200.check_status(qkv.device) == 0
    for name, g, w, bound in zip("qkv", got, outs, out_bounds):
        assert_within(g, w, bound, name)
    for name, g, w, bound in zip(("dqkv", "dqw", "dkw"), back, (dqkv, *dws), (dqkv_bound, *dw_bounds)):
        assert_within(g, w, bound, name)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_one_bad_axis_is_reported_in_both_directions(b200, seed, axis, interleaved):  # noqa: F811
    # Token 7 of batch entry 1 has a bad position on one axis: all its rotated values are NaN,
    # as are the gradients that pass its norm; every other token is as without it.
    import torch

    case = (2, 20, 3, 2, 64, interleaved, "fp32", "int32", (10, 6, 16))
    qkv, cos, sin, how, grads = make(case, 22)
    want = seed.qkv_norm_rope(qkv, 3, 2, cos, sin, **how)
    want_back = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    how["positions"][axis, 1, 7] = cos.shape[0]
    got = seed.qkv_norm_rope(qkv, 3, 2, cos, sin, **how)
    with pytest.raises(b200.B200AttentionError, match="position"):
        b200.check_status(qkv.device)
    back = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    with pytest.raises(b200.B200AttentionError, match="position"):
        b200.check_status(qkv.device)
    for g, w in zip(got[:2], want[:2]):
        assert bool(torch.isnan(g[1, :, 7, :64]).all()) and torch.equal(g[1, :, 7, 64:], w[1, :, 7, 64:])
        g[1, :, 7] = w[1, :, 7]
        assert torch.equal(g, w)
    assert torch.equal(got[2], want[2])
    dqkv, dqw, dkw = back
    assert bool(torch.isnan(dqkv[1, 7, :5, :64]).all())
    assert bool(torch.isnan(dqw[:64]).all()) and bool(torch.isnan(dkw[:64]).all())
    dqkv[1, 7, :5] = want_back[0][1, 7, :5]
    assert torch.equal(dqkv, want_back[0])
