"""grouped_attention on a B200 against 64 bits, with the bounds that its formulas give and no slack.

With u = 2^-8 (half a bf16 step), eps = 2^-24, A = scale * sum_d |q k| and M = max_j |s| of a row,
a probability's fp32 value before the division by the row sum has the relative error

    e_j = 2.5e-7 (the exponential) + 128 eps A_j (the dot product) + 3 eps |s_j| (the scale's
          roundings) + eps (|s_j| + M + 11) (the exponent: the row's reference value lies within
          2^15, that is 10.4 in natural units, of its maximum)

and joining the pieces of a row multiplies by at most eight exponentials, e_m = 8 (2.5e-7 +
eps (2 M + 11)).  The row sum l adds n keys: its relative error is L = sum_j P_j e_j + n eps + e_m.
P is rounded to bf16 for the product with V, whose n terms are added in fp32; the output is
divided by l (two roundings) and rounded once:

    |O err|   <= 1.01 (sum_j P_j |V_j| (u + e_j + e_m + n eps) + |O| (L + 2 eps)) + u |O|
    |LSE err| <= L + 8 eps (|LSE| + M + 1)

where 1.01 covers the products of two of these errors.
"""

from __future__ import annotations

import math

import pytest
from test_gpu_attention_backward import CASES, EPS32, U, make

pytestmark = pytest.mark.gpu

# Causal, from two items of 256 rows per multiprocessor on: whole items in lists, several query
# heads to a key/value head among them.
LISTS = [
    # batch, heads, kv_heads, seq_q, seq_kv, causal
    (2, 16, 4, 2400, 2400, True),
    (4, 32, 8, 1111, 1500, True),
    (2, 96, 1, 513, 300, True),      # rows that see no key, one key/value head for all
    (37, 8, 2, 129, 700, True),
    (1, 512, 128, 1025, 1025, True),
]


@pytest.fixture(scope="module")
def seed():
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention_seed.py"
    spec = importlib.util.spec_from_file_location("avo_candidate_b200_seed_grouped", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def check(b200, q, k, v, causal, got, got_lse):
    """Compares out and lse with the formula, one batch entry and key/value head at a time."""
    import torch

    scale = b200.default_scale()
    batch, heads, seq_q, _ = q.shape
    kv_heads, n = k.shape[1], k.shape[2]
    group = heads // kv_heads
    hidden = torch.arange(n, device=q.device) > torch.arange(seq_q, device=q.device)[:, None] + n - seq_q
    for b in range(batch):
        for g in range(kv_heads):
            mine = slice(g * group, (g + 1) * group)
            qh, kh, vh = q[b, mine].double(), k[b, g].double(), v[b, g].double()
            s = scale * (qh @ kh.T)
            if causal:
                s = s.masked_fill(hidden, -math.inf)
            lse = torch.logsumexp(s, -1)
            empty = lse == -math.inf
            p = torch.exp(s - torch.where(empty, 0.0, lse)[..., None])
            out = p @ vh
            size = s.abs().masked_fill(s == -math.inf, 0.0)
            most = size.amax(-1) if n else torch.zeros_like(lse)
            e = 2.5e-7 + 128 * EPS32 * scale * (qh.abs() @ kh.abs().T) + EPS32 * (4 * size + most[..., None] + 11)
            e_m = 8 * (2.5e-7 + EPS32 * (2 * most + 11))
            total = (p * e).sum(-1) + n * EPS32 + e_m
            bound = 1.01 * ((p * (U + e + e_m[..., None] + n * EPS32)) @ vh.abs()
                            + out.abs() * (total[..., None] + 2 * EPS32)) + U * out.abs()
            err = (got[b, mine].double() - out).abs()
            assert bool((err <= bound + 1e-30).all()), ("out", b, g, float((err / (bound + 1e-30)).max()))
            mine_lse = got_lse[b, mine]
            assert torch.equal(mine_lse == -math.inf, empty) and bool((got[b, mine][empty] == 0).all())
            err = (mine_lse.double() - lse).abs()[~empty]
            allowed = (total + 8 * EPS32 * (lse.abs() + most + 1))[~empty]
            assert bool((err <= allowed).all()), ("lse", b, g, float((err / allowed).max()))


@pytest.mark.parametrize("case", CASES + LISTS)
def test_forward_within_the_derived_bounds(b200, seed, case):
    import torch

    q, k, v, _ = make(case, seed=31)
    if case in LISTS:
        assert b200.grouped_plan(*case, sm_count=torch.cuda.get_device_properties(0).multi_processor_count,
                                 split=False)[0] == 2
    got, got_lse = seed.grouped_attention(q, k, v, case[5])
    again, again_lse = seed.grouped_attention(q, k, v, case[5])
    torch.cuda.synchronize()
    b200.check_status(q.device)
    assert torch.equal(got, again) and torch.equal(got_lse, again_lse)
    check(b200, q, k, v, case[5], got, got_lse)


@pytest.mark.parametrize("case,splits", [((1, 4, 1, 512, 512, True), False), ((4, 16, 16, 1184, 256, False), False),
                                         ((1, 8, 2, 3, 9001, False), True), ((1, 16, 2, 1, 9001, True), True)])
def test_scratch_is_taken_only_where_the_plan_splits(b200, seed, case, splits):
    # The split plan's scratch is some 38 MB; beside it a call allocates out and lse, each
    # rounded up to a block of at most 2 MB more.
    import torch

    q, k, v, _ = make(case, seed=32)
    seed.grouped_attention(q, k, v, case[5])
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out, lse = seed.grouped_attention(q, k, v, case[5])
    taken = torch.cuda.max_memory_allocated() - before
    results = out.numel() * 2 + lse.numel() * 4
    scratch = b200.workspace(0).numel()
    assert b200.grouped_plan(*case)[0] == (1 if splits else 0)
    assert taken >= results + scratch if splits else taken <= results + (4 << 20)


# NaN: in whole items, in lists, and in the first and in a later piece of split work.
NAN_CASES = [((1, 2, 1, 40, 40, True), (0, 1, 2, 17, 39)), ((1, 2, 2, 300, 300, True), (0, 1, 129, 288)),
             ((2, 74, 37, 300, 300, True), (16, 130)), ((1, 2, 1, 1, 1, False), (0,)),
             ((1, 8, 2, 3, 9001, False), (0, 1, 4800, 9000))]


@pytest.mark.parametrize("case,places", NAN_CASES)
def test_nan_reaches_exactly_the_rows_that_see_it(b200, seed, case, places):
    # A score that is NaN makes its row NaN, LSE included, wherever its key lies in a tile; rows
    # that do not see the key, or belong to another query, keep their bits.
    import torch

    q, k, v, _ = make(case, seed=33)
    seq_q, seq_kv, causal = case[3:]
    clean, clean_lse = seed.grouped_attention(q, k, v, causal)
    row = torch.arange(seq_q, device="cuda")
    for at in places:
        for what in ("key", "query"):
            x = (k if what == "key" else q).clone()
            if what == "query" and at >= seq_q:
                continue
            x[-1, -1, at, 5] = float("nan")
            out, lse = seed.grouped_attention(*((q, x) if what == "key" else (x, k)), v, causal)
            bad = torch.zeros(case[0], case[1], seq_q, dtype=torch.bool, device="cuda")
            if what == "query":
                bad[-1, -1, at] = True
            else:
                bad[-1, -(case[1] // case[2]):] = row + seq_kv - seq_q >= at if causal else True
            torch.cuda.synchronize()
            assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(lse), bad), (what, at)
            assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad]), (what, at)
    b200.check_status(q.device)


@pytest.mark.parametrize("case", [(1, 2, 1, 40, 40, True), (1, 8, 2, 3, 9001, False)])
def test_infinite_scores_make_a_row_nan(b200, seed, case):
    # Scores of +infinity, as the softmax of the definition: infinity - infinity is NaN.
    import torch

    q, k, v, _ = make(case, seed=34)
    q[0, 0, 2, 7] = float("inf")
    out, lse = seed.grouped_attention(q, k.abs(), v, case[5])
    torch.cuda.synchronize()
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    bad[0, 0, 2] = True
    assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(lse), bad)


@pytest.mark.parametrize("at", [0, 1, 2, 150])
def test_gradients_of_a_nan_query(b200, seed, at):
    # Its own gradient is NaN, no gradient of a key that it sees is finite; the other queries'
    # gradients and the other key/value heads keep their bits.
    import torch

    q, k, v, do = make((1, 4, 2, 300, 300, True), seed=35)
    out, lse = seed.grouped_attention(q, k, v, True)
    clean = seed.attention_backward(do, q, k, v, out, lse, True)
    q[0, 3, at, 5] = float("nan")
    out, lse = seed.grouped_attention(q, k, v, True)
    dq, dk, dv = seed.attention_backward(do, q, k, v, out, lse, True)
    torch.cuda.synchronize()
    b200.check_status(q.device)
    assert bool(torch.isnan(dq[0, 3, at]).all())
    dq[0, 3, at] = clean[0][0, 3, at]
    assert torch.equal(dq, clean[0])
    for got, want in ((dk, clean[1]), (dv, clean[2])):
        assert torch.equal(got[0, 0], want[0, 0]) and not bool(torch.isfinite(got[0, 1, :at + 1]).any())


def test_offsets_past_32_bits_within_the_derived_bounds(b200, seed):
    # q and out have more than 2^31 elements; the last heads of the last batch entry.
    import torch

    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    q, k, v, _ = make((16, 1024, 256, 1100, 1100, True), seed=36)
    assert q.numel() > 2**31
    out, lse = seed.grouped_attention(q, k, v, True)
    torch.cuda.synchronize()
    b200.check_status(q.device)
    few = (t[-1:, h] for t, h in ((q, slice(-8, None)), (k, slice(-2, None)), (v, slice(-2, None))))
    check(b200, *few, True, out[-1:, -8:], lse[-1:, -8:])


@pytest.mark.parametrize("case", [(1, 2, 1, 130, 130, True), (1, 4, 2, 90, 300, True), (2, 74, 37, 300, 300, True)])
def test_hidden_values_add_nothing_however_large(b200, seed, case):
    # Rows that do not see the last keys keep their bits when those hold the type's largest and
    # lowest values; 2^-125 of them would be 8.
    import torch

    q, k, v, _ = make(case, seed=37)
    out, lse = seed.grouped_attention(q, k, v, True)
    few = 40
    v[:, :, -few:, ::2] = torch.finfo(torch.bfloat16).max
    v[:, :, -few:, 1::2] = torch.finfo(torch.bfloat16).min
    got, got_lse = seed.grouped_attention(q, k, v, True)
    torch.cuda.synchronize()
    assert torch.equal(got[:, :, :-few], out[:, :, :-few]) and torch.equal(got_lse, lse)
