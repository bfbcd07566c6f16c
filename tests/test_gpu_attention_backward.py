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
    (1, 16, 2, 1, 3000, True),    # one token of a long context, eight heads to a key
    (2, 9, 3, 5, 1111, False),
    (1, 1, 1, 3000, 3000, True),     # one head: both passes split along the sequence
    (1, 8, 1, 1500, 1200, True),
    (1, 4, 2, 130, 6000, False),
    (1, 148, 148, 100, 100, True),   # causal pairs of tiles: a single tile per head,
    (2, 74, 74, 129, 129, True),     # two,
    (2, 74, 37, 300, 300, True),     # three, whose middle one has no partner,
    (1, 37, 37, 1000, 1000, True),   # eight
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


@pytest.mark.parametrize("case", CASES)
def test_grouped_forward_matches_fp64(b200, training, case):
    # O: P rounded to bf16 (the row sum is taken over unrounded P), then O rounded once:
    # |err| <= sum_j P (u + e) |V| + u |O|.  LSE: the exponentials' relative error and fp32.
    import torch

    q, k, v, do = make(case, seed=2)
    out, lse, _, _ = plain(q, k, v, do, case[5], b200.default_scale())
    got, got_lse = training.grouped_attention(q, k, v, case[5])
    torch.cuda.synchronize()
    b200.check_status(q.device)
    group = case[1] // case[2]
    kx, vx = (t.double().repeat_interleave(group, 1) for t in (k, v))
    s = b200.default_scale() * (q.double() @ kx.transpose(-1, -2))
    if case[5]:
        i = torch.arange(case[3], device=q.device)[:, None] + case[4] - case[3]
        s = s.masked_fill(torch.arange(case[4], device=q.device)[None, :] > i, -math.inf)
    p = torch.where(lse[..., None] == -math.inf, torch.zeros_like(s), torch.exp(s - lse[..., None]))
    e = 2e-4 + 128 * EPS32 * b200.default_scale() * (q.double().abs() @ kx.abs().transpose(-1, -2))
    e = e + case[4] * EPS32
    assert_within(got, out, 2 * ((p * (U + e)) @ vx.abs()) + U * out.abs(), "out")
    empty = lse == -math.inf
    assert torch.equal(got_lse == -math.inf, empty) and bool((got[empty] == 0).all())
    assert float((got_lse.double() - lse)[~empty].abs().max()) <= 1e-3


def test_equal_shapes_agree_with_the_candidate_forward(b200, training):
    # The same kernel but for the polynomial of its exponentials (relative errors 2.2e-7 and
    # 7.5e-5): both round P and the output to bf16, the LSEs differ by the larger error.
    import torch

    for case in [(1, 4, 4, 512, 512, False), (1, 4, 4, 500, 500, True)]:
        q, k, v, do = make(case, seed=3)
        exact, lse64, _, _ = plain(q, k, v, do, case[5], b200.default_scale())
        out, lse = training.grouped_attention(q, k, v, case[5])
        want, want_lse = b200.attention_forward(q, k, v, case[5])
        s = q.double() @ k.double().transpose(-1, -2) * b200.default_scale()
        p = torch.exp(s - lse64[..., None])
        if case[5]:
            p = p.tril()
        bound = 2 * (U + 1.5e-4) * (p @ v.double().abs()) + 2 * U * exact.abs()
        assert bool(((out.double() - want.double()).abs() <= bound).all())
        assert float((lse - want_lse).abs().max()) <= 1e-4


@pytest.mark.parametrize("seq", [1, 4, 64, 300, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_lse_has_fp32_precision(b200, training, seq, causal):
    # Inputs of a few bits: the scores are exact.  What is left: 2.5e-7 of every exponential,
    # one step per addition of the row sum, and a few of the terms of LSE = m + log(sum).
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seq)
    q, k, v = (torch.randint(-2, 3, (2, 4, seq, 128), device="cuda", generator=gen).bfloat16() / 2 for _ in range(3))
    out, lse = training.grouped_attention(q, k, v, causal)
    s = q.double() @ k.double().transpose(-1, -2) * b200.default_scale()
    if causal:
        s = s.masked_fill(torch.ones((seq, seq), device="cuda", dtype=torch.bool).triu(1), -math.inf)
    want = torch.logsumexp(s, -1)
    most = s.masked_fill(s == -math.inf, 0).abs().amax(-1)
    bound = 2.5e-7 + seq * EPS32 + 8 * EPS32 * (want.abs() + most)
    assert bool(((lse.double() - want).abs() <= bound).all())


def test_rows_without_keys_get_zero_gradients(b200, training):
    import torch

    case = (1, 2, 1, 300, 100, True)  # rows 0..199 see nothing
    q, k, v, do = make(case, seed=4)
    q[:, :, :200] = 1e30   # what no key sees must not matter, however large
    do[:, :, :200] = 1e30
    out, lse = training.grouped_attention(q, k, v, True)
    assert bool((out[:, :, :200] == 0).all()) and bool((lse[:, :, :200] == -math.inf).all())
    dq, dk, dv = training.attention_backward(do, q, k, v, out, lse, True)
    tail = [t[:, :, 200:].contiguous() for t in (do, q, out, lse)]
    dq2, dk2, dv2 = training.attention_backward(tail[0], tail[1], k, v, tail[2], tail[3], True)
    torch.cuda.synchronize()
    b200.check_status(q.device)
    assert bool((dq[:, :, :200] == 0).all())
    _, _, grads, bounds = plain(tail[1], k, v, tail[0], True, b200.default_scale())
    for name, g, w, bound in zip(("dq", "dk", "dv"), (dq[:, :, 200:], dk, dv), grads, bounds):
        assert_within(g, w, 2 * bound, name)  # out and lse are the forward kernel's here
    for g, h in zip((dk, dv), (dk2, dv2)):
        assert bool(torch.isfinite(g.float()).all()) and bool(torch.isfinite(h.float()).all())


def test_large_scores_and_inputs(b200, training):
    # k x 3 makes rows peaked: P is then 0 or 1 almost everywhere.
    import torch

    case = (1, 2, 2, 384, 384, True)
    q, k, v, do = make(case, seed=5, std_do=1e4)
    k = (k * 3).contiguous()
    out, lse, grads, bounds = plain(q, k, v, do, True, b200.default_scale())
    got = training.attention_backward(do, q, k, v, out.bfloat16(), lse.float(), True)
    torch.cuda.synchronize()
    for name, g, w, bound in zip(("dq", "dk", "dv"), got, grads, bounds):
        assert_within(g, w, bound, name)


def test_gradient_against_differences(b200, training):
    # L(q, k, v) = sum dO . O in fp64: a central difference along a random direction d is
    # <grad, d> up to the kernel's bound sum |d| bound and the difference's own error
    # (h^2 / 6 times the third derivative, below 1e-6 of the value at h = 1e-3 here).
    import torch

    case = (1, 4, 2, 150, 210, True)
    q, k, v, do = make(case, seed=6)
    scale = b200.default_scale()
    out, lse, _, bounds = plain(q, k, v, do, True, scale)
    got = training.attention_backward(do, q, k, v, out.bfloat16(), lse.float(), True)
    gen = torch.Generator(device="cuda").manual_seed(7)
    base = [t.double() for t in (q, k, v)]
    for i in range(3):
        d = torch.randn(base[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        value = []
        for h in (1e-3, -1e-3):
            x = list(base)
            x[i] = x[i] + h * d
            value.append(float((plain(*x, do, True, scale)[0] * do.double()).sum()))
        slope = (value[0] - value[1]) / 2e-3
        mine = float((got[i].double() * d).sum())
        assert abs(mine - slope) <= float((bounds[i] * d.abs()).sum()) + 1e-4 * abs(slope), (i, mine, slope)


def test_same_inputs_give_the_same_bits(b200, training):
    import torch

    case = (2, 8, 2, 900, 900, True)
    q, k, v, do = make(case, seed=8)
    out, lse = training.grouped_attention(q, k, v, True)
    first = training.attention_backward(do, q, k, v, out, lse, True)
    for _ in range(3):
        again = training.attention_backward(do, q, k, v, out, lse, True)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


# One head over long sequences, and few rows over many keys: both plans split their work and
# join the pieces from scratch.
SPLIT = [(1, 1, 1, 2500, 2500, True), (1, 8, 2, 3, 9001, False), (1, 2, 1, 300, 5000, True)]


@pytest.mark.parametrize("case", SPLIT)
def test_split_work_on_streams_and_replayed_gives_the_same_bits(b200, training, case):
    import torch

    causal = case[5]
    q, k, v, do = make(case, seed=17)

    def layer():
        out, lse = training.grouped_attention(q, k, v, causal)
        return (out, lse, *training.attention_backward(do, q, k, v, out, lse, causal))

    want = layer()
    torch.cuda.synchronize()
    graphs, kept = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(layer())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):  # two replays and an eager call at once
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        again = layer()
        torch.cuda.synchronize()
        for got in (*kept, again):
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        for results in kept:
            for t in results:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
    del graphs


def test_two_streams_at_once(b200, training):
    import torch

    cases = [(1, 8, 2, 1024, 1024, True), (1, 8, 8, 640, 900, False)]
    sets, want = [], []
    for case in cases:
        q, k, v, do = make(case, seed=9)
        out, lse = training.grouped_attention(q, k, v, case[5])
        sets.append((do, q, k, v, out, lse))
        want.append(training.attention_backward(*sets[-1], case[5]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = training.attention_backward(*sets[i], cases[i][5])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_outputs_into_given_tensors_and_back_to_back_use(b200, training):
    # The gradients are read by the next work in the stream at once: both passes of the
    # backward have to be complete by then.
    import torch

    case = (1, 16, 4, 2048, 2048, True)
    q, k, v, do = make(case, seed=10)
    out, lse = training.grouped_attention(q, k, v, True)
    want = training.attention_backward(do, q, k, v, out, lse, True)
    torch.cuda.synchronize()
    grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
    for _ in range(5):
        for g in grads:
            g.fill_(float("nan"))
        result = training.attention_backward(do, q, k, v, out, lse, True, dq=grads[0], dk=grads[1], dv=grads[2])
        copies = [g.clone() for g in grads]
        # The forward kernel starts early (programmatic launch) behind the backward: it may
        # only see complete gradients.
        after, _ = training.grouped_attention(grads[0], grads[1], grads[2], True)
        torch.cuda.synchronize()
        assert all(r is g for r, g in zip(result, grads))
        assert all(torch.equal(c, w) for c, w in zip(copies, want))
        assert torch.equal(after, training.grouped_attention(want[0], want[1], want[2], True)[0])


def test_captured_backward_replays(b200, training):
    import torch

    case = (1, 8, 4, 700, 700, True)
    q, k, v, do = make(case, seed=11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = training.grouped_attention(q, k, v, True)
        training.attention_backward(do, q, k, v, out, lse, True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):  # two graphs share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = training.grouped_attention(q, k, v, True)
            results.append(training.attention_backward(do, q, k, v, out, lse, True))
        graphs.append(graph)
    for seed in (12, 13):
        fresh = make(case, seed=seed)
        for dst, src in zip((q, k, v, do), fresh):
            dst.copy_(src)
        for graph in graphs:
            graph.replay()
        nq, nk, nv, ndo = fresh
        out, lse = training.grouped_attention(nq, nk, nv, True)
        want = training.attention_backward(ndo, nq, nk, nv, out, lse, True)
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    del graphs


def test_autograd_and_its_refusals(b200, training):
    import torch

    case = (1, 4, 2, 200, 200, True)
    q, k, v, do = make(case, seed=14)
    out, lse = training.grouped_attention(q, k, v, True)
    want = training.attention_backward(do, q, k, v, out, lse, True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    got, got_lse = training.grouped_attention(*leaves, True)
    assert torch.equal(got, out) and not got_lse.requires_grad
    got.backward(do.transpose(1, 2).contiguous().transpose(1, 2))  # a gradient in another layout
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, want))
    # A broadcast gradient.
    for leaf in leaves:
        leaf.grad = None
    got, _ = training.grouped_attention(*leaves, True)
    got.sum().backward()
    ones = training.attention_backward(torch.ones_like(q), q, k, v, out, lse, True)
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, ones))
    # Only the log-sum-exp used: no gradient flows, none is invented.
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            training.grouped_attention(*leaves, True)
        with torch.no_grad():
            training.grouped_attention(*leaves, True)
    del graph


def test_refusals(b200, training):
    import torch

    q, k, v, do = make((1, 4, 2, 64, 96, False), seed=15)
    out, lse = training.grouped_attention(q, k, v, False)
    both = torch.empty((2 * k.numel(),), dtype=k.dtype, device="cuda")
    first, second = (both[at:at + k.numel()].view(k.shape) for at in (0, k.numel() // 2))

    def shifted(t):  # contiguous, but off the 16-byte grid
        return torch.empty((t.numel() + 4,), dtype=t.dtype, device="cuda")[4:].view(t.shape)

    bad = [
        (lambda: training.grouped_attention(q.cpu(), k, v, False), "q must be a CUDA tensor"),
        (lambda: training.grouped_attention(q.half(), k, v, False), "q must be bf16"),
        (lambda: training.grouped_attention(q.transpose(1, 2), k, v, False), "q must be contiguous"),
        (lambda: training.grouped_attention(q[:, :3].contiguous(), k, v, False), "multiple of the key/value heads"),
        (lambda: training.grouped_attention(q, k, v[:, :, :95].contiguous(), False), "same shape"),
        (lambda: training.grouped_attention(q, k, v, False, softmax_scale=0.0), "softmax_scale"),
        (lambda: training.grouped_attention(q[..., :64].contiguous(), k, v, False), "head_dim must be 128"),
        (lambda: training.attention_backward(do[:, :2].contiguous(), q, k, v, out, lse, False), "dout must have"),
        (lambda: training.attention_backward(do.float(), q, k, v, out, lse, False), "dout must be bf16"),
        (lambda: training.attention_backward(do, q, k, v, out, lse[:, :2].contiguous(), False), "lse must have"),
        (lambda: training.attention_backward(do, q, k, v, out, lse.double(), False), "lse must be float32"),
        (lambda: training.attention_backward(do, q, k, v, out, lse, False, dk=torch.empty_like(q)), "dk must have"),
        (lambda: training.attention_backward(do, q, k, v, out, lse, False, dq=q), "dq must not overlap"),
        (lambda: training.attention_backward(do, q, k, v, out, lse, False, dk=v), "dk must not overlap"),
        (lambda: training.attention_backward(do, q, k, v, out, lse, False, dk=first, dv=second), "dv must not"),
        (lambda: training.grouped_attention(shifted(q), k, v, False), "avo_b200_attn_fwd_grouped"),
        (lambda: training.attention_backward(do, q, shifted(k), v, out, lse, False), "avo_b200_attn_bwd"),
    ]
    for call, match in bad:
        with pytest.raises(RuntimeError, match=match):
            call()


def test_empty_sizes(b200, training):
    import torch

    for shape in [(0, 2, 1, 4, 4), (1, 2, 1, 0, 4), (1, 2, 1, 4, 0), (1, 2, 1, 0, 0)]:
        q, k, v, do = make((*shape, True), seed=16)
        out, lse = training.grouped_attention(q, k, v, True)
        grads = training.attention_backward(do, q, k, v, out, lse, True)
        torch.cuda.synchronize()
        assert out.shape == q.shape and lse.shape == q.shape[:3]
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
        for g, like in zip(grads, (q, k, v)):
            assert g.shape == like.shape and bool((g == 0).all())


def test_offsets_past_32_bits(b200, training):
    # q, out and their gradients have more than 2^31 elements; the last heads against the formula.
    import torch

    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 60 GB of device memory")
    case = (16, 1024, 256, 1100, 1100, True)
    q, k, v, do = make(case, seed=21)
    assert q.numel() > 2**31
    out, lse = training.grouped_attention(q, k, v, True)
    heads, kv_heads = slice(-8, None), slice(-2, None)
    sq, sk, sv, sdo = (t[-1:, h].contiguous() for t, h in ((q, heads), (k, kv_heads), (v, kv_heads), (do, heads)))
    exact, lse64, want, bounds = plain(sq, sk, sv, sdo, True, b200.default_scale())
    assert float((out[-1:, heads].double() - exact).abs().max()) <= 2e-2
    assert float((lse[-1:, heads].double() - lse64).abs().max()) <= 1e-3
    out[-1:, heads] = exact.bfloat16()
    lse[-1:, heads] = lse64.float()
    grads = training.attention_backward(do, q, k, v, out, lse, True)
    torch.cuda.synchronize()
    for name, g, h, w, bound in zip(("dq", "dk", "dv"), grads, (heads, kv_heads, kv_heads), want, bounds):
        assert_within(g[-1:, h], w, bound, name)
