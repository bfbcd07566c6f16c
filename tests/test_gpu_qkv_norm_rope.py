"""qkv_norm_rope and its gradient on a B200 against a plain implementation in 64 bits.

Tolerances, per element, from the formulas (e = 2^-24, u = 2^-8 half a bf16 step): with
Y = r (|x w cos| + |p w_p sin|) every fp32 path to y has fewer than 40 roundings (128 squares
summed 8 in a row and 4 across lanes, the root, the products), so |y err| <= 40 e Y + u |y|.
With G = |dy cos| + |p(dy) sin|: |dx err| <= 64 e r (G w + |x_hat| mean(G w |x_hat|)) + u |dx|,
and a weight's gradient, a sum of fewer than 128 terms in a row at any level here, is within
256 e sum G |x_hat|.
"""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-8
E = 2.0**-24

CASES = [
    # batch, seq, heads, kv_heads, rotary, interleaved, weights, positions, sections
    (1, 1, 1, 1, 128, False, "fp32", None, None),
    (1, 1, 16, 4, 128, False, "bf16", "int64", None),
    (2, 7, 3, 1, 64, False, "fp32", "int32", None),
    (3, 33, 4, 2, 96, True, "bf16", "int64", None),
    (1, 129, 5, 5, 32, False, None, None, None),
    (2, 50, 8, 2, 128, True, None, "shared", None),
    (2, 65, 4, 4, 128, False, "fp32", "int64", (16, 24, 24)),
    (1, 77, 6, 3, 128, True, "bf16", "int32", (10, 27, 27)),
    (2, 20, 2, 1, 16, False, "fp32", "shared", (3, 5)),
    (2, 20, 2, 1, 64, True, "fp32", "int64", (8, 0, 20, 4)),
    (1, 40, 0, 3, 128, False, "fp32", None, None),
    (1, 40, 3, 0, 128, False, "fp32", None, None),
    (4, 600, 17, 3, 128, False, "fp32", "int64", None),
    (1, 5000, 32, 8, 128, False, "bf16", None, None),
]


@pytest.fixture(scope="module")
def seed():
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates" / "cuda_b200_attention_seed.py"
    spec = importlib.util.spec_from_file_location("avo_candidate_b200_seed_rope", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def make(case, seed_value, table=None):
    import torch

    batch, seq, heads, kv_heads, rotary, interleaved, weights, positions, sections = case
    gen = torch.Generator(device="cuda").manual_seed(seed_value)
    qkv = torch.randn((batch, seq, heads + 2 * kv_heads, 128), device="cuda", generator=gen).bfloat16()
    table = table or max(seq, 97)
    angle = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        10000.0, -torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    how = {"interleaved": interleaved, "sections": sections}
    if weights:
        dtype = {"fp32": torch.float32, "bf16": torch.bfloat16}[weights]
        for name in ("q_weight", "k_weight"):
            how[name] = (1 + 0.2 * torch.randn(128, device="cuda", generator=gen)).to(dtype)
    if positions:
        shape = (seq,) if positions == "shared" else (batch, seq)
        if sections:
            shape = (len(sections), *shape)
        how["positions"] = torch.randint(0, table, shape, device="cuda", generator=gen).to(
            torch.int32 if positions == "int32" else torch.int64)
    grads = [torch.randn((batch, n, seq, 128), device="cuda", generator=gen).bfloat16()
             for n in (heads, kv_heads, kv_heads)]
    return qkv, angle.cos().float(), angle.sin().float(), how, grads


def turn(case, cos, sin, how):
    """cos and sin per pair, fp64, [B, S, 1, rotary / 2]."""
    import torch

    batch, seq, rotary, sections = case[0], case[1], case[4], case[8]
    pairs = rotary // 2
    pos = how.get("positions")
    if pos is None:
        pos = torch.arange(seq, device="cuda")
    if not sections:
        pos, sections = pos[None], (pairs,)
    pos = pos.expand(len(sections), batch, seq) if pos.dim() == 3 else pos[:, None].expand(-1, batch, -1)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    row = pos[axis].permute(1, 2, 0).long()
    col = torch.arange(pairs, device="cuda")
    return cos.double()[row, col][:, :, None], sin.double()[row, col][:, :, None]


def halves(x, rotary, interleaved):
    return (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])


def join(a, b, rest, interleaved):
    import torch

    return torch.cat((torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1), rest), -1)


def rotate(x, c, s, case):
    rotary, inter = case[4], case[5]
    a, b = halves(x, rotary, inter)
    return join(a * c - b * s, b * c + a * s, x[..., rotary:], inter)


def rotate_abs(x, c, s, case):
    """Sum of the absolute values of the terms of each rotated element."""
    rotary, inter = case[4], case[5]
    a, b = halves(x.abs(), rotary, inter)
    c, s = c.abs(), s.abs()
    return join(a * c + b * s, b * c + a * s, x[..., rotary:].abs(), inter)


def plain(case, qkv, cos, sin, how, grads, eps=1e-6):
    import torch

    heads, kv_heads = case[2], case[3]
    c, s = turn(case, cos, sin, how)
    x = qkv.double()
    parts = x[:, :, :heads], x[:, :, heads:heads + kv_heads]
    outs, out_bounds, dxs, dx_bounds, dws, dw_bounds = [], [], [], [], [], []
    for part, weight, dy in zip(parts, ("q_weight", "k_weight"), grads):
        w = how[weight].double() if weight in how else torch.ones(128, device="cuda", dtype=torch.float64)
        r = (part.square().mean(-1, keepdim=True) + eps).rsqrt() if weight in how else torch.ones_like(part[..., :1])
        xh = part * r
        y = rotate(xh * w, c, s, case)
        outs.append(y.transpose(1, 2))
        out_bounds.append((40 * E * rotate_abs(xh * w, c, s, case) + U * y.abs()).transpose(1, 2))
        d = dy.double().transpose(1, 2)
        g, big = rotate(d, c, -s, case), rotate_abs(d, c, s, case)
        if weight in how:
            dx = r * (g * w - xh * (g * w * xh).mean(-1, keepdim=True))
            bound = 64 * E * r * (big * w.abs() + xh.abs() * (big * w.abs() * xh.abs()).mean(-1, keepdim=True))
            dws.append((g * xh).sum((0, 1, 2)))
            dw_bounds.append(256 * E * (big * xh.abs()).sum((0, 1, 2)))
        else:
            dx, bound = g, 64 * E * big
        dxs.append(dx)
        dx_bounds.append(bound + U * dx.abs())
    v = qkv[:, :, heads + kv_heads:].transpose(1, 2)
    outs.append(v.double())
    out_bounds.append(torch.zeros_like(outs[-1]))
    dv = grads[2].double().transpose(1, 2)
    return (outs, out_bounds, torch.cat((*dxs, dv), 2), torch.cat((*dx_bounds, torch.zeros_like(dv)), 2), dws,
            dw_bounds)


def assert_within(got, want, bound, what):
    err = (got.double() - want).abs()
    over = err > bound * 1.001 + 1e-38
    assert not bool(over.any()), (what, int(over.sum()), float((err / (bound + 1e-38)).max()))


@pytest.mark.parametrize("case", CASES)
def test_matches_fp64(b200, seed, case):
    import torch

    qkv, cos, sin, how, grads = make(case, 1)
    outs, out_bounds, dqkv, dqkv_bound, dws, dw_bounds = plain(case, qkv, cos, sin, how, grads)
    got = seed.qkv_norm_rope(qkv, case[2], case[3], cos, sin, **how)
    back = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    torch.cuda.synchronize()
    b200.check_status(qkv.device)
    for name, g, w, bound in zip("qkv", got, outs, out_bounds):
        assert g.is_contiguous() and g.dtype == torch.bfloat16 and g.shape == w.shape
        assert_within(g, w, bound, name)
    assert back[0].is_contiguous() and back[0].shape == qkv.shape
    assert_within(back[0], dqkv, dqkv_bound, "dqkv")
    if case[6] is None:
        assert back[1] is None and back[2] is None
    else:
        for name, g, w, bound in zip(("dq_weight", "dk_weight"), back[1:], dws, dw_bounds):
            assert g.dtype == torch.float32
            assert_within(g, w, bound, name)


def test_strided_projection_and_positions(b200, seed):
    import torch

    case = (2, 37, 4, 2, 128, False, "fp32", "int64", None)
    qkv, cos, sin, how, grads = make(case, 2)
    want = seed.qkv_norm_rope(qkv, 4, 2, cos, sin, **how)
    want_back = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    # The projection as a part of wider rows, tokens in front of the batch; positions strided.
    wide = torch.full((37, 2, 8 * 128 + 40), float("nan"), device="cuda", dtype=torch.bfloat16)
    view = wide[:, :, 8:8 + 8 * 128].unflatten(2, (8, 128)).transpose(0, 1)
    view.copy_(qkv)
    pos = torch.zeros((37, 2, 3), device="cuda", dtype=torch.int64)
    pos[:, :, 1] = how["positions"].transpose(0, 1)
    how["positions"] = pos[:, :, 1].transpose(0, 1)
    got = seed.qkv_norm_rope(view, 4, 2, cos, sin, **how)
    back = seed.qkv_norm_rope_backward(*grads, view, cos, sin, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(back, want_back))
    # Positions of one row of a batch, expanded.
    how["positions"] = how["positions"][:1].contiguous()
    one = seed.qkv_norm_rope(qkv[:1].contiguous(), 4, 2, cos, sin, **how)
    how["positions"] = how["positions"].expand(2, -1)
    both = seed.qkv_norm_rope(qkv[:1].expand(2, -1, -1, -1), 4, 2, cos, sin, **how)
    for a, b in zip(one, both):
        assert torch.equal(b[0], a[0]) and torch.equal(b[1], a[0])


def test_positions_outside_the_table_are_reported(b200, seed):
    import torch

    case = (1, 6, 2, 1, 64, False, "fp32", "int64", None)
    qkv, cos, sin, how, grads = make(case, 3, table=50)
    how["positions"] = torch.tensor([[0, 49, 50, -1, 2**40, 7]], device="cuda")
    q, k, v = seed.qkv_norm_rope(qkv, 2, 1, cos, sin, **how)
    with pytest.raises(b200.B200AttentionError, match="position"):
        b200.check_status(qkv.device)
    assert b200.check_status(qkv.device) == 0  # reported once
    bad = torch.tensor([False, False, True, True, True, False], device="cuda")
    for t in (q, k):
        assert torch.equal(torch.isnan(t[0, 0]).all(-1) | torch.isnan(t[0, 0, :, :64]).all(-1), bad)
        assert not bool(torch.isnan(t[:, :, :, 64:]).any())
    assert torch.equal(v, qkv[:, :, 3:].transpose(1, 2))
    dqkv, _, _ = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    with pytest.raises(b200.B200AttentionError, match="position"):
        b200.check_status(qkv.device)
    assert torch.equal(torch.isnan(dqkv[0, :, 0]).any(-1), bad)


def test_zero_rows_and_large_values(b200, seed):
    import torch

    case = (1, 9, 2, 1, 128, False, "fp32", None, None)
    qkv, cos, sin, how, grads = make(case, 4)
    qkv[0, 3] = 0
    qkv[0, 4] *= 1e15
    qkv[0, 5] *= 1e-15
    outs, bounds, dqkv, dqkv_bound, dws, dw_bounds = plain(case, qkv, cos, sin, how, grads)
    got = seed.qkv_norm_rope(qkv, 2, 1, cos, sin, **how)
    back = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    for g, w, bound in zip(got, outs, bounds):
        assert_within(g, w, bound, "out")
    assert_within(back[0], dqkv, dqkv_bound, "dqkv")
    for g, w, bound in zip(back[1:], dws, dw_bounds):
        assert_within(g, w, bound, "weight")


def test_gradient_against_differences(b200, seed):
    # L = sum dy . y in fp64 along random directions; the central difference at h = 1e-4 is
    # off by h^2 times third derivatives (below 1e-6 of the value).
    import torch

    case = (1, 12, 3, 2, 64, True, "fp32", "int64", (12, 20))
    qkv, cos, sin, how, grads = make(case, 5)
    dqkv, dqw, dkw = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
    _, _, _, dqkv_bound, _, dw_bounds = plain(case, qkv, cos, sin, how, grads)
    gen = torch.Generator(device="cuda").manual_seed(6)

    def loss(x, hw):
        return sum(float((y * d.double()).sum()) for y, d in zip(plain(case, x, cos, sin, hw, grads)[0], grads))

    for what, mine, bound in (("qkv", dqkv, dqkv_bound), ("q_weight", dqw, dw_bounds[0]), ("k_weight", dkw, dw_bounds[1])):
        base = qkv.double() if what == "qkv" else how[what].double()
        d = torch.randn(base.shape, device="cuda", generator=gen, dtype=torch.float64)
        value = []
        for h in (1e-4, -1e-4):
            x = base + h * d
            value.append(loss(x, how) if what == "qkv" else loss(qkv.double(), {**how, what: x}))
        slope = (value[0] - value[1]) / 2e-4
        got = float((mine.double() * d).sum())
        assert abs(got - slope) <= float((bound * d.abs()).sum()) + 1e-5 * abs(slope) + 1e-7, (what, got, slope)


def test_layer_forward_and_backward_together(b200, seed):
    # The layer's training step as a user runs it: projection -> q, k, v -> attention -> loss,
    # by autograd, against the plain calls (bit for bit) and against fp64 autograd.  The
    # roundings on the way (q and k perturb a score s by at most 2 u |s|; P, dS, out, the
    # attention gradients and dqkv are rounded once each) bound the 2-norm of the error by
    # (5 + 2 max |s|) u of the gradient's.
    import torch

    case = (2, 300, 8, 2, 128, False, "fp32", "int64", None)
    batch, seq, heads, kv_heads = case[:4]
    qkv, cos, sin, how, grads = make(case, 7)
    dout = grads[0]
    leaves = [qkv.clone().requires_grad_(), *(how[n].clone().requires_grad_() for n in ("q_weight", "k_weight"))]
    named = {**how, "q_weight": leaves[1], "k_weight": leaves[2]}
    q, k, v = seed.qkv_norm_rope(leaves[0], heads, kv_heads, cos, sin, **named)
    out, lse = seed.grouped_attention(q, k, v, True)
    out.backward(dout)

    with torch.no_grad():
        q, k, v = seed.qkv_norm_rope(qkv, heads, kv_heads, cos, sin, **how)
        o, lse = seed.grouped_attention(q, k, v, True)
        dq, dk, dv = seed.attention_backward(dout, q, k, v, o, lse, True)
        want = seed.qkv_norm_rope_backward(dq, dk, dv, qkv, cos, sin, **how)
    torch.cuda.synchronize()
    b200.check_status(qkv.device)
    assert torch.equal(out.detach(), o)
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, want))

    x = qkv.double().requires_grad_()
    ws = [how[n].double().requires_grad_() for n in ("q_weight", "k_weight")]
    (q6, k6, v6), *_ = plain(case, x, cos, sin, {**how, "q_weight": ws[0], "k_weight": ws[1]}, grads)
    v6 = x[:, :, heads + kv_heads:].transpose(1, 2)
    s = (q6 @ k6.repeat_interleave(heads // kv_heads, 1).transpose(-1, -2)) * b200.default_scale()
    most = float(s.abs().max())
    s = s.masked_fill(torch.ones(seq, seq, device="cuda").triu(1).bool(), float("-inf"))
    (s.softmax(-1) @ v6.repeat_interleave(heads // kv_heads, 1)).backward(dout.double())
    for leaf, w in zip(leaves, (x.grad, ws[0].grad, ws[1].grad)):
        assert float((leaf.grad.double() - w).norm() / w.norm()) <= (5 + 2 * most) * U


def test_captured_layer_replays_and_streams(b200, seed):
    import torch

    case = (2, 130, 4, 2, 128, False, "fp32", "int64", None)
    qkv, cos, sin, how, grads = make(case, 8)

    def step(x, pos, dout):
        h = {**how, "positions": pos}
        q, k, v = seed.qkv_norm_rope(x, 4, 2, cos, sin, **h)
        o, lse = seed.grouped_attention(q, k, v, True)
        return seed.qkv_norm_rope_backward(*seed.attention_backward(dout, q, k, v, o, lse, True), x, cos, sin, **h)

    pos, dout = how["positions"], grads[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step(qkv, pos, dout)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step(qkv, pos, dout)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(qkv, pos, dout)
    for value in (9, 10):
        nqkv, _, _, nhow, ngrads = make(case, value)
        qkv.copy_(nqkv)
        pos.copy_(nhow["positions"])
        dout.copy_(ngrads[0])
        graph.replay()
        want = step(nqkv, nhow["positions"], ngrads[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
    del graph


def test_autograd_refuses_capture_and_runs_in_parts(b200, seed):
    import torch

    case = (1, 20, 2, 1, 128, False, "bf16", None, None)
    qkv, cos, sin, how, grads = make(case, 11)
    leaf = qkv.clone().requires_grad_()
    q, k, v = seed.qkv_norm_rope(leaf, 2, 1, cos, sin, **how)
    q.sum().backward()  # k and v unused: their gradients are zero
    zero = [torch.zeros_like(t) for t in (k, v)]
    want = seed.qkv_norm_rope_backward(torch.ones_like(q), *(z.detach() for z in zero), qkv, cos, sin, **how)
    assert torch.equal(leaf.grad, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            seed.qkv_norm_rope(leaf, 2, 1, cos, sin, **how)
    del graph


def test_refusals(b200, seed):
    import torch

    case = (2, 10, 4, 2, 64, False, "fp32", "int64", None)
    qkv, cos, sin, how, grads = make(case, 12)
    plain_how = {"q_weight": how["q_weight"], "k_weight": how["k_weight"]}
    ok = how["positions"]
    bad = [
        (dict(), (qkv.cpu(), 4, 2, cos, sin), "qkv must be a CUDA tensor"),
        (dict(), (qkv.float(), 4, 2, cos, sin), "qkv must be bf16"),
        (dict(), (qkv, 4, 1, cos, sin), "qkv must have shape"),
        (dict(), (qkv.transpose(2, 3).contiguous().transpose(2, 3), 4, 2, cos, sin), "must be contiguous"),
        (dict(), (qkv, 4, 2, cos.double(), sin), "cos must be float32"),
        (dict(), (qkv, 4, 2, cos[:, :5].contiguous(), sin[:, :5].contiguous()), "rotary_dim"),
        (dict(), (qkv, 4, 2, cos, sin[:5]), "same shape"),
        (dict(), (qkv, 4, 2, cos[:9], sin[:9]), "fewer rows"),
        (dict(q_weight=how["q_weight"], k_weight=None), (qkv, 4, 2, cos, sin), "together"),
        (dict(q_weight=how["q_weight"], k_weight=how["k_weight"].bfloat16()), (qkv, 4, 2, cos, sin), "k_weight must be"),
        (dict(eps=-1.0), (qkv, 4, 2, cos, sin), "eps"),
        (dict(positions=ok.float()), (qkv, 4, 2, cos, sin), "int32 or int64"),
        (dict(positions=ok.cpu()), (qkv, 4, 2, cos, sin), "positions must be on"),
        (dict(positions=ok[:, :9]), (qkv, 4, 2, cos, sin), "positions must have shape"),
        (dict(positions=ok[None], sections=(16, 16)), (qkv, 4, 2, cos, sin), "positions must have shape"),
        (dict(positions=ok[None].expand(2, -1, -1), sections=(16, 15)), (qkv, 4, 2, cos, sin), "sections"),
        (dict(sections=(16, 16)), (qkv, 4, 2, cos, sin), "sections need positions"),
    ]
    for more, args, match in bad:
        with pytest.raises(RuntimeError, match=match):
            seed.qkv_norm_rope(*args, **{**plain_how, **more})
    for table in ((cos.clone().requires_grad_(), sin), (cos, sin.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient for cos and sin"):
            seed.qkv_norm_rope(qkv, 4, 2, *table, **plain_how, positions=ok)
        with torch.no_grad():
            seed.qkv_norm_rope(qkv, 4, 2, *table, **plain_how, positions=ok)
    with pytest.raises(RuntimeError, match="match qkv"):
        seed.qkv_norm_rope_backward(grads[0][:, :, :9].contiguous(), *grads[1:], qkv, cos, sin, **how)
    with pytest.raises(RuntimeError, match="dq must be contiguous"):
        seed.qkv_norm_rope_backward(grads[0].transpose(1, 2), *grads[1:], qkv, cos, sin, **how)


def test_empty_sizes(b200, seed):
    import torch

    for batch, seq in ((0, 4), (2, 0)):
        case = (batch, seq, 2, 1, 64, False, "fp32", None, None)
        qkv, cos, sin, how, grads = make(case, 13)
        q, k, v = seed.qkv_norm_rope(qkv, 2, 1, cos, sin, **how)
        assert q.shape == (batch, 2, seq, 128) and k.shape == v.shape == (batch, 1, seq, 128)
        dqkv, dqw, dkw = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, **how)
        assert dqkv.shape == qkv.shape and bool((dqw == 0).all()) and bool((dkw == 0).all())


def test_offsets_past_32_bits(b200, seed):
    # A projection of more than 2^31 elements: its last tokens equal a call on them alone.
    import torch

    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of device memory")
    gen = torch.Generator(device="cuda").manual_seed(5)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16)

    batch, seq, heads, kv_heads, last = 2, 351_001, 16, 4, 70
    qkv = randn(batch, seq, heads + 2 * kv_heads, 128)
    assert qkv.numel() > 2**31
    angle = torch.rand((1000, 64), device="cuda", generator=gen) * 6
    cos, sin = angle.cos(), angle.sin()
    positions = torch.arange(seq, device="cuda") % 1000
    w = 1 + torch.rand(128, device="cuda", generator=gen)
    how = dict(q_weight=w, k_weight=w)
    outs = seed.qkv_norm_rope(qkv, heads, kv_heads, cos, sin, positions=positions, **how)
    tail = seed.qkv_norm_rope(qkv[-1:, -last:], heads, kv_heads, cos, sin, positions=positions[-last:], **how)
    for got, want in zip(outs, tail):
        assert torch.equal(got[-1:, :, -last:], want)
    grads = [randn(*t.shape) for t in outs]
    del outs
    dqkv, _, _ = seed.qkv_norm_rope_backward(*grads, qkv, cos, sin, positions=positions, **how)
    few = [g[-1:, :, -last:].contiguous() for g in grads]
    want, _, _ = seed.qkv_norm_rope_backward(*few, qkv[-1:, -last:], cos, sin, positions=positions[-last:], **how)
    assert torch.equal(dqkv[-1:, -last:], want)
