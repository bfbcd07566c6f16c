"""What is measured of the training side of attention: the operators, their plain forms and their exact values.

Four operators around ``attention()``, head_dim 128, bf16 in memory:

``grouped_attention``       softmax(scale * q k^T [+ causal mask]) v with H query heads sharing Hkv key/value
                            heads and seq_q != seq_kv allowed; the causal mask is aligned at the end (the last
                            query sees every key), so with seq_q > seq_kv the first queries see nothing.
``attention_backward``      its gradient from out and the log-sum-exp: the probabilities are recomputed.
``qkv_norm_rope``           the fused projection [B, S, H + 2 Hkv, 128] to attention's q, k, v [B, heads, S, 128]:
                            RMS norm of each query and key head, rotation by position (one axis or several),
                            heads moved in front of the tokens, in one pass.
``qkv_norm_rope_backward``  its gradient: dqkv and the gradients of the two norm weights.

``run`` computes them with elementary torch operations in fp32 (long sums in fp64) unless ``own`` is set, when
it calls this repository's entry points.  ``exact`` gives the same outputs in fp64, by autograd over the
operator's definition.
"""

import math
from pathlib import Path

import torch

own = False

D = 128


def listed():
    return [
        # The smallest training call of the repository's own cases (B1 H4 S512): latency counts.
        _attn("bwd", "attn_bwd_b1_h4_s512", 1, 4, 4, 512, 512, False),
        # The repository's mid-size workload, every query against every key (an encoder, an image model).
        _attn("bwd", "attn_bwd_b4_h16_s4096", 4, 16, 16, 4096, 4096, False),
        # The repository's long causal workload: language-model training.
        _attn("bwd", "attn_bwd_b2_h16_s8192_causal", 2, 16, 16, 8192, 8192, True),
        # Shared key/value heads and a length that ends inside a tile.
        _attn("bwd", "attn_bwd_b2_h16_kv4_s4001_causal", 2, 16, 4, 4001, 4001, True),
        # A chunk of queries at the end of a longer context, one key/value head for eight query heads, odd sizes.
        _attn("bwd", "attn_bwd_b1_h16_kv2_q777_kv5003_causal", 1, 16, 2, 777, 5003, True, 0.07),
        # The forward of the shared-head layer.
        _attn("fwd", "attn_fwd_b2_h16_kv4_s4096_causal", 2, 16, 4, 4096, 4096, True),
        # Cross attention: odd lengths, one shared key/value head.
        _attn("fwd", "attn_fwd_b1_h12_kv1_q1001_kv9003", 1, 12, 1, 1001, 9003, False),
        # One token of one sequence: the smallest call there is.
        _rope("rope_fwd", "norm_rope_fwd_b1_s1_h16_kv4", 1, 1, 16, 4, positions="int64"),
        # The layer input of the B4 H16 S4096 workload with shared key/value heads.
        _rope("rope_fwd", "norm_rope_fwd_b4_s4096_h16_kv4", 4, 4096, 16, 4),
        # Video tokens: time, height and width each turn a part of the pairs; neighbouring elements are a pair.
        _rope("rope_fwd", "norm_rope_fwd_b2_s6007_h16_kv16_3axes", 2, 6007, 16, 16, positions="int32", axes="16,24,24",
              interleaved=True, wdtype="bf16"),
        # The gradients of a short and of the ordinary layer input.
        _rope("rope_bwd", "norm_rope_bwd_b1_s333_h16_kv16_3axes", 1, 333, 16, 16, positions="int64", axes="16,24,24"),
        _rope("rope_bwd", "norm_rope_bwd_b4_s4096_h16_kv4", 4, 4096, 16, 4),
    ]


def _attn(op, name, batch, heads, kv_heads, seq_q, seq_kv, causal, scale=0.08838834764831845):
    return {"name": name, "op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq_q": seq_q,
            "seq_kv": seq_kv, "causal": causal, "scale": scale}


def _rope(op, name, batch, seq, heads, kv_heads, positions="none", axes="", rotary=128, interleaved=False,
          wdtype="fp32"):
    return {"name": name, "op": op, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
            "positions": positions, "axes": axes, "rotary": rotary, "interleaved": interleaved, "wdtype": wdtype}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bwd", "bwd", "fwd", "rope_fwd", "rope_bwd"])
    batch = rng.choice([1, 1, 2, 3, 4])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    if op in ("bwd", "fwd"):
        heads = kv_heads * rng.choice([1, 1, 2, 4] if kv_heads <= 4 else [1, 2])
        seq_q = _log(rng, 1, 8192)
        seq_kv = seq_q if rng.random() < 0.6 else _log(rng, 4, 8192)
        seq_kv = max(seq_kv, 4)  # with a single key dq and dk are zero: differences of equal numbers, nothing to measure
        while batch * heads * seq_q * seq_kv > 1 << 30:
            seq_q, seq_kv = (seq_q + 1) // 2, (seq_kv + 1) // 2
        case = _attn(op, "", batch, heads, kv_heads, seq_q, seq_kv, rng.random() < 0.6,
                     rng.choice([0.08838834764831845, 0.05, 0.11]))
    else:
        heads = kv_heads * rng.choice([1, 2, 4] if kv_heads <= 8 else [1, 2])
        seq = _log(rng, 1, 16384)
        while batch * seq * (heads + 2 * kv_heads) > 4 * 16384 * 24:
            seq = (seq + 1) // 2
        kind, axes = rng.choice([("none", ""), ("int32", ""), ("int64", ""), ("int32", "2"), ("int64", "3")])
        rotary = rng.choice([128, 128, 64, 96, 32])
        if axes:
            pairs = rotary // 2
            first = rng.randint(1, pairs // 2)
            rest = pairs - first
            axes = "%d,%d" % (first, rest) if axes == "2" else "%d,%d,%d" % (first, rest // 2, rest - rest // 2)
        case = _rope(op, "", batch, seq, heads, kv_heads, kind, axes, rotary, rng.random() < 0.4,
                     rng.choice(["fp32", "bf16"]))
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    b, h, g = case["batch"], case["heads"], case["kv_heads"]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * std).bfloat16()

    if case["op"] in ("bwd", "fwd"):
        state["q"] = randn(b, h, case["seq_q"], D)  # normed queries and keys: unit root mean square
        state["k"] = randn(b, g, case["seq_kv"], D)
        state["v"] = randn(b, g, case["seq_kv"], D)
        if case["op"] == "bwd":
            state["do"] = randn(b, h, case["seq_q"], D, std=0.02)
            state["out"], state["lse"] = _attention(state)
        return state
    s, rot = case["seq"], case["rotary"]
    state["qkv"] = randn(b, s, h + 2 * g, D)
    wdtype = torch.bfloat16 if case["wdtype"] == "bf16" else torch.float32
    state["q_weight"], state["k_weight"] = (
        (1.0 + 0.1 * torch.randn(D, device="cuda", generator=gen)).to(wdtype) for _ in range(2))
    table = max(2 * s, 64)
    sections = [int(x) for x in case["axes"].split(",")] if case["axes"] else None
    state["sections"] = sections
    angles = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        10000.0, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
    state["position_ids"] = None
    if case["positions"] != "none":
        shape = (len(sections), b, s) if sections else (b, s)
        state["position_ids"] = torch.randint(0, table, shape, device="cuda", generator=gen).to(
            torch.int32 if case["positions"] == "int32" else torch.int64)
    if case["op"] == "rope_bwd":
        state["dq"], state["dk"], state["dv"] = (randn(b, n, s, D, std=0.02) for n in (h, g, g))
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"fwd": _attention, "bwd": _attention_backward, "rope_fwd": _norm_rope,
            "rope_bwd": _norm_rope_backward}[state["op"]](state)


def _framework():
    import importlib.util
    import sys

    name = "avo_candidate_cuda_b200_attention_seed"
    if name not in sys.modules:
        path = (Path(__file__).resolve().parents[1] / "avo-ampere_b200" / "candidates"
                / "cuda_b200_attention_seed.py")
        spec = importlib.util.spec_from_file_location(name, path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        sys.modules[name] = module
    return sys.modules[name]


def _own(s):
    f = _framework()
    if s["op"] == "fwd":
        return f.grouped_attention(s["q"], s["k"], s["v"], s["causal"], softmax_scale=s["scale"])
    if s["op"] == "bwd":
        return f.attention_backward(s["do"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["causal"],
                                    softmax_scale=s["scale"])
    how = dict(q_weight=s["q_weight"], k_weight=s["k_weight"], positions=s["position_ids"], sections=s["sections"],
               eps=1e-6, interleaved=s["interleaved"])
    if s["op"] == "rope_fwd":
        return f.qkv_norm_rope(s["qkv"], s["heads"], s["kv_heads"], s["cos"], s["sin"], **how)
    return f.qkv_norm_rope_backward(s["dq"], s["dk"], s["dv"], s["qkv"], s["cos"], s["sin"], **how)


def _hidden(s):
    """True where a query does not see a key, [seq_q, seq_kv]; the last query sees every key."""
    i = torch.arange(s["seq_q"], device="cuda")[:, None] + (s["seq_kv"] - s["seq_q"])
    return torch.arange(s["seq_kv"], device="cuda")[None, :] > i


def _by_group(t, s):
    """[B, H, S, ...] as [B, Hkv, H / Hkv, S, ...]."""
    return t.float().unflatten(1, (s["kv_heads"], -1))


def _attention(s):
    q, k, v = _by_group(s["q"], s), _by_group(s["k"], s), _by_group(s["v"], s)
    scores = (q * s["scale"]) @ k.transpose(-1, -2)
    if s["causal"]:
        scores.masked_fill_(_hidden(s), -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log()).squeeze(-1)
    return out.flatten(1, 2).bfloat16(), lse.flatten(1, 2)


def _attention_backward(s):
    q, k, v, do, out = (_by_group(s[n], s) for n in ("q", "k", "v", "do", "out"))
    lse = _by_group(s["lse"], s)[..., None]
    p = (q * s["scale"]) @ k.transpose(-1, -2)
    p.sub_(torch.where(lse == -math.inf, torch.full_like(lse, math.inf), lse)).exp_()
    if s["causal"]:
        p.masked_fill_(_hidden(s), 0.0)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = do @ v.transpose(-1, -2)
    ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return dq.flatten(1, 2).bfloat16(), dk.bfloat16(), dv.bfloat16()


def _cos_sin(s):
    """[B or 1, S, 1, rotary / 2] each."""
    pairs = s["rotary"] // 2
    pos = s["position_ids"]
    if pos is None:
        return s["cos"][None, :s["seq"], None], s["sin"][None, :s["seq"], None]
    if s["sections"] is None:
        return s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device="cuda"),
                                   torch.tensor(s["sections"], device="cuda"))
    row = pos[axis].permute(1, 2, 0).long()
    col = torch.arange(pairs, device="cuda")
    return s["cos"][row, col][:, :, None], s["sin"][row, col][:, :, None]


def _rotate(x, s, sign):
    cos, sin = _cos_sin(s)
    sin = sin * sign
    rot = s["rotary"]
    if s["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _split(s, t):
    h, g = s["heads"], s["kv_heads"]
    return t[:, :, :h], t[:, :, h:h + g], t[:, :, h + g:]


def _norm_rope(s):
    def one(x, weight):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        return _rotate(x, s, 1.0).bfloat16().transpose(1, 2).contiguous()

    q, k, v = _split(s, s["qkv"])
    return one(q, s["q_weight"]), one(k, s["k_weight"]), v.transpose(1, 2).contiguous()


def _norm_rope_backward(s):
    def one(x, weight, dy):
        x = x.float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        x = x * r
        g = _rotate(dy.float().transpose(1, 2), s, -1.0)
        dw = (g * x).double().sum((0, 1, 2)).float()
        g = g * weight.float()
        return (r * (g - x * (g * x).mean(-1, keepdim=True))).bfloat16(), dw

    q, k, _ = _split(s, s["qkv"])
    dq, dqw = one(q, s["q_weight"], s["dq"])
    dk, dkw = one(k, s["k_weight"], s["dk"])
    return torch.cat((dq, dk, s["dv"].transpose(1, 2)), 2), dqw, dkw


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    b, h, g = case["batch"], case["heads"], case["kv_heads"]
    if case["op"] in ("bwd", "fwd"):
        sq, skv = case["seq_q"], case["seq_kv"]
        seen = sq * skv
        if case["causal"]:  # query i sees skv - sq + 1 + i keys, none at least
            empty = max(0, sq - skv)
            rows = sq - empty
            seen = rows * (max(0, skv - sq) + 1) + rows * (rows - 1) // 2
        products = 5 if case["op"] == "bwd" else 2
        q_rows, kv_rows = b * h * sq, b * g * skv
        bytes_ = (4 * q_rows + 4 * kv_rows if case["op"] == "bwd" else 2 * q_rows + 2 * kv_rows) * D * 2 + 4 * q_rows
        return {"bytes": bytes_, "flops": products * 2 * D * b * h * seen}
    s = case["seq"]
    rows, turned = b * s * (h + 2 * g), b * s * (h + g)
    table = s * case["rotary"] // 2 * 2 * 4
    if case["op"] == "rope_fwd":
        return {"bytes": rows * D * 2 * 2 + table, "flops": turned * D * 8}
    return {"bytes": rows * D * 2 * 2 + turned * D * 2 + table, "flops": turned * D * 16}


# ---------------------------------------------------------------- exact values, fp64
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("bwd", "fwd"):
        return _exact_attention(s)
    return _exact_norm_rope(s)


def _exact_attention(s):
    sq, skv, group = s["seq_q"], s["seq_kv"], s["heads"] // s["kv_heads"]
    backward = s["op"] == "bwd"
    first = max(0, sq - skv) if s["causal"] else 0  # rows before it see no key
    q64 = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    dk, dv = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    offset = torch.arange(first, sq, device="cuda") + (skv - sq)
    for b in range(s["batch"]):
        for h in range(s["heads"]):
            q = s["q"][b, h, first:].double().requires_grad_(backward)
            k = s["k"][b, h // group].double().requires_grad_(backward)
            v = s["v"][b, h // group].double().requires_grad_(backward)
            logits = torch.einsum("id,jd->ij", q, k) * s["scale"]
            if s["causal"]:
                logits = torch.where(torch.arange(skv, device="cuda") <= offset[:, None], logits, -math.inf)
            o = torch.softmax(logits, 1) @ v
            if backward:
                o.backward(s["do"][b, h, first:].double())
                q64[b, h, first:] = q.grad
                dk[b, h // group] += k.grad
                dv[b, h // group] += v.grad
            else:
                q64[b, h, first:] = o
                lse[b, h, first:] = torch.logsumexp(logits, 1)
    return (q64, dk, dv) if backward else (q64, lse)


def _exact_norm_rope(s):
    h, g, rot = s["heads"], s["kv_heads"], s["rotary"]
    backward = s["op"] == "rope_bwd"
    qkv = s["qkv"].double().requires_grad_(backward)
    weights = [s[n].double().requires_grad_(backward) for n in ("q_weight", "k_weight")]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    pos = s["position_ids"]
    if pos is None:
        turn = turn[:s["seq"]].expand(s["batch"], -1, -1)
    else:
        parts, at = [], 0
        for axis, n in enumerate(s["sections"] or [rot // 2]):
            ids = (pos[axis] if s["sections"] else pos).long()
            parts.append(turn[:, at:at + n][ids])
            at += n
        turn = torch.cat(parts, -1)
    turn = turn[:, :, None]

    def one(x, weight):
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * weight
        if s["interleaved"]:
            z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., rot:]), -1).transpose(1, 2)

    outs = [one(qkv[:, :, :h], weights[0]), one(qkv[:, :, h:h + g], weights[1]), qkv[:, :, h + g:].transpose(1, 2)]
    if not backward:
        return tuple(outs)
    torch.autograd.backward(outs, [s[n].double() for n in ("dq", "dk", "dv")])
    return (qkv.grad, *(w.grad for w in weights))
