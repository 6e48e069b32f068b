"""The operators of a mixture-of-experts layer around the block-scaled matmuls, on one GPU: what is timed, their plain forms in
elementary torch operations, and their values in 64 bits.

A case is a dict of plain values:
  op       "norm"     residual addition, root-mean-square norm, MX quantiser (capi.add_rms_norm_mx_quant)
           "route"    router scores to experts and weights, and the rows of the dispatch (capi.moe_route, capi.moe_row_plan)
           "grouped"  every expert's product on its own rows (capi.mx_grouped_gemm)
           "combine"  the weighted sum of a token's expert rows (capi.moe_combine)
           "matvec"   products of one or a few tokens with FP4 weights (capi.mx_fp4_matvec)
  m n k    rows or tokens, output columns (norm: width), contraction length
  experts, top_k, and the fields of one operator that its part of draw() shows
  codes    element type of 8-bit activation codes: "e4m3" or "e5m2"
  out      element type of a product: "bf16" or "fp16"
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
EMAX = {"e4m3": 8, "e5m2": 15}
MOST = {"e4m3": 448.0, "e5m2": 57344.0}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decode step of 16 sequences in front of a projection: two small launches' worth of work
        dict(name="norm_decode", op="norm", m=16, n=7168, residual=True, keep=True, codes="e4m3"),
        # a long ragged prefill chunk; the router is elsewhere, so the 16-bit output is not kept
        dict(name="norm_prefill", op="norm", m=8190, n=5120, residual=True, keep=False, codes="e5m2"),
        # the router of a decode step: sigmoid scores, balance bias, 4 of 8 groups, 8 of 256 experts
        dict(name="route_decode", op="route", m=16, experts=256, top_k=8, score="sigmoid", bias=True, groups=8, top_groups=4,
             group_best=2, renormalize=True, scale=2.5, logits="fp32", first=0, local=256),
        # the same router over a long prefill, on a rank that holds 32 of the experts
        dict(name="route_prefill", op="route", m=16384, experts=256, top_k=8, score="sigmoid", bias=True, groups=8, top_groups=4,
             group_best=2, renormalize=True, scale=2.5, logits="fp32", first=64, local=32),
        # a softmax router with 16-bit logits and an odd number of tokens
        dict(name="route_softmax", op="route", m=2671, experts=64, top_k=6, score="softmax", bias=False, groups=1, top_groups=1,
             group_best=1, renormalize=False, scale=1.0, logits="bf16", first=0, local=64),
        # 16 sequences' routes on a rank with 32 experts: the weights stream
        dict(name="grouped_decode", op="grouped", m=128, n=4096, k=7168, experts=32, codes="e4m3", out="bf16", packed=False),
        # a prefill of 2048 tokens with 8 routes each, packed rows as the dispatch writes them
        dict(name="grouped_prefill", op="grouped", m=16384, n=2304, k=7168, experts=32, codes="e4m3", out="bf16", packed=True),
        # the second product of a layer with few experts, ragged rows, E5M2 activations, 16-bit floats out
        dict(name="grouped_ragged", op="grouped", m=3001, n=7168, k=2304, experts=8, codes="e5m2", out="fp16", packed=False),
        # the end of a decode step's expert layer
        dict(name="combine_decode", op="combine", m=16, n=7168, top_k=8, shared=True, out="bf16"),
        # of a prefill, with dropped routes
        dict(name="combine_prefill", op="combine", m=4095, n=7168, top_k=8, shared=False, out="bf16"),
        # one token through a dense projection with FP4 weights
        dict(name="matvec_one", op="matvec", m=1, n=4096, k=7168, experts=0, top_k=0, out="bf16"),
        # four tokens through the experts that they chose
        dict(name="matvec_experts", op="matvec", m=4, n=2304, k=7168, experts=32, top_k=8, out="bf16"),
    ]


MOST_FLOPS = 2.0 * 16384 * 2304 * 7168  # of grouped_prefill
MOST_BYTES = 32 * 4096 * 7168 * 33.0 / 32  # of grouped_decode


def _spread(rng, low, high, step=1):
    """A multiple of `step` between the two, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    while True:
        op = rng.choice(("norm", "route", "grouped", "combine", "matvec"))
        c = dict(op=op)
        if op == "norm":
            c.update(m=_spread(rng, 1, 16384), n=_spread(rng, 32, 8192, 32), residual=rng.random() < 0.7, keep=rng.random() < 0.5,
                     codes=rng.choice(("e4m3", "e4m3", "e5m2")))
        elif op == "route":
            groups = rng.choice((1, 1, 2, 4, 8))
            experts = groups * _spread(rng, 8 if groups == 1 else 4, 384 // groups)
            top_groups = rng.randint(1, groups)
            bias = rng.random() < 0.6
            first = rng.choice((0, rng.randrange(experts)))
            c.update(m=_spread(rng, 1, 16384), experts=experts, top_k=min(_spread(rng, 1, 12), experts // groups * top_groups),
                     score=rng.choice(("softmax", "sigmoid")), bias=bias, groups=groups, top_groups=top_groups,
                     group_best=rng.choice((1, 2)), renormalize=rng.random() < 0.6, scale=rng.choice((1.0, 2.5)),
                     logits=rng.choice(("fp32", "bf16")), first=first, local=experts - first)
        elif op == "grouped":
            c.update(m=_spread(rng, 1, 16384), n=_spread(rng, 256, 7168, 16), k=_spread(rng, 256, 7168, 128),
                     experts=_spread(rng, 1, 64), codes=rng.choice(("e4m3", "e4m3", "e5m2")), out=rng.choice(("bf16", "fp16")),
                     packed=rng.random() < 0.5)
        elif op == "combine":
            c.update(m=_spread(rng, 1, 8192), n=_spread(rng, 256, 8192, 8), top_k=rng.randint(1, 8), shared=rng.random() < 0.5,
                     out=rng.choice(("bf16", "fp16")))
        else:
            many = rng.random() < 0.5
            c.update(m=_spread(rng, 1, 8 if many else 16), n=_spread(rng, 512, 7168, 16), k=_spread(rng, 512, 8192, 64),
                     experts=_spread(rng, 4, 64) if many else 0, out=rng.choice(("bf16", "fp16")))
            c["top_k"] = rng.randint(1, min(8, c["experts"])) if many else 0
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and c.get("experts", 0) * c.get("k", 0) * c.get("n", 0) <= 32 * 4096 * 7168:
            return c


def work(case):
    """Each input read once, each output written once, and the products."""
    op, m = case["op"], case["m"]
    if op == "norm":
        per = 2.0 + 1.0 + 1.0 / 32 + (4.0 if case["residual"] else 0.0) + (2.0 if case["keep"] else 0.0)
        return {"bytes": m * case["n"] * per + 2.0 * case["n"], "flops": 6.0 * m * case["n"]}
    if op == "route":
        per = (2.0 if case["logits"] == "bf16" else 4.0) * case["experts"] + 12.0 * case["top_k"]
        return {"bytes": m * per + 4.0 * case["local"], "flops": 0.0}
    if op == "combine":
        return {"bytes": m * (case["n"] * (2.0 * case["top_k"] + 2.0 + (2.0 if case["shared"] else 0.0)) + 8.0 * case["top_k"]),
                "flops": 2.0 * m * case["n"] * case["top_k"]}
    n, k, e = case["n"], case["k"], case["experts"]
    if op == "grouped":
        return {"bytes": m * k * 33.0 / 32 + min(e, m) * n * k * 33.0 / 32 + 2.0 * m * n, "flops": 2.0 * m * n * k}
    routes = m * case["top_k"] if e else m
    weights = e * (1.0 - (1.0 - 1.0 / e) ** routes) if e else 1.0  # distinct experts among the routes, about
    return {"bytes": weights * n * k * (0.5 + 1.0 / 32) + 2.0 * (m * k + routes * n), "flops": 2.0 * routes * n * k}


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _activations(m, k, gen):
    """Hidden states: normal, with one channel in a thousand much larger."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    x[:, torch.randperm(k, generator=gen, device="cuda")[: math.ceil(0.001 * k)]] *= 30.0
    return x


def _mx_codes(x, codes):
    """float [..., 32 i] -> E4M3 or E5M2 codes (uint8, same shape) and E8M0 scales [..., i]."""
    block = x.unflatten(-1, (-1, 32))
    e = torch.frexp(block.abs().amax(dim=-1).clamp_min(1e-12))[1] - 1 - EMAX[codes]
    q = torch.ldexp(block, -e.unsqueeze(-1)).clamp(-MOST[codes], MOST[codes]).flatten(-2).to(F8[codes]).view(torch.uint8)
    return q, (e + 127).to(torch.uint8)


def _weights8(e, k, n, gen):
    """N(0, 0.02), quantised along k: codes [e, k, n], scales [e, k / 64, n, 2]."""
    b = torch.empty((e, k, n), dtype=torch.uint8, device="cuda")
    s = torch.empty((e, k // 64, n, 2), dtype=torch.uint8, device="cuda")
    for i in range(e):
        q, f = _mx_codes(torch.randn((n, k), generator=gen, device="cuda") * 0.02, "e4m3")
        b[i], s[i] = q.t(), f.view(n, k // 64, 2).permute(1, 0, 2)
    return b, s


def _weights4(e, k, n, gen):
    """The same in E2M1, two columns to a byte (the low nibble is the even one): codes [e, k, n / 2], scales [e, k / 64, n, 2]."""
    b = torch.empty((e, k, n // 2), dtype=torch.uint8, device="cuda")
    s = torch.empty((e, k // 64, n, 2), dtype=torch.uint8, device="cuda")
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    for i in range(e):
        block = (torch.randn((n, k), generator=gen, device="cuda") * 0.02).view(n, k // 32, 32)
        x = torch.frexp(block.abs().amax(dim=2))[1] - 3
        v = torch.ldexp(block, -x.unsqueeze(2)).view(n, k).t()
        q = torch.bucketize(v.abs().contiguous(), edges).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
        b[i] = q[:, 0::2] | (q[:, 1::2] << 4)
        s[i] = (x + 127).to(torch.uint8).view(n, k // 64, 2).permute(1, 0, 2)
    return b, s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    op, m = case["op"], case["m"]
    if op == "norm":
        s["x"] = _activations(m, case["n"], gen).to(torch.bfloat16)
        s["stream"] = (_activations(m, case["n"], gen) * 2.0).to(torch.bfloat16) if case["residual"] else None
        s["stream_out"] = torch.empty_like(s["stream"]) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(case["n"], generator=gen, device="cuda")).to(torch.bfloat16)
        s["norm"] = torch.zeros((m, case["n"]), dtype=torch.bfloat16, device="cuda") if case["keep"] else None
    elif op == "route":
        logits = torch.randn((m, case["experts"]), generator=gen, device="cuda") * 1.5
        s["l"] = logits.to(torch.bfloat16) if case["logits"] == "bf16" else logits
        s["b"] = 0.05 * torch.randn(case["experts"], generator=gen, device="cuda") if case["bias"] else None
    elif op == "grouped":
        e, n, k = case["experts"], case["n"], case["k"]
        # some experts are chosen far more often than others, some not at all
        popular = torch.softmax(torch.randn(e, generator=gen, device="cuda"), 0)
        expert = torch.multinomial(popular, m, replacement=True, generator=gen).sort().values
        s["offsets"] = torch.searchsorted(expert, torch.arange(e + 1, device="cuda")).to(torch.int32)
        s["cap"] = int(torch.bincount(expert, minlength=e).max())  # only the plain form needs it
        q, f = _mx_codes(_activations(m, k, gen), case["codes"])
        if case["packed"]:  # rows [codes | scales, padded to an even count | zeros to 32 bytes] of the dispatch
            row = (k + (k // 32 + 1) // 2 * 2 + 31) // 32 * 32
            packed = torch.zeros((m, row), dtype=torch.uint8, device="cuda")
            packed[:, :k], packed[:, k : k + k // 32] = q, f
            q, f = packed[:, :k], packed[:, k : k + k // 32]
        s["a"], s["a_scales"] = q, f
        s["w"], s["w_scales"] = _weights8(e, k, n, gen)
        s["c"] = torch.zeros((m, n), dtype=DTYPE[case["out"]], device="cuda")
    elif op == "combine":
        rows = m * case["top_k"]
        s["y"] = _activations(rows, case["n"], gen).to(DTYPE[case["out"]])
        index = torch.randperm(rows, generator=gen, device="cuda").to(torch.int32)
        index[torch.rand(rows, generator=gen, device="cuda") < 0.02] = -1
        s["index"] = index.view(m, case["top_k"])
        s["gate"] = torch.softmax(torch.randn((m, case["top_k"]), generator=gen, device="cuda"), 1)
        s["shared_out"] = torch.randn((m, case["n"]), generator=gen, device="cuda").to(DTYPE[case["out"]]) if case["shared"] else None
    else:
        e, n, k = case["experts"], case["n"], case["k"]
        s["x"] = _activations(m, k, gen).to(torch.bfloat16)
        s["w"], s["w_scales"] = _weights4(max(1, e), k, n, gen)
        s["ids"] = None
        if e:
            s["ids"] = torch.rand((m, e), generator=gen, device="cuda").argsort(dim=1)[:, : case["top_k"]].to(torch.int32).contiguous()
        else:
            s["w"], s["w_scales"] = s["w"][0], s["w_scales"][0]
    return s


# ---- the calls that a user makes --------------------------------------------------------------------------------------------
_options = {}


def _types(capi, s):
    """The element types are the library's options: a program sets them once, here when the case changes."""
    want = {"a_dtype": 1 if s.get("codes") == "e5m2" else 0, "b_dtype": 0, "c_dtype": 1 if s.get("out") == "fp16" else 0}
    if _options != want:
        for key, value in want.items():
            capi.set_option(key, value)
        _options.update(want)


def _run_own(s):
    from catccos_b200 import capi

    _types(capi, s)
    op = s["op"]
    if op == "norm":
        codes, scales = capi.add_rms_norm_mx_quant(s["x"], s["stream"], s["weight"], EPS, residual_out=s["stream_out"], norm_out=s["norm"])
        return _eight_bits(codes, scales, s["codes"]) | {"residual": s["stream_out"], "norm": s["norm"]}
    if op == "route":
        ids, weights = capi.moe_route(s["l"], s["top_k"], bias=s["b"], score=s["score"], groups=s["groups"],
                                      top_groups=s["top_groups"], group_best=s["group_best"], renormalize=s["renormalize"],
                                      scale=s["scale"])
        index, offsets = capi.moe_row_plan(ids, s["local"], first_expert=s["first"])
        return {"ids": ids, "weights": weights, "index": index, "offsets": offsets}
    if op == "grouped":
        return capi.mx_grouped_gemm(s["a"], s["a_scales"], s["w"], s["w_scales"], s["offsets"], out=s["c"])
    if op == "combine":
        return capi.moe_combine(s["y"], s["index"], s["gate"], shared=s["shared_out"])
    return capi.mx_fp4_matvec(s["x"], s["w"], s["w_scales"], ids=s["ids"], out_dtype=DTYPE[s["out"]])


def _eight_bits(codes, scales, kind):
    """Codes and scales as the numbers that their bytes stand for."""
    return {"codes": codes.view(F8[kind]), "scales": scales.view(torch.float8_e8m0fnu)}


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _power(scales):
    """E8M0 bytes 1 .. 254 as fp32."""
    return (scales.to(torch.int32) << 23).view(torch.float32)


def _dequantised_weights(s):
    """[..., k, n] in fp32."""
    if s["op"] == "matvec":
        value = torch.tensor(E2M1, device="cuda")
        value = torch.cat((value, -value))
        w = torch.stack((value[(s["w"] & 15).long()], value[(s["w"] >> 4).long()]), dim=-1).flatten(-2)
    else:
        w = s["w"].view(torch.float8_e4m3fn).float()
    scale = _power(s["w_scales"]).transpose(-1, -2).flatten(-3, -2)  # [..., k / 32, n]
    return (w.unflatten(-2, (-1, 32)) * scale.unsqueeze(-2)).flatten(-3, -2)


def _plain_norm(s):
    h = s["x"]
    if s["residual"]:
        h = (s["x"].float() + s["stream"].float()).to(torch.bfloat16)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    block = y.unflatten(1, (-1, 32))
    top = block.abs().amax(dim=2)
    small = top < 1e-12  # such a block has scale 1 and codes of zero
    e = torch.where(small, 0, torch.frexp(top)[1] - 1 - EMAX[s["codes"]])
    q = (block * _power(127 - e).unsqueeze(2)).masked_fill(small.unsqueeze(2), 0.0)
    q = q.flatten(1).clamp(-MOST[s["codes"]], MOST[s["codes"]]).to(F8[s["codes"]])
    return _eight_bits(q.view(torch.uint8), (e + 127).to(torch.uint8), s["codes"]) | {
        "residual": h if s["residual"] else None, "norm": y.to(torch.bfloat16) if s["keep"] else None}


def _plain_route(s):
    l = s["l"].double()  # neighbouring scores are told apart in 64 bits
    score = torch.softmax(l, dim=1) if s["score"] == "softmax" else torch.sigmoid(l)
    choice = score + s["b"].double() if s["bias"] else score
    if s["groups"] > 1:
        of_group = choice.unflatten(1, (s["groups"], -1))
        best = of_group.sort(dim=2, descending=True).values[:, :, : s["group_best"]].sum(dim=2)
        taken = best.sort(dim=1, descending=True, stable=True).indices[:, : s["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, taken, True)
        choice = of_group.masked_fill(~open_.unsqueeze(2), -math.inf).flatten(1)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, : s["top_k"]]
    weights = score.gather(1, ids)
    if s["renormalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    # the dispatch: routes of this rank's experts in the order of experts, then of tokens
    local = ids.flatten() - s["first"]
    mine = (local >= 0) & (local < s["local"])
    key = torch.where(mine, local, s["local"])
    order = key.sort(stable=True).indices
    index = torch.empty_like(key).scatter_(0, order, torch.arange(key.numel(), device="cuda"))
    counts = torch.zeros(s["local"] + 1, dtype=torch.long, device="cuda").scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat((counts.new_zeros(1), counts[:-1].cumsum(0)))
    return {"ids": ids.to(torch.int32), "weights": (weights * s["scale"]).float(),
            "index": torch.where(mine, index, -1).view_as(ids).to(torch.int32), "offsets": offsets.to(torch.int32)}


def _plain_grouped(s):
    a = (s["a"].view(F8[s["codes"]]).float().unflatten(1, (-1, 32)) * _power(s["a_scales"]).unsqueeze(2)).flatten(1)
    begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    row = begin[:, None] + torch.arange(s["cap"], device="cuda")
    inside = row < end[:, None]
    c = torch.bmm(a[row.clamp(max=s["m"] - 1)], _dequantised_weights(s))
    out = torch.zeros((s["m"], s["n"]), dtype=DTYPE[s["out"]], device="cuda")
    out[row[inside]] = c[inside].to(out.dtype)
    return out


def _plain_combine(s):
    index = s["index"].long()
    part = s["y"][index.clamp(min=0)].float() * (s["gate"] * (index >= 0)).unsqueeze(2)
    total = part.sum(dim=1)
    return (total + s["shared_out"].float() if s["shared"] else total).to(s["y"].dtype)


def _plain_matvec(s):
    w, x = _dequantised_weights(s), s["x"].float()
    if s["ids"] is not None:
        return torch.bmm(x.repeat_interleave(s["top_k"], 0).unsqueeze(1), w[s["ids"].flatten().long()]).squeeze(1).to(DTYPE[s["out"]])
    return (x @ w).to(DTYPE[s["out"]])


def run(s):
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "route": _plain_route, "grouped": _plain_grouped, "combine": _plain_combine,
            "matvec": _plain_matvec}[s["op"]](s)


# ---- values in 64 bits ------------------------------------------------------------------------------------------------------
def _round_to(v, digits, lowest, most):
    """To the nearest value with `digits` bits behind the leading one (ties to even), steps no finer than below 2^lowest."""
    e = torch.frexp(v)[1] - 1
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=v.device), e.clamp(min=lowest) - digits)
    return (torch.round(v / step) * step).clamp(-most, most)


def _exact_norm(s):
    h = s["x"].double()
    total = h
    if s["residual"]:
        total = h + s["stream"].double()
        h = _round_to(total, 7, -126, math.inf)
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / s["n"] + EPS) * s["weight"].double()
    block = y.view(s["m"], -1, 32)
    top = block.abs().max(dim=2).values
    e = torch.where(top < 1e-12, 0, torch.floor(torch.log2(top.clamp_min(1e-300))) - EMAX[s["codes"]])
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=y.device), e)
    q = torch.where((top < 1e-12)[:, :, None], 0.0, block / scale[:, :, None])
    q = _round_to(q, 3, -6, 448.0) if s["codes"] == "e4m3" else _round_to(q, 2, -14, 57344.0)
    return {"codes": q.view(s["m"], s["n"]), "scales": scale, "residual": total if s["residual"] else None,
            "norm": y if s["keep"] else None}


def _exact_route(s):
    l = s["l"].double().cpu().numpy()
    if s["score"] == "softmax":
        score = np.exp(l - l.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    else:
        score = 1.0 / (1.0 + np.exp(-l))
    choice = score + s["b"].double().cpu().numpy() if s["bias"] else score.copy()
    m, experts, groups = s["m"], s["experts"], s["groups"]
    parts = np.sort(choice.reshape(m, groups, experts // groups), axis=2)[:, :, ::-1][:, :, : s["group_best"]].sum(axis=2)
    rank = np.argsort(np.argsort(-parts, axis=1, kind="stable"), axis=1, kind="stable")
    choice[np.repeat(rank >= s["top_groups"], experts // groups, axis=1)] = -np.inf
    ids = np.argsort(-choice, axis=1, kind="stable")[:, : s["top_k"]]
    weights = np.take_along_axis(score, ids, axis=1)
    if s["renormalize"]:
        weights = weights / weights.sum(1, keepdims=True)
    return {"ids": None, "weights": torch.from_numpy(weights * s["scale"]), "index": None, "offsets": None}


def _exact_weights(s, e):
    """Expert e's weight [k, n] (or the only one, e None)."""
    w, f = (s["w"], s["w_scales"]) if e is None else (s["w"][e], s["w_scales"][e])
    if s["op"] == "matvec":
        nibble = torch.empty((w.shape[0], 2 * w.shape[1]), dtype=torch.long, device=w.device)
        nibble[:, 0::2], nibble[:, 1::2] = w.long() % 16, w.long() // 16
        low, high = nibble % 2, nibble // 2 % 4
        value = torch.where(high == 0, low * 0.5, (1 + low * 0.5) * torch.pow(2.0, (high - 1).double()))
        value = torch.where(nibble >= 8, -value, value)
    else:
        value = w.view(torch.float8_e4m3fn).double()
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=w.device), f.double() - 127.0)
    return value * power.permute(0, 2, 1).reshape(-1, value.shape[1]).repeat_interleave(32, dim=0)


def _exact_grouped(s):
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), s["a_scales"].double() - 127.0)
    a = s["a"].view(F8[s["codes"]]).double() * power.repeat_interleave(32, dim=1)
    out = torch.zeros((s["m"], s["n"]), dtype=torch.float64, device="cuda")
    edges = s["offsets"].tolist()
    for e, (begin, end) in enumerate(zip(edges, edges[1:])):
        if end > begin:
            out[begin:end] = a[begin:end] @ _exact_weights(s, e)
    return out


def _exact_combine(s):
    out = s["shared_out"].double() if s["shared"] else torch.zeros((s["m"], s["n"]), dtype=torch.float64, device="cuda")
    for r in range(s["top_k"]):
        at = s["index"][:, r].long()
        live = at >= 0
        out[live] += s["y"][at[live]].double() * s["gate"][live, r].double()[:, None]
    return out


def _exact_matvec(s):
    x = s["x"].double()
    if s["ids"] is None:
        return x @ _exact_weights(s, None)
    out = torch.zeros((s["m"] * s["top_k"], s["n"]), dtype=torch.float64, device="cuda")
    for r, e in enumerate(s["ids"].flatten().tolist()):
        out[r] = x[r // s["top_k"]] @ _exact_weights(s, e)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "route": _exact_route, "grouped": _exact_grouped, "combine": _exact_combine,
            "matvec": _exact_matvec}[s["op"]](s)
