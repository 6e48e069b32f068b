"""Products of 8-bit codes with one fp32 scale for each block of 128, and the way of an expert layer's rows there and back with its gradients, on
one GPU: what is timed, their plain forms in elementary torch operations, and their values in 64 bits.

A case is a dict of plain values:
  op       "quant"     blocks of 128 to 8-bit codes and fp32 scales (capi.block_quant)
           "gemm"      products of such operands (capi.block_gemm)
           "grouped"   every expert's product on its own rows (capi.block_grouped_gemm)
           "dispatch"  rows to their places in the experts' order, or the gradient of that (capi.moe_dispatch, capi.moe_dispatch_grad)
           "combine"   the gradients of the weighted sum of a token's expert rows (capi.moe_combine_grad)
  m n k    rows or tokens, output columns (dispatch, combine: width), contraction length (quant: width)
  x        element type of 16- or 32-bit values: "bf16", "fp16" or "fp32"; of a product: the output's
  codes    element type of 8-bit activation codes: "e4m3" or "e5m2"
  block    quant: "row" (1 x 128), "column" (128 x 1) or "square" (128 x 128)
  top_k    routes of a token; quant: 0, or each token's codes go to the rows of its routes
  pass     gemm: "forward" (x W), "input" (dy W^T) or "weight" (x^T dy); grouped: "forward" or "input"; dispatch: "forward" or "backward"
"""
import math

import torch

own = False

MOST = {"e4m3": 448.0, "e5m2": 57344.0}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
LEAST = 2.0**-100  # a block's largest value counts as at least this


def listed():
    return [
        # a prefill chunk on its way into the expert layer: quantised once, written to the rows of its routes
        dict(name="quant_dispatch", op="quant", m=4096, k=7168, x="bf16", codes="e4m3", block="row", top_k=8),
        # one side of a weight's gradient: a batch's output gradients, quantised along the tokens (a ragged last block)
        dict(name="quant_columns", op="quant", m=8190, k=2304, x="bf16", codes="e5m2", block="column", top_k=0),
        # one decode step of 16 sequences through a projection: the weight streams
        dict(name="gemm_decode", op="gemm", m=16, n=4096, k=7168, codes="e4m3", x="bf16", **{"pass": "forward"}),
        # a long prefill chunk
        dict(name="gemm_prefill", op="gemm", m=8192, n=2304, k=7168, codes="e4m3", x="bf16", **{"pass": "forward"}),
        # training: the gradient of a projection's input, an odd number of tokens, the weight read the other way round
        dict(name="gemm_input_grad", op="gemm", m=3001, n=7168, k=2304, codes="e5m2", x="bf16", **{"pass": "input"}),
        # training: the gradient of a projection's weight over 4096 tokens
        dict(name="gemm_weight_grad", op="gemm", m=7168, n=2304, k=4096, codes="e4m3", x="fp32", **{"pass": "weight"}),
        # 16 sequences' routes on a rank with 32 experts: the weights stream
        dict(name="grouped_decode", op="grouped", m=128, n=4096, k=7168, experts=32, codes="e4m3", x="bf16", **{"pass": "forward"}),
        # a prefill of 2048 tokens with 8 routes each
        dict(name="grouped_prefill", op="grouped", m=16384, n=2304, k=7168, experts=32, codes="e4m3", x="bf16", **{"pass": "forward"}),
        # the rows of a prefill sorted by expert, with dropped routes
        dict(name="dispatch_prefill", op="dispatch", m=4095, n=7168, top_k=8, x="bf16", **{"pass": "forward"}),
        # the gradient of that for a small batch
        dict(name="dispatch_backward", op="dispatch", m=64, n=7168, top_k=8, x="bf16", **{"pass": "backward"}),
        # the end of the expert layer backwards: a small batch, and a long one with an odd number of tokens
        dict(name="combine_grad_small", op="combine", m=64, n=7168, top_k=8, x="bf16"),
        dict(name="combine_grad_large", op="combine", m=4095, n=5120, top_k=6, x="fp16"),
    ]


MOST_FLOPS = 2.0 * 16384 * 2304 * 7168  # of grouped_prefill
MOST_BYTES = 32 * 4096 * 7168 * 1.0  # of grouped_decode


def _spread(rng, low, high, step=1):
    """A multiple of `step` between the two, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    while True:
        op = rng.choice(("quant", "gemm", "gemm", "grouped", "dispatch", "combine"))
        c = dict(op=op)
        codes = rng.choice(("e4m3", "e4m3", "e5m2"))
        if op == "quant":
            block = rng.choice(("row", "row", "column", "square"))
            top_k = rng.randint(1, 8) if block == "row" and rng.random() < 0.5 else 0
            c.update(m=_spread(rng, 1, 16384 if top_k == 0 else 4096), k=_spread(rng, 16, 8192, 16),
                     x=rng.choice(("bf16", "bf16", "fp16", "fp32")), codes=codes, block=block, top_k=top_k)
        elif op == "gemm":
            which = rng.choice(("forward", "forward", "input", "weight"))
            c.update(m=_spread(rng, 256, 8192, 16) if which == "weight" else _spread(rng, 1, 16384), n=_spread(rng, 128, 8192, 16),
                     k=_spread(rng, 16, 16384, 16) if which == "weight" else _spread(rng, 128, 8192, 16), codes=codes,
                     x="fp32" if which == "weight" else rng.choice(("bf16", "fp16")))
            c["pass"] = which
        elif op == "grouped":
            c.update(m=_spread(rng, 1, 16384), n=_spread(rng, 256, 7168, 16), k=_spread(rng, 256, 7168, 16),
                     experts=_spread(rng, 1, 64), codes=codes, x=rng.choice(("bf16", "fp16")))
            c["pass"] = rng.choice(("forward", "input"))
        else:
            c.update(m=_spread(rng, 1, 8192), n=_spread(rng, 64, 8192, 8), top_k=rng.randint(1, 8), x=rng.choice(("bf16", "fp16")))
            if op == "dispatch":
                c["pass"] = rng.choice(("forward", "backward"))
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and c.get("experts", 0) * c.get("k", 0) * c.get("n", 0) <= 32 * 4096 * 7168:
            return c


def _blocks(n):
    return (n + 127) // 128


def work(case):
    """Each input read once, each output written once, and the products."""
    op, m, k, n = case["op"], case["m"], case.get("k", 0), case.get("n", 0)
    if op == "quant":
        scales = {"row": m * _blocks(k), "column": _blocks(m) * k, "square": _blocks(m) * _blocks(k)}[case["block"]]
        copies = max(1, case["top_k"])
        return {"bytes": float(m * k * (SIZE[case["x"]] + copies) + 4 * copies * scales + 4 * m * case["top_k"]), "flops": 0.0}
    if op == "gemm":
        scales = m * _blocks(k) + _blocks(k) * (n if case["pass"] == "weight" else _blocks(n))
        return {"bytes": float(m * k + k * n + 4 * scales + SIZE[case["x"]] * m * n), "flops": 2.0 * m * n * k}
    if op == "grouped":
        weights = min(case["experts"], m) * (n * k + 4 * _blocks(n) * _blocks(k))
        return {"bytes": float(m * k + 4 * m * _blocks(k) + weights + 2 * m * n), "flops": 2.0 * m * n * k}
    routes = m * case["top_k"]
    if op == "dispatch":
        return {"bytes": float(2 * n * (m + routes) + 4 * routes), "flops": float(routes * n if case["pass"] == "backward" else 0)}
    return {"bytes": float(2 * n * (m + 2 * routes) + 12 * routes), "flops": 3.0 * routes * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _activations(m, k, gen):
    """Hidden states: normal, with one channel in a thousand much larger."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    x[:, torch.randperm(k, generator=gen, device="cuda")[: math.ceil(0.001 * k)]] *= 30.0
    return x


def _gradients(m, k, gen):
    """Small, with rows of very different size."""
    return torch.randn((m, k), generator=gen, device="cuda") * torch.exp(2.0 * torch.randn((m, 1), generator=gen, device="cuda")) * 1e-4


def _padded(x, block):
    """x in blocks [.., rows in a block, .., columns in a block], zeros behind its edges."""
    rows, cols = (1 if block == "row" else 128), (1 if block == "column" else 128)
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // cols, cols)


def _codes(x, codes, block):
    """fp32 [m, k] -> 8-bit codes [m, k] and the blocks' scales."""
    v = _padded(x, block)
    top = v.abs().amax(dim=(1, 3), keepdim=True).clamp_min(LEAST)
    q = (v * (MOST[codes] / top)).clamp(-MOST[codes], MOST[codes]).to(F8[codes])
    q = q.reshape(v.shape[0] * v.shape[1], -1)[: x.shape[0], : x.shape[1]].contiguous()
    return q, (top / MOST[codes]).squeeze(3).squeeze(1).contiguous()


def _routes(m, top_k, gen, drop):
    """Every route's row, -1 for one that is dropped."""
    index = torch.randperm(m * top_k, generator=gen, device="cuda").to(torch.int32)
    if drop:
        index[torch.rand(m * top_k, generator=gen, device="cuda") < 0.02] = -1
    return index.view(m, top_k)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    op, m = case["op"], case["m"]
    if op == "quant":
        k, top_k = case["k"], case["top_k"]
        s["in"] = (_gradients(m, k, gen) if case["codes"] == "e5m2" else _activations(m, k, gen)).to(DTYPE[case["x"]])
        if top_k:  # rows that no route names stay as they are
            s["index"] = _routes(m, top_k, gen, True)
            s["rows"] = torch.zeros((m * top_k, k), dtype=torch.uint8, device="cuda").view(F8[case["codes"]])
            s["row_scales"] = torch.zeros((m * top_k, _blocks(k)), device="cuda")
    elif op == "gemm":
        n, k = case["n"], case["k"]
        if case["pass"] == "weight":  # x [k, m] and dy [k, n], both quantised along k
            a, s["a_scales"] = _codes(_activations(k, m, gen), "e4m3", "column")
            s["a"], s["a_scales"] = a.t(), s["a_scales"].t()
            s["b"], s["b_scales"] = _codes(_gradients(k, n, gen), case["codes"], "column")
        else:
            values = _gradients(m, k, gen) if case["pass"] == "input" else _activations(m, k, gen)
            s["a"], s["a_scales"] = _codes(values, case["codes"], "row")
            shape = (k, n) if case["pass"] == "forward" else (n, k)
            s["b"], s["b_scales"] = _codes(torch.randn(shape, generator=gen, device="cuda") * 0.02, "e4m3", "square")
            if case["pass"] == "input":
                s["b"], s["b_scales"] = s["b"].t(), s["b_scales"].t()
    elif op == "grouped":
        e, n, k = case["experts"], case["n"], case["k"]
        # some experts are chosen far more often than others, some not at all
        popular = torch.softmax(torch.randn(e, generator=gen, device="cuda"), 0)
        expert = torch.multinomial(popular, m, replacement=True, generator=gen).sort().values
        s["offsets"] = torch.searchsorted(expert, torch.arange(e + 1, device="cuda")).to(torch.int32)
        s["cap"] = int(torch.bincount(expert, minlength=e).max())  # only the plain form needs it
        s["a"], s["a_scales"] = _codes(_gradients(m, k, gen) if case["pass"] == "input" else _activations(m, k, gen), case["codes"], "row")
        rows, cols = (k, n) if case["pass"] == "forward" else (n, k)
        b = torch.empty((e, rows, cols), dtype=torch.uint8, device="cuda")
        f = torch.empty((e, _blocks(rows), _blocks(cols)), device="cuda")
        for i in range(e):
            q, f[i] = _codes(torch.randn((rows, cols), generator=gen, device="cuda") * 0.02, "e4m3", "square")
            b[i] = q.view(torch.uint8)
        b = b.view(torch.float8_e4m3fn)
        s["b"], s["b_scales"] = (b, f) if case["pass"] == "forward" else (b.transpose(1, 2), f.transpose(1, 2))
    else:
        n, top_k, kind = case["n"], case["top_k"], DTYPE[case["x"]]
        s["index"] = _routes(m, top_k, gen, True)
        if op == "dispatch" and case["pass"] == "forward":
            s["in"] = _activations(m, n, gen).to(kind)
            s["rows"] = torch.zeros((m * top_k, n), dtype=kind, device="cuda")
        elif op == "dispatch":
            s["in"] = _gradients(m * top_k, n, gen).to(kind)
        else:
            s["y"] = _activations(m * top_k, n, gen).to(kind)
            s["gate"] = torch.softmax(torch.randn((m, top_k), generator=gen, device="cuda"), 1)
            s["d_out"] = (_gradients(m, n, gen) * 100.0).to(kind)
            s["rows"] = torch.zeros((m * top_k, n), dtype=kind, device="cuda")
    return s


# ---- the calls that a user makes --------------------------------------------------------------------------------------------
def _run_own(s):
    from catccos_b200 import capi

    op = s["op"]
    if op == "quant":
        if s["top_k"]:
            codes, scales = capi.block_quant(s["in"], dtype=F8[s["codes"]], row_index=s["index"], out=(s["rows"], s["row_scales"]))
        else:
            codes, scales = capi.block_quant(s["in"], dtype=F8[s["codes"]], block=s["block"])
        return {"codes": codes, "scales": scales}
    if op == "gemm":
        return capi.block_gemm(s["a"], s["a_scales"], s["b"], s["b_scales"], out_dtype=DTYPE[s["x"]])
    if op == "grouped":
        return capi.block_grouped_gemm(s["a"], s["a_scales"], s["b"], s["b_scales"], s["offsets"], out_dtype=DTYPE[s["x"]])
    if op == "dispatch":
        if s["pass"] == "forward":
            return capi.moe_dispatch(s["in"], s["index"], out=s["rows"])
        return capi.moe_dispatch_grad(s["in"], s["index"])
    d_rows, d_gate = capi.moe_combine_grad(s["d_out"], s["y"], s["index"], s["gate"], out=s["rows"])
    return {"rows": d_rows, "weights": d_gate}


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _spread_scales(scales, rows, cols):
    """Scales of 128 x 128 blocks, one for each value of [.., rows, cols]."""
    return scales.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)[..., :cols]


def _plain_quant(s):
    codes, scales = _codes(s["in"].float(), s["codes"], s["block"])
    if not s["top_k"]:
        return {"codes": codes, "scales": scales}
    index = s["index"].long().flatten()
    live = index >= 0
    token = torch.arange(s["m"], device="cuda").repeat_interleave(s["top_k"])[live]
    rows = torch.zeros((s["m"] * s["top_k"], s["k"]), dtype=torch.uint8, device="cuda")
    rows[index[live]] = codes.view(torch.uint8)[token]
    row_scales = torch.zeros((s["m"] * s["top_k"], scales.shape[1]), device="cuda")
    row_scales[index[live]] = scales[token]
    return {"codes": rows.view(F8[s["codes"]]), "scales": row_scales}


def _plain_gemm(s):
    a = s["a"].float() * s["a_scales"].repeat_interleave(128, 1)[:, : s["k"]]
    if s["pass"] == "weight":
        b = s["b"].float() * s["b_scales"].repeat_interleave(128, 0)[: s["k"]]
    else:
        b = s["b"].float() * _spread_scales(s["b_scales"], s["k"], s["n"])
    return (a @ b).to(DTYPE[s["x"]])


def _plain_grouped(s):
    a = s["a"].float() * s["a_scales"].repeat_interleave(128, 1)[:, : s["k"]]
    b = s["b"].float() * _spread_scales(s["b_scales"], s["k"], s["n"])
    begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    row = begin[:, None] + torch.arange(s["cap"], device="cuda")
    inside = row < end[:, None]
    c = torch.bmm(a[row.clamp(max=s["m"] - 1)], b)
    out = torch.empty((s["m"], s["n"]), dtype=DTYPE[s["x"]], device="cuda")
    out[row[inside]] = c[inside].to(out.dtype)
    return out


def _plain_dispatch(s):
    index = s["index"].long()
    if s["pass"] == "backward":
        return (s["in"][index.clamp(min=0)].float() * (index >= 0).unsqueeze(2)).sum(dim=1).to(s["in"].dtype)
    out = torch.zeros((s["m"] * s["top_k"], s["n"]), dtype=s["in"].dtype, device="cuda")
    live = index.flatten() >= 0
    out[index.flatten()[live]] = s["in"].repeat_interleave(s["top_k"], 0)[live]
    return out


def _plain_combine(s):
    index = s["index"].long()
    live = index >= 0
    d = s["d_out"].float().unsqueeze(1)
    weights = (s["y"][index.clamp(min=0)].float() * d).sum(dim=2) * live
    rows = torch.zeros((s["m"] * s["top_k"], s["n"]), dtype=s["y"].dtype, device="cuda")
    rows[index[live]] = (s["gate"].unsqueeze(2) * d)[live].to(rows.dtype)
    return {"rows": rows, "weights": weights}


def run(s):
    if own:
        return _run_own(s)
    return {"quant": _plain_quant, "gemm": _plain_gemm, "grouped": _plain_grouped, "dispatch": _plain_dispatch,
            "combine": _plain_combine}[s["op"]](s)


# ---- values in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_quant(s):
    m, k, most = s["m"], s["k"], MOST[s["codes"]]
    x = s["in"].double()
    codes = torch.empty_like(x)
    rows, cols = (1 if s["block"] == "row" else 128), (1 if s["block"] == "column" else 128)
    whole = torch.zeros((-(-m // rows) * rows, -(-k // cols) * cols), dtype=torch.float64, device="cuda")
    whole[:m, :k] = x
    top = whole.abs().unflatten(1, (-1, cols)).amax(2).unflatten(0, (-1, rows)).amax(1)
    scales = torch.maximum(top, torch.full_like(top, LEAST)) / most
    codes = x / scales.repeat_interleave(rows, 0)[:m].repeat_interleave(cols, 1)[:, :k]
    digits, lowest = (3, -6) if s["codes"] == "e4m3" else (2, -14)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), (torch.frexp(codes)[1] - 1).clamp(min=lowest) - digits)
    codes = (torch.round(codes / step) * step).clamp(-most, most)
    if not s["top_k"]:
        return {"codes": codes, "scales": scales}
    out = torch.zeros((m * s["top_k"], k), dtype=torch.float64, device="cuda")
    out_scales = torch.zeros((m * s["top_k"], scales.shape[1]), dtype=torch.float64, device="cuda")
    for r in range(s["top_k"]):
        at = s["index"][:, r].long()
        live = at >= 0
        out[at[live]], out_scales[at[live]] = codes[live], scales[live]
    return {"codes": out, "scales": out_scales}


def _exact_product(a, a_scales, b, b_scales):
    """A sum over blocks of 128: each block's product, scaled on both sides."""
    k, n = b.shape
    out = torch.zeros((a.shape[0], n), dtype=torch.float64, device="cuda")
    for i, k0 in enumerate(range(0, k, 128)):
        f = b_scales[i].double()
        if f.numel() != n:
            f = f.repeat_interleave(128)[:n]
        out += (a[:, k0 : k0 + 128].double() * a_scales[:, i].double()[:, None]) @ (b[k0 : k0 + 128].double() * f)
    return out


def _exact_grouped(s):
    out = torch.zeros((s["m"], s["n"]), dtype=torch.float64, device="cuda")
    edges = s["offsets"].tolist()
    for e, (begin, end) in enumerate(zip(edges, edges[1:])):
        if end > begin:
            out[begin:end] = _exact_product(s["a"][begin:end], s["a_scales"][begin:end], s["b"][e], s["b_scales"][e])
    return out


def _exact_dispatch(s):
    forward = s["pass"] == "forward"
    out = torch.zeros((s["m"] * (s["top_k"] if forward else 1), s["n"]), dtype=torch.float64, device="cuda")
    for r in range(s["top_k"]):
        at = s["index"][:, r].long()
        live = at >= 0
        if forward:
            out[at[live]] = s["in"][live].double()
        else:
            out[live] += s["in"][at[live]].double()
    return out


def _exact_combine(s):
    rows = torch.zeros((s["m"] * s["top_k"], s["n"]), dtype=torch.float64, device="cuda")
    weights = torch.zeros((s["m"], s["top_k"]), dtype=torch.float64, device="cuda")
    d = s["d_out"].double()
    for r in range(s["top_k"]):
        at = s["index"][:, r].long()
        live = at >= 0
        rows[at[live]] = d[live] * s["gate"][live, r].double()[:, None]
        weights[live, r] = torch.einsum("tn,tn->t", d[live], s["y"][at[live]].double())
    return {"rows": rows, "weights": weights}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        return _exact_product(s["a"], s["a_scales"], s["b"], s["b_scales"])
    return {"quant": _exact_quant, "grouped": _exact_grouped, "dispatch": _exact_dispatch, "combine": _exact_combine}[case["op"]](s)
