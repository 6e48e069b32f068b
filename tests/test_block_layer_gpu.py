"""GPU test of an expert layer with weights in blocks of 128, there and back: routing, rows of the dispatch, quantised dispatch, the experts'
products, the combination; then the combination's gradient, the products with the weights read the other way round, the dispatch's
gradient.  Every stage is checked against its definition in 64 bits on what the stage before wrote, on a rank that has all experts and on
one that has some; the whole is captured in a CUDA graph and replayed."""
import pytest

pytestmark = pytest.mark.gpu

HIDDEN, INNER, EXPERTS, TOP_K = 528, 272, 12, 4  # blocks that are not full on every axis
HALF = 2.0**-8


class Layer:
    def __init__(self, torch, capi, seed, first=0, local=EXPERTS):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.capi, self.first, self.local = torch, capi, first, local
        self.router = torch.randn((HIDDEN, EXPERTS), generator=gen, device="cuda") * 0.1
        self.up = self._weights(torch.randn((local, HIDDEN, 2 * INNER), generator=gen, device="cuda") * 0.05)  # [K, N]
        self.down = self._weights(torch.randn((local, HIDDEN, INNER), generator=gen, device="cuda") * 0.05)    # a checkpoint's [N, K]
        self.down = tuple(t.transpose(1, 2) for t in self.down)

    def _weights(self, w):
        both = [self.capi.block_quant(m, block="square") for m in w]  # from fp32
        return self.torch.stack([c.view(self.torch.uint8) for c, _ in both]).view(self.torch.float8_e4m3fn), self.torch.stack([s for _, s in both])

    def forward(self, h):
        torch, capi = self.torch, self.capi
        s = {"h": h}
        s["ids"], s["weights"] = capi.moe_route(h.float() @ self.router, TOP_K, score="sigmoid", scale=2.0)
        s["index"], s["offsets"] = capi.moe_row_plan(s["ids"], self.local, first_expert=self.first)
        rows = h.shape[0] * TOP_K
        # rows that belong to no expert here hold anything
        out = (torch.full((rows, HIDDEN), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.full((rows, 5), float("nan"), device="cuda"))
        s["a"], s["a_scales"] = capi.block_quant(h, row_index=s["index"], out=out)
        s["gate_up"] = capi.block_grouped_gemm(s["a"], s["a_scales"], *self.up, s["offsets"], out=torch.full((rows, 2 * INNER), float("nan"), dtype=torch.bfloat16, device="cuda"))
        gate, up = s["gate_up"].float().split(INNER, 1)
        s["inner"], s["inner_scales"] = capi.block_quant((torch.nn.functional.silu(gate) * up).to(torch.bfloat16))
        s["y"] = capi.block_grouped_gemm(s["inner"], s["inner_scales"], *self.down, s["offsets"], out=torch.full((rows, HIDDEN), float("nan"), dtype=torch.bfloat16, device="cuda"))
        s["out"] = capi.moe_combine(s["y"], s["index"], s["weights"], shared=h)
        return s

    def backward(self, s, d_out):
        torch, capi = self.torch, self.capi
        rows = s["y"].shape[0]
        nan = lambda n: torch.full((rows, n), float("nan"), dtype=torch.bfloat16, device="cuda")
        g = {"d_out": d_out}
        g["d_y"], g["d_weights"] = capi.moe_combine_grad(d_out, s["y"], s["index"], s["weights"], out=nan(HIDDEN))
        g["d_y_codes"], g["d_y_scales"] = capi.block_quant(g["d_y"], dtype=torch.float8_e5m2)
        down, scales = (t.transpose(1, 2) for t in self.down)
        g["d_inner"] = capi.block_grouped_gemm(g["d_y_codes"], g["d_y_scales"], down, scales, s["offsets"], out=nan(INNER))
        gate, up = s["gate_up"].float().split(INNER, 1)
        sig, d = torch.sigmoid(gate), g["d_inner"].float()
        g["d_gate_up"] = torch.cat((d * up * sig * (1 + gate * (1 - sig)), d * gate * sig), 1).to(torch.bfloat16)
        g["d_gate_up_codes"], g["d_gate_up_scales"] = capi.block_quant(g["d_gate_up"], dtype=torch.float8_e5m2)
        g["d_rows"] = capi.block_grouped_gemm(g["d_gate_up_codes"], g["d_gate_up_scales"], *(t.transpose(1, 2) for t in self.up), s["offsets"], out=nan(HIDDEN))
        g["d_h"] = capi.moe_dispatch_grad(g["d_rows"], s["index"], shared=d_out)
        return g


def _value(codes, scales, square=False):
    k = codes.shape[-1]
    s = scales.double().repeat_interleave(128, -1)[..., :k]
    if square:
        s = s.repeat_interleave(128, -2)[..., : codes.shape[-2], :]
    return codes.double() * s


def _check_products(torch, got, a, a_scales, w, w_scales, offsets):
    k = a.shape[1]
    edges = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(edges, edges[1:])):
        if hi > lo:
            x, m = _value(a[lo:hi], a_scales[lo:hi]), _value(w[e], w_scales[e], True)
            want, slack = x @ m, (k + 2 * ((k + 127) // 128)) * 2.0**-23 * (x.abs() @ m.abs())
            assert bool(((got[lo:hi].double() - want).abs() <= slack + HALF * (want.abs() + slack)).all())
    assert bool(got[edges[-1] :].isnan().all())


@pytest.mark.parametrize("first,local", [(0, EXPERTS), (5, 3)])
@pytest.mark.parametrize("tokens", [1, 37, 300, 3000])
def test_layer(capi, cuda, tokens, first, local):
    torch = cuda
    layer = Layer(torch, capi, tokens, first, local)
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    h, d_out = (torch.randn((tokens, HIDDEN), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    s = layer.forward(h)
    g = layer.backward(s, d_out)
    assert capi.last_status()[0] == 0
    index, offsets = s["index"], s["offsets"]
    live = index >= 0
    at, token = index[live].long(), torch.arange(tokens, device="cuda")[:, None].expand(-1, TOP_K)[live]
    mine = int(offsets[-1])
    # the dispatch, quantised before and after
    codes, scales = capi.block_quant(h)
    rows, row_scales = capi.block_quant(capi.moe_dispatch(h, index, out=torch.zeros((tokens * TOP_K, HIDDEN), dtype=h.dtype, device="cuda")))
    for got_codes, got_scales in ((s["a"], s["a_scales"]), (rows, row_scales)):
        assert torch.equal(got_codes.view(torch.uint8)[at], codes.view(torch.uint8)[token]) and torch.equal(got_scales[at], scales[token])
    _check_products(torch, s["gate_up"], s["a"], s["a_scales"], *layer.up, offsets)
    _check_products(torch, s["y"], s["inner"], s["inner_scales"], *(t.contiguous() for t in layer.down), offsets)
    parts = torch.zeros((tokens, TOP_K, HIDDEN), dtype=torch.float64, device="cuda")
    parts[live] = s["y"].double()[at] * s["weights"].double()[live].unsqueeze(1)
    want = parts.sum(1) + h.double()
    slack = (TOP_K + 1) * 2.0**-24 * (parts.abs().sum(1) + h.double().abs())
    assert bool(((s["out"].double() - want).abs() <= slack + HALF * (want.abs() + slack)).all())
    # and back
    want = d_out.double()[token] * s["weights"].double()[live].unsqueeze(1)
    slack = 2.0**-24 * want.abs()
    assert bool(((g["d_y"].double()[at] - want).abs() <= slack + HALF * (want.abs() + slack)).all())
    products = d_out.double()[token] * s["y"].double()[at]
    assert bool(((g["d_weights"].double()[live] - products.sum(1)).abs() <= HIDDEN * 2.0**-24 * products.abs().sum(1)).all())
    assert bool((g["d_weights"][~live] == 0).all())
    _check_products(torch, g["d_inner"], g["d_y_codes"], g["d_y_scales"], *(t.transpose(1, 2).contiguous() for t in layer.down), offsets)
    _check_products(torch, g["d_rows"], g["d_gate_up_codes"], g["d_gate_up_scales"], *(t.transpose(1, 2).contiguous() for t in layer.up), offsets)
    parts.zero_()
    parts[live] = g["d_rows"].double()[at]
    want = parts.sum(1) + d_out.double()
    slack = (TOP_K + 1) * 2.0**-24 * (parts.abs().sum(1) + d_out.double().abs())
    assert bool(((g["d_h"].double() - want).abs() <= slack + HALF * (want.abs() + slack)).all())
    assert mine == at.numel()


@pytest.mark.parametrize("tokens", [40, 2000])  # the products' forms for few rows and for many
def test_layer_in_a_graph(capi, cuda, tokens):
    torch = cuda
    layer = Layer(torch, capi, 1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    inputs = [tuple(torch.randn((tokens, HIDDEN), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)) for _ in range(3)]

    def step(h, d_out):
        s = layer.forward(h)
        g = layer.backward(s, d_out)
        return s["out"], g["d_h"], g["d_weights"]

    want = [step(*i) for i in inputs]
    h, d_out = (t.clone() for t in inputs[0])
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(h, d_out)
        graphs.append((graph, out))
    got = []
    for i in (0, 1, 2, 1, 0, 2):
        h.copy_(inputs[i][0])
        d_out.copy_(inputs[i][1])
        graph, out = graphs[len(got) % 2]
        graph.replay()
        got.append((i, [t.clone() for t in out]))
        step(*inputs[0])  # an eager step between two replays
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    assert capi.last_status()[0] == 0


def test_gradients_of_a_dense_layer(capi, cuda):
    # x W, and the gradients of x and of W from the same codes: against the plain products of what the codes stand for
    torch = cuda
    m, k, n = 400, 528, 272
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, w, dy = (torch.randn(s, generator=gen, device="cuda").to(torch.bfloat16) for s in ((m, k), (k, n), (m, n)))
    wc, ws = capi.block_quant(w, block="square")
    for got, (a, a_scales), (b, b_scales), a64, b64 in (
        (lambda a, b: capi.block_gemm(*a, *b), capi.block_quant(x), (wc, ws), lambda c, s: _value(c, s), lambda c, s: _value(c, s, True)),
        (lambda a, b: capi.block_gemm(*a, b[0].t(), b[1].t()), capi.block_quant(dy, dtype=torch.float8_e5m2), (wc, ws), lambda c, s: _value(c, s),
         lambda c, s: _value(c, s, True).t()),
        (lambda a, b: capi.block_gemm(a[0].t(), a[1].t(), *b, out_dtype=torch.float32), capi.block_quant(x, block="column"),
         capi.block_quant(dy, dtype=torch.float8_e5m2, block="column"), lambda c, s: (c.double() * s.double().repeat_interleave(128, 0)[:m]).t(),
         lambda c, s: c.double() * s.double().repeat_interleave(128, 0)[:m])):
        c = got((a, a_scales), (b, b_scales))
        l, r = a64(a, a_scales), b64(b, b_scales)
        want, slack = l @ r, (l.shape[1] + 2 * ((l.shape[1] + 127) // 128)) * 2.0**-23 * (l.abs() @ r.abs())
        half = 2.0**-24 if c.dtype == torch.float32 else HALF
        assert bool(((c.double() - want).abs() <= slack + half * (want.abs() + slack)).all())


def test_tensors_of_another_stream(capi, cuda):
    # a call runs on the current stream of its tensors' device, behind what was put there
    torch = cuda
    x = torch.randn((3000, 1024), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    want = capi.block_quant(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20000000)
        late = x.clone()
        got = capi.block_quant(late)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
