"""GPU test of the mixture-of-experts steps run together, as a layer uses them: norm, routing, rows of the dispatch, packed scatter,
the experts' products, the combination; and a token's way through FP4 experts.  Every stage is checked against its definition in
64 bits on what the stage before wrote; the whole is captured in a CUDA graph and replayed, and run on two streams at once."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIDDEN, INNER, EXPERTS, TOP_K = 512, 256, 12, 4
EPS = 1e-5


def _mx(torch, capi, w):
    """[experts, n, k] -> codes [experts, k, n], scales [experts, k / 64, n, 2], and the values in 64 bits [experts, k, n]."""
    e, n, k = w.shape
    q, s = capi.mx_quant(w.reshape(e * n, k).to(torch.bfloat16))
    value = q.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    return (q.view(e, n, k).transpose(1, 2).contiguous(), s.view(e, n, k // 64, 2).permute(0, 2, 1, 3).contiguous(),
            value.view(e, n, k).transpose(1, 2))


class Layer:
    def __init__(self, torch, capi, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.capi = torch, capi
        self.norm_weight = (1 + 0.1 * torch.randn(HIDDEN, generator=gen, device="cuda")).to(torch.bfloat16)
        self.router = torch.randn((HIDDEN, EXPERTS), generator=gen, device="cuda") * 0.1
        self.bias = torch.randn(EXPERTS, generator=gen, device="cuda") * 0.1
        self.up = _mx(torch, capi, torch.randn((EXPERTS, 2 * INNER, HIDDEN), generator=gen, device="cuda") * 0.05)
        self.down = _mx(torch, capi, torch.randn((EXPERTS, HIDDEN, INNER), generator=gen, device="cuda") * 0.05)

    def __call__(self, x, stream, seen=None):
        torch, capi = self.torch, self.capi
        tokens = x.shape[0]
        h = torch.empty_like(x)
        codes, scales = capi.add_rms_norm_mx_quant(x, stream, self.norm_weight, EPS, norm_out=h)
        logits = h.float() @ self.router
        ids, weights = capi.moe_route(logits, TOP_K, bias=self.bias, score="sigmoid", groups=4, top_groups=2, group_best=2, scale=2.0)
        index, offsets = capi.moe_row_plan(ids, EXPERTS)
        packed = torch.zeros((tokens * TOP_K, capi.packed_row_bytes(HIDDEN)), dtype=torch.uint8, device="cuda")
        capi.mx_quant_scatter_packed(h, index, packed, TOP_K)
        a, a_scales = packed[:, :HIDDEN], packed[:, HIDDEN : HIDDEN + HIDDEN // 32]
        gate_up = capi.mx_grouped_gemm(a, a_scales, self.up[0], self.up[1], offsets)
        inner = (torch.nn.functional.silu(gate_up[:, :INNER].float()) * gate_up[:, INNER:].float()).to(torch.bfloat16)
        inner_codes, inner_scales = capi.mx_quant(inner)
        y = capi.mx_grouped_gemm(inner_codes, inner_scales, self.down[0], self.down[1], offsets)
        out = capi.moe_combine(y, index, weights, shared=h)
        if seen is not None:
            seen.update(h=h, codes=codes, scales=scales, logits=logits, ids=ids, weights=weights, index=index, offsets=offsets, a=a,
                        a_scales=a_scales, gate_up=gate_up, inner_codes=inner_codes, inner_scales=inner_scales, y=y)
        return out


def _products(torch, a, a_scales, w64, offsets):
    a64 = a.contiguous().view(torch.float8_e4m3fn).double() * torch.exp2(a_scales.double() - 127).repeat_interleave(32, 1)
    want = torch.empty((a.shape[0], w64.shape[2]), dtype=torch.float64, device="cuda")
    size = torch.empty_like(want)
    edges = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(edges, edges[1:])):
        want[lo:hi], size[lo:hi] = a64[lo:hi] @ w64[e], a64[lo:hi].abs() @ w64[e].abs()
    return want, size


@pytest.mark.parametrize("tokens", [1, 37, 300, 5000])
def test_layer(capi, cuda, tokens):
    torch = cuda
    layer = Layer(torch, capi, tokens)
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x, stream = (torch.randn((tokens, HIDDEN), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    seen = {}
    out = layer(x, stream, seen)
    # the dispatch: every route has a row, rows are in the experts' order, and a row holds its token's codes
    ids, index, offsets = seen["ids"], seen["index"].long(), seen["offsets"]
    assert torch.equal(index.flatten().sort().values, torch.arange(tokens * TOP_K, device="cuda"))
    assert torch.equal((index.unsqueeze(2) >= offsets[1:].long()).sum(dim=2).int(), ids)
    assert int(offsets[-1]) == tokens * TOP_K
    codes, scales = capi.mx_quant(seen["h"])
    assert torch.equal(seen["a"][index], codes.unsqueeze(1).expand(-1, TOP_K, -1))
    assert torch.equal(seen["a_scales"][index], scales.unsqueeze(1).expand(-1, TOP_K, -1))
    # the products: K steps of 2^-23 of what is added up, and half a step of bf16
    for a, a_scales, w64, got in ((seen["a"], seen["a_scales"], layer.up[2], seen["gate_up"]),
                                  (seen["inner_codes"], seen["inner_scales"], layer.down[2], seen["y"])):
        want, size = _products(torch, a, a_scales, w64, offsets)
        slack = a.shape[1] * 2.0**-23 * size
        assert bool(((got.double() - want).abs() <= slack + 2.0**-8 * (want.abs() + slack)).all())
    parts = seen["y"].double()[index] * seen["weights"].double().unsqueeze(2)
    want, size = parts.sum(1) + seen["h"].double(), parts.abs().sum(1) + seen["h"].double().abs()
    slack = (TOP_K + 1) * 2.0**-24 * size
    assert bool(((out.double() - want).abs() <= slack + 2.0**-8 * (want.abs() + slack)).all())


@pytest.mark.parametrize("tokens", [40, 4400])  # one CTA and a cluster of sixteen for the plan; single CTAs and pairs for the products
def test_layer_in_a_graph(capi, cuda, tokens):
    torch = cuda
    layer = Layer(torch, capi, 1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    inputs = [tuple(torch.randn((tokens, HIDDEN), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)) for _ in range(3)]
    want = [(layer(x, r := s.clone()), r) for x, s in inputs]
    x, stream = inputs[0][0].clone(), inputs[0][1].clone()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, stream)
        graphs.append((graph, out))
    got = []
    for i in (0, 1, 2, 1, 0, 2):
        x.copy_(inputs[i][0])
        stream.copy_(inputs[i][1])
        graph, out = graphs[len(got) % 2]
        graph.replay()
        got.append((i, out.clone(), stream.clone()))
        layer(inputs[0][0], inputs[0][1].clone())  # an eager call between two replays
    torch.cuda.synchronize()
    for i, out, stream_out in got:
        assert torch.equal(out, want[i][0]) and torch.equal(stream_out, want[i][1])
    assert capi.last_status()[0] == 0


def test_layer_on_two_streams(capi, cuda):
    torch = cuda
    layers = [Layer(torch, capi, s) for s in (3, 4)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    inputs = [tuple(torch.randn((t, HIDDEN), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)) for t in (64, 150)]
    want = [layer(x, s.clone()) for layer, (x, s) in zip(layers, inputs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(layers[i](inputs[i][0], inputs[i][1].clone()))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def _fp4(torch, gen, experts, n, k):
    w = torch.randint(0, 256, (experts, k, n // 2), generator=gen, device="cuda", dtype=torch.uint8)
    return w, torch.randint(119, 122, (experts, k // 64, n, 2), generator=gen, device="cuda", dtype=torch.uint8)


def test_tokens_through_fp4_experts(capi, cuda):
    torch = cuda
    tokens = 3
    gen = torch.Generator(device="cuda").manual_seed(8)
    up, down = _fp4(torch, gen, EXPERTS, 2 * INNER, HIDDEN), _fp4(torch, gen, EXPERTS, HIDDEN, INNER)
    x = torch.randn((tokens, HIDDEN), generator=gen, device="cuda").to(torch.bfloat16)
    logits = torch.randn((tokens, EXPERTS), generator=gen, device="cuda")
    logits[0, 2:] = float("-inf")  # two experts left for four places
    rows = torch.arange(tokens * TOP_K, dtype=torch.int32, device="cuda").view(tokens, TOP_K)

    def step():
        ids, weights = capi.moe_route(logits, TOP_K)
        gate_up = capi.mx_fp4_matvec(x, *up, ids=ids)
        inner = (torch.nn.functional.silu(gate_up[:, :INNER].float()) * gate_up[:, INNER:].float()).to(torch.bfloat16)
        y = capi.mx_fp4_matvec(inner, *down, ids=ids)
        return ids, gate_up, inner, y, weights, capi.moe_combine(y, rows, weights)

    ids, gate_up, inner, y, weights, out = step()
    assert ids[0, 2:].tolist() == [-1, -1] and bool((y[2:4] == 0).all()) and bool((weights[0, 2:] == 0).all())
    # the experts' single products agree with the dense ones on the expert's own weight
    for r, e in enumerate(ids.flatten().tolist()):
        if e >= 0:
            assert torch.equal(gate_up[r], capi.mx_fp4_matvec(x[r // TOP_K : r // TOP_K + 1], up[0][e], up[1][e])[0])
            assert torch.equal(y[r], capi.mx_fp4_matvec(inner[r : r + 1], down[0][e], down[1][e])[0])
    parts = y.double().view(tokens, TOP_K, HIDDEN) * weights.double().unsqueeze(2)
    slack = (TOP_K + 1) * 2.0**-24 * parts.abs().sum(1)
    assert bool(((out.double() - parts.sum(1)).abs() <= slack + 2.0**-8 * (parts.sum(1).abs() + slack)).all())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, (ids, gate_up, inner, y, weights, out)))


FIRST_CALLS = """
import threading, torch
from catccos_b200 import capi
capi.load()
gen = torch.Generator(device="cuda").manual_seed(4)
logits = torch.randn((500, 64), generator=gen, device="cuda")
x = torch.randn((33, 256), generator=gen, device="cuda").to(torch.bfloat16)
weight = torch.ones(256, dtype=torch.bfloat16, device="cuda")
torch.cuda.synchronize()
start, out = threading.Barrier(16), [None] * 16

def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        out[i] = capi.moe_route(logits, 6) if i % 2 else capi.add_rms_norm_mx_quant(x, None, weight, 1e-6)
        torch.cuda.current_stream().synchronize()

threads = [threading.Thread(target=work, args=(i,)) for i in range(16)]
for t in threads:
    t.start()
for t in threads:
    t.join()
for i in range(2, 16):
    assert all(torch.equal(a, b) for a, b in zip(out[i], out[i % 2])), i
print("first calls ok")
"""


def test_first_calls_of_several_threads(capi, cuda):
    # a process of their own: the calls that set the library up
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "first calls ok" in run.stdout, run.stdout + run.stderr


FIRST_PRODUCTS = """
import threading, torch
from catccos_b200 import capi
capi.load()
gen = torch.Generator(device="cuda").manual_seed(4)
n, k, experts = 256, 256, 2
codes = lambda *shape: torch.randint(0, 120, shape, generator=gen, device="cuda", dtype=torch.uint8)
scales = lambda *shape: torch.randint(118, 122, shape, generator=gen, device="cuda", dtype=torch.uint8)
small = (codes(40, k), scales(40, k // 32), codes(experts, k, n), scales(experts, k // 64, n, 2), torch.tensor([0, 9, 40], dtype=torch.int32, device="cuda"))
large = (codes(9000, k), scales(9000, k // 32), *small[2:4], torch.tensor([0, 9, 9000], dtype=torch.int32, device="cuda"))
ids = torch.randint(-1, 9, (9000, 2), generator=gen, device="cuda", dtype=torch.int32)
x = torch.randn((6, k), generator=gen, device="cuda").to(torch.bfloat16)
w, w_scales = codes(k, n // 2), scales(k // 64, n, 2)
calls = [lambda: capi.mx_grouped_gemm(*small), lambda: capi.mx_grouped_gemm(*large), lambda: capi.moe_row_plan(ids, 9),
         lambda: capi.mx_fp4_matvec(x, w, w_scales)]
torch.cuda.synchronize()
start, out = threading.Barrier(16), [None] * 16

def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        got = calls[i % 4]()
        out[i] = got if isinstance(got, tuple) else (got,)
        torch.cuda.current_stream().synchronize()

threads = [threading.Thread(target=work, args=(i,)) for i in range(16)]
for t in threads:
    t.start()
for t in threads:
    t.join()
for i in range(4, 16):
    assert all(torch.equal(a, b) for a, b in zip(out[i], out[i % 4])), i
assert all(bool(torch.isfinite(o[0]).all()) for o in out) and capi.last_status()[0] == 0
print("first products ok")
"""


def test_first_products_of_several_threads(capi, cuda):
    # the entry points of the driver, what kernels may use and the tensor maps are found out by threads that call at once
    run = subprocess.run([sys.executable, "-c", FIRST_PRODUCTS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "first products ok" in run.stdout, run.stdout + run.stderr
