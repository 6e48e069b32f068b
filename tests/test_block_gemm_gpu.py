"""GPU tests of the products of 8-bit codes with an fp32 scale for each block of 128, dense and per expert, against the dequantised
operands in 64 bits.

A result may be off by: K + 2 B steps of 2^-23 of the sum of its products' magnitudes (the accumulator takes K products and
truncates; B = K / 128 blocks are each scaled, by a product of two scales, and added, in fp32), half a step of its type, and, in
fp16, half of the smallest step there."""
import threading

import pytest

pytestmark = pytest.mark.gpu

# the kernels' forms: tiles of 16, 32 and 64 rows, K cut over CTAs, pairs of CTAs, and what the library chooses
FORMS = [dict(block_rows=16, split_k=1), dict(block_rows=32, split_k=1), dict(block_rows=64, split_k=1), dict(block_rows=16, split_k=8),
         dict(block_rows=32, split_k=2), dict(block_rows=64, split_k=4), dict(cta_pair=1), dict()]
IDS = ["16", "32", "64", "16x8", "32x2", "64x4", "pair", "auto"]
HALF = {"bfloat16": 2.0**-8, "float16": 2.0**-11, "float32": 2.0**-24}
LEAST = {"bfloat16": 0.0, "float16": 2.0**-25, "float32": 0.0}


class Options:
    def __init__(self, capi, options):
        self.capi, self.options = capi, options

    def __enter__(self):
        for key, value in self.options.items():
            self.capi.set_option(key, value)

    def __exit__(self, *_):
        for key in self.options:
            self.capi.set_option(key, 0)


def _codes(torch, shape, dtype, gen):
    """Codes of every size, none infinite or NaN."""
    bits = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    if dtype == "float8_e4m3fn":
        bits = torch.where((bits & 0x7F) == 0x7F, bits ^ 1, bits)
    else:  # within a few octaves of each other: 57344 beside 2^-16 would leave nothing but the largest
        bits = (bits & 0x83) | (0x30 + (bits & 0x0C))
    return bits.view(getattr(torch, dtype))


def _scales(torch, shape, gen):
    return torch.exp(torch.randn(shape, generator=gen, device="cuda")) * 2.0**-8


def _spread(scales, n):
    """One scale for each of n values."""
    return scales.repeat_interleave(128, -1)[..., :n]


def _want(torch, a, a_scales, b, b_scales):
    k, n = b.shape
    a64 = a.double() * _spread(a_scales.double(), k)
    fb = b_scales.double().repeat_interleave(128, 0)[:k]
    b64 = b.double() * (fb if fb.shape[1] == n else _spread(fb, n))
    return a64 @ b64, a64.abs() @ b64.abs()


def _close(torch, c, want, size, k):
    kind = str(c.dtype).split(".")[1]
    slack = (k + 2 * ((k + 127) // 128)) * 2.0**-23 * size
    off = (c.double() - want).abs()
    bound = slack + HALF[kind] * (want.abs() + slack) + LEAST[kind]
    assert bool((off <= bound).all()), float((off / bound).max())


def _framed(torch, t, pad, fill):
    """The same matrix inside a larger one, whose other values are `fill`: lines further apart, and more lines behind the last."""
    by_row = t.stride(-1) == 1
    s = t if by_row else t.transpose(-1, -2)
    frame = torch.full((*s.shape[:-2], s.shape[-2] + 3, s.shape[-1] + pad), fill, dtype=torch.uint8, device="cuda")
    frame[..., : s.shape[-2], : s.shape[-1]] = s.view(torch.uint8)
    s = frame[..., : s.shape[-2], : s.shape[-1]].view(t.dtype)
    return s if by_row else s.transpose(-1, -2)


def _operands(torch, m, n, k, a_type="float8_e4m3fn", b_type="float8_e4m3fn", a_t=False, b_t=False, by_column=False, experts=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + m + 7 * n + 13 * k)
    blocks, lead = (k + 127) // 128, () if experts is None else (experts,)
    a = _codes(torch, (k, m) if a_t else (m, k), a_type, gen)
    b = _codes(torch, (*lead, n, k) if b_t else (*lead, k, n), b_type, gen)
    return (a.t() if a_t else a, _scales(torch, (m, blocks), gen), b.transpose(-1, -2) if b_t else b,
            _scales(torch, (*lead, blocks, n if by_column else (n + 127) // 128), gen))


def _run(torch, capi, form, m, n, k, out="bfloat16", framed=0, **kw):
    a, a_scales, b, b_scales = _operands(torch, m, n, k, **kw)
    want, size = _want(torch, a, a_scales, b, b_scales)
    if framed:
        a, b = _framed(torch, a, framed, 0x7F), _framed(torch, b, framed, 0x7F)  # NaN in both types
    c = torch.full((m + 2, n), 7.0, dtype=getattr(torch, out), device="cuda")
    with Options(capi, form):
        assert capi.block_gemm(a, a_scales, b, b_scales, out=c[1 : m + 1] if n % 32 == 0 else c[:m]) is not None
    torch.cuda.synchronize()
    assert capi.last_status()[0] == 0
    got, rest = (c[1 : m + 1], c[[0, m + 1]]) if n % 32 == 0 else (c[:m], c[m:])
    assert bool((rest == 7.0).all())
    _close(torch, got, want, size, k)
    return got


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (1, 128, 128), (7, 48, 144), (33, 272, 384), (128, 144, 1040), (129, 400, 2304), (257, 272, 512), (300, 1040, 640)])
def test_sizes(capi, cuda, m, n, k, form):
    _run(cuda, capi, form, m, n, k)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("a_t,b_t", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("m,n,k", [(16, 16, 16), (48, 272, 400), (144, 208, 1152), (272, 528, 784)])
def test_orders(capi, cuda, m, n, k, a_t, b_t, form):
    _run(cuda, capi, form, m, n, k, a_t=a_t, b_t=b_t)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("a_t,b_t", [(True, False), (False, False), (False, True)])
@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(16, 16, 48), (144, 400, 1030 // 16 * 16), (528, 272, 384)])
def test_scales_by_column(capi, cuda, m, n, k, out, a_t, b_t, form):
    _run(cuda, capi, form, m, n, k, out=out, a_t=a_t, b_t=b_t, by_column=True)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("a_type,b_type", [("float8_e5m2", "float8_e4m3fn"), ("float8_e4m3fn", "float8_e5m2"), ("float8_e5m2", "float8_e5m2")])
def test_types(capi, cuda, a_type, b_type, out, form):
    _run(cuda, capi, form, 150, 336, 656, out=out, a_type=a_type, b_type=b_type)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("a_t,b_t", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("m,n,k", [(48, 160, 208), (272, 288, 528)])
def test_lines_apart_and_what_lies_between_them(capi, cuda, m, n, k, a_t, b_t, form):
    _run(cuda, capi, form, m, n, k, a_t=a_t, b_t=b_t, framed=48)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1000, 2320, 256), (2500, 784, 1168)])
def test_several_rounds_of_tiles(capi, cuda, m, n, k, form):
    _run(cuda, capi, form, m, n, k)
    _run(cuda, capi, form, m // 16 * 16, n, k, a_t=True, by_column=True, out="float32")


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_scales_of_any_distance(capi, cuda, form):
    torch = cuda
    m, n, k = 200, 384, 1280
    a, a_scales, b, b_scales = _operands(torch, m, n, k)
    with Options(capi, form):
        want = capi.block_gemm(a, a_scales, b, b_scales)
        wide = torch.zeros((m, 37), device="cuda")
        wide[:, 3:13] = a_scales
        shifted = torch.zeros((12, 5), device="cuda")
        shifted[1:11, 2:] = b_scales
        for xs in (wide[:, 3:13], a_scales.t().contiguous().t()):
            for bs in (shifted[1:11, 2:], b_scales.t().contiguous().t()):
                assert torch.equal(capi.block_gemm(a, xs, b, bs), want)
        one = a_scales[:1, :1]  # one scale for everything, and one for each row
        assert torch.equal(capi.block_gemm(a, one.expand(m, 10), b, b_scales), capi.block_gemm(a, one.repeat(m, 10), b, b_scales))
        assert torch.equal(capi.block_gemm(a, a_scales[:, :1].expand(m, 10), b, b_scales[:, :1].expand(10, 3)),
                           capi.block_gemm(a, a_scales[:, :1].repeat(1, 10), b, b_scales[:, :1].repeat(1, 3)))


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_rows_that_are_not_finite_stay_alone(capi, cuda, form):
    torch = cuda
    m, n, k = 70, 272, 400
    a, a_scales, b, b_scales = _operands(torch, m, n, k)
    with Options(capi, form):
        clean = capi.block_gemm(a, a_scales, b, b_scales)
        a.view(torch.uint8)[3, 250] = 0x7F
        a_scales[40, 1] = float("nan")
        a_scales[41, 2] = float("inf")
        a_scales[42, :] = 0.0
        got = capi.block_gemm(a, a_scales, b, b_scales)
    bad = [3, 40]
    rest = [i for i in range(m) if i not in (3, 40, 41, 42)]
    assert bool(got[bad].isnan().all()) and not bool(torch.isfinite(got[41]).any()) and bool((got[42] == 0).all())
    assert torch.equal(got[rest], clean[rest])


def test_the_same_result_every_time(capi, cuda):
    torch = cuda
    for shape in ((16, 4096, 7168), (300, 1024, 4096), (1024, 2304, 1024)):
        operands = _operands(torch, *shape)
        want = capi.block_gemm(*operands)
        for _ in range(10):
            assert torch.equal(capi.block_gemm(*operands), want)


def test_more_values_than_32_bits_count(capi, cuda):
    torch = cuda
    m, n, k = 33000, 65536, 256  # 2^31 results and some
    a, a_scales, b, b_scales = _operands(torch, m, n, k)
    c = capi.block_gemm(a, a_scales, b, b_scales)
    rows = torch.tensor([0, 255, 32767, 32768, 32999], device="cuda")
    want, size = _want(torch, a[rows], a_scales[rows], b, b_scales)
    _close(torch, c[rows], want, size, k)
    del c, want, size
    m, n, k = 270000, 48, 8192  # 2^31 codes and some
    a, a_scales, b, b_scales = _operands(torch, m, n, k)
    c = capi.block_gemm(a, a_scales, b, b_scales)
    rows = torch.tensor([0, 262143, 262144, 269999], device="cuda")
    want, size = _want(torch, a[rows], a_scales[rows], b, b_scales)
    _close(torch, c[rows], want, size, k)


def _grouped(torch, capi, form, m, n, k, offsets, out="bfloat16", framed=0, **kw):
    experts = len(offsets) - 1
    a, a_scales, b, b_scales = _operands(torch, m, n, k, experts=experts, **kw)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    want = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    mine = torch.zeros(m, dtype=torch.bool, device="cuda")
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi > lo:
            want[lo:hi], size[lo:hi] = _want(torch, a[lo:hi], a_scales[lo:hi], b[e], b_scales[e])
            mine[lo:hi] = True
    a.view(torch.uint8)[~mine] = 0x7F  # rows that nobody has may hold anything
    a_scales[~mine] = float("nan")
    if framed:
        a, b = _framed(torch, a, framed, 0x7F), _framed(torch, b, framed, 0x7F)
    c = torch.full((m, n), 7.0, dtype=getattr(torch, out), device="cuda")
    with Options(capi, form):
        assert capi.block_grouped_gemm(a, a_scales, b, b_scales, off, out=c) is c
    torch.cuda.synchronize()
    assert capi.last_status()[0] == 0
    assert bool((c[~mine] == 7.0).all())
    _close(torch, c[mine], want[mine], size[mine], k)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("m,n,k,offsets", [
    (1, 16, 16, [0, 1]),
    (9, 272, 272, [0, 1, 1, 4, 9]),                          # one row, none, a few
    (400, 528, 384, [3, 3, 35, 68, 197, 325, 325, 390]),     # 32, 33, 129, 128 rows; rows in front and behind that nobody has
    (700, 2320, 512, [0, 0, 0, 700]),                        # one expert has them all; the last tiles are ragged
    (130, 64, 1152, [0, 97, 130, 130]),
    (1300, 784, 656, [0, 128, 129, 385, 642, 1300]),         # an end on each side of a pair's halves
])
def test_rows_of_each_expert(capi, cuda, m, n, k, offsets, form):
    _grouped(cuda, capi, form, m, n, k, offsets)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("out", ["float32", "float16"])
@pytest.mark.parametrize("m,n,k,offsets", [(300, 304, 656, [0, 20, 20, 160, 300]), (16, 1040, 1024, list(range(0, 17, 2)))])
def test_experts_transposed(capi, cuda, m, n, k, offsets, out, form):
    _grouped(cuda, capi, form, m, n, k, offsets, out=out, b_t=True, a_type="float8_e5m2")
    _grouped(cuda, capi, form, m, n, k, offsets, out=out, b_t=True, framed=16)
    _grouped(cuda, capi, form, m, n, k, offsets, out=out, framed=32)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_many_experts(capi, cuda, form):
    counts = [(i * 7919) % 5 if i % 3 == 0 else 0 for i in range(200)] + [150]
    offsets = [0]
    for v in counts:
        offsets.append(offsets[-1] + v)
    _grouped(cuda, capi, form, offsets[-1] + 5, 336, 144, offsets)
    counts = [(i * 7919) % 41 if i % 97 == 5 else 0 for i in range(1024)]
    offsets = [0]
    for v in counts:
        offsets.append(offsets[-1] + v)
    _grouped(cuda, capi, form, offsets[-1], 32, 128, offsets)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_offsets_that_do_not_ascend_stay_inside(capi, cuda, form):
    torch = cuda
    m, n, k, experts = 200, 64, 256, 4
    a, a_scales, b, b_scales = _operands(torch, m, n, k, experts=experts)
    guard = torch.full((3 * m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    with Options(capi, form):
        for offsets in ([0, 150, 50, 300, 200], [-5, 10, 2**31 - 1, 20, 10], [300, 200, 100, 0, -1]):
            off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
            capi.block_grouped_gemm(a, a_scales, b, b_scales, off, out=guard[m : 2 * m])
            torch.cuda.synchronize()
            assert bool((guard[:m] == 7.0).all()) and bool((guard[2 * m :] == 7.0).all())
    assert capi.last_status()[0] == 0


def test_uint8_codes_follow_the_options(capi, cuda):
    torch = cuda
    a, a_scales, b, b_scales = _operands(torch, 40, 272, 256, a_type="float8_e5m2")
    want = capi.block_gemm(a, a_scales, b, b_scales)
    with Options(capi, dict(a_dtype=1)):
        assert torch.equal(capi.block_gemm(a.view(torch.uint8), a_scales, b.view(torch.uint8), b_scales), want)
    assert not torch.equal(capi.block_gemm(a.view(torch.uint8), a_scales, b, b_scales), want)
    for dtype in (torch.float16, torch.float32, torch.bfloat16):
        assert capi.block_gemm(a, a_scales, b, b_scales, out_dtype=dtype).dtype == dtype


def test_streams_graphs_and_threads(capi, cuda):
    torch = cuda
    shapes = [(16, 1024, 2048), (300, 784, 1040), (2048, 2304, 512)]
    operands = [_operands(torch, *s, seed=i) for i, s in enumerate(shapes)]
    off = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    grouped = (*_operands(torch, 300, 528, 640, experts=2), off)
    calls = [lambda o=o: capi.block_gemm(*o) for o in operands] + [lambda: capi.block_grouped_gemm(*grouped)]
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(5):  # side by side on the GPU
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(len(calls)) for x in got[i])
    graphs = []
    for _ in range(2):  # two graphs of the same calls, replayed on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [call() for call in calls]
        graphs.append((graph, out))
    for graph, out in graphs:
        for t in out:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        assert torch.equal(calls[0](), want[0])
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for _, out in graphs for x, w in zip(out, want))
    out = [None] * 12

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out[i] = calls[i % len(calls)]()
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(out))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(out[i], want[i % len(calls)]) for i in range(len(out)))
    assert capi.last_status()[0] == 0


def test_refusals(capi, cuda):
    torch = cuda
    a, a_scales, b, b_scales = _operands(torch, 32, 64, 256)
    ok = dict(a=a, a_scales=a_scales, b=b, b_scales=b_scales)
    out = torch.zeros((32, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (dict(a=a.cpu()), dict(a=a[0]), dict(a=a.float()), dict(a=a[:, :128]), dict(a_scales=a_scales[:16]), dict(a_scales=a_scales.half()),
                dict(b=b[:128]), dict(b_scales=b_scales[:1]), dict(b_scales=b_scales.double()), dict(out=out[:16]), dict(out=out.t()),
                dict(out=out.int()), dict(out_dtype=torch.int32), dict(a=a[::2, ::2], a_scales=a_scales[:16, :1], b=b[:128], b_scales=b_scales[:1]),
                dict(a="a")):
        with pytest.raises((ValueError, TypeError)):
            capi.block_gemm(**{**ok, **bad})
    packed = torch.zeros((32, 264), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    odd = torch.zeros(32 * 64 + 8, dtype=torch.bfloat16, device="cuda")[8:].view(32, 64)
    three = a.t().contiguous().t()[:24]
    by_column = torch.ones((2, 65), device="cuda")[:, 1:]
    for bad in (dict(a=packed[:, :256]), dict(a=a[:, :40], a_scales=a_scales[:, :1], b=b[:40], b_scales=b_scales[:1]), dict(b=b[:, :24]),
                dict(out=odd), dict(a=three, a_scales=a_scales[:24]), dict(b_scales=by_column)):
        with pytest.raises((ValueError, capi.CatccosError)):
            capi.block_gemm(**{**ok, **bad})
    # c in an operand's memory
    both = torch.zeros((64, 256), dtype=torch.uint8, device="cuda")
    with pytest.raises(capi.CatccosError):
        capi.block_gemm(both[:32].view(torch.float8_e4m3fn), a_scales, b, b_scales, out=both.view(torch.bfloat16).view(-1)[: 32 * 64].view(32, 64))
    e, es, w, ws = _operands(torch, 32, 64, 256, experts=3)
    off = torch.tensor([0, 4, 9, 32], dtype=torch.int32, device="cuda")
    ok = dict(a=e, a_scales=es, b=w, b_scales=ws, offsets=off)
    for bad in (dict(offsets=off[:3]), dict(offsets=off.long()), dict(b=w[:2]), dict(b_scales=ws[:, :1]), dict(b=w[0]), dict(b_scales=torch.ones((3, 2, 64), device="cuda"))):
        with pytest.raises(ValueError):
            capi.block_grouped_gemm(**{**ok, **bad})
    with pytest.raises(capi.CatccosError):
        capi.block_grouped_gemm(**{**ok, "a": e.t().contiguous().t()})
    with pytest.raises(capi.CatccosError):
        capi.block_grouped_gemm(**{**ok, "b": w[:1].expand(3, 256, 64)})  # one matrix three times: matrices that overlap
    assert capi.block_gemm(a[:0], a_scales[:0], b, b_scales).shape == (0, 64)
    assert capi.block_grouped_gemm(e[:0], es[:0], w, ws, off * 0).shape == (0, 64)
