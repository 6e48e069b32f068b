"""GPU tests of the experts' products: every expert's rows against the product of the dequantised operands in 64 bits, and, bit for
bit, against the single-CTA GEMM on the expert's operands (the same tile, the same order of the sums).

Against 64 bits a result may be off by K * 2^-23 of the sum of its products' magnitudes (K steps of an fp32 accumulator that
truncates) and half a step of its type."""
import threading

import pytest

pytestmark = pytest.mark.gpu

SINGLE_CTA = dict(cta_pair=2, small_tile=2, split_k=1)


def _operands(torch, capi, rows, n, k, experts, a_dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x[:, :: max(1, k // 7)] *= 20
    capi.set_option("a_dtype", a_dtype)
    a, a_scales = capi.mx_quant(x.to(torch.bfloat16))
    capi.set_option("a_dtype", 0)
    w = torch.randn((experts * n, k), generator=gen, device="cuda") * 0.05
    q, s = capi.mx_quant(w.to(torch.bfloat16))
    b = q.view(experts, n, k).transpose(1, 2).contiguous()
    b_scales = s.view(experts, n, k // 64, 2).permute(0, 2, 1, 3).contiguous()
    return a, a_scales, b, b_scales


def _packed(torch, capi, a, a_scales):
    rows, k = a.shape
    packed = torch.full((rows, capi.packed_row_bytes(k)), 0xAB, dtype=torch.uint8, device="cuda")
    packed[:, :k], packed[:, k : k + k // 32] = a, a_scales
    return packed[:, :k], packed[:, k : k + k // 32]


def _dequantised(torch, a, a_scales, a_dtype):
    f8 = torch.float8_e4m3fn if a_dtype == 0 else torch.float8_e5m2
    return a.view(f8).double() * torch.exp2(a_scales.double() - 127).repeat_interleave(32, 1)


def _set(capi, options):
    for key, value in options.items():
        capi.set_option(key, value)


def _run(torch, capi, rows, n, k, offsets, a_dtype=0, out="bfloat16", packed=False, block_n=0, cta_pair=0, seed=0):
    experts = len(offsets) - 1
    a, a_scales, b, b_scales = _operands(torch, capi, rows, n, k, experts, a_dtype, seed + rows + n + k)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    dtype = getattr(torch, out)
    c = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
    single = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
    options = dict(a_dtype=a_dtype, c_dtype=1 if out == "float16" else 0, block_n=block_n, cta_pair=cta_pair)
    _set(capi, options)
    try:
        assert capi.mx_grouped_gemm(*(_packed(torch, capi, a, a_scales) if packed else (a, a_scales)), b, b_scales, off, out=c) is c
        _set(capi, SINGLE_CTA)
        for e in range(experts):
            lo, hi = offsets[e], offsets[e + 1]
            if hi > lo:
                capi.mx_gemm(a[lo:hi].contiguous(), a_scales[lo:hi].contiguous(), b[e], b_scales[e], out=single[lo:hi])
    finally:
        _set(capi, {key: 0 for key in (*options, *SINGLE_CTA)})
    assert capi.last_status()[0] == 0
    assert torch.equal(c, single)  # rows of no expert keep their sevens on both sides
    half = 2.0**-8 if out == "bfloat16" else 2.0**-11
    a64 = _dequantised(torch, a, a_scales, a_dtype)
    for e in range(experts):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            w64 = b[e].view(torch.float8_e4m3fn).double() * torch.exp2(b_scales[e].double() - 127).permute(0, 2, 1).reshape(k // 32, n).repeat_interleave(32, 0)
            want, size = a64[lo:hi] @ w64, a64[lo:hi].abs() @ w64.abs()
            slack = k * 2.0**-23 * size
            assert bool(((c[lo:hi].double() - want).abs() <= slack + half * (want.abs() + slack) + 2.0**-25).all()), e


@pytest.mark.parametrize("block_n,cta_pair", [(64, 2), (128, 2), (256, 2), (0, 1)])
@pytest.mark.parametrize("rows,n,k,offsets", [
    (1, 16, 128, [0, 1]),
    (9, 272, 256, [0, 1, 1, 4, 9]),                          # one row, none, a few
    (400, 528, 384, [3, 3, 35, 68, 197, 325, 325, 390]),     # 32, 33, 129, 128 rows; rows in front and behind that nobody has
    (700, 2320, 512, [0, 0, 0, 700]),                        # one expert has them all; the last tiles are ragged
    (130, 64, 1152, [0, 97, 130, 130]),
    (1300, 784, 640, [0, 128, 129, 385, 642, 1300]),         # an end on each side of a pair's halves
])
def test_rows_of_each_expert(capi, cuda, rows, n, k, offsets, block_n, cta_pair):
    _run(cuda, capi, rows, n, k, offsets, block_n=block_n, cta_pair=cta_pair)


@pytest.mark.parametrize("cta_pair", [1, 2])
@pytest.mark.parametrize("a_dtype,out,packed", [(0, "bfloat16", True), (1, "float16", False), (1, "bfloat16", True), (0, "float16", True)])
@pytest.mark.parametrize("rows,n,k,offsets", [(300, 304, 640, [0, 20, 20, 160, 300]), (16, 1040, 1024, list(range(0, 17, 2)))])
def test_types_and_packed_rows(capi, cuda, rows, n, k, offsets, a_dtype, out, packed, cta_pair):
    _run(cuda, capi, rows, n, k, offsets, a_dtype, out, packed, cta_pair=cta_pair)


@pytest.mark.parametrize("cta_pair", [1, 2])
def test_many_experts(capi, cuda, cta_pair):
    # more experts than a warp counts at a time, most of them without rows; several rounds of units a CTA
    counts = [(i * 7919) % 5 if i % 3 == 0 else 0 for i in range(200)] + [150]
    offsets = [0]
    for v in counts:
        offsets.append(offsets[-1] + v)
    _run(cuda, capi, offsets[-1] + 5, 336, 128, offsets, cta_pair=cta_pair)


@pytest.mark.parametrize("cta_pair", [1, 2])
def test_as_many_experts_as_there_may_be(capi, cuda, cta_pair):
    counts = [(i * 7919) % 41 if i % 97 == 5 else 0 for i in range(1024)]
    offsets = [0]
    for v in counts:
        offsets.append(offsets[-1] + v)
    _run(cuda, capi, offsets[-1], 32, 128, offsets, cta_pair=cta_pair)


@pytest.mark.parametrize("block_n,cta_pair", [(0, 0), (64, 2), (128, 2), (0, 1)])
def test_several_rounds_of_tiles(capi, cuda, block_n, cta_pair):
    _run(cuda, capi, 2500, 2304, 256, [0, 100, 612, 613, 1500, 2500], block_n=block_n, cta_pair=cta_pair)


@pytest.mark.parametrize("block_n,cta_pair", [(64, 2), (128, 2), (256, 2), (0, 1)])
def test_long_rows_of_few_tokens(capi, cuda, block_n, cta_pair):
    # more K tiles than the ring has stages, several times over
    _run(cuda, capi, 21, 784, 7168, [0, 1, 21], block_n=block_n, cta_pair=cta_pair)


@pytest.mark.parametrize("cta_pair", [0, 1, 2])
@pytest.mark.parametrize("live", [0, 1, 500, 4096])
def test_rows_that_nobody_has(capi, cuda, live, cta_pair):
    # a rank with some of the experts hands over room for every route and uses a part: the rest stays as it is
    offsets = [0, live // 8, live // 8, live // 2, live // 2 + live % 3, live, live, live, live]
    _run(cuda, capi, 4096, 1056, 512, offsets, cta_pair=cta_pair)


def test_one_row_of_a_wider_tensor(capi, cuda):
    torch = cuda
    a, a_scales, b, b_scales = _operands(torch, capi, 1, 32, 128, 2, 0, 1)
    off = torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    want = capi.mx_grouped_gemm(a, a_scales, b, b_scales, off)
    got = capi.mx_grouped_gemm(*_packed(torch, capi, a, a_scales), b, b_scales, off)
    assert torch.equal(got, want)


@pytest.mark.parametrize("cta_pair", [1, 2])
def test_offsets_that_are_none(capi, cuda, cta_pair):
    # cut to the matrix in the kernel: unspecified results, no access outside; nothing at all is written where none is left
    torch = cuda
    a, a_scales, b, b_scales = _operands(torch, capi, 40, 64, 128, 3, 0, 2)
    guard = torch.full((42, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    c = guard[:40]
    capi.set_option("cta_pair", cta_pair)
    for bad in ([-5, -3, -1, -1], [40, 40, 40, 2**31 - 1], [50, 60, 70, 80]):
        capi.mx_grouped_gemm(a, a_scales, b, b_scales, torch.tensor(bad, dtype=torch.int32, device="cuda"), out=c)
        assert bool((guard == 7).all())
    for bad in ([0, 10, 5, 20], [-(2**31), 2**31 - 1, 2**31 - 1, 2**31 - 1], [30, 10, 2**31 - 1, 5]):
        capi.mx_grouped_gemm(a, a_scales, b, b_scales, torch.tensor(bad, dtype=torch.int32, device="cuda"), out=c)
    capi.set_option("cta_pair", 0)
    assert bool((guard[40:] == 7).all())
    assert capi.last_status()[0] == 0


def test_calls_of_several_threads(capi, cuda):
    # more operands than a table of tensor maps holds, other ones in every thread; each result as one thread alone gets it
    torch = cuda
    threads, sets, rounds = 8, 8, 40
    work = []
    for t in range(threads):
        for i in range(sets):
            rows, n, k = 33 + 40 * i + t, 64 + 16 * t, 128 * (1 + (i + t) % 3)
            a, a_scales, b, b_scales = _operands(torch, capi, rows, n, k, 2, 0, t * sets + i)
            offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
            operands = (a, a_scales, b, b_scales, offsets)
            work.append((operands, capi.mx_grouped_gemm(*operands)))
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(threads), [None] * threads

    def run(t):
        stream, bad = torch.cuda.Stream(), 0
        with torch.cuda.stream(stream):
            start.wait()
            for r in range(rounds):
                got = [capi.mx_grouped_gemm(*operands) for operands, _ in work[t * sets : (t + 1) * sets]]
                bad += sum(not torch.equal(g, want) for g, (_, want) in zip(got, work[t * sets : (t + 1) * sets]))
            stream.synchronize()
        wrong[t] = bad

    running = [threading.Thread(target=run, args=(t,)) for t in range(threads)]
    for thread in running:
        thread.start()
    for thread in running:
        thread.join()
    assert wrong == [0] * threads and capi.last_status()[0] == 0


def test_refusals(capi, cuda):
    torch = cuda
    a, a_scales, b, b_scales = _operands(torch, capi, 8, 64, 128, 2, 0, 3)
    off = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
    for bad in ((a.t(), a_scales, b, b_scales, off), (a, a_scales[:4], b, b_scales, off), (a, a_scales, b[:1], b_scales, off),
                (a, a_scales, b, b_scales.transpose(1, 2), off), (a, a_scales, b, b_scales, off[:2]), (a, a_scales, b, b_scales, off.long()),
                (a, a_scales, b, b_scales.cpu(), off), (a.float(), a_scales, b, b_scales, off)):
        with pytest.raises(ValueError):
            capi.mx_grouped_gemm(*bad, out=torch.empty((8, 64), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        capi.mx_grouped_gemm(a, a_scales, b, b_scales, off, out=torch.empty((8, 64), device="cuda"))
    wide = torch.zeros((8, 136), dtype=torch.uint8, device="cuda")
    for x, xs in ((wide[:, :128], a_scales), (a, torch.zeros((8, 6), dtype=torch.uint8, device="cuda")[:, :4])):
        with pytest.raises(capi.CatccosError) as e:  # rows that are 136 bytes, or scales that are 6 bytes, apart
            capi.mx_grouped_gemm(x, xs, b, b_scales, off)
        assert e.value.code == -1
    for option in ("a_dtype", "b_dtype"):
        capi.set_option(option, 2)
        try:
            with pytest.raises(capi.CatccosError):
                capi.mx_grouped_gemm(a, a_scales, b, b_scales, off)
        finally:
            capi.set_option(option, 0)
    assert capi.mx_grouped_gemm(a[:0], a_scales[:0], b, b_scales, off * 0).shape == (0, 64)
