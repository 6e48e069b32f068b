"""GPU tests of the products of a few tokens with FP4 weights, against the dequantised weights' products in 64 bits.

The tokens' values go in as f16 after a power of two, off by at most 2^-40 of the largest of their 64; products are exact in fp32;
two sums of 16 in the tensor core, 2 K / 64 sums of those, and 8 + 8 partial sums, each step off by 2^-23 of what is added up; then
half a step of the result's type."""
import pytest

pytestmark = pytest.mark.gpu

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _weights(torch, gen, lead, k, n, scales=(118, 130)):
    w = torch.randint(0, 256, (*lead, k, n // 2), generator=gen, device="cuda", dtype=torch.uint8)
    s = torch.randint(scales[0], scales[1], (*lead, k // 64, n, 2), generator=gen, device="cuda", dtype=torch.uint8)
    return w, s


def _dequantised(torch, w, s):
    value = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    even, odd = value[(w & 15).long()], value[(w >> 4).long()]
    full = torch.stack((even, odd), dim=-1).flatten(-2)
    scale = torch.exp2(s.double() - 127).transpose(-1, -2).flatten(-3, -2)
    return full * scale.repeat_interleave(32, dim=-2)


def _compare(torch, out, x, w64, k):
    want, size = x.double() @ w64, x.double().abs() @ w64.abs()
    half = (2.0**-8, 2.0**-134) if out.dtype == torch.bfloat16 else (2.0**-11, 2.0**-25)
    slack = (32 + 2 * k // 64 + 16) * 2.0**-23 * size + 2.0**-40 * x.double().abs().amax() * w64.abs().sum(0)
    assert bool(((out.double() - want).abs() <= slack + half[0] * (want.abs() + slack) + half[1]).all())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rows,n,k", [(1, 16, 64), (1, 4096, 7168), (2, 48, 192), (3, 144, 128), (4, 2304, 1024), (5, 16, 8256), (8, 272, 640),
                                      (9, 128, 4096), (17, 528, 576), (1, 16, 65536)])
def test_dense(capi, cuda, rows, n, k, f16):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows + n + k)
    w, s = _weights(torch, gen, (), k, n, (113, 121))
    x = torch.randn((rows, k), generator=gen, device="cuda").to(torch.bfloat16)
    x[:, ::50] *= 100
    capi.set_option("c_dtype", 1 if f16 else 0)
    try:
        out = capi.mx_fp4_matvec(x, w, s, out_dtype=torch.float16 if f16 else torch.bfloat16)
        again = capi.mx_fp4_matvec(x, w, s, out=torch.empty_like(out))
    finally:
        capi.set_option("c_dtype", 0)
    assert out.shape == (rows, n) and torch.equal(out, again)
    _compare(torch, out, x, _dequantised(torch, w, s), k)


@pytest.mark.parametrize("tokens,top_k,experts,n,k", [(1, 1, 1, 16, 64), (1, 8, 32, 2304, 1024), (4, 6, 8, 144, 320), (33, 2, 3, 32, 128)])
@pytest.mark.parametrize("per_route", [False, True])
def test_experts(capi, cuda, tokens, top_k, experts, n, k, per_route):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(tokens + n + k)
    w, s = _weights(torch, gen, (experts,), k, n)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen, device="cuda", dtype=torch.int32)  # an expert twice, too
    if tokens > 1:
        ids[0, 0], ids[1, top_k - 1], ids[2, 0] = -1, experts, -(2**31)
    x = torch.randn((tokens * top_k if per_route else tokens, k), generator=gen, device="cuda").to(torch.bfloat16)
    out = capi.mx_fp4_matvec(x, w, s, ids=ids)
    w64 = _dequantised(torch, w, s)
    for r, e in enumerate(ids.flatten().tolist()):
        if 0 <= e < experts:
            _compare(torch, out[r : r + 1], x[r : r + 1] if per_route else x[r // top_k : r // top_k + 1], w64[e], k)
        else:
            assert bool((out[r] == 0).all())


@pytest.mark.parametrize("routes,experts,top_k,n,k", [(1023, 1, 1, 16, 64), (1025, 5, 1, 48, 128), (1500, 7, 4, 144, 64), (2049, 700, 1, 16, 128),
                                                      (65535, 3, 1, 16, 64)])
@pytest.mark.parametrize("kind", ["random", "one expert", "mostly dropped"])
def test_more_routes_than_a_window(capi, cuda, routes, experts, top_k, n, k, kind):
    # rows that share a weight find one another among 1024 routes: here they go on in the next ones
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(routes + experts)
    w, s = _weights(torch, gen, (experts,), k, n)
    ids = torch.randint(-1, experts + 1, (routes,), generator=gen, device="cuda", dtype=torch.int32)
    if kind == "one expert":
        ids[:] = experts - 1
    elif kind == "mostly dropped":
        ids[torch.rand(routes, generator=gen, device="cuda") < 7 / 8] = -1
    x = torch.randn((routes // top_k, k), generator=gen, device="cuda").to(torch.bfloat16)
    guard = torch.full((routes + 1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    out = capi.mx_fp4_matvec(x, w, s, ids=ids, out=guard[:routes])
    w64, x_row = _dequantised(torch, w, s), torch.arange(routes, device="cuda") // top_k
    for e in range(experts):
        rows = (ids == e).nonzero().flatten()
        if rows.numel():
            _compare(torch, out[rows], x[x_row[rows]], w64[e], k)
    assert bool((out[(ids < 0) | (ids >= experts)] == 0).all()) and bool((guard[routes:] == 7).all())


def test_every_code_at_every_place(capi, cuda):
    # weights read back one k at a time: unit vectors give the weight itself
    torch = cuda
    k, n = 128, 272
    gen = torch.Generator(device="cuda").manual_seed(4)
    w, s = _weights(torch, gen, (), k, n, (100, 150))
    x = torch.eye(k, dtype=torch.bfloat16, device="cuda")
    out = capi.mx_fp4_matvec(x, w, s)
    assert torch.equal(out.double(), _dequantised(torch, w, s))


@pytest.mark.parametrize("magnitude", [2.0**-126, 2.0**-100, 1.0, 2.0**60])
def test_magnitudes(capi, cuda, magnitude):
    # one power of two for 64 values of a token: rows, and stretches of one row, of very different size
    torch = cuda
    k, n = 512, 64
    gen = torch.Generator(device="cuda").manual_seed(6)
    w, s = _weights(torch, gen, (), k, n, (120, 130))
    x = torch.randn((3, k), generator=gen, device="cuda")
    x[1] *= 2.0**-20
    x[2] = 0
    x[0, :64] *= 2.0**-30
    x = (x.double() * magnitude).to(torch.bfloat16)
    out = capi.mx_fp4_matvec(x, w, s)
    w64 = _dequantised(torch, w, s)
    for r in range(3):
        _compare(torch, out[r : r + 1], x[r : r + 1], w64, k)
    assert bool((out[2] == 0).all())


def test_scales_at_their_ends(capi, cuda):
    torch = cuda
    k, n = 128, 32
    w = torch.full((k, n // 2), 0x22, dtype=torch.uint8, device="cuda")  # ones
    s = torch.full((2, n, 2), 127, dtype=torch.uint8, device="cuda")
    s[:, 0], s[:, 1], s[1, 2, 1] = 0, 254, 255
    x = torch.zeros((2, k), dtype=torch.bfloat16, device="cuda")
    x[0, 0], x[1, 0] = 2.0**100, 2.0**-100
    out = capi.mx_fp4_matvec(x, w, s).double()
    assert out[0, 0] == 2.0**-27 and out[0, 1] == float("inf") and out[0, 3] == 2.0**100
    assert out[1, 0] == 0 and out[1, 1] == 2.0**27 and out[1, 3] == 2.0**-100
    assert bool(torch.isnan(out[:, 2]).all())  # a scale of 0xFF is NaN, whatever it scales


@pytest.mark.parametrize("rows", [1, 5])  # one and two sets of four tokens
def test_large_values_with_small_scales(capi, cuda, rows):
    # the activations' power of two is undone before the weights' scale is applied: what lies between stays in range
    torch = cuda
    k, n = 256, 32
    w = torch.zeros((k, n // 2), dtype=torch.uint8, device="cuda")
    w[0], w[64] = 0x76, 0xE2  # 4 and 6; 1 and -4
    s = torch.full((k // 64, n, 2), 107, dtype=torch.uint8, device="cuda")
    s[:, 2:4], s[:, 4] = 0, 254
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.tensor([2.0**127, 2.0**115, 2.0**113, 2.0**-100, 1.0][:rows])
    x[:, 64] = torch.tensor([-(2.0**126), 2.0**127, 1.0, 2.0**127, 2.0**-133][:rows])
    want = x.double() @ _dequantised(torch, w, s)
    got = capi.mx_fp4_matvec(x, w, s).double()
    inside = want.abs() < 2.0**127
    # two products, exact in the tensor core, and one sum of theirs in fp32: two roundings of 2^-24 and half a step of bf16
    assert bool(((got - want).abs() <= (2.0**-8 + 2.0**-22) * want.abs())[inside].all())
    assert bool(inside[:, :4].all()) and not bool(inside[:, 4].any())
    # column 4: a product of 2^129 and more is infinite in the fp32 sums; row 0 has one of either sign (2^256 - 2^253), and no sum
    w64 = _dequantised(torch, w, s)
    sums = (x[:, :1].double() * w64[0]).float() + (x[:, 64:65].double() * w64[64]).float()
    assert torch.equal(torch.nan_to_num(got[:, 4], nan=-1.0), torch.nan_to_num(sums[:, 4].double(), nan=-1.0))


def test_values_that_are_not_finite(capi, cuda):
    torch = cuda
    k, n = 192, 32
    inf = float("inf")
    w = torch.zeros((k, n // 2), dtype=torch.uint8, device="cuda")
    w[70] = 0x2A  # even columns -1, odd columns 1; zeros elsewhere
    w[71] = 0x22
    s = torch.full((3, n, 2), 127, dtype=torch.uint8, device="cuda")
    x = torch.ones((5, k), dtype=torch.bfloat16, device="cuda")
    x[1, 70] = inf
    x[2, 3] = inf  # meets zeros only
    x[3, 71] = float("nan")
    x[4, 70], x[4, 71] = 3e38, -inf
    out = capi.mx_fp4_matvec(x, w, s)
    assert bool((out[0, ::2] == 0).all()) and bool((out[0, 1::2] == 2).all())
    assert bool((out[1, ::2] == -inf).all()) and bool((out[1, 1::2] == inf).all())
    assert bool(torch.isnan(out[2]).all()) and bool(torch.isnan(out[3]).all())
    assert bool((out[4] == -inf).all())  # a large value beside an infinity stays finite


def test_refusals(capi, cuda):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(1)
    w, s = _weights(torch, gen, (2,), 128, 64)
    x = torch.zeros((2, 128), dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in ((x.float(), w[0], s[0]), (x, w, s), (x[:, :64], w[0], s[0]), (x, w[0], s[0, :1]), (x, w[0].cpu(), s[0]), (x.t(), w[0], s[0])):
        with pytest.raises(ValueError):
            capi.mx_fp4_matvec(*bad, out=torch.empty((2, 64), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        capi.mx_fp4_matvec(x, w, s, ids=ids.long())
    with pytest.raises(ValueError):
        capi.mx_fp4_matvec(x, w, s[:1], ids=ids)
    with pytest.raises(capi.CatccosError) as e:  # three routes of two rows
        capi.mx_fp4_matvec(x, w, s, ids=ids[:3])
    assert e.value.code == -1
    with pytest.raises(capi.CatccosError):
        capi.mx_fp4_matvec(x[:, :96].contiguous(), w[0, :96].contiguous(), s[0, :1].contiguous())
    assert capi.mx_fp4_matvec(x[:0], w[0], s[0]).shape == (0, 64)
    assert capi.mx_fp4_matvec(x, w, s, ids=ids[:0]).shape == (0, 64)
