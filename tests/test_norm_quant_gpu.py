"""GPU test of the norm that quantises: h = bf16(x + residual), y = h / sqrt(mean(h^2) + eps) * weight, codes and scales of y,
against the same formulas in 64 bits.

The kernel's y is off by at most (74 / 2 + 6) * 2^-24 of itself (74: the longest chain of additions in the sum of squares, whose
relative error the root halves; 6: the mean, eps, root, quotient and two products) = 2.6e-6, below DELTA.  Rounding is monotonic:
a code has to lie between those of y (1 - DELTA) and y (1 + DELTA), and a scale between those of the block's largest |y|."""
import pytest

pytestmark = pytest.mark.gpu

DELTA = 4e-6
EPS = 1e-6
EMAX = {0: 8, 1: 15}
MOST = {0: 448.0, 1: 57344.0}


def _reference(torch, x, residual, weight):
    h = x if residual is None else (x.float() + residual.float()).to(torch.bfloat16)
    d = h.double()
    return h, d / torch.sqrt((d * d).mean(dim=1, keepdim=True) + EPS) * weight.double()


def _exponent(torch, top, a_dtype):
    """The scale byte of a block whose largest magnitude is `top` (golden rule for tiny blocks)."""
    return torch.where(top < 1e-12, 127, torch.frexp(top)[1] - 1 - EMAX[a_dtype] + 127)


def _code_values(torch, y, byte, a_dtype):
    f8 = torch.float8_e4m3fn if a_dtype == 0 else torch.float8_e5m2
    scaled = y.unflatten(1, (-1, 32)) * torch.exp2(127.0 - byte.double()).unsqueeze(2)
    return scaled.flatten(1).clamp(-MOST[a_dtype], MOST[a_dtype]).to(f8).double()


def _check(torch, x, residual, weight, codes, scales, h_out, norm_out, a_dtype):
    h, y = _reference(torch, x, residual, weight)
    if h_out is not None:
        assert torch.equal(h_out, h)
    if norm_out is not None:
        # half a step of bf16 is 2^-8 of the value; below the smallest normal half of 2^-133
        assert bool(((norm_out.double() - y).abs() <= (2.0**-8 + DELTA) * y.abs() + 2.0**-134).all())
    top = y.unflatten(1, (-1, 32)).abs().amax(dim=2)
    got = scales.long()
    low, high = (_exponent(torch, top * f, a_dtype) for f in (1 - DELTA, 1 + DELTA))
    assert bool(((got >= torch.minimum(low, high)) & (got <= torch.maximum(low, high))).all())
    value = codes.view(torch.float8_e4m3fn if a_dtype == 0 else torch.float8_e5m2).double()
    tiny = (top < 1e-12).unsqueeze(2).expand(-1, -1, 32).flatten(1)
    assert bool((value[tiny] == 0).all())
    ends = [_code_values(torch, y * f, got, a_dtype) for f in (1 - DELTA, 1 + DELTA)]
    inside = (value >= torch.minimum(*ends)) & (value <= torch.maximum(*ends))
    assert bool((inside | tiny).all())


# one lane's half block to several passes; one warp to sixteen a row; rows that share a CTA; ragged last warps
SIZES = [(1, 32), (3, 64), (300, 96), (5, 512), (9, 544), (37, 1056), (16, 7168), (2, 8192), (3, 8224), (2, 16416), (1, 32768), (509, 2080)]


@pytest.mark.parametrize("a_dtype", [0, 1])
@pytest.mark.parametrize("rows,n", SIZES)
def test_against_64_bits(capi, cuda, rows, n, a_dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows * 65536 + n + a_dtype)
    x = (torch.randn((rows, n), generator=gen, device="cuda") * 3).to(torch.bfloat16)
    x[:, ::61] *= 40
    residual = torch.randn((rows, n), generator=gen, device="cuda").to(torch.bfloat16)
    weight = (1 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(torch.bfloat16)
    capi.set_option("a_dtype", a_dtype)
    try:
        plain = capi.add_rms_norm_mx_quant(x, None, weight, EPS)
        norm, stream, apart = torch.empty_like(x), residual.clone(), torch.empty_like(x)
        added = capi.add_rms_norm_mx_quant(x, stream, weight, EPS, norm_out=norm)  # the stream is updated in place
        again = capi.add_rms_norm_mx_quant(x, residual, weight, EPS, residual_out=apart)
        into_x = x.clone()
        third = capi.add_rms_norm_mx_quant(into_x, residual, weight, EPS, residual_out=into_x)
    finally:
        capi.set_option("a_dtype", 0)
    _check(torch, x, None, weight, *plain, None, None, a_dtype)
    _check(torch, x, residual, weight, *added, stream, norm, a_dtype)
    for other, h in ((again, apart), (third, into_x)):
        assert torch.equal(other[0], added[0]) and torch.equal(other[1], added[1]) and torch.equal(h, stream)


def test_rows_at_odd_addresses(capi, cuda):
    # 16-byte aligned, not 32: the loads of a half block are then two
    torch = cuda
    rows, n = 7, 160
    gen = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn((4, rows * n + 8), generator=gen, device="cuda").to(torch.bfloat16)
    x, residual, h, norm = (base[i, :-8].view(rows, n) if i % 2 else base[i, 8:].view(rows, n) for i in range(4))
    assert all(t.data_ptr() % 32 == 16 for t in (x, residual, h, norm))
    weight = torch.randn(n + 8, generator=gen, device="cuda").to(torch.bfloat16)[8:]
    x0, r0 = x.clone(), residual.clone()
    codes, scales = capi.add_rms_norm_mx_quant(x, residual, weight, EPS, residual_out=h, norm_out=norm)
    _check(torch, x0, r0, weight, codes, scales, h, norm, 0)


def test_rows_of_zeros_and_values_that_are_not_finite(capi, cuda):
    torch = cuda
    n = 1024
    x = torch.randn((6, n), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    x[0] = 0
    x[1] = 1e-30  # the mean square is far below eps: blocks below 1e-12
    x[2, 5], x[3, 40], x[4, 1000] = float("inf"), float("-inf"), float("nan")
    weight = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    norm = torch.empty_like(x)
    codes, scales = capi.add_rms_norm_mx_quant(x, None, weight, EPS, norm_out=norm)
    assert bool((codes[:2] & 0x7F == 0).all()) and bool((scales[:2] == 0x7F).all()) and bool((norm[0] == 0).all())
    # an infinity: its row's 1 / rms is zero, itself NaN; a NaN: the whole row
    for row, column in ((2, 5), (3, 40)):
        block = column // 32
        assert bool((scales[row, block] == 0xFF).all()) and bool((codes[row, block * 32 : block * 32 + 32] == 0x7F).all())
        rest = [i for i in range(n // 32) if i != block]
        assert bool((scales[row, rest] == 0x7F).all())
        assert bool(torch.isnan(norm[row, column])) and int(torch.isnan(norm[row]).sum()) == 1
    assert bool((scales[4] == 0xFF).all()) and bool((codes[4] == 0x7F).all()) and bool(torch.isnan(norm[4]).all())
    _check(torch, x[5:], None, weight, codes[5:], scales[5:], None, norm[5:], 0)


@pytest.mark.parametrize("n", [96, 512, 2080, 16416])
def test_squares_beyond_fp32(capi, cuda, n):
    # 1 / rms may be as small as 2^-128, which fp32 holds to 2^-22: 4 * 2^-24 more, 2.8e-6 in all
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(n)
    x, residual = (torch.randn((5, n), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    x[0], x[2], x[3] = x[0] * 2.0**60, x[2] * 2.0**64, x[3] * 2.0**125  # sums of squares around 2^128 and far beyond
    x[4, 3], x[1, n - 1] = 3e38, -1e20  # one large value among ordinary ones
    residual[3], residual[4, 3] = 1e30, 0.0
    weight = (1 + 0.2 * torch.randn(n, generator=gen, device="cuda")).to(torch.bfloat16)
    h, norm = torch.empty_like(x), torch.empty_like(x)
    assert bool(torch.isfinite(x.float() + residual.float()).all())
    codes, scales = capi.add_rms_norm_mx_quant(x, residual, weight, EPS, residual_out=h, norm_out=norm)
    _check(torch, x, residual, weight, codes, scales, h, norm, 0)


def test_tiny_blocks_of_the_device_rule(capi, cuda):
    torch = cuda
    n = 256
    x = torch.ones((1, n), dtype=torch.bfloat16, device="cuda")
    weight = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    weight[:32], weight[32:64], weight[64:96] = 2.0**-50, 2.0**-119, 2.0**-125
    capi.set_option("tiny_block_rule", 1)
    try:
        codes, scales = capi.add_rms_norm_mx_quant(x, None, weight, 1e-30)
    finally:
        capi.set_option("tiny_block_rule", 0)
    # byte = max(exponent - 8, 0); a byte of zero has codes of zero
    assert scales[0].tolist() == [127 - 50 - 8, 0, 0] + [127 - 8] * 5
    assert bool((codes[0, :32] == 0x78).all()) and bool((codes[0, 32:96] == 0).all())  # 0x78 = 256
    capi_codes, capi_scales = capi.add_rms_norm_mx_quant(x, None, weight, 1e-30)
    assert capi_scales[0].tolist() == [127] * 3 + [127 - 8] * 5 and bool((capi_codes[0, :96] == 0).all())


def test_feeds_the_matmul(capi, cuda):
    torch = cuda
    m, n, k = 24, 64, 512
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((m, k), generator=gen, device="cuda").to(torch.bfloat16)
    weight = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    w_codes, w_scales = capi.mx_quant((torch.randn((n, k), generator=gen, device="cuda")).to(torch.bfloat16))
    b, b_scales = w_codes.t().contiguous(), w_scales.view(n, k // 64, 2).permute(1, 0, 2).contiguous()
    codes, scales = capi.add_rms_norm_mx_quant(x, None, weight, EPS)
    c = capi.mx_gemm(codes, scales, b, b_scales)
    a64 = codes.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    w64 = w_codes.view(torch.float8_e4m3fn).double() * torch.exp2(w_scales.double() - 127).repeat_interleave(32, 1)
    want = a64 @ w64.t()
    # a sum of k products, each step off by 2^-23 of what is added up, and the rounding to bf16
    slack = k * 2.0**-23 * (a64.abs() @ w64.abs().t()) + 2.0**-8 * want.abs()
    assert bool(((c.double() - want).abs() <= slack).all())


def test_refusals(capi, cuda):
    torch = cuda
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    weight = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        capi.add_rms_norm_mx_quant(x.float(), None, weight, EPS)
    with pytest.raises(ValueError):
        capi.add_rms_norm_mx_quant(x.t(), None, weight, EPS)
    with pytest.raises(ValueError):
        capi.add_rms_norm_mx_quant(x.cpu(), None, weight, EPS)
    with pytest.raises(ValueError):
        capi.add_rms_norm_mx_quant(x, x[:2], weight, EPS)
    with pytest.raises(ValueError):
        capi.add_rms_norm_mx_quant(x, None, weight[:32], EPS)
    with pytest.raises(ValueError):
        capi.add_rms_norm_mx_quant(x, None, weight, EPS, residual_out=x)
    with pytest.raises(TypeError):
        capi.add_rms_norm_mx_quant(x, None, None, EPS)
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(capi.CatccosError) as e:
            capi.add_rms_norm_mx_quant(x, None, weight, eps)
        assert e.value.code == -1
    with pytest.raises(capi.CatccosError):
        capi.add_rms_norm_mx_quant(x[:, :48].contiguous(), None, weight[:48], EPS)
    capi.set_option("a_dtype", 2)
    try:
        with pytest.raises(capi.CatccosError):
            capi.add_rms_norm_mx_quant(x, None, weight, EPS)
    finally:
        capi.set_option("a_dtype", 0)
    codes, scales = capi.add_rms_norm_mx_quant(x[:0], None, weight, EPS)
    assert codes.shape == (0, 64) and scales.shape == (0, 2)
