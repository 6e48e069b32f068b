"""GPU tests of the element types of the grouped product and the FP4 matvec on torch tensors: what a tensor's own type says, or
out_dtype, holds whatever the process-wide options are; codes in plain bytes go by the options."""
import pytest

pytestmark = pytest.mark.gpu

ROWS, N, K, EXPERTS = 40, 64, 256, 3
HALF = {"bfloat16": 2.0**-8, "float16": 2.0**-11}


@pytest.fixture
def options(capi):
    def set_(**values):
        for key, value in values.items():
            capi.set_option(key, value)

    yield set_
    set_(a_dtype=0, b_dtype=0, c_dtype=0)


def _codes(torch, gen, shape, kind):
    """Finite codes of a type, as bytes, and their values in 64 bits."""
    b = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    f8 = getattr(torch, kind)
    b[~torch.isfinite(b.view(f8).float()) | (b.view(f8).float().abs() > 448)] = 0x38
    return b, b.view(f8).double()


def _grouped(torch, a_kind, b_kind):
    gen = torch.Generator(device="cuda").manual_seed(len(a_kind + b_kind))
    a, a64 = _codes(torch, gen, (ROWS, K), a_kind)
    b, b64 = _codes(torch, gen, (EXPERTS, K, N), b_kind)
    sa = torch.randint(118, 122, (ROWS, K // 32), generator=gen, device="cuda", dtype=torch.uint8)
    sb = torch.randint(118, 122, (EXPERTS, K // 64, N, 2), generator=gen, device="cuda", dtype=torch.uint8)
    offsets = torch.tensor([0, 7, 7, ROWS], dtype=torch.int32, device="cuda")
    a64 = a64 * torch.exp2(sa.double() - 127).repeat_interleave(32, 1)
    b64 = b64 * torch.exp2(sb.double() - 127).transpose(2, 3).flatten(1, 2).repeat_interleave(32, 1)
    want, size = torch.cat((a64[:7] @ b64[0], a64[7:] @ b64[2])), torch.cat((a64[:7].abs() @ b64[0].abs(), a64[7:].abs() @ b64[2].abs()))
    return (a, sa, b, sb, offsets), want, size


def _close(got, want, size, half):
    # K steps of an fp32 accumulator that truncates, half a step of the result's type (fp16 is never in its denormals here but at
    # less than its smallest normal number's step)
    slack = K * 2.0**-23 * size
    return bool(((got.double() - want).abs() <= slack + half * (want.abs() + slack) + 2.0**-25).all())


@pytest.mark.parametrize("c_dtype", [0, 1])
@pytest.mark.parametrize("given", ["out", "out_dtype"])
@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
def test_output_type_of_the_grouped_product(capi, cuda, options, kind, given, c_dtype):
    torch = cuda
    operands, want, size = _grouped(torch, "float8_e4m3fn", "float8_e4m3fn")
    dtype = getattr(torch, kind)
    options(c_dtype=c_dtype)
    out = torch.empty((ROWS, N), dtype=dtype, device="cuda")
    got = capi.mx_grouped_gemm(*operands, **(dict(out=out) if given == "out" else dict(out_dtype=dtype)))
    assert got.dtype == dtype and _close(got, want, size, HALF[kind])


@pytest.mark.parametrize("c_dtype", [0, 1])
def test_output_type_without_a_word_is_bf16(capi, cuda, options, c_dtype):
    torch = cuda
    operands, want, size = _grouped(torch, "float8_e4m3fn", "float8_e4m3fn")
    options(c_dtype=c_dtype)
    got = capi.mx_grouped_gemm(*operands)
    assert got.dtype == torch.bfloat16 and _close(got, want, size, HALF["bfloat16"])


@pytest.mark.parametrize("pair", [1, 2])
@pytest.mark.parametrize("a_dtype,b_dtype", [(0, 0), (1, 1), (0, 1)])
@pytest.mark.parametrize("a_kind", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("b_kind", ["float8_e4m3fn", "float8_e5m2"])
def test_types_of_the_codes(capi, cuda, options, a_kind, b_kind, a_dtype, b_dtype, pair):
    torch = cuda
    (a, sa, b, sb, offsets), want, size = _grouped(torch, a_kind, b_kind)
    options(cta_pair=pair)
    try:
        # tensors that say what they are
        options(a_dtype=a_dtype, b_dtype=b_dtype)
        typed = capi.mx_grouped_gemm(a.view(getattr(torch, a_kind)), sa, b.view(getattr(torch, b_kind)), sb, offsets)
        # bytes, and the options
        options(a_dtype=1 if a_kind == "float8_e5m2" else 0, b_dtype=1 if b_kind == "float8_e5m2" else 0)
        plain = capi.mx_grouped_gemm(a, sa, b, sb, offsets)
    finally:
        options(cta_pair=0)
    assert _close(plain, want, size, HALF["bfloat16"]) and torch.equal(typed, plain)


@pytest.mark.parametrize("c_dtype", [0, 1])
@pytest.mark.parametrize("given", ["out", "out_dtype", "nothing"])
@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
def test_output_type_of_the_matvec(capi, cuda, options, kind, given, c_dtype):
    torch = cuda
    dtype = getattr(torch, kind)
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device="cuda")
    x[0, 3], x[1, 60] = 1.0, -3.0
    w = torch.full((64, 8), 0x53, dtype=torch.uint8, device="cuda")  # 1.5 and 3
    s = torch.full((1, 16, 2), 127, dtype=torch.uint8, device="cuda")
    options(c_dtype=c_dtype)
    if given == "nothing":
        got, dtype = capi.mx_fp4_matvec(x, w, s), torch.bfloat16
    else:
        out = torch.empty((2, 16), dtype=dtype, device="cuda")
        got = capi.mx_fp4_matvec(x, w, s, **(dict(out=out) if given == "out" else dict(out_dtype=dtype)))
    assert got.dtype == dtype
    assert torch.equal(got.double().cpu(), torch.tensor([[1.5, 3.0] * 8, [-4.5, -9.0] * 8], dtype=torch.float64))
