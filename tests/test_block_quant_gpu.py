"""GPU tests of the quantiser for blocks of 128 with fp32 scales: bit for bit against its definition in fp32, and its values against
the input in 64 bits (a code is off by half a step of its type, and by the two roundings, of F / top and of the product, before it)."""
import math

import pytest

pytestmark = pytest.mark.gpu

LEAST = 2.0**-100
MOST = {"float8_e4m3fn": 448.0, "float8_e5m2": 57344.0}
HALF = {"float8_e4m3fn": (2.0**-4, 2.0**-10), "float8_e5m2": (2.0**-3, 2.0**-17)}  # of a value; of the smallest steps


def _rows_cols(block):
    return (1 if block == "row" else 128), (1 if block == "column" else 128)


def _spread(torch, scales, shape, block):
    rows, cols = _rows_cols(block)
    return scales.repeat_interleave(rows, 0)[: shape[0]].repeat_interleave(cols, 1)[:, : shape[1]]


def _tops(torch, x, block):
    rows, cols = _rows_cols(block)
    v = torch.nn.functional.pad(x.float(), (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))
    return v.abs().unflatten(1, (-1, cols)).amax(2).unflatten(0, (-1, rows)).amax(1)


def _expected(torch, x, dtype, block):
    top = _tops(torch, x, block).clamp_min(LEAST)
    most = torch.full_like(top, MOST[dtype])  # a tensor: torch divides by (or from) a number with two roundings
    q = x.float() * _spread(torch, most / top, x.shape, block)
    return q.clamp(-MOST[dtype], MOST[dtype]).to(getattr(torch, dtype)), top / most


def _check(torch, capi, x, dtype, block):
    codes, scales = capi.block_quant(x, dtype=getattr(torch, dtype), block=block)
    want, want_scales = _expected(torch, x, dtype, block)
    assert codes.dtype == getattr(torch, dtype) and codes.shape == x.shape and scales.dtype == torch.float32
    assert torch.equal(scales, want_scales)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
    x64, s64 = x.double(), _spread(torch, scales.double(), x.shape, block)
    rel, least = HALF[dtype]
    off = (codes.double() * s64 - x64).abs()
    assert bool((off <= (rel + 3 * 2.0**-24) * x64.abs() + least * s64).all())
    return codes, scales


def _values(torch, rows, k, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x *= torch.exp(3 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x[:, :: max(1, k // 5)] *= 30
    return x.clamp(-60000, 60000).to(getattr(torch, dtype))


@pytest.mark.parametrize("block", ["row", "column", "square"])
@pytest.mark.parametrize("dtype", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 128), (3, 144), (127, 112), (128, 256), (129, 1040), (300, 2304), (1000, 528)])
def test_blocks(capi, cuda, rows, k, kind, dtype, block):
    _check(cuda, capi, _values(cuda, rows, k, kind, rows + k), dtype, block)


@pytest.mark.parametrize("block", ["row", "column", "square"])
def test_every_finite_bf16(capi, cuda, block):
    torch = cuda
    bits = torch.arange(1 << 16, device="cuda", dtype=torch.int32)
    bits = bits[(bits & 0x7F80) != 0x7F80].to(torch.int16)  # 255 * 256 values
    x = bits.view(torch.bfloat16)[torch.randperm(bits.numel(), generator=torch.Generator("cuda").manual_seed(1), device="cuda")]
    _check(torch, capi, x.view(255, 256), "float8_e4m3fn", block)
    _check(torch, capi, bits.view(torch.bfloat16).view(255, 256), "float8_e5m2", block)  # neighbours of one size


@pytest.mark.parametrize("dtype", ["float8_e4m3fn", "float8_e5m2"])
def test_extremes(capi, cuda, dtype):
    torch = cuda
    x = torch.zeros((8, 384), device="cuda")
    x[1, 5] = 3.4028234663852886e38
    x[2, 130] = -1.4e-45
    x[3, :] = 2.0**-101
    x[4, :] = 2.0**-99
    x[5, 0], x[5, 1] = -0.0, 2.0**-120
    x[6, ::3] = -1e38
    codes, scales = _check(torch, capi, x, dtype, "row")
    assert bool((codes[0].float() == 0).all()) and bool((scales[0] == LEAST / MOST[dtype]).all()) and bool(torch.isfinite(scales).all())


@pytest.mark.parametrize("block", ["row", "column", "square"])
@pytest.mark.parametrize("kind", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_block_that_is_not_finite_is_nan_and_no_other(capi, cuda, bad, kind, block):
    torch = cuda
    x = _values(torch, 260, 272, kind, 3)
    clean, clean_scales = capi.block_quant(x, block=block)
    x[131, 140] = bad
    codes, scales = capi.block_quant(x, block=block)
    hit = torch.zeros_like(scales, dtype=torch.bool)
    rows, cols = _rows_cols(block)
    hit[131 // rows, 140 // cols] = True
    assert bool(scales[hit].isnan().all()) and torch.equal(scales[~hit], clean_scales[~hit])
    hit = _spread(torch, hit, x.shape, block)
    assert bool(codes.float()[hit].isnan().all()) and torch.equal(codes.view(torch.uint8)[~hit], clean.view(torch.uint8)[~hit])


@pytest.mark.parametrize("block", ["row", "column", "square"])
def test_rows_of_a_wider_matrix(capi, cuda, block):
    torch = cuda
    wide = _values(torch, 140, 1024, "bfloat16", 4)
    for first, k in ((0, 400), (8, 400), (24, 128), (512, 512)):  # 16- and 32-byte aligned rows
        x = wide[:, first : first + k]
        codes, scales = capi.block_quant(x, block=block)
        want, want_scales = capi.block_quant(x.contiguous(), block=block)
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)


@pytest.mark.parametrize("tokens,k,top_k", [(1, 16, 1), (5, 144, 3), (300, 2304, 8), (64, 7168, 2)])
def test_dispatch(capi, cuda, tokens, k, top_k):
    torch = cuda
    x = _values(torch, tokens, k, "bfloat16", 5)
    index = torch.randperm(tokens * top_k, generator=torch.Generator("cuda").manual_seed(6), device="cuda").to(torch.int32).view(tokens, top_k)
    index[:, -1] = torch.where(torch.arange(tokens, device="cuda") % 3 == 0, -1, index[:, -1])
    rows = tokens * top_k - 1  # the last row is outside: such a route is dropped
    codes = torch.full((rows, k), 0x55, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.full((rows, -(-k // 128)), 7.0, device="cuda")
    got = capi.block_quant(x, row_index=index, out=(codes, scales))
    assert got[0].data_ptr() == codes.data_ptr() and got[1].data_ptr() == scales.data_ptr()
    plain, plain_scales = capi.block_quant(x)
    want, want_scales = torch.full((rows, k), 0x55, dtype=torch.uint8, device="cuda"), torch.full_like(scales, 7.0)
    live = (index >= 0) & (index < rows)
    token = torch.arange(tokens, device="cuda")[:, None].expand(-1, top_k)[live]
    want[index[live].long()] = plain.view(torch.uint8)[token]
    want_scales[index[live].long()] = plain_scales[token]
    assert torch.equal(codes.view(torch.uint8), want) and torch.equal(scales, want_scales)
    codes, scales = capi.block_quant(x, row_index=index, rows=rows)
    assert codes.shape == (rows, k) and torch.equal(codes.view(torch.uint8)[index[live].long()], plain.view(torch.uint8)[token])


def test_more_values_than_32_bits_count(capi, cuda):
    torch = cuda
    rows, k = 262145 + 7, 8192  # 2^31 codes and some, 4 GiB of input
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    x[-3:] = _values(torch, 3, k, "bfloat16", 7)
    for block in ("row", "column", "square"):
        codes, scales = capi.block_quant(x, block=block)
        first = (rows - 3) // 128 * 128
        want, want_scales = capi.block_quant(x[first:], block=block)
        assert torch.equal(codes[first:].view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(scales[-want_scales.shape[0] :], want_scales)
        del codes, scales, want, want_scales


def test_refusals(capi, cuda):
    torch = cuda
    x = torch.zeros((8, 256), dtype=torch.bfloat16, device="cuda")
    index = torch.zeros((8, 2), dtype=torch.int32, device="cuda")
    codes, scales = capi.block_quant(x)
    for bad in (dict(x=x.cpu()), dict(x=x[0]), dict(x=x.t()), dict(x=x.int()), dict(dtype=torch.uint8), dict(dtype=torch.float16), dict(dtype=3),
                dict(block="rows"), dict(row_index=index[:4]), dict(row_index=index.long()), dict(rows=4), dict(row_index=index, rows=-1),
                dict(out=(codes[:4], scales)), dict(out=(codes, scales.double())), dict(out=(codes.view(torch.uint8), scales)),
                dict(out=(codes, scales[:, :1]))):
        with pytest.raises((ValueError, TypeError)):
            capi.block_quant(**{"x": x, **bad})
    for bad in (dict(x=x[:, :24]), dict(x=x[:, 4:20]), dict(row_index=index, block="column"), dict(row_index=index[:, :0])):
        with pytest.raises(capi.CatccosError):
            capi.block_quant(**{"x": x, **bad})
    for block, shape in (("row", (0, 2)), ("column", (0, 256)), ("square", (0, 2))):
        codes, scales = capi.block_quant(x[:0], block=block)
        assert codes.shape == (0, 256) and scales.shape == shape
