"""GPU tests of products of blocks of 128 whose scales are finite, but multiply to what fp32 does not hold: the result has to be that of the
definition in 64 bits wherever it and the sums on the way to it are in fp32's range."""
import pytest

from block_products import bound, codes, scales, sums
from test_block_gemm_gpu import FORMS, IDS, Options

pytestmark = pytest.mark.gpu

PAIR = [FORMS[IDS.index("pair")]]  # the only form for scales by column and a stored by column


def _power(torch, e):
    e = torch.as_tensor(e, device="cuda")
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e).float()


def _check(torch, c, a, a_scales, b, b_scales):
    want, size = sums(a, a_scales, b, b_scales)
    inside = size < 2.0**127  # nothing on the way overflows
    off, limit = (c.double() - want).abs(), bound(want, size, b.shape[0], "float32")
    assert bool((off <= limit)[inside].all()), int((~(off <= limit))[inside].sum())
    return inside


def _far(torch, m, n, k, by_column=False, seed=0):
    """Scales from 2^-149 to 2^127, most of a block's two of opposite sizes."""
    gen = torch.Generator(device="cuda").manual_seed(seed + m + n + k)
    blocks = (k + 127) // 128
    a_e = torch.randint(-140, 125, (m, blocks), generator=gen, device="cuda")
    b_e = torch.randint(-140, 125, (blocks, n if by_column else (n + 127) // 128), generator=gen, device="cuda")
    fraction = lambda shape: 1 + torch.rand(shape, generator=gen, device="cuda")
    return gen, fraction(a_e.shape) * _power(torch, a_e), fraction(b_e.shape) * _power(torch, b_e)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("kind", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (40, 400, 128), (70, 272, 1040), (300, 144, 640)])
def test_scales_of_every_size(capi, cuda, m, n, k, kind, form):
    torch = cuda
    gen, a_scales, b_scales = _far(torch, m, n, k)
    a, b = codes(torch, (m, k), kind, gen), codes(torch, (k, n), kind, gen)
    with Options(capi, form):
        c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    _check(torch, c, a, a_scales, b, b_scales)


@pytest.mark.parametrize("kind", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("m,n,k", [(16, 16, 16), (48, 400, 128), (272, 272, 1040)])
def test_scales_of_every_size_by_column(capi, cuda, m, n, k, kind):
    torch = cuda
    gen, a_scales, b_scales = _far(torch, m, n, k, True)
    a, b = codes(torch, (k, m), kind, gen).t(), codes(torch, (k, n), kind, gen)
    c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    _check(torch, c, a, a_scales, b, b_scales)


@pytest.mark.parametrize("form,by_column", [(f, False) for f in FORMS] + [(f, True) for f in PAIR], ids=IDS + ["by_column"])
@pytest.mark.parametrize("a_e,b_e", [(100, 30), (30, 100), (127, 127), (64, 64), (-100, -40), (-40, -100), (-149, -149), (-70, -57), (127, -149)])
def test_blocks_of_zeros_between_others(capi, cuda, a_e, b_e, form, by_column):
    # block 1 of row 3 is zero, with scales that multiply to 0 or infinity; its other blocks are ordinary, and so are the other rows
    torch = cuda
    m, n, k = 36, 272, 400
    gen = torch.Generator(device="cuda").manual_seed(1)
    a, b = codes(torch, (m, k), "float8_e4m3fn", gen), codes(torch, (k, n), "float8_e4m3fn", gen)
    a_scales, b_scales = scales(torch, (m, 4), gen), scales(torch, (4, n if by_column else 3), gen)
    b_scales[1, :] = _power(torch, b_e)
    a_scales[:, 1] = 1 / b_scales[1, 0] if -126 <= b_e <= 126 else 2.0 ** (100 if b_e < 0 else -100)
    a.view(torch.uint8)[3, 128:256] = 0
    with Options(capi, form):
        clean = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
        a_scales[3, 1] = _power(torch, a_e)
        c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    assert bool(torch.isfinite(c).all()) and bool(_check(torch, c, a, a_scales, b, b_scales).all())
    if not by_column:  # a row's result does not depend on the others
        others = torch.arange(m, device="cuda") != 3
        assert torch.equal(c[others], clean[others])


@pytest.mark.parametrize("form,by_column", [(f, False) for f in FORMS] + [(f, True) for f in PAIR], ids=IDS + ["by_column"])
def test_small_values_with_large_scales_and_large_ones_with_small(capi, cuda, form, by_column):
    # one product a block: 2^-16 * 2^-16 with scales of 2^70 each (2^108), 57344^2 with scales of 1.2 * 2^-80 and 1.7 * 2^-60
    torch = cuda
    m, n, k = 20, 144, 272
    a, b = (torch.zeros(s, dtype=torch.uint8, device="cuda") for s in ((m, k), (k, n)))
    a_scales, b_scales = torch.ones((m, 3), device="cuda"), torch.ones((3, n if by_column else 2), device="cuda")
    a[2, 5], b[5, :] = 0x01, 0x81  # 2^-16, -2^-16
    a_scales[2, 0], b_scales[0, :] = 2.0**70, 2.0**70
    a[7, 200], b[200, :] = 0x7B, 0x7B  # 57344
    a_scales[7, 1], b_scales[1, :] = 1.2 * 2.0**-80, 1.7 * 2.0**-60
    a, b = a.view(torch.float8_e5m2), b.view(torch.float8_e5m2)
    with Options(capi, form):
        c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    assert bool((c[2] == -(2.0**108)).all())
    want = 57344.0**2 * float(a_scales[7, 1]) * float(b_scales[1, 0])
    assert bool(((c[7].double() - want).abs() <= 4 * 2.0**-24 * want).all())
    c[2], c[7] = 0, 0
    assert bool((c == 0).all())


@pytest.mark.parametrize("form,by_column", [(f, False) for f in FORMS] + [(f, True) for f in PAIR], ids=IDS + ["by_column"])
def test_what_is_not_finite_or_zero_counts_as_such_beside_them(capi, cuda, form, by_column):
    torch = cuda
    m, n, k = 24, 144, 272
    gen = torch.Generator(device="cuda").manual_seed(2)
    a, b = codes(torch, (m, k), "float8_e4m3fn", gen, (5, 9)), codes(torch, (k, n), "float8_e4m3fn", gen, (5, 9))
    a_scales, b_scales = torch.ones((m, 3), device="cuda"), torch.ones((3, n if by_column else 2), device="cuda")
    b_scales[1, :] = 2.0**100
    a_scales[:, 1] = 2.0**-100
    a_scales[0, 1], a_scales[1, 1], a_scales[2, 1], a_scales[3, 1], a_scales[4, 1] = 2.0**100, float("nan"), float("inf"), 0.0, -(2.0**-100)
    with Options(capi, form):
        c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    assert bool(c[1].isnan().all()) and not bool(torch.isfinite(c[2]).any()) and not bool(torch.isfinite(c[0]).any())
    _check(torch, c[3:], a[3:], a_scales[3:], b, b_scales)
    assert bool(torch.isfinite(c[3:]).all())


@pytest.mark.parametrize("form,by_column", [(f, False) for f in FORMS] + [(f, True) for f in PAIR], ids=IDS + ["by_column"])
@pytest.mark.parametrize("m,n,k", [(40, 272, 8192), (1000, 2320, 1168)])
def test_some_groups_of_some_tiles(capi, cuda, m, n, k, form, by_column):
    # tiles with such scales in front, in the middle, at the end and without any, several of them a CTA
    torch = cuda
    blocks = (k + 127) // 128
    gen = torch.Generator(device="cuda").manual_seed(3)
    a, b = codes(torch, (m, k), "float8_e4m3fn", gen), codes(torch, (k, n), "float8_e4m3fn", gen)
    a_scales, b_scales = scales(torch, (m, blocks), gen), scales(torch, (blocks, n if by_column else (n + 127) // 128), gen)
    rows = torch.randperm(m, generator=gen, device="cuda")[: max(2, m // 100)]
    at = torch.randint(0, blocks, rows.shape, generator=gen, device="cuda")
    at[0], at[1] = 0, blocks - 1
    with Options(capi, form):
        clean = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
        a_scales[rows, at] = torch.where(torch.arange(rows.numel(), device="cuda") % 2 == 0, 2.0**90, 2.0**-149)
        c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    assert bool(_check(torch, c, a, a_scales, b, b_scales).all())
    others = torch.ones(m, dtype=torch.bool, device="cuda")
    others[rows] = False
    if not by_column:
        assert torch.equal(c[others], clean[others])


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_experts(capi, cuda, form):
    torch = cuda
    m, n, k, offsets = 330, 272, 656, [0, 20, 20, 180, 330]
    gen, a_scales, _ = _far(torch, m, n, k)
    a, b = codes(torch, (m, k), "float8_e5m2", gen), codes(torch, (4, k, n), "float8_e4m3fn", gen)
    b_scales = torch.stack([_far(torch, m, n, k, seed=i)[2] for i in range(1, 5)])
    with Options(capi, form):
        c = capi.block_grouped_gemm(a, a_scales, b, b_scales, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi > lo:
            _check(torch, c[lo:hi], a[lo:hi], a_scales[lo:hi], b[e], b_scales[e])
