"""GPU tests of the accuracy of products of blocks of 128 over long sums: within what 128 products on the tensor core and the additions in
fp32 may be off (block_products), which scales or sums in 16 bits are not (test_block_accuracy_cpu).  Codes of every exponent, infinities and
NaN among them."""
import pytest

from block_products import bound, codes, scales, sums
from test_block_gemm_gpu import FORMS, IDS, Options

pytestmark = pytest.mark.gpu

LONG = [(16, 272, 7168), (16, 4096, 7168), (64, 144, 8192), (300, 272, 7680)]
E4M3, E5M2 = "float8_e4m3fn", "float8_e5m2"


def _close(c, want, size, k):
    kind = str(c.dtype).split(".")[1]
    off, limit = (c.double() - want).abs(), bound(want, size, k, kind)
    assert bool((off <= limit).all()), float((off / limit).max())


def _operands(torch, m, n, k, a_type=E4M3, b_type=E4M3, a_t=False, b_t=False, by_column=False, lead=(), seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + m + 7 * n + 13 * k)
    blocks = (k + 127) // 128
    a, b = codes(torch, (k, m) if a_t else (m, k), a_type, gen), codes(torch, (*lead, n, k) if b_t else (*lead, k, n), b_type, gen)
    return (a.t() if a_t else a, scales(torch, (m, blocks), gen), b.transpose(-1, -2) if b_t else b,
            scales(torch, (*lead, blocks, n if by_column else (n + 127) // 128), gen))


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", LONG)
def test_long_sums(capi, cuda, m, n, k, out, form):
    o = _operands(cuda, m, n, k)
    if out == "float16":
        o[1].mul_(2.0**-8)  # results within its range
    with Options(capi, form):
        c = capi.block_gemm(*o, out_dtype=getattr(cuda, out))
    _close(c, *sums(*o), k)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("a_type,b_type", [(E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
def test_types_with_every_exponent(capi, cuda, a_type, b_type, form):
    o = _operands(cuda, 144, 400, 7168, a_type, b_type, b_t=True)
    with Options(capi, form):
        c = capi.block_gemm(*o, out_dtype=cuda.float32)
    _close(c, *sums(*o), 7168)


@pytest.mark.parametrize("a_t,b_t", [(True, False), (True, True), (False, True), (False, False)])
@pytest.mark.parametrize("m,n,k", [(144, 272, 8192), (528, 400, 4104 // 16 * 16)])
def test_weight_gradients(capi, cuda, m, n, k, a_t, b_t):
    o = _operands(cuda, m, n, k, E4M3, E5M2, a_t=a_t, b_t=b_t, by_column=True)
    _close(capi.block_gemm(*o, out_dtype=cuda.float32), *sums(*o), k)


@pytest.mark.parametrize("form", FORMS, ids=IDS)
@pytest.mark.parametrize("b_t", [False, True])
def test_experts(capi, cuda, b_t, form):
    torch = cuda
    m, n, k, offsets = 400, 272, 7168, [0, 16, 16, 80, 400]
    o = _operands(torch, m, n, k, E5M2 if b_t else E4M3, b_t=b_t, lead=(4,))
    with Options(capi, form):
        c = capi.block_grouped_gemm(*o, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    a, a_scales, b, b_scales = o
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi > lo:
            _close(c[lo:hi], *sums(a[lo:hi], a_scales[lo:hi], b[e], b_scales[e]), k)


@pytest.mark.parametrize("form,by_column", [(f, False) for f in FORMS] + [(dict(cta_pair=1), True)], ids=IDS + ["by_column"])  # pairs alone scale by column
@pytest.mark.parametrize("bits", [0x7C, 0xFC, 0x7E, 0xFF])  # E5M2: infinities, NaN
def test_codes_that_are_not_finite(capi, cuda, bits, form, by_column):
    torch = cuda
    m, n, k = 40, 272, 400
    gen = torch.Generator(device="cuda").manual_seed(bits)
    a, b = codes(torch, (m, k), E5M2, gen, (10, 20)), codes(torch, (k, n), E4M3, gen, (5, 9))
    a_scales, b_scales = scales(torch, (m, 4), gen), scales(torch, (4, n if by_column else 3), gen)
    a.view(torch.uint8)[5, 17] = a.view(torch.uint8)[30, 399] = bits
    b.view(torch.uint8)[17, 100] = 0  # infinity times 0
    with Options(capi, form):
        c = capi.block_gemm(a, a_scales, b, b_scales, out_dtype=torch.float32)
    hit = torch.zeros(m, dtype=torch.bool, device="cuda")
    hit[[5, 30]] = True
    _close(c[~hit], *sums(a[~hit], a_scales[~hit], b, b_scales), k)
    code = a.view(torch.uint8).view(a.dtype)[5, 17].double()
    for row, at in ((5, 17), (30, 399)):
        want = code * b[at].double()  # the term that decides
        assert torch.equal(c[row].isnan(), want.isnan()) and torch.equal(c[row].nan_to_num(0, 1, -1).sign(), want.nan_to_num(0, 1, -1).sign())
        assert not bool(torch.isfinite(c[row]).any())
