"""CPU tests of the bound that the products of blocks of 128 are held to: it passes what the kernels do (blocks summed with truncation, scaled and
added in fp32) and sees scales that were rounded to 16 bits, sums over blocks held in 16 bits, and a block that was left out."""
import pytest
import torch

from block_products import bound, codes, scales, sums

CASES = [(16, 48, 7168), (64, 32, 8192), (16, 32, 2304)]


def _case(m, n, k):
    gen = torch.Generator().manual_seed(m + n + k)
    blocks = (k + 127) // 128
    return (codes(torch, (m, k), "float8_e4m3fn", gen), scales(torch, (m, blocks), gen), codes(torch, (k, n), "float8_e4m3fn", gen),
            scales(torch, (blocks, (n + 127) // 128), gen))


def _truncated(x, digits=24):
    """To so many binary digits, towards zero."""
    f, e = torch.frexp(x)
    return torch.ldexp(torch.trunc(f * 2.0**digits), e - digits)


def _result(a, a_scales, b, b_scales, rounded=lambda s: s, held=torch.float32, leave_out=-1):
    m, k = a.shape
    out = torch.zeros((m, b.shape[1]), dtype=held)
    for t in range((k + 127) // 128):
        if t == leave_out:
            continue
        v = torch.zeros(out.shape, dtype=torch.float64)
        for i in range(128 * t, min(k, 128 * t + 128), 32):  # 32 products at a time, cut to 24 digits
            v = _truncated(v + a[:, i : i + 32].double() @ b[i : i + 32].double())
        f = rounded(a_scales[:, t : t + 1]) * rounded(b_scales[t]).repeat_interleave(128)[: b.shape[1]]
        out = (out.double() + v * f.double()).to(held)
    return out


def _passes(result, case, kind="float32"):
    want, size = sums(*case)
    return bool(((result.to(getattr(torch, kind)).double() - want).abs() <= bound(want, size, case[0].shape[1], kind)).all())


@pytest.mark.parametrize("m,n,k", CASES)
def test_what_the_bound_passes(m, n, k):
    case = _case(m, n, k)
    assert all(_passes(_result(*case), case, kind) for kind in ("float32", "bfloat16"))


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("m,n,k", CASES)
def test_what_the_bound_sees(m, n, k, kind):
    case = _case(m, n, k)
    assert not _passes(_result(*case, rounded=lambda s: s.bfloat16().float()), case, kind)
    assert not _passes(_result(*case, leave_out=3), case, kind)
    small = (case[0], case[1] * 2.0**-12, *case[2:])  # within fp16's range
    assert not _passes(_result(*small, held=torch.float16), small, kind)
    assert not _passes(_result(*case, held=torch.bfloat16), case, kind)
    if kind == "float32":
        assert not _passes(_result(*case, rounded=lambda s: s.half().float()), case, kind)
