"""Operands of the products of blocks of 128, their result in 64 bits and how far a result may be off, on any device.

The tensor core sums the 128 products of a block and truncates: off by 128 steps of 2^-23 of the sum of their magnitudes at most.  A block's
sum then meets its scales (three roundings at most) and the blocks, then the parts of K (eight at most), are added one after the other,
each addition off by 2^-24 of what has been added so far.  So a result is off by
    ((min(K, 128) + 2) * 2^-23 + (B + 8) * 2^-24) * sum of all magnitudes,   B = ceil(K / 128)
half a step of its type, and half of the smallest step there; where values are below fp32's normal numbers, each of the 2 B roundings by half
of 2^-149 as well."""

HALF = {"bfloat16": 2.0**-8, "float16": 2.0**-11, "float32": 2.0**-24}
LEAST = {"bfloat16": 2.0**-134, "float16": 2.0**-25, "float32": 2.0**-150}


def codes(torch, shape, dtype, gen, exponents=None):
    """Finite codes of every size, or with those exponent fields only."""
    bits = torch.randint(0, 256, shape, generator=gen, device=gen.device, dtype=torch.uint8)
    digits = 3 if dtype == "float8_e4m3fn" else 2
    if exponents is not None:
        low, high = exponents
        field = torch.randint(low, high + 1, shape, generator=gen, device=gen.device, dtype=torch.uint8)
        bits = (bits & (0x80 | ((1 << digits) - 1))) | (field << digits)
    if dtype == "float8_e4m3fn":
        bits = torch.where((bits & 0x7F) == 0x7F, bits ^ 1, bits)
    else:
        bits = torch.where((bits & 0x7C) == 0x7C, bits ^ 4, bits)
    return bits.view(getattr(torch, dtype))


def scales(torch, shape, gen):
    return torch.exp(torch.randn(shape, generator=gen, device=gen.device)) * 2.0**-8


def spread(s, n):
    """One scale for each of n values."""
    return s.repeat_interleave(128, -1)[..., :n]


def sums(a, a_scales, b, b_scales):
    """The product and the sum of its terms' magnitudes, in 64 bits: a [m, k], b [k, n], b_scales of columns or of blocks of them."""
    k, n = b.shape
    a64 = a.double() * spread(a_scales.double(), k)
    f = b_scales.double().repeat_interleave(128, 0)[:k]
    b64 = b.double() * (f if f.shape[1] == n else spread(f, n))
    return a64 @ b64, a64.abs() @ b64.abs()


def bound(want, size, k, kind):
    blocks = (k + 127) // 128
    slack = ((min(k, 128) + 2) * 2.0**-23 + (blocks + 8) * 2.0**-24) * size + 2 * blocks * 2.0**-150
    return slack + HALF[kind] * (want.abs() + slack) + LEAST[kind]
