"""GPU tests of the dispatch in 16 bits, its gradient and the gradient of the combination, against their definitions in 64 bits and
against differences."""
import pytest

pytestmark = pytest.mark.gpu

HALF = {"bfloat16": 2.0**-8, "float16": 2.0**-11}
LEAST = {"bfloat16": 0.0, "float16": 2.0**-25}
SIZES = [(1, 8, 1), (1, 7168, 8), (3, 72, 2), (37, 1000, 5), (64, 2304, 8), (129, 136, 3), (700, 1032, 6), (5, 512, 33), (4, 16384, 4)]


def _case(torch, tokens, n, top_k, kind, seed=0, drop=True):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + tokens + n + top_k)
    rows = tokens * top_k
    index = torch.randperm(rows, generator=gen, device="cuda").to(torch.int32)
    if drop:
        index[torch.rand(rows, generator=gen, device="cuda") < 0.2] = -1
        index = torch.where(index == 0, rows + 5, index)  # behind the last row: dropped as well
    dtype = getattr(torch, kind)
    values = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(dtype)
    return index.view(tokens, top_k), values(tokens, n), values(rows, n), torch.rand((tokens, top_k), generator=gen, device="cuda")


def _live(index, rows):
    return (index >= 0) & (index < rows)


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,n,top_k", SIZES)
def test_dispatch(capi, cuda, tokens, n, top_k, kind):
    torch = cuda
    index, x, _, _ = _case(torch, tokens, n, top_k, kind)
    rows = tokens * top_k
    out = torch.full((rows + 2, n), 7.0, dtype=x.dtype, device="cuda")
    assert capi.moe_dispatch(x, index, out=out[:rows]).data_ptr() == out.data_ptr()
    want = torch.full_like(out, 7.0)
    live = _live(index, rows)
    want[index[live].long()] = x[torch.arange(tokens, device="cuda")[:, None].expand(-1, top_k)[live]]
    assert torch.equal(out, want)
    assert capi.moe_dispatch(x, index).shape == (rows, n) and capi.moe_dispatch(x, index, rows=rows + 9).shape == (rows + 9, n)


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("with_shared", [False, True])
@pytest.mark.parametrize("tokens,n,top_k", SIZES)
def test_dispatch_grad(capi, cuda, tokens, n, top_k, with_shared, kind):
    torch = cuda
    index, shared, d_rows, _ = _case(torch, tokens, n, top_k, kind, 1)
    live = _live(index, tokens * top_k)
    d_rows[_unused(torch, index, tokens * top_k)] = float("nan")  # nobody's rows are not read
    parts = d_rows.double()[index.long().clamp(0, tokens * top_k - 1)].where(live.unsqueeze(2), 0.0)
    want, size = parts.sum(1), parts.abs().sum(1)
    if with_shared:
        want, size = want + shared.double(), size + shared.double().abs()
    got = capi.moe_dispatch_grad(d_rows, index, shared=shared if with_shared else None)
    slack = (top_k + 1) * 2.0**-24 * size
    assert bool(((got.double() - want).abs() <= slack + HALF[kind] * (want.abs() + slack) + LEAST[kind]).all())
    if with_shared:
        assert torch.equal(capi.moe_dispatch_grad(d_rows, index, shared=shared, out=shared), got)


def _unused(torch, index, rows):
    used = torch.zeros(rows, dtype=torch.bool, device="cuda")
    used[index[_live(index, rows)].long()] = True
    return ~used


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,n,top_k", SIZES)
def test_combine_grad(capi, cuda, tokens, n, top_k, kind):
    torch = cuda
    index, d_out, y, weights = _case(torch, tokens, n, top_k, kind, 2)
    rows = tokens * top_k
    live, unused = _live(index, rows), _unused(torch, index, rows)
    y[unused] = float("nan")
    weights = torch.where(live, weights, float("nan"))  # nor a dropped route's weight
    out = torch.full((rows + 2, n), 7.0, dtype=y.dtype, device="cuda")
    d_y, d_weights = capi.moe_combine_grad(d_out, y, index, weights, out=out[:rows])
    assert d_y.data_ptr() == out.data_ptr() and bool((out[:rows][unused] == 7.0).all()) and bool((out[rows:] == 7.0).all())
    at = index[live].long()
    token = torch.arange(tokens, device="cuda")[:, None].expand(-1, top_k)[live]
    want = d_out.double()[token] * weights.double()[live].unsqueeze(1)
    slack = 2.0**-24 * want.abs()
    assert bool(((d_y[at].double() - want).abs() <= slack + HALF[kind] * (want.abs() + slack) + LEAST[kind]).all())
    assert bool((d_weights[~live] == 0).all())
    products = d_out.double()[token] * y.double()[at]
    # a sum of n products, in any order: n roundings of at most the sum of their magnitudes
    assert bool(((d_weights[live].double() - products.sum(1)).abs() <= n * 2.0**-24 * products.abs().sum(1)).all())
    # in place, and again: the same values
    again, again_weights = capi.moe_combine_grad(d_out, y, index, weights, out=y)
    assert torch.equal(again[at], d_y[at]) and torch.equal(again_weights, d_weights)


def test_gradients_against_differences(capi, cuda):
    # the combination and the dispatch are linear in each argument: for a step s, f(a + s) - f(a - s) = 2 <s, gradient>; in
    # 64 bits, on values (eighths up to 1) that the 16-bit forms hold without rounding
    torch = cuda
    tokens, n, top_k = 6, 64, 3
    gen = torch.Generator(device="cuda").manual_seed(9)
    eighths = lambda *shape: torch.randint(-8, 9, shape, generator=gen, device="cuda").double() / 8
    index, _, _, _ = _case(torch, tokens, n, top_k, "float16", 3)
    rows = tokens * top_k
    live = _live(index, rows).unsqueeze(2)
    at = index.long().clamp(0, rows - 1)
    x, y, weights, d_out, d_rows = eighths(tokens, n), eighths(rows, n), eighths(tokens, top_k), eighths(tokens, n), eighths(rows, n)

    def combined(y, weights):
        return ((y[at] * weights.unsqueeze(2)).where(live, 0.0).sum(1) * d_out).sum()

    def dispatched(x):
        return (d_rows[at] * x.unsqueeze(1)).where(live, 0.0).sum()

    h = lambda t: t.to(torch.float16)
    d_y, d_weights = capi.moe_combine_grad(h(d_out), h(y), index, weights.float(), out=torch.zeros((rows, n), dtype=torch.float16, device="cuda"))
    d_x = capi.moe_dispatch_grad(h(d_rows), index)
    for _ in range(5):
        s = eighths(rows, n)
        assert float(combined(y + s, weights) - combined(y - s, weights)) == float(2 * (s * d_y.double()).sum())
        s = eighths(tokens, top_k)
        assert float(combined(y, weights + s) - combined(y, weights - s)) == float(2 * (s * d_weights.double()).sum())
        s = eighths(tokens, n)
        assert float(dispatched(x + s) - dispatched(x - s)) == float(2 * (s * d_x.double()).sum())


def test_more_values_than_32_bits_count(capi, cuda):
    torch = cuda
    tokens, n, top_k = 40000, 8192, 7  # 2.3e9 values in the rows
    index = torch.arange(tokens * top_k, dtype=torch.int32, device="cuda").view(tokens, top_k)
    x = torch.randn((tokens, n), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    out = capi.moe_dispatch(x, index)
    for t in (0, 37448, 37449, tokens - 1):  # around 2^31 values
        assert torch.equal(out[t * top_k : (t + 1) * top_k], x[t].expand(top_k, n))
    got = capi.moe_dispatch_grad(out, index)
    assert torch.equal(got[-1], (x[-1].float() * top_k).to(torch.bfloat16))
    weights = torch.full((tokens, top_k), 0.5, device="cuda")
    d_y, d_weights = capi.moe_combine_grad(x, out, index, weights, out=out)
    assert torch.equal(d_y[-1], x[-1] / 2) and torch.equal(d_y[37449 * top_k], x[37449] / 2)
    want = x[-1].double().square().sum()
    assert abs(float(d_weights[-1, 0]) - float(want)) <= n * 2.0**-24 * float(want)


def test_refusals(capi, cuda):
    torch = cuda
    index, x, y, weights = _case(torch, 4, 64, 2, "bfloat16")
    for call, ok, bads in (
        (capi.moe_dispatch, dict(x=x, row_index=index), [dict(x=x.float()), dict(x=x[0]), dict(x=x.t()), dict(x=x.cpu()), dict(row_index=index[:3]), dict(row_index=index.long()),
                                                         dict(rows=-1), dict(out=y.half()), dict(out=y[:, :32])]),
        (capi.moe_dispatch_grad, dict(d_rows=y, row_index=index), [dict(d_rows=y.float()), dict(d_rows=y[:, :32]), dict(row_index=index.t()), dict(shared=x[:3]),
                                                                   dict(shared=x.half()), dict(out=x[:3])]),
        (capi.moe_combine_grad, dict(d_out=x, expert_out=y, row_index=index, weights=weights),
         [dict(d_out=x.float()), dict(d_out=x[:3]), dict(expert_out=y.half()), dict(expert_out=y[:, :32]), dict(row_index=index[:, :1]), dict(weights=weights.double()),
          dict(weights=weights[:3]), dict(out=y[:3]), dict(out=y.half())])):
        for bad in bads:
            with pytest.raises((ValueError, TypeError)):
                call(**{**ok, **bad})
    for call in (lambda: capi.moe_dispatch(x[:, :12].contiguous(), index), lambda: capi.moe_dispatch(x, index[:, :0]), lambda: capi.moe_dispatch(x, index, out=x),
                 lambda: capi.moe_dispatch_grad(y[:, :12].contiguous(), index), lambda: capi.moe_dispatch_grad(y, index, out=y[:4]),
                 lambda: capi.moe_combine_grad(y[:4], y, index, weights, out=y)):
        with pytest.raises(capi.CatccosError):
            call()
    assert capi.moe_dispatch(x[:0], index[:0]).shape == (0, 64) and capi.moe_dispatch_grad(y, index[:0]).shape == (0, 64)
    d_y, d_weights = capi.moe_combine_grad(x[:0], y, index[:0], weights[:0])
    assert d_y.shape == y.shape and d_weights.shape == (0, 2)
    # no rows at all: every route is dropped
    assert bool((capi.moe_dispatch_grad(y[:0], index) == 0).all()) and bool((capi.moe_combine_grad(x, y[:0], index, weights)[1] == 0).all())
