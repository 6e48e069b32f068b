"""GPU tests of routing, of the rows of the dispatch and of the combination of the experts' rows, against plain forms in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _route(logits, bias, top_k, score, groups, top_groups, group_best, renormalize, scale):
    """The definition, token by token, in 64 bits; also each weight's relative error bound in fp32 (see test_routes)."""
    tokens, experts = logits.shape
    size = experts // groups
    ids = np.full((tokens, top_k), -1, np.int32)
    weights = np.zeros((tokens, top_k))
    spread = np.zeros((tokens, 1))
    for t in range(tokens):
        l = logits[t].astype(np.float64)
        seen = l > -np.inf  # not NaN either
        if not seen.any():
            continue
        top = l[seen].max()
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.where(l == top, 1.0, np.exp(np.where(seen, l, -np.inf) - top))
            e[~seen] = 0.0
            s = e / e.sum() if score == "softmax" else 1.0 / (1.0 + np.exp(-np.where(seen, l, -np.inf)))
        order = np.where(seen, l if bias is None and (top_groups == groups or group_best == 1) else s, -np.inf)
        if bias is not None:
            b = bias.astype(np.float64)
            order = np.where(seen & (b > -np.inf), s + np.where(b > -np.inf, b, 0.0), -np.inf)
        if top_groups < groups:
            best = -np.sort(-order.reshape(groups, size), axis=1)[:, :group_best]
            value = np.array([g[0] if g[0] == -np.inf else g[g > -np.inf].sum() for g in best])
            keep = [g for g in np.argsort(-value, kind="stable")[:top_groups] if value[g] > -np.inf]
            order = np.where(np.isin(np.arange(experts) // size, keep), order, -np.inf)
        pick = [x for x in np.argsort(-order, kind="stable")[:top_k] if order[x] > -np.inf]
        ids[t, : len(pick)] = pick
        if not pick:
            continue
        w = s[pick]
        if renormalize:
            lp = l[pick]
            with np.errstate(invalid="ignore", over="ignore"):
                if score == "softmax":
                    w = np.where(lp == lp.max(), 1.0, np.exp(lp - lp.max()))
                elif lp.max() < 0:
                    w = np.exp(lp - lp.max()) / (1.0 + np.exp(lp))
            w = w / w.sum()
        weights[t, : len(pick)] = w * scale
        finite = l[np.isfinite(l)]
        # (a difference of more than 104 leaves nothing in fp32)
        spread[t] = min(104.0, np.abs(finite).max() * 2) if finite.size else 0.0
    return ids, weights, spread


def _check_route(capi, torch, logits, bias=None, top_k=1, score="softmax", groups=1, top_groups=1, group_best=1, renormalize=True,
                 scale=1.0):
    ids, weights = capi.moe_route(logits, top_k, bias=bias, score=score, groups=groups, top_groups=top_groups, group_best=group_best,
                                  renormalize=renormalize, scale=scale)
    want_ids, want, spread = _route(logits.float().cpu().numpy(), None if bias is None else bias.cpu().numpy(), top_k, score, groups,
                                    top_groups, group_best, renormalize, scale)
    assert ids.dtype == torch.int32 and weights.dtype == torch.float32
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    got = weights.double().cpu().numpy()
    # 2^-23 for each of: the sum's additions (at most 37 + 5), two exponentials of two units each, their arguments' rounding
    # (the logits' spread), quotients and products; a result below 2^-126 is off by 2^-126 more
    slack = (64 + spread) * 2.0**-23 * np.abs(want) + 2.0**-126 * abs(scale)
    assert (np.abs(got - want) <= slack).all()


ROUTERS = [
    # tokens, experts, top_k, score, bias, groups, top_groups, group_best, renormalize
    (1, 8, 2, "softmax", False, 1, 1, 1, True),
    (5, 1, 1, "sigmoid", True, 1, 1, 1, False),
    (33, 60, 4, "softmax", False, 1, 1, 1, False),
    (67, 64, 6, "softmax", True, 1, 1, 1, True),
    (130, 256, 8, "sigmoid", True, 8, 4, 2, True),
    (130, 160, 6, "softmax", False, 8, 3, 1, False),
    (31, 160, 6, "sigmoid", False, 5, 2, 2, True),
    (9, 384, 12, "sigmoid", True, 3, 2, 1, True),
    (7, 96, 3, "softmax", True, 32, 7, 2, True),
    (4, 512, 32, "softmax", False, 1, 1, 1, True),
    (3, 1024, 32, "sigmoid", True, 2, 1, 2, False),
    (11, 40, 5, "sigmoid", False, 1, 1, 1, True),
    (21, 97, 5, "softmax", True, 1, 1, 1, True),  # no whole lanes
    (6, 32, 32, "sigmoid", True, 1, 1, 1, True),
]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens,experts,top_k,score,with_bias,groups,top_groups,group_best,renormalize", ROUTERS)
def test_routes(capi, cuda, tokens, experts, top_k, score, with_bias, groups, top_groups, group_best, renormalize, dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(tokens * 4096 + experts)
    logits = (torch.randn((tokens, experts), generator=gen, device="cuda") * 2).to(getattr(torch, dtype))
    bias = torch.randn(experts, generator=gen, device="cuda") * 0.1 if with_bias else None
    _check_route(capi, torch, logits, bias, top_k, score, groups, top_groups, group_best, renormalize, 2.5)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_at_odd_addresses(capi, cuda, dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(9 * 128 + 1, generator=gen, device="cuda").to(getattr(torch, dtype))
    _check_route(capi, torch, base[1:].view(9, 128), torch.randn(129, generator=gen, device="cuda")[1:], 8, "sigmoid", 4, 2, 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,group_best", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
def test_equal_scores_go_to_the_lowest_index(capi, cuda, score, groups, top_groups, group_best):
    torch = cuda
    logits = torch.tensor([[0.0, 1.0, 1.0, 0.0] * 8, [0.0] * 32, [-0.0, 0.0] * 16, [100.0] * 32, [-100.0] * 32], device="cuda")
    for bias in (None, torch.zeros(32, device="cuda"), torch.full((32,), 0.25, device="cuda")):
        _check_route(capi, torch, logits, bias, 7, score, groups, top_groups, group_best)


@pytest.mark.parametrize("experts,groups,top_groups,group_best", [(256, 1, 1, 1), (256, 8, 3, 2), (1024, 1, 1, 1), (60, 4, 2, 2)])
def test_choices_closer_than_fp32_tells_apart(capi, cuda, experts, groups, top_groups, group_best):
    # the bias makes all of a token's choice values equal up to its own rounding: some 1e-9 between neighbours
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(experts + groups)
    row = torch.randn(experts, generator=gen, device="cuda")
    for score, s in (("sigmoid", torch.sigmoid(row.double())), ("softmax", torch.softmax(row.double(), 0))):
        bias = (0.7 - s).float()
        logits = torch.stack((row, row + 1.0, torch.randn(experts, generator=gen, device="cuda")))
        _check_route(capi, torch, logits, bias, 8, score, groups, top_groups, group_best)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,top_groups,group_best", [(1, 1, 1), (4, 2, 1), (4, 3, 2)])
@pytest.mark.parametrize("renormalize", [False, True])
def test_masked_experts(capi, cuda, score, with_bias, groups, top_groups, group_best, renormalize):
    torch = cuda
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn((9, 32), generator=gen, device="cuda")
    logits[0] = -inf  # nothing left
    logits[1] = nan
    logits[2, 1:] = -inf  # one expert left
    logits[3, ::2] = nan
    logits[4, 8:] = -inf  # one group left
    logits[5, :30] = low  # the type's lowest value is a value
    logits[6, 4], logits[6, 20] = inf, inf
    logits[7, 3] = 3e38
    bias = None
    if with_bias:
        bias = torch.randn(32, generator=gen, device="cuda")
        bias[5], bias[6], bias[30] = -inf, nan, inf
    _check_route(capi, torch, logits, bias, 6, score, groups, top_groups, group_best, renormalize)


def _choice(logits, bias, top_k, score, groups, top_groups):
    """ids by the two best of each group, for finite logits and biases, in 64 bits; and how far apart the groups at the border are."""
    l, b = logits.astype(np.float64), bias.astype(np.float64)
    e = np.exp(l - l.max(1, keepdims=True))
    choice = (e / e.sum(1, keepdims=True) if score == "softmax" else 1.0 / (1.0 + np.exp(-l))) + b
    tokens, experts = l.shape
    best = np.sort(choice.reshape(tokens, groups, -1), axis=2)[:, :, -2:].sum(axis=2)
    order = np.argsort(-best, axis=1, kind="stable")
    open_ = np.zeros((tokens, groups), bool)
    np.put_along_axis(open_, order[:, :top_groups], True, 1)
    choice[~np.repeat(open_, experts // groups, axis=1)] = -np.inf
    ranked = np.take_along_axis(best, order, 1)
    return np.argsort(-choice, axis=1, kind="stable")[:, :top_k].astype(np.int32), ranked[:, top_groups - 1] - ranked[:, top_groups]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups", [(32, 4, 2), (40, 5, 3)])  # whole lanes, and not
@pytest.mark.parametrize("size", [64.0, 1000.0, 10000.0])
def test_group_sums_that_cancel(capi, cuda, score, experts, groups, top_groups, size):
    # one expert a group far up, the others far down: a group's two best add up to far less than either, whose rounding stays
    torch = cuda
    rng = np.random.default_rng(int(size) + experts)
    logits = (0.2 + 1e-3 * rng.standard_normal((4096, experts))).astype(np.float32)
    bias = np.full(experts, -size, np.float32)
    bias[:: experts // groups] = size
    want, apart = _choice(logits, bias, top_groups, score, groups, top_groups)
    keep = apart > 64 * size * 2.0**-52  # where 64 bits themselves decide
    assert keep.mean() > 0.99
    ids, _ = capi.moe_route(torch.from_numpy(logits).cuda(), top_groups, bias=torch.from_numpy(bias).cuda(), score=score, groups=groups,
                            top_groups=top_groups, group_best=2)
    np.testing.assert_array_equal(ids.cpu().numpy()[keep], want[keep])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_one_large_group_hides_no_close_pair(capi, cuda, score):
    # the groups at the border are small and apart; a group further down is so large that its sum may belong above them
    torch = cuda
    rng = np.random.default_rng(5)
    logits = (0.2 + 1e-3 * rng.standard_normal((4096, 32))).astype(np.float32)
    bias = np.zeros(32, np.float32)
    bias[8:16] = 0.001
    bias[16:24], bias[16] = -20000.0, 20000.0
    want, apart = _choice(logits, bias, 8, score, 4, 1)
    keep = apart > 64 * 20000 * 2.0**-52
    assert keep.mean() > 0.99
    ids, _ = capi.moe_route(torch.from_numpy(logits).cuda(), 8, bias=torch.from_numpy(bias).cuda(), score=score, groups=4, group_best=2)
    np.testing.assert_array_equal(ids.cpu().numpy()[keep], want[keep])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_best", [1, 2])
@pytest.mark.parametrize("experts,groups", [(32, 4), (60, 5)])  # whole lanes, and not
def test_groups_masked_by_the_lowest_value(capi, cuda, score, group_best, experts, groups):
    # the type's lowest value is a value: the sum of two of them passes fp32's range, and the group still counts as one with experts
    torch = cuda
    low = torch.finfo(torch.float32).min
    logits = torch.randn((33, experts), generator=torch.Generator(device="cuda").manual_seed(experts), device="cuda")
    bias = torch.full((experts,), low, device="cuda")
    bias[experts // groups : 2 * (experts // groups)] = 0.0
    _check_route(capi, torch, logits, bias, experts // groups + 2, score, groups, 2, group_best)
    bias[: experts // groups] = float("-inf")  # and comes before one that has none
    _check_route(capi, torch, logits, bias, experts // groups + 2, score, groups, 2, group_best)
    _check_route(capi, torch, logits, -bias.clamp(min=low), 5, score, groups, 2, group_best)  # as far up


def test_route_refusals_and_empty_batch(capi, cuda):
    torch = cuda
    l = torch.zeros((4, 32), device="cuda")
    for bad in (dict(top_k=0), dict(top_k=33), dict(top_k=9, groups=4, top_groups=1), dict(top_k=1, groups=3), dict(top_k=1, groups=0),
                dict(top_k=1, groups=4, top_groups=5), dict(top_k=1, top_groups=0), dict(top_k=1, group_best=3),
                dict(top_k=1, scale=float("nan"))):
        with pytest.raises(capi.CatccosError) as e:
            capi.moe_route(l, **bad)
        assert e.value.code == -1, bad
    with pytest.raises(capi.CatccosError):
        capi.moe_route(torch.zeros((1, 1025), device="cuda"), 1)
    for bad in (l.half(), l.t(), l[0], l.cpu()):
        with pytest.raises(ValueError):
            capi.moe_route(bad, 1)
    for bias in (l[0, :31], l[0].half(), l[0].cpu()):
        with pytest.raises(ValueError):
            capi.moe_route(l, 1, bias=bias)
    with pytest.raises(ValueError):
        capi.moe_route(l, 1, score="tanh")
    with pytest.raises(ValueError):
        capi.moe_route(l, -1)
    ids, weights = capi.moe_route(l[:0], 3)
    assert ids.shape == weights.shape == (0, 3)


# ---- rows of the dispatch ----------------------------------------------------------------------------------------------------
def _plan(ids, experts, first):
    local = ids.astype(np.int64).reshape(-1) - first
    mine = (ids.reshape(-1) >= 0) & (local >= 0) & (local < experts)
    key = np.where(mine, local, experts)
    order = np.argsort(key, kind="stable")
    index = np.empty(key.size, np.int32)
    index[order] = np.arange(key.size, dtype=np.int32)
    index[~mine] = -1
    return index.reshape(ids.shape), np.concatenate(([0], np.cumsum(np.bincount(key, minlength=experts + 1)[:experts]))).astype(np.int32)


PLANS = [(0, 4, 0), (1, 1, 0), (31, 3, 0), (33, 1024, 0), (128, 256, 64), (1000, 7, 2), (4096, 64, 0), (4097, 64, 0), (33000, 1024, 100),
         (131072, 32, 64), (300001, 5, 0)]


@pytest.mark.parametrize("routes,experts,first", PLANS)
def test_rows_of_the_dispatch(capi, cuda, routes, experts, first):
    torch = cuda
    rng = np.random.default_rng(routes + experts)
    for kind in range(4):
        if kind == 0:  # some below, some above this rank's experts, some dropped
            ids = rng.integers(-1, first + experts + 3, routes)
        elif kind == 1:  # one expert has them all
            ids = np.full(routes, first + experts - 1)
        elif kind == 2:  # nobody has any; the numbers are as far out as they come
            ids = rng.choice(np.array([-1, -(2**31), 2**31 - 1, first + experts] + ([first - 1] if first else [])), routes)
        else:
            ids = first + rng.permutation(np.arange(routes) % experts)
        ids = ids.astype(np.int32).reshape(-1, 1)
        index, offsets = capi.moe_row_plan(torch.from_numpy(ids).cuda(), experts, first_expert=first)
        want_index, want_offsets = _plan(ids, experts, first)
        np.testing.assert_array_equal(index.cpu().numpy(), want_index)
        np.testing.assert_array_equal(offsets.cpu().numpy(), want_offsets)


@pytest.mark.parametrize("routes", [100, 70001])
def test_row_plan_in_place(capi, cuda, routes):
    torch = cuda
    ids = torch.randint(-1, 40, (routes,), generator=torch.Generator(device="cuda").manual_seed(routes), device="cuda", dtype=torch.int32)
    index, offsets = capi.moe_row_plan(ids, 30, first_expert=3)
    other = torch.empty_like(offsets)
    code = capi.load().catccos_b200_moe_row_plan(torch.cuda.current_stream().cuda_stream, ids.data_ptr(), routes, 30, 3, ids.data_ptr(), other.data_ptr())
    assert code == 0 and torch.equal(ids, index) and torch.equal(other, offsets)


def test_row_plan_refusals(capi, cuda):
    torch = cuda
    ids = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for experts in (0, 1025, 2**31 - 1):
        with pytest.raises(capi.CatccosError) as e:
            capi.moe_row_plan(ids, experts)
        assert e.value.code == -1
    for bad in (ids.long(), ids.t(), ids.cpu()):
        with pytest.raises(ValueError):
            capi.moe_row_plan(bad, 4)
    with pytest.raises(ValueError):
        capi.moe_row_plan(ids, 4, first_expert=-1)


# ---- combine -----------------------------------------------------------------------------------------------------------------
def _check_combine(capi, torch, y, index, weights, shared, **more):
    out = capi.moe_combine(y, index, weights, shared=shared, **more)
    live = (index >= 0) & (index < y.shape[0])
    rows = y.double()[index.long().clamp(0, max(0, y.shape[0] - 1))] if y.shape[0] else torch.zeros((*index.shape, y.shape[1]), dtype=torch.float64, device="cuda")
    parts = torch.where(live.unsqueeze(2), rows * weights.double().unsqueeze(2), 0.0)
    want, size = parts.sum(dim=1), parts.abs().sum(dim=1)
    if shared is not None:
        want, size = want + shared.double(), size + shared.double().abs()
    # top_k + 1 roundings of 2^-24 of what is added up, then half a step of the type (below its smallest normal: half of that step)
    half = {torch.bfloat16: (2.0**-8, 2.0**-134), torch.float16: (2.0**-11, 2.0**-25)}[y.dtype]
    slack = (index.shape[1] + 1) * 2.0**-24 * size
    assert bool(((out.double() - want).abs() <= slack + half[0] * (want.abs() + slack) + half[1]).all())
    return out


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,n,top_k,rows", [(1, 8, 1, 1), (3, 256, 2, 6), (130, 520, 8, 1040), (5, 1016, 9, 50), (2, 1024, 17, 40),
                                                 (16, 7168, 8, 128), (300, 24, 3, 900), (4, 1032, 4, 0)])
def test_combines(capi, cuda, tokens, n, top_k, rows, dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(tokens * 8192 + n)
    y = torch.randn((rows, n), generator=gen, device="cuda").to(getattr(torch, dtype))
    index = torch.randint(-1, rows + 2, (tokens, top_k), generator=gen, device="cuda", dtype=torch.int32)  # some dropped, some outside
    weights = torch.rand((tokens, top_k), generator=gen, device="cuda") - 0.25
    shared = torch.randn((tokens, n), generator=gen, device="cuda").to(y.dtype)
    _check_combine(capi, torch, y, index, weights, None)
    out = _check_combine(capi, torch, y, index, weights, shared)
    kept = shared.clone()
    assert capi.moe_combine(y, index, weights, shared=kept, out=kept) is kept and torch.equal(kept, out)
    none = capi.moe_combine(y, torch.full_like(index, -1), weights)
    assert bool((none == 0).all())


def test_dropped_routes_do_not_touch_their_values(capi, cuda):
    torch = cuda
    y = torch.ones((4, 64), dtype=torch.bfloat16, device="cuda")
    y[0] = float("nan")
    index = torch.tensor([[-1, 1], [2, -1], [0, 1]], dtype=torch.int32, device="cuda")
    weights = torch.tensor([[float("nan"), 2.0], [0.5, float("inf")], [0.0, 1.0]], device="cuda")
    out = capi.moe_combine(y, index, weights)
    assert bool((out[0] == 2).all()) and bool((out[1] == 0.5).all())
    assert bool(torch.isnan(out[2]).all())  # a row that is routed counts, whatever its weight


def test_rows_behind_four_gibibytes(capi, cuda):
    torch = cuda
    n, rows = 8192, 300000  # 4.9 GB
    y = torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")
    y[rows - 1], y[1] = 3.0, 1.0
    index = torch.tensor([[rows - 1, 1]], dtype=torch.int32, device="cuda")
    out = capi.moe_combine(y, index, torch.tensor([[1.0, 0.5]], device="cuda"))
    assert bool((out == 3.5).all())
    del y
    torch.cuda.empty_cache()  # a test behind this one measures what is left


def test_combine_refusals(capi, cuda):
    torch = cuda
    y = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    index, weights = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros((2, 2), device="cuda")
    for bad in ((y.float(), index, weights), (y, index.long(), weights), (y, index, weights.half()), (y, index, weights[:1]),
                (y[:, :32], index, weights), (y, index.cpu(), weights)):
        with pytest.raises(ValueError):
            capi.moe_combine(*bad)
    with pytest.raises(ValueError):
        capi.moe_combine(y, index, weights, shared=y)
    with pytest.raises(ValueError):
        capi.moe_combine(y, index, weights, out=torch.zeros((2, 64), dtype=torch.float16, device="cuda"))
    with pytest.raises(capi.CatccosError) as e:
        capi.moe_combine(y[:, :4].contiguous(), index, weights)
    assert e.value.code == -1
    assert capi.moe_combine(y, index[:0], weights[:0]).shape == (0, 64)
