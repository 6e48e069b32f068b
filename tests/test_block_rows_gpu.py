"""GPU test of the rows that a dispatch allocates when it is not told how many: tokens * top_k, refused where row_index cannot name them."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k", [2**30, 2**30 - 1, 2**29])  # 2^32 rows, 2^32 - 4, 2^31
def test_more_rows_than_an_index_names(capi, cuda, top_k):
    torch = cuda
    x = torch.zeros((4, 16), dtype=torch.bfloat16, device="cuda")
    index = torch.empty((4, top_k), dtype=torch.int32, device="cuda")  # never read
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for call in (lambda: capi.moe_dispatch(x, index), lambda: capi.block_quant(x, row_index=index)):
        with pytest.raises(ValueError, match="rows"):
            call()
    assert torch.cuda.max_memory_allocated() == before  # nothing of that size was allocated first
    del index
    torch.cuda.empty_cache()


def test_rows_that_are_told_hold(capi, cuda):
    torch = cuda
    x = torch.randn((4, 16), device="cuda").to(torch.bfloat16)
    index = torch.tensor([[5, -1], [2, 9], [0, 1], [3, 7]], dtype=torch.int32, device="cuda")
    for rows in (6, 8, 12):
        out = torch.zeros((rows, 16), dtype=x.dtype, device="cuda")
        want = out.clone()
        for t, route in enumerate(index.tolist()):
            for r in route:
                if 0 <= r < rows:
                    want[r] = x[t]
        assert torch.equal(capi.moe_dispatch(x, index, out=out), want)
        assert capi.moe_dispatch(x, index, rows=rows).shape == (rows, 16) and capi.block_quant(x, row_index=index, rows=rows)[0].shape == (rows, 16)
    assert capi.moe_dispatch(x, index).shape == (8, 16)
    for rows in (2**31, -1):
        for call in (lambda: capi.moe_dispatch(x, index, rows=rows), lambda: capi.block_quant(x, row_index=index, rows=rows)):
            with pytest.raises(ValueError, match="rows"):
                call()
