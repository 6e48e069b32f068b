"""GPU tests of the combination's gradient on both sides of the sizes at which a CTA takes one, two or four routes."""
import pytest

import test_moe_grad_gpu as grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,n,top_k", [(2048, 64, 4), (2047, 64, 4), (1366, 72, 3), (1365, 72, 3), (1639, 512, 5), (1500, 528, 6), (4100, 136, 2), (700, 1024, 3),
                                            (700, 1040, 3), (171, 520, 3), (170, 520, 3), (1366, 1032, 3), (700, 1024, 1), (5, 64, 7)])
def test_combine_grad(capi, cuda, tokens, n, top_k, kind):
    grad.test_combine_grad(capi, cuda, tokens, n, top_k, kind)
