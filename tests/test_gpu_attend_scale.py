"""Unusual score scales of the paged attention (GPU)."""

import math

import pytest

from test_gpu_attend_nonfinite import check
from test_gpu_serving import BF16, F16, I8, gen, gpu, i32, pool  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("cache", [I8, BF16, F16], ids=str)
def test_scales_of_zero_below_zero_and_nan(pkg, cache):
    """sm_scale 0 weighs all positions alike whatever the query is; a negative one turns the scores; NaN gives NaN."""
    n = 77
    c, table, ref = pool(pkg, [n], 16, 2, 64, cache, 10)
    q = torch.randn((1, 8, 64), generator=gen(11), device="cuda")
    q[0, 1], q[0, 2], q[0, 3] = 0.0, q[0, 2] * 1e-30, q[0, 3] * 1e6
    for scale in (0.0, -0.3, 1e-30):
        out, lse = c.attend(q, table, i32([n]), sm_scale=scale, return_lse=True)
        assert check(out[0], lse[0], q[0], *ref[0], scale).all()
    out, lse = c.attend(q, table, i32([n]), sm_scale=math.nan, return_lse=True)
    assert out.isnan().all() and lse.isnan().all()
