"""Weights of the paged attention over bfloat16 pools (GPU): a 16-bit output is the correctly rounded value wherever
float32 arithmetic decides it.
"""

import pytest

from test_gpu_serving import BF16, F16, gen, gpu, i32, pool, u  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("qt", [BF16, F16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 4, 64), (32, 8, 128), (32, 2, 128)])
def test_bf16_pool_rounds_once(pkg, qt, heads, kv_heads, d):
    """Two or three positions a row and scores near zero, so that nothing averages out. With A <= 0.05 the score
    errors are below u; a weight carries 6u from its exponent (2^(8 + s') from a float32 argument), 4u from the
    exponential, 2u from each of sum, join and division and 4u from the products' accumulation: 20u of max|v| in
    all, taken as 32u as in test_gpu_serving.py. A value farther than that from every border between two roundings
    has to be the rounded one. (16-bit weights are off by up to 64u.)"""
    rows = 256
    lens = [2 + r % 2 for r in range(rows)]
    c, table, ref = pool(pkg, lens, 16, kv_heads, d, BF16, 5)
    q = (torch.randn((rows, heads, d), generator=gen(6), device="cuda") * 0.01).to(qt)
    out = c.attend(q, table, i32(lens))
    group, wrong = heads // kv_heads, 0
    for r in range(rows):
        k, v = (x.repeat_interleave(group, 1).transpose(0, 1) for x in ref[r])  # [heads, n, d]
        s = (k * q[r].double().unsqueeze(1)).sum(-1) * d ** -0.5
        want = (torch.softmax(s, -1).unsqueeze(-1) * v).sum(1)
        e = 32 * u * v.abs().amax(1)
        low, high = (want - e).float().to(qt), (want + e).float().to(qt)  # rounding is monotone
        wrong += int(((out[r] < low) | (out[r] > high)).sum())
    assert wrong == 0
