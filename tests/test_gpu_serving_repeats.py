"""Repeated calls of the paged attention and the log probabilities give the same
bits (GPU): both keep a ring of tiles per warp that copies refill while the
warp works, and results that depend on when a copy lands show only in some of
many calls. Full-size calls, since idle SMs hide it.
"""

import pytest

from test_gpu_serving import BF16, F16, F32, I8, gen, gpu, i32, pool  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def differing(call, times):
    """How many of `times` further calls differ from the first in a bit of any result."""
    first = [t.clone() for t in call()]
    count = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(times):
        count += torch.stack([(a != b).any() for a, b in zip(call(), first)]).any()
    return int(count)


@pytest.mark.parametrize("dt,rows,vocab,top_k", [(F32, 2048, 32000, 5), (F32, 1500, 20011, 20), (BF16, 2048, 32000, 5),
                                                 (F16, 40, 50021, 5)], ids=str)
def test_logprobs_repeat(pkg, dt, rows, vocab, top_k):
    x = (torch.randn((rows, vocab), generator=gen(1), device="cuda") * 2.5).to(dt)
    tokens = torch.randint(0, vocab, (rows,), generator=gen(2), device="cuda").to(torch.int32)
    assert differing(lambda: pkg.token_logprobs(x, tokens, top_k), 3000) == 0
    pkg.shim.check(pkg.load_library().tl_device_error(), "tl_device_error")


@pytest.mark.parametrize("cache,heads,kv_heads,d,page", [(I8, 32, 4, 64, 16), (F16, 40, 8, 128, 16),
                                                         (BF16, 32, 2, 128, 48), (I8, 32, 4, 64, 17)], ids=str)
def test_attend_repeat(pkg, cache, heads, kv_heads, d, page):
    lens = [(211 * i) % 2048 + 1 for i in range(48)]
    c, table, _ = pool(pkg, lens, page, kv_heads, d, cache, 11)
    q = torch.randn((len(lens), heads, d), generator=gen(3), device="cuda")
    lengths = i32(lens)
    assert differing(lambda: c.attend(q, table, lengths, return_lse=True), 3000) == 0
    pkg.shim.check(pkg.load_library().tl_device_error(), "tl_device_error")
