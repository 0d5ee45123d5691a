"""Log probabilities of rows in which one token stands far above the rest (GPU): logprob and entropy are small
differences there, and their signs are known.
"""

import pytest

from test_gpu_serving import BF16, F16, F32, gen, gpu, u  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (40, 50021), (700, 4099), (1500, 32000)])
def test_confident_rows(pkg, dt, rows, vocab):
    """One token 15 to 20 above the largest of the others, late in the row. With the row's maximum as the reference its
    own term is exactly 1, and the sum of the others is rounded to 1's step: once for each batch of a thread that holds
    the maximum (at most vocab / 4096 + 1 of 16 or 32 elements) and for about 16 joins, u each (2u for the pair). The
    other terms (in all below 2^-3 of it) carry 8u of themselves. So |err| <= (2 (vocab / 4096 + 1) + 24) u + 8u |value|."""
    x = (torch.randn((rows, vocab), generator=gen(vocab), device="cuda") * 2).to(dt)
    g = gen(rows)
    at = vocab - 1 - torch.randint(0, vocab // 8, (rows,), generator=g, device="cuda")
    above = torch.rand(rows, generator=g, device="cuda") * 5 + 15
    peak = (x.float().amax(1) + above).to(dt)
    x[torch.arange(rows, device="cuda"), at] = peak
    r = pkg.token_logprobs(x, at.to(torch.int32), 3)
    logp = torch.log_softmax(x.double(), 1)
    want = logp.gather(1, at.unsqueeze(1)).squeeze(1)
    entropy = torch.special.entr(logp.exp()).sum(1)
    step = (2 * (vocab // 4096 + 1) + 24) * u
    assert torch.all((r.logprob.double() - want).abs() <= step + 8 * u * want.abs())
    assert torch.all((r.entropy.double() - entropy).abs() <= step + 8 * u * entropy)
    assert torch.equal(r.top_logprobs[:, 0], r.logprob)
    assert torch.all(r.logprob <= 0) and torch.all(r.entropy >= 0) and torch.all(r.top_logprobs <= 0)


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_signs_of_ordinary_rows(pkg, dt):
    """No distribution has a log probability above 0 or an entropy below 0, whatever the spread."""
    for spread in (1e-3, 0.5, 4.0, 12.0, 40.0):
        x = (torch.randn((500, 3001), generator=gen(int(spread * 1000)), device="cuda") * spread).to(dt)
        r = pkg.token_logprobs(x, x.argmax(1).to(torch.int32), 5)
        assert torch.all(r.logprob <= 0) and torch.all(r.entropy >= 0) and torch.all(r.top_logprobs <= 0)
