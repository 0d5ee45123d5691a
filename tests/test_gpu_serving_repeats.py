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


@pytest.mark.parametrize("cache,rows,heads,kv_heads,d,page", [(I8, 64, 32, 4, 64, 16), (BF16, 3, 32, 8, 128, 48)],
                         ids=str)
def test_calls_in_a_row(pkg, cache, rows, heads, kv_heads, d, page):
    """A step's calls placed behind one another as the stream takes them give what they give with the GPU idle
    between them (each call's blocks may be there before the call before has ended)."""
    steps, context = 100, 500
    pages = -(-(context + steps) // page)
    table = torch.randperm(rows * pages, generator=gen(21), device="cuda").to(torch.int32).view(rows, pages)
    cos, sin = (torch.from_numpy(t).cuda() for t in pkg.rope_tables(context + steps, d, 10000.0))
    seq = torch.arange(rows, dtype=torch.int32, device="cuda")
    prompt = torch.randn((rows * context, kv_heads, d), generator=gen(22), device="cuda")
    qkv = torch.randn((steps, rows, heads + 2 * kv_heads, d), generator=gen(23), device="cuda")
    pos = torch.arange(context, context + steps, dtype=torch.int32, device="cuda")[:, None].repeat(1, rows)
    lengths = pos + 1

    def run(idle):
        c = pkg.PagedKVCache(rows * pages, page, kv_heads, d, cache)
        at = torch.arange(context, dtype=torch.int32, device="cuda").repeat(rows)
        c.append(prompt, prompt, table, seq.repeat_interleave(context), at, cos, sin)
        q = torch.empty((rows, heads, d), device="cuda")
        out, lse = torch.empty((steps, rows, heads, d), device="cuda"), torch.empty((steps, rows, heads), device="cuda")
        k, v = (torch.empty((steps, rows, kv_heads, d), device="cuda") for _ in range(2))
        for i in range(steps):
            x = qkv[i]
            c.append(x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], table, seq, pos[i], cos, sin, q=x[:, :heads],
                     q_out=q)
            idle()
            c.attend(q, table, lengths[i], out=out[i], lse=lse[i])
            idle()
            c.read(table, seq, pos[i], k_out=k[i], v_out=v[i])
            idle()
        return out, lse, k, v

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))
