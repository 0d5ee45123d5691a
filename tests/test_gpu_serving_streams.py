"""A paged cache dropped while its calls run on another stream than the one it was made on (GPU)."""

import weakref

import pytest

from test_gpu_serving import BF16, I8, gen, gpu, i32, pool  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def check(c, calls, want):
    """Drops the only reference to cache ``c`` while ``calls(c)`` wait on a busy side stream: none of the memory that it
    has allocated goes to anybody else before they have ended."""
    held = [(t.data_ptr(), t.numel() * t.element_size()) for t in c._owned]
    busy = torch.randn((8192, 8192), device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(10):  # some 20 ms and more of work in front
            busy @ busy
        got = calls(c)
        end = torch.cuda.Event()
        end.record()
    gone = weakref.ref(c)
    del c
    assert gone() is None
    others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _, size in held for _ in range(4)]
    assert not end.query(), "the side stream had ended already"
    assert not {t.data_ptr() for t in others} & {p for p, _ in held}
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_scratch_outlives_a_dropped_cache(pkg):
    made, table, _ = pool(pkg, [500], 16, 2, 64, BF16, 2)
    q, le = torch.randn((1, 8, 64), generator=gen(3), device="cuda"), i32([500])
    check(pkg.PagedKVCache.from_tensors(made.k, made.v), lambda c: [c.attend(q, table, le), c.attend(q, table, le)],
          [made.attend(q, table, le)] * 2)


@pytest.mark.parametrize("cache", [BF16, I8], ids=str)
def test_pool_outlives_a_dropped_cache(pkg, cache):
    n = 100
    table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    k, v = (torch.randn((n, 2, 64), generator=gen(s), device="cuda") for s in (4, 5))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)

    def calls(c):
        c.append(k, v, table, seq, pos)
        return c.read(table, seq, pos)

    check(pkg.PagedKVCache(7, 16, 2, 64, cache), calls, calls(pkg.PagedKVCache(7, 16, 2, 64, cache)))
