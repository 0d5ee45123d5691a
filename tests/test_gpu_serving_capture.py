"""A paged cache whose first calls are captured in a graph (GPU)."""

import pytest

from test_gpu_serving import BF16, I8, check_attend, gen, gpu, i32, pool  # noqa: F401 (gpu: the module's fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("cache", [I8, BF16], ids=str)
def test_first_call_captured_then_an_ordinary_one(pkg, cache):
    """Nothing that a later call needs is left to the graph: an ordinary call between capture and first replay, and both
    with more heads than before, allocate nothing beyond their outputs and give the rows."""
    lens = [9001, 40]  # the first is split over many blocks
    c, table, ref = pool(pkg, lens, 16, 2, 64, cache, 3)
    le = i32(lens)
    qs = [torch.randn((2, h, 64), generator=gen(h), device="cuda") for h in (4, 40)]
    outs = [torch.zeros_like(q) for q in qs]
    captured = [torch.zeros_like(q) for q in qs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.cuda.memory_allocated()
        for q, o in zip(qs, captured):
            c.attend(q, table, le, out=o)
        assert torch.cuda.memory_allocated() == held
    held = torch.cuda.memory_allocated()
    for q, o in zip(qs, outs):
        c.attend(q, table, le, out=o)
    assert torch.cuda.memory_allocated() == held
    graph.replay()
    torch.cuda.synchronize()
    for q, o, got in zip(qs, outs, captured):
        check_attend(o, None, q, [tuple(x) for x in ref], 0.125)
        assert torch.equal(o, got)


def test_no_cache_is_made_under_capture(pkg):
    c, _, _ = pool(pkg, [20], 16, 2, 64, BF16, 1)
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError):
            pkg.PagedKVCache(4, 16, 2, 64)
        with pytest.raises(RuntimeError):
            pkg.PagedKVCache.from_tensors(c.k, c.v)
    graph.replay()
    assert x.tolist() == [1, 1, 1, 1]
