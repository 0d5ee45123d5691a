"""Infinities and NaN in the paged attention's operands (GPU)."""

import math

import pytest

from test_gpu_serving import BF16, F16, F32, I8, TINY, U, gen, gpu, i32, pool, u  # noqa: F401 (gpu: the fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def check(out, lse, q, k, v, scale):
    """One row against float64: out and q [heads, d], k and v [n, kv heads, d]. A score of -infinity has weight 0, one of
    +infinity or NaN makes the head NaN, and a head that only -infinity is left of gives zeros. Finite elements carry the
    bounds of test_gpu_serving.py, taken over the positions that have weight."""
    heads, d = q.shape
    kk, vv = (x.repeat_interleave(heads // x.shape[1], 1).transpose(0, 1) for x in (k, v))
    terms = kk * q.double().unsqueeze(1)
    s = terms.sum(-1) * scale
    live = torch.isfinite(s)
    A = (terms.abs().sum(-1) * abs(scale)).masked_fill(~live, 0).amax(-1, keepdim=True)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    none = (total == 0).squeeze(-1)
    want = (p.unsqueeze(-1) * vv).sum(1) / torch.where(total == 0, torch.ones_like(total), total)
    want[none] = 0
    want_lse = (top + torch.log(total)).squeeze(-1)
    assert torch.equal(lse.double().isnan(), want_lse.isnan())
    fine = want_lse.isfinite()
    assert torch.all((lse.double() - want_lse).abs()[fine] <= (8 * A[fine, 0] + 32) * u + 2 * u * want_lse[fine].abs())
    assert torch.all(lse[none] == -math.inf) and torch.all(out[none] == 0)
    got = out.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[want.isinf()], want[want.isinf()])
    vmax = vv.abs().masked_fill(~vv.isfinite(), 0).amax((1, 2)).unsqueeze(1)
    err = torch.where(want.isfinite(), (got - want).abs(), torch.zeros_like(want))
    bound = (16 * A + 32) * u * vmax + U[out.dtype] * want.abs() + TINY[out.dtype]
    assert torch.all((err <= bound) | ~want.isfinite())
    return fine


def rows_of(c, table, n, page):
    p = torch.arange(n, device="cuda")
    return table[0, p // page].long(), p % page


@pytest.mark.parametrize("cache", [BF16, F16], ids=str)
@pytest.mark.parametrize("qt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("n,heads,kv_heads,d,page", [(70, 8, 1, 64, 16), (70, 32, 2, 128, 24), (9000, 16, 1, 128, 32),
                                                      (3, 4, 4, 64, 7)])
def test_infinite_keys_and_values(pkg, cache, qt, n, heads, kv_heads, d, page):
    """An infinite key element scores its position +-infinity by the query's sign there; an infinite value element makes
    its column +-infinity, and NaN where both signs meet."""
    c, table, ref = pool(pkg, [n], page, kv_heads, d, cache, n + d)
    q = torch.randn((1, heads, d), generator=gen(1), device="cuda").to(qt)
    q[..., 5] = torch.where(q[..., 5] < 0, q[..., 5] - 1, q[..., 5] + 1)  # (no element near zero meets the infinity)
    pg, off = rows_of(c, table, n, page)

    def put(tensor, of, position, element, value):
        tensor[pg[position], :, off[position], element] = value
        of[position, :, element] = value

    out, lse = c.attend(q, table, i32([n]), return_lse=True)
    assert check(out[0], lse[0], q[0], *ref[0], d ** -0.5).all()
    put(c.v, ref[0][1], n // 2, 7, math.inf)
    put(c.v, ref[0][1], n - 1, d - 1, -math.inf)
    put(c.v, ref[0][1], 0, 11, math.inf)
    put(c.v, ref[0][1], n - 1, 11, -math.inf)
    put(c.v, ref[0][1], 1, 20, math.nan)
    out, lse = c.attend(q, table, i32([n]), return_lse=True)
    assert check(out[0], lse[0], q[0], *ref[0], d ** -0.5).all()
    assert torch.all(out[0, :, 7] == math.inf) and torch.all(out[0, :, d - 1] == -math.inf)
    put(c.k, ref[0][0], n // 3, 5, -math.inf)
    out, lse = c.attend(q, table, i32([n]), return_lse=True)
    fine = check(out[0], lse[0], q[0], *ref[0], d ** -0.5)
    assert torch.equal(fine, q[0, :, 5] > 0)
    # the position alone: weight 0 leaves nothing
    lone = table.clone()
    lone[0, 0] = pg[n // 3]
    if page <= n // 3 and int(off[n // 3]) == 0:
        out, lse = c.attend(q, lone, i32([1]), return_lse=True)
        check(out[0], lse[0], q[0], ref[0][0][n // 3:n // 3 + 1], ref[0][1][n // 3:n // 3 + 1], d ** -0.5)


def test_position_of_infinite_score_alone(pkg):
    for cache in (BF16, F16):
        c, table, ref = pool(pkg, [1], 16, 2, 64, cache, 3)
        q = torch.randn((1, 8, 64), generator=gen(2), device="cuda")
        q[..., 5] = torch.where(torch.arange(8, device="cuda") % 2 == 0, 1.0, -1.0)
        c.k[table[0, 0], :, 0, 5] = -math.inf
        c.v[table[0, 0], :, 0, 9] = math.inf
        out, lse = c.attend(q, table, i32([1]), return_lse=True)
        assert torch.all(out[0, ::2] == 0) and torch.all(lse[0, ::2] == -math.inf)
        assert out[0, 1::2].isnan().all() and lse[0, 1::2].isnan().all()


def test_float16_overflow_of_append(pkg):
    """A key and a value beyond 65504 become infinities of a float16 pool and keep their meaning."""
    n, d = 40, 64
    c, table, _ = pool(pkg, [n], 16, 1, d, F16, 4)
    k, v = (torch.randn((n, 1, d), generator=gen(s), device="cuda") for s in (5, 6))
    k[9, 0, 3], v[20, 0, 8], v[21, 0, 9] = -1e6, 1e6, -1e6
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    c.append(k, v, table, torch.zeros_like(pos), pos)
    q = torch.randn((1, 8, d), generator=gen(7), device="cuda")
    q[..., 3] = 1.0
    out, lse = c.attend(q, table, i32([n]), return_lse=True)
    kk, vv = k.to(F16).double(), v.to(F16).double()
    assert check(out[0], lse[0], q[0], kk, vv, d ** -0.5).all()
    assert torch.all(out[0, :, 8] == math.inf) and torch.all(out[0, :, 9] == -math.inf)


@pytest.mark.parametrize("cache", [I8, BF16, F16], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite_query(pkg, cache, bad):
    """A NaN or an infinity in a query head makes that head NaN, the other heads stay; a row without positions is zeros."""
    lens = [1, 50, 200]
    c, table, ref = pool(pkg, lens, 16, 2, 64, cache, 8)
    q = torch.randn((4, 6, 64), generator=gen(9), device="cuda")
    want, want_lse = c.attend(q, table, i32(lens + [0]), seq=i32([0, 1, 2, -1]), return_lse=True)
    q[:, 4, 33] = bad
    out, lse = c.attend(q, table, i32(lens + [0]), seq=i32([0, 1, 2, -1]), return_lse=True)
    keep = [0, 1, 2, 3, 5]
    assert torch.equal(out[:, keep], want[:, keep]) and torch.equal(lse[:, keep], want_lse[:, keep])
    assert out[:3, 4].isnan().all() and lse[:3, 4].isnan().all()
    assert torch.all(out[3, 4] == 0) and lse[3, 4] == -math.inf


def test_split_row_of_infinite_scores(pkg):
    """A context over many blocks none of whose positions has weight, some with infinite values."""
    n = 20000
    for cache in (BF16, F16):
        c, table, ref = pool(pkg, [n], 16, 1, 64, cache, 12)
        q = torch.randn((1, 8, 64), generator=gen(13), device="cuda")
        q[..., 5] = torch.where(torch.arange(8, device="cuda") % 2 == 0, 1.0, -1.0)
        pg, off = rows_of(c, table, n, 16)
        c.k[pg, :, off, 5] = -math.inf
        c.v[pg[::777], :, off[::777], 9] = math.inf
        out, lse = c.attend(q, table, i32([n]), return_lse=True)
        assert torch.all(out[0, ::2] == 0) and torch.all(lse[0, ::2] == -math.inf)
        assert out[0, 1::2].isnan().all() and lse[0, 1::2].isnan().all()
