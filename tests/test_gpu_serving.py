"""The paged-cache operators and token log probabilities against plain float64
implementations (GPU).

Tolerances, with u = 2^-24 (float32) and U the unit roundoff of the output's
type (2^-8 bfloat16, 2^-11 float16, u float32):

* appended rows: two products and one sum in float32, then one rounding:
  |err| <= 3u (|a cos| + |b sin|) + U |value| (at least half a subnormal step
  where the type has one in reach); an INT8 row is within half a step
  (1 + 1e-4) of the rotated value and uses the quantize_int8 scale;
* attention: a score is a sum of head_dim products of exact factors (the query
  in at least 22 bits) accumulated in float32. With A = max_j sum_i |q_i k_ji| *
  sm_scale its error is at most 8 u A (query split 4u, head_dim / 16 accumulation
  steps and the base change), which moves the softmax weights by twice that;
  the weights themselves and their sum carry 32 u. So
  |out err| <= (16 A + 32) u max|v| + U |out|, |lse err| <= (8 A + 32) u + 2 u |lse|;
* log probabilities: |err| <= 1e-5 + 2u(|x| + |lse|): the sum of up to 2^17 terms
  in partial sums of at most 2^10 terms (statistically 2^5 u) and exp within 4u.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, BF16, F16, I8 = torch.float32, torch.bfloat16, torch.float16, torch.int8
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 0.0, BF16: 0.0, F16: 2.0 ** -25}  # half the spacing of float16 below its smallest normal number
u = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(pkg, lens, page, kv_heads, d, dtype, seed, poison=True, spare=2):
    """A cache whose sequences hold random rows (float64 copies returned) in pages of random
    order; every row that belongs to no position is poisoned (NaN, or a NaN scale)."""
    g = gen(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    c = pkg.PagedKVCache(pages, page, kv_heads, d, dtype)
    if poison:
        if dtype == I8:
            c.k.fill_(127), c.v.fill_(-127), c.k_scale.fill_(math.nan), c.v_scale.fill_(math.nan)
        else:
            c.k.fill_(math.nan), c.v.fill_(math.nan)
    at, ref = 0, []
    for s, n in enumerate(lens):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
        p = torch.arange(n, device="cuda")
        page_of, off = table[s, (p // page)].long(), p % page
        got = []
        for t, sc in ((c.k, c.k_scale), (c.v, c.v_scale)):
            if dtype == I8:
                q = torch.randint(-127, 128, (n, kv_heads, d), generator=g, device="cuda").to(I8)
                z = torch.rand((n, kv_heads), generator=g, device="cuda") * 0.03 + 1e-3
                t[page_of, :, off], sc[page_of, :, off] = q, z
                got.append(q.double() * z.double().unsqueeze(-1))
            else:
                x = torch.randn((n, kv_heads, d), generator=g, device="cuda").to(dtype)
                t[page_of, :, off] = x
                got.append(x.double())
        ref.append(got)
    return c, table, ref


def check_attend(out, lse, q, ref_rows, scale):
    """Each row against float64; ref_rows[r] = (k, v) float64 [n, kv_heads, d] or None for an empty row."""
    n, heads, d = q.shape
    for r in range(n):
        if ref_rows[r] is None or ref_rows[r][0].shape[0] == 0:
            assert torch.all(out[r] == 0)
            assert lse is None or torch.all(lse[r] == -math.inf)
            continue
        k, v = ref_rows[r]
        group = heads // k.shape[1]
        kk, vv = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))  # [heads, n, d]
        qq = q[r].double().unsqueeze(1)
        s = (kk * qq).sum(-1) * scale
        A = ((kk * qq).abs().sum(-1) * scale).amax(-1, keepdim=True)
        want = (torch.softmax(s, -1).unsqueeze(-1) * vv).sum(1)
        vmax = vv.abs().amax((1, 2)).unsqueeze(1)
        err = (out[r].double() - want).abs()
        assert torch.all(err <= (16 * A + 32) * u * vmax + U[out.dtype] * want.abs() + TINY[out.dtype]), (r, float(err.max()))
        if lse is not None:
            wl = torch.logsumexp(s, -1)
            assert torch.all((lse[r].double() - wl).abs() <= (8 * A[:, 0] + 32) * u + 2 * u * wl.abs()), r


ALL_LENS = [1, 0, 15, 16, 17, 300, 63, 64, 65, 127, 128, 129, 2, 500]


@pytest.mark.parametrize("cache", [I8, BF16, F16], ids=str)
@pytest.mark.parametrize("qt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,d,page", [(32, 4, 64, 16), (8, 1, 128, 64), (3, 3, 64, 7), (12, 4, 128, 1),
                                                   (32, 2, 128, 24), (24, 1, 64, 100), (10, 2, 128, 128)])
def test_attend(pkg, cache, qt, heads, kv_heads, d, page):
    c, table, ref = pool(pkg, ALL_LENS, page, kv_heads, d, cache, heads * page + d)
    q = (torch.randn((len(ALL_LENS), heads, d), generator=gen(3), device="cuda") * 1.5).to(qt)
    out, lse = c.attend(q, table, i32(ALL_LENS), return_lse=True)
    check_attend(out, lse, q, ref, d ** -0.5)
    # the same inputs again give the same bits (the workspace is left as it was found)
    again, lse2 = c.attend(q, table, i32(ALL_LENS), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("cache", [I8, BF16, F16], ids=str)
@pytest.mark.parametrize("rows,n,heads,kv_heads,d,page", [(1, 40001, 32, 4, 64, 16), (1, 33333, 40, 8, 128, 48),
                                                          (3, 9000, 16, 1, 128, 32), (150, 700, 8, 8, 64, 16),
                                                          (1, 1, 1, 1, 128, 16), (700, 33, 4, 4, 64, 8)])
def test_attend_long_and_wide(pkg, cache, rows, n, heads, kv_heads, d, page):
    """Contexts split over many CTAs, and many short rows shared by one."""
    lens = [max(1, n - 37 * (r % 11)) for r in range(rows)]
    c, table, ref = pool(pkg, lens, page, kv_heads, d, cache, n)
    q = torch.randn((rows, heads, d), generator=gen(n), device="cuda") * 1.5
    out, lse = c.attend(q, table, i32(lens), return_lse=True)
    check_attend(out, lse, q, ref, d ** -0.5)


@pytest.mark.parametrize("cache", [I8, BF16, F16], ids=str)
def test_attend_rows_that_name_nothing(pkg, cache):
    """seq out of range, lengths beyond the table, negative lengths, pages that do not exist."""
    lens = [100, 64, 31]
    c, table, ref = pool(pkg, lens, 16, 2, 64, cache, 5, spare=3)
    cut = table[0].clone()  # sequence 0 loses its third page: positions 32..47 are left out
    table[0, 2] = -1
    table[1, 1] = c.num_pages + 7
    keep0 = torch.tensor([p for p in range(100) if not 32 <= p < 48], device="cuda")
    keep1 = torch.tensor([p for p in range(64) if not 16 <= p < 32], device="cuda")
    seq = i32([0, -1, 3, 1, 2, 2, 0, 1, 2**31 - 1])
    le = i32([100, 50, 50, 64, 31, -5, 0, 16, 7])
    q = torch.randn((9, 6, 64), generator=gen(1), device="cuda")
    out, lse = c.attend(q, table, le, seq=seq, return_lse=True)
    k0, v0 = ref[0]
    k1, v1 = ref[1]
    rows = [(k0[keep0], v0[keep0]), None, None, (k1[keep1], v1[keep1]), tuple(ref[2]), None, None,
            (k1[:16], v1[:16]), None]
    check_attend(out, lse, q, rows, 0.125)
    # a length beyond the table's width is cut to it: exactly the table's positions
    full, tab2, ref2 = pool(pkg, [48, 48], 16, 2, 64, cache, 6)
    o, l = full.attend(q[:2], tab2, i32([48, 2**31 - 1]), return_lse=True)
    check_attend(o, l, q[:2], [tuple(x) for x in ref2], 0.125)
    # a row all of whose pages are missing is an empty row
    tab2[1] = -1
    o, l = full.attend(q[:2], tab2, i32([48, 48]), return_lse=True)
    check_attend(o, l, q[:2], [tuple(ref2[0]), None], 0.125)
    del cut


def test_attend_views_scale_and_outputs(pkg):
    """A query that is a column block of a fused projection, a table that is a slice, sm_scale,
    outputs given, no lse, prompt rows as causal rows of one sequence."""
    c, table, ref = pool(pkg, [200, 90], 16, 4, 64, BF16, 8)
    wide = torch.zeros((2, 40), dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = table
    qkv = torch.randn((5, 32 + 8, 64), generator=gen(2), device="cuda").to(BF16)
    q = qkv[:, 4:36]
    le, seq = i32([200, 199, 1, 90, 45]), i32([0, 0, 0, 1, 1])
    out = torch.full((5, 32, 64), 7.0, dtype=BF16, device="cuda")
    got = c.attend(q, wide[:, 3:3 + table.shape[1]], le, seq=seq, sm_scale=0.3, out=out)
    assert got is out
    rows = [tuple(x[:n] for x in ref[s]) for s, n in zip(seq.tolist(), le.tolist())]
    check_attend(out, None, q, rows, 0.3)


def test_attend_large_scores_do_not_overflow(pkg):
    """Scores in the thousands: the weights are those of the running maximum; a peaked row returns its value row."""
    c, table, ref = pool(pkg, [333], 16, 1, 64, F16, 9, poison=False)
    q = torch.randn((1, 8, 64), generator=gen(4), device="cuda") * 3e3
    out, lse = c.attend(q, table, i32([333]), return_lse=True)
    k, v = ref[0]
    s = torch.einsum("hd,nd->hn", q[0].double(), k[:, 0]) / 8
    A = float((torch.einsum("hd,nd->hn", q[0].double().abs(), k[:, 0].abs()) / 8).max())
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert torch.all((lse[0].double() - torch.logsumexp(s, -1)).abs() <= 8 * A * u + 2 * u * lse[0].abs().double())
    top2 = s.topk(2, -1).values
    sure = (top2[:, 0] - top2[:, 1]) > 60
    assert sure.any()
    want = v[s.argmax(-1), 0]
    assert torch.all((out[0].double() - want).abs()[sure] <= 1e-5)


@pytest.mark.parametrize("cache", [BF16, F16, I8], ids=str)
def test_attend_extreme_magnitudes(pkg, cache):
    """Queries and values far from one: tiny and large query rows, value scales over six decades."""
    lens = [257]
    c, table, ref = pool(pkg, lens, 16, 2, 64, cache, 10)
    if cache == I8:
        z = 10.0 ** (torch.rand(257, 2, generator=gen(11), device="cuda") * 6 - 4)
        p = torch.arange(257, device="cuda")
        pg, off = table[0, p // 16].long(), p % 16
        q8 = c.v[pg, :, off].double()
        c.v_scale[pg, :, off] = z
        ref[0][1] = q8 * z.double().unsqueeze(-1)
    for mag in (1e-6, 1e-3, 20.0):
        q = torch.randn((1, 10, 64), generator=gen(12), device="cuda") * mag
        out, lse = c.attend(q, table, i32(lens), return_lse=True)
        check_attend(out, lse, q, [tuple(ref[0])], 0.125)


def test_attend_other_stream_and_graph(pkg):
    """Calls on a side stream, and a captured call replayed with new contents of the same tensors."""
    lens = [400, 77, 0]
    c, table, ref = pool(pkg, lens, 16, 4, 128, BF16, 21)
    q = torch.randn((3, 16, 128), generator=gen(22), device="cuda").to(BF16)
    le = i32(lens)
    want, lse = c.attend(q, table, le, return_lse=True)
    check_attend(want, lse, q, [tuple(x) for x in ref], 128 ** -0.5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = c.attend(q, table, le)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(q, table, le, out=out)
    q.copy_(torch.randn((3, 16, 128), generator=gen(23), device="cuda").to(BF16))
    le.copy_(i32([399, 0, 3]))
    graph.replay()
    torch.cuda.synchronize()
    # sequence 2 holds no page: its three positions are left out
    check_attend(out, None, q, [tuple(x[:399] for x in ref[0]), None, None], 128 ** -0.5)


# ------------------------------------------------------------------- append
def angles(n, d, theta=10000.0):
    inv = theta ** (-np.arange(0, d, 2, dtype=np.float32) / d)
    a = np.outer(np.arange(n, dtype=np.float32), inv)
    a = np.concatenate([a, a], -1)
    return (torch.from_numpy(f(a).astype(np.float32)).cuda() for f in (np.cos, np.sin))


def rotated(x, cos, sin, pos):
    """float64 rotation, and the sum of its terms' magnitudes."""
    h = x.shape[-1] // 2
    c, s = cos[pos].double()[:, None, :h], sin[pos].double()[:, None, :h]
    a, b = x[..., :h].double(), x[..., h:].double()
    return (torch.cat([a * c - b * s, b * c + a * s], -1),
            torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1))


def check_stored(c, table, seq, pos, want, mag, which):
    """Rows in the pool against float64 values ``want`` (terms of magnitude ``mag``)."""
    t, sc = (c.k, c.k_scale) if which == "k" else (c.v, c.v_scale)
    pg = table[seq.long(), (pos // c.page_size).long()].long()
    got = t[pg, :, (pos % c.page_size).long()]
    if c.dtype == I8:
        z = sc[pg, :, (pos % c.page_size).long()]
        peak = want.abs().amax(-1)
        tol = 3 * u * mag.amax(-1)
        step = torch.where(peak == 0, torch.ones_like(peak), peak / 127)
        assert torch.all((z.double() - step).abs() <= tol / 127 + 2 * u * step)
        err = (got.double() * z.double().unsqueeze(-1) - want).abs()
        assert torch.all(err <= 0.5 * (1 + 1e-4) * z.double().unsqueeze(-1) + 3 * u * mag)
        assert int(got.abs().max()) <= 127
    else:
        assert torch.all((got.double() - want).abs() <= 3 * u * mag + U[c.dtype] * want.abs() * (1 + 1e-3) + TINY[c.dtype])


@pytest.mark.parametrize("cache", [I8, BF16, F16], ids=str)
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("heads,kv_heads,d,page,lens", [(32, 4, 64, 16, [1]), (8, 8, 128, 7, [5, 64, 1, 130]),
                                                        (3, 1, 64, 64, [700, 3]), (16, 2, 128, 1, [9])])
def test_append_prompts_and_read(pkg, cache, dt, heads, kv_heads, d, page, lens):
    c, table, _ = pool(pkg, lens, page, kv_heads, d, cache, 31)
    before = [t.clone() for t in (c.k, c.v)]
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(torch.int32).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).cuda()
    n = seq.numel()
    cos, sin = angles(max(lens) + 3, d)
    # columns of one fused projection, with extra columns between them
    qkv = (torch.randn((n, heads + 2 * kv_heads + 2, d), generator=gen(32), device="cuda") * 2).to(dt)
    q, k, v = qkv[:, 1:1 + heads], qkv[:, 1 + heads:1 + heads + kv_heads], qkv[:, 2 + heads + kv_heads:]
    k[0, 0] = 0  # a row of zeros
    keep = qkv.clone()
    qr = c.append(k, v, table, seq, pos, cos, sin, q=q)
    assert torch.equal(qkv, keep) and qr.dtype == dt and qr.shape == (n, heads, d)
    for x, which in ((k, "k"), (v, "v")):
        want, mag = rotated(x, cos, sin, pos.long()) if which == "k" else (x.double(), torch.zeros_like(x).double())
        check_stored(c, table, seq, pos, want, mag, which)
    wq, mq = rotated(q, cos, sin, pos.long())
    assert torch.all((qr.double() - wq).abs() <= 3 * u * mq + U[dt] * wq.abs() * (1 + 1e-3) + TINY[dt])
    # every row that was not appended is as it was
    pg, off = table[seq.long(), (pos // page).long()].long(), (pos % page).long()
    for t, b in zip((c.k, c.v), before):
        rest = torch.ones(t.shape[0], t.shape[2], dtype=torch.bool, device="cuda")
        rest[pg, off] = False
        x, y = (z.transpose(1, 2)[rest] for z in (t, b))
        assert torch.equal(x.nan_to_num(5.0) if x.is_floating_point() else x, y.nan_to_num(5.0) if y.is_floating_point() else y)
    # read back: what is stored, times its scale, rounded once
    for out_dt in (F32, BF16, F16):
        rk, rv = c.read(table, seq, pos, dtype=out_dt)
        for got, t, sc in ((rk, c.k, c.k_scale), (rv, c.v, c.v_scale)):
            x = t[pg, :, off].float()
            if cache == I8:
                x = x * sc[pg, :, off].unsqueeze(-1)
            assert torch.equal(got, x.to(out_dt))
    # rows that were read go into another pool as they are, without angles
    d2, tab2, _ = pool(pkg, lens, 5, kv_heads, d, F16 if cache == F16 else BF16, 33)
    rk, rv = c.read(table, seq, pos, dtype=F32)
    assert d2.append(rk, rv, tab2, seq, pos) is None
    ak, av = d2.read(tab2, seq, pos, dtype=F32)
    assert torch.equal(ak, rk.to(d2.dtype).float()) and torch.equal(av, rv.to(d2.dtype).float())


def test_append_int8_is_the_quantize_rule(pkg):
    """The INT8 rows and scales are bit for bit the float32 rule of quantize_int8 on each rotated row."""
    from oracle import golden as G
    n, kv, d = 200, 4, 64
    c, table, _ = pool(pkg, [n], 16, kv, d, I8, 41)
    cos, sin = angles(n, d)
    k, v = (torch.randn((n, kv, d), generator=gen(s), device="cuda") * 3 for s in (42, 43))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    c.append(k, v, table, torch.zeros_like(pos), pos, cos, sin)
    x, cs, sn = k.cpu().numpy(), cos.cpu().numpy()[:, None], sin.cpu().numpy()[:, None]
    rot = np.concatenate([-x[..., d // 2:], x[..., :d // 2]], -1)
    pg, off = table[0, (pos // 16).long()].long(), (pos % 16).long()
    for y, t, sc in ((x * cs + rot * sn, c.k, c.k_scale), (v.cpu().numpy(), c.v, c.v_scale)):
        got, z = t[pg, :, off].cpu().numpy(), sc[pg, :, off].cpu().numpy()
        for i in range(n):
            for h in range(kv):
                want, scale = G.quantize_int8(y[i, h])
                assert np.float32(scale) == z[i, h]
                np.testing.assert_array_equal(got[i, h], want)


def test_append_skips_what_names_no_row(pkg):
    lens = [40, 20]
    c, table, ref = pool(pkg, lens, 16, 2, 64, BF16, 51)
    table[1, 1] = -1
    cos, sin = angles(30, 64)
    #            fine  pad  no such seq  no angle  no page  beyond the table  negative position
    seq = i32([0, -1, 2, 0, 1, 1, 0])
    pos = i32([5, 3, 3, 33, 17, 29, -1])
    before = c.k.clone(), c.v.clone()
    k, v, q = (torch.randn((7, h, 64), generator=gen(h), device="cuda") for h in (2, 2, 6))
    qr = c.append(k[:, :2], v, table, seq, pos, cos, sin, q=q)
    changed = [(x.nan_to_num(9.0) != y.nan_to_num(9.0)).any(-1).any(1) for x, y in zip((c.k, c.v), before)]
    for ch in changed:
        assert ch.nonzero().tolist() == [[int(table[0, 0]), 5]]
    want, mag = rotated(q, cos, sin, pos.long().clamp(0, 29))
    live = torch.tensor([0, 1, 2, 4, 5], device="cuda")
    assert torch.all((qr.double() - want).abs()[live] <= 4 * u * mag[live] + 1e-30)
    assert torch.all(qr[3] == 0) and torch.all(qr[6] == 0)
    rk, rv = c.read(table, seq, pos, dtype=F16)
    assert torch.all(rk[[1, 2, 4, 5, 6]] == 0) and torch.all(rv[[1, 2, 4, 5, 6]] == 0)
    assert torch.equal(rk[3], ref[0][0][33].to(F16))  # no angle: read as it was


def test_append_in_place_and_nonfinite(pkg):
    c, table, _ = pool(pkg, [33], 16, 2, 128, I8, 61)
    cos, sin = angles(33, 128)
    pos = torch.arange(33, dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(pos)
    q = torch.randn((33, 4, 128), generator=gen(62), device="cuda")
    k, v = (torch.randn((33, 2, 128), generator=gen(s), device="cuda") for s in (63, 64))
    k[7, 1, 5], v[9, 0, 127] = math.nan, -math.inf
    want = c.append(k, v, table, zero, pos, cos, sin, q=q.clone())
    got = c.append(k, v, table, zero, pos, cos, sin, q=q, q_out=q)
    assert got is q and torch.equal(q, want)
    rk, rv = c.read(table, zero, pos)
    bad = torch.zeros((33, 2), dtype=torch.bool, device="cuda")
    bad[7, 1] = True
    assert torch.equal(torch.isnan(rk).all(-1), bad) and torch.isfinite(rk[~bad]).all()
    bad[7, 1], bad[9, 0] = False, True
    assert torch.equal(torch.isnan(rv).all(-1), bad) and torch.isfinite(rv[~bad]).all()


@pytest.mark.parametrize("cache", [I8, BF16], ids=str)
def test_offsets_beyond_32_bits(pkg, cache):
    """A pool of more than 2^31 elements (and, in 16 bits, 2^32 bytes): rows in its last pages."""
    kv, d, page = 8, 128, 64
    pages = 2 ** 31 // (kv * d * page) + 40
    c = pkg.PagedKVCache(pages, page, kv, d, cache)
    n = 300
    table = torch.arange(pages - 1, pages - 1 - 5, -1, dtype=torch.int32, device="cuda").unsqueeze(0).contiguous()
    cos, sin = angles(n, d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    k, v = (torch.randn((n, kv, d), generator=gen(s), device="cuda") for s in (71, 72))
    c.append(k, v, table, torch.zeros_like(pos), pos, cos, sin)
    assert not c.k[: pages - 5].any()
    rk, rv = c.read(table, torch.zeros_like(pos), pos)
    tol = 0.6 * 5 / 127 if cache == I8 else 2.0 ** -8 * 6
    assert torch.all((rv - v).abs() <= tol) and torch.all((rk - rotated(k, cos, sin, pos.long())[0]).abs() <= tol)
    q = torch.randn((1, 16, d), generator=gen(73), device="cuda")
    out, lse = c.attend(q, table, i32([n]), return_lse=True)
    check_attend(out, lse, q, [(rk.double(), rv.double())], d ** -0.5)


# ----------------------------------------------------------------- logprobs
def check_logprobs(r, x, tokens, top_k):
    """A row-by-row float64 reference with the documented rules."""
    xd = x.double()
    rows, vocab = x.shape
    for i in range(rows):
        row = xd[i]
        bad = bool(torch.isnan(row).any() or (row == math.inf).any())
        none = not bad and bool((row == -math.inf).all())
        lse = float(torch.logsumexp(row, 0))
        if tokens is not None:
            t, got = int(tokens[i]), float(r.logprob[i])
            if t < 0:
                assert got == 0
            elif bad or t >= vocab:
                assert math.isnan(got)
            elif none or float(row[t]) == -math.inf:
                assert got == -math.inf
            else:
                assert abs(got - (float(row[t]) - lse)) <= 1e-5 + 2 * u * (abs(float(row[t])) + abs(lse))
        got = float(r.entropy[i])
        if bad:
            assert math.isnan(got)
        elif none:
            assert got == 0
        else:
            p = torch.softmax(row, 0)  # takes the maximum off first: the log-sum-exp of a row near 1e38 absorbs its logarithm
            h = float(torch.special.entr(p).sum())
            assert abs(got - h) <= 1e-5 * (1 + h)
        if not top_k:
            continue
        ids, lps = r.top_ids[i].tolist(), r.top_logprobs[i].double()
        if bad:
            assert ids == [-1] * top_k and bool(torch.isnan(lps).all())
            continue
        order = torch.sort(row + 0.0, descending=True, stable=True)
        live = min(top_k, int((row > -math.inf).sum()))
        assert ids == order.indices[:live].tolist() + [-1] * (top_k - live)
        want = order.values[:live] - lse
        assert torch.all((lps[:live] - want).abs() <= 1e-5 + 2 * u * (order.values[:live].abs() + abs(lse)))
        assert torch.all(lps[live:] == -math.inf)


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (1, 32000, 20), (3, 31, 32), (2, 50021, 5), (5, 257, 7),
                                              (300, 2049, 3), (1, 131071, 32), (17, 8, 0), (64, 1000, 1)])
def test_logprobs(pkg, dt, rows, vocab, top_k):
    x = (torch.randn((rows, vocab), generator=gen(vocab), device="cuda") * 4).to(dt)
    tokens = torch.randint(0, vocab, (rows,), generator=gen(rows), device="cuda").to(torch.int32)
    check_logprobs(pkg.token_logprobs(x, tokens, top_k), x, tokens, top_k)


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_logprobs_many_rows_agree_with_one(pkg, dt):
    """Every row of a large call is the row's own call, bit for bit in ids and within rounding in values."""
    x = (torch.randn((700, 4099), generator=gen(81), device="cuda") * 3).to(dt)
    tokens = torch.randint(0, 4099, (700,), generator=gen(82), device="cuda").to(torch.int32)
    many = pkg.token_logprobs(x, tokens, 9)
    check_logprobs(many, x, tokens, 9)
    for i in (0, 5, 699):
        one = pkg.token_logprobs(x[i:i + 1], tokens[i:i + 1], 9)
        assert torch.equal(one.top_ids[0], many.top_ids[i])
        assert torch.allclose(one.top_logprobs[0], many.top_logprobs[i], rtol=0, atol=2e-5)


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("vocab", [40, 3001, 70000])
def test_logprobs_masks_ties_and_nonfinite(pkg, dt, vocab):
    g = gen(91)
    x = (torch.randn((16, vocab), generator=g, device="cuda") * 3).to(dt)
    low = torch.finfo(dt).min
    x[0] = -math.inf                                   # nothing left
    x[1] = -math.inf
    x[1, vocab - 1] = 2.0                              # one token left
    x[2, 1:] = -math.inf
    x[3] = low                                         # the type's lowest value everywhere: a uniform row
    x[4] = low
    x[4, vocab // 2] = 1.0
    x[5] = 1.5                                         # all equal: ids 0, 1, 2, ...
    x[6, vocab // 3] = math.nan
    x[7, 3] = math.inf
    x[8, 5], x[8, 6] = math.inf, math.nan
    x[9] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.9, torch.tensor(-math.inf, device="cuda").to(dt), x[9])
    x[10] = torch.arange(vocab, device="cuda").to(dt).neg()          # descending (with ties in 16 bits)
    x[11] = torch.arange(vocab, device="cuda").float().clamp_max(60000).to(dt)  # ascending
    x[12] = 0.0
    x[12, ::2] = -0.0                                  # zeros of both signs are equal
    x[13] = torch.randint(0, 3, (vocab,), generator=g, device="cuda").to(dt)    # three values
    x[14] = -math.inf
    x[14, ::7] = low
    tokens = torch.randint(0, vocab, (16,), generator=g, device="cuda").to(torch.int32)
    tokens[15], tokens[13] = vocab, -1
    tokens[1] = vocab - 1
    for top_k in (1, 5, 32):
        check_logprobs(pkg.token_logprobs(x, tokens, top_k), x, tokens, top_k)
    r = pkg.token_logprobs(x, None, 4)
    assert r.logprob is None
    check_logprobs(r, x, None, 4)


def test_logprobs_strided_and_unaligned(pkg):
    """Rows of a wider matrix that start at any element."""
    for dt in (F32, BF16, F16):
        wide = (torch.randn((6, 5003), generator=gen(95), device="cuda") * 3).to(dt)
        for start, n in ((0, 5003), (1, 5000), (3, 4097), (7, 33), (5002, 1)):
            x = wide[:, start:start + n]
            tokens = torch.randint(0, n, (6,), generator=gen(96), device="cuda").to(torch.int32)
            check_logprobs(pkg.token_logprobs(x, tokens, 6), x, tokens, 6)


def test_logprobs_large_offsets(pkg):
    """Rows whose element offsets pass 2^31."""
    x = torch.zeros((2, 40), dtype=BF16, device="cuda")
    big = torch.empty(2 ** 31 + 4096, dtype=BF16, device="cuda")
    view = big.as_strided((2, 40), (2 ** 31 + 8, 1))
    x.copy_(torch.randn((2, 40), generator=gen(97), device="cuda"))
    view.copy_(x)
    tokens = i32([3, 39])
    check_logprobs(pkg.token_logprobs(view, tokens, 3), x, tokens, 3)


# ----------------------------------------------------------------- refusals
def test_refusals(pkg):
    c, table, _ = pool(pkg, [20], 16, 2, 64, BF16, 1)
    q = torch.zeros((1, 4, 64), device="cuda")
    kv = torch.zeros((1, 2, 64), device="cuda")
    one, cos = i32([1]), torch.zeros((8, 64), device="cuda")
    bad = [
        lambda: pkg.PagedKVCache(4, 16, 2, 96),
        lambda: pkg.PagedKVCache(0, 16, 2, 64),
        lambda: pkg.PagedKVCache(4, 16, 2, 64, torch.float32),
        lambda: pkg.PagedKVCache.from_tensors(c.k, c.v[:, :1].contiguous()),
        lambda: pkg.PagedKVCache.from_tensors(c.k.transpose(1, 2), c.v.transpose(1, 2)),
        lambda: pkg.PagedKVCache.from_tensors(c.k.to(I8), c.v.to(I8)),
        lambda: pkg.PagedKVCache.from_tensors(c.k, c.v, torch.zeros(c.k.shape[:3], device="cuda"), None),
        lambda: c.attend(q[:, :3], table, one),                       # heads not a multiple
        lambda: c.attend(q[..., :32].contiguous(), table, one),       # head_dim
        lambda: c.attend(q.double(), table, one),
        lambda: c.attend(q.cpu(), table, one),
        lambda: c.attend(q, table.long(), one),
        lambda: c.attend(q, table[0], one),
        lambda: c.attend(q, table, one.long()),
        lambda: c.attend(q, table, i32([1, 2])),
        lambda: c.attend(q.expand(2, 4, 64), table, i32([1, 2])),     # rows that overlap
        lambda: c.attend(torch.zeros((2, 4, 64), device="cuda"), table, i32([1, 1])),  # more rows than sequences
        lambda: c.attend(torch.zeros((1, 4, 128), device="cuda")[..., ::2], table, one),
        lambda: c.attend(torch.zeros(4 * 64 + 1, device="cuda")[1:].view(1, 4, 64), table, one),
        lambda: c.attend(q, table, one, out=torch.zeros((1, 4, 64), dtype=BF16, device="cuda")),
        lambda: c.append(kv, kv[:, :1], table, one, one, cos, cos),
        lambda: c.append(kv, kv.half(), table, one, one, cos, cos),
        lambda: c.append(kv, kv, table, one, one, cos, None),
        lambda: c.append(kv, kv, table, one, one, cos[:, :32].contiguous(), cos[:, :32].contiguous()),
        lambda: c.append(kv, kv, table, one, one, q=q),
        lambda: c.append(kv, kv, table, one, one, cos, cos, q=q.half()),
        lambda: c.append(kv, kv, table, one, one, cos, cos, q_out=q),
        lambda: c.read(table, one, one, dtype=I8),
        lambda: c.read(table, one, i32([1, 2])),
        lambda: pkg.token_logprobs(cos, one),
        lambda: pkg.token_logprobs(cos, None, 33),
        lambda: pkg.token_logprobs(cos, None, -1),
        lambda: pkg.token_logprobs(cos.double(), None),
        lambda: pkg.token_logprobs(cos.cpu(), None),
        lambda: pkg.token_logprobs(cos.t(), None),
        lambda: pkg.token_logprobs(cos.expand(8, 64)[:1].expand(8, 64), None),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    # nothing to do is no error
    assert c.attend(q[:0], table, one[:0]).shape == (0, 4, 64)
    assert c.append(kv[:0], kv[:0], table, one[:0], one[:0], cos, cos, q=q[:0]).shape == (0, 4, 64)
    assert c.read(table, one[:0], one[:0])[0].shape == (0, 2, 64)
    assert pkg.token_logprobs(cos[:0], None, 2).top_ids.shape == (0, 2)


def test_c_entry_refuses_bad_arguments(pkg):
    """The C entries return a status for every argument the header excludes."""
    lib = pkg.load_library()
    c, table, _ = pool(pkg, [20], 16, 2, 64, BF16, 1)
    q = torch.zeros((1, 4, 64), device="cuda")
    one = i32([1])
    need = lib.tl_paged_attn_workspace_bytes(4, 2, 64)
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    good = dict(q=q.data_ptr(), seq=one.data_ptr(), le=one.data_ptr(), tab=table.data_ptr(), out=out.data_ptr(), lse=0,
                w=work.data_ptr(), wb=need, qs=256, ts=2, dt=0, n=1, mp=2, rows=1, heads=4, sc=0.125)

    def call(cache=c._ref, **kw):
        return lib.tl_paged_attn_decode(cache, pkg.serving._ATTEND.pack(*{**good, **kw}.values()), None)

    assert call() == 0
    assert call(cache=None) == 16 and lib.tl_paged_attn_decode(c._ref, None, None) == 16
    for kw in (dict(q=0), dict(dt=3), dict(dt=9), dict(qs=255), dict(qs=128), dict(le=0), dict(tab=0), dict(n=0),
               dict(mp=0), dict(ts=1), dict(rows=0), dict(heads=3), dict(heads=0), dict(out=0), dict(w=0),
               dict(q=q.data_ptr() + 4)):
        assert call(**kw) == 16, kw
    assert call(wb=need - 1) == 17 and call(seq=0, rows=2) == 17 and call(mp=2**30, ts=2**30) == 17
    for fn in (lib.tl_paged_append, lib.tl_paged_read):
        assert fn(c._ref, None, None) == 16 and fn(None, b"\0" * 256, None) == 16 and fn(c._ref, b"\0" * 256, None) == 16
    assert lib.tl_token_logprobs(None, None) == 16 and lib.tl_token_logprobs(b"\0" * 256, None) == 16
    for h, kv, d in ((0, 1, 64), (4, 0, 64), (5, 2, 64), (4, 2, 80)):
        assert lib.tl_paged_attn_workspace_bytes(h, kv, d) == 0
    torch.cuda.synchronize()
