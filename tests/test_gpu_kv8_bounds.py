"""Where 16-bit attention over the paged 8-bit KV cache can lose a result:
scores far from 0, large and tiny score caps, pages whose values are of very
unlike size or NaN, long histories, values near fp32's end, a
capacity far above the lengths.  Against plain implementations in 64 bits, as in test_gpu_kv8.py,
with tolerances that depend on what a row sees alone."""

import math

import pytest

from test_gpu_kv8 import HALF, I32, PAGE, TYPES, Cache, clean_status, near, status  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -23  # a step of fp32: what an addition that cuts loses at most
FAST_CAP = 128.0  # up to here 16-bit rows take cap - 2 cap / (e^2y + 1)


def exact(c, i, q, pos, window=0, prefix=0, cap=0.0, tc=False):
    """q [m, h, hd] of positions pos -> out, lse and their tolerances, in 64 bits.

    A score is a sum of hd products in fp32: each addition may be cut, a step U of the sum of magnitudes; eight more
    for its factors.  tanh does not widen that, and adds: up to a cap of FAST_CAP the difference of two numbers of the
    cap's size, each off by a step or two (4 U cap); above it eight steps of the score itself.  A weight is off by
    twice the largest score error of its row, and in the 16-bit types by half an fp16 step (2^-11); the capped prompt
    form's polynomial adds 2^-18.  A weight's fp16 form ends at 2^-39 of the largest weight (2^14 times it are held,
    and fp16's last half step is 2^-25), in the tcgen05 form (`tc`) at 2^-28 (the largest is held at 2^3 at least).
    Sums: a product of 16 keys is one addition to fp32 that may be cut, in runs of at most 16,384 keys; pages, and
    such runs, are joined by rounding additions.  The stored value is off by half a step of its type."""
    k, v = c.values(i)
    n, (m, h, hd) = k.shape[0], q.shape
    r = h // c.kv
    kk, vv = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
    s = torch.einsum("mhd,thd->mht", q.double(), kk) * hd ** -0.5
    mag = torch.einsum("mhd,thd->mht", q.double().abs(), kk.abs()) * hd ** -0.5
    if cap:
        s = cap * torch.tanh(s / cap)
    t = torch.arange(n, device="cuda")
    p = torch.as_tensor(list(pos), device="cuda")[:, None]
    see = (t < prefix) | ((t <= p) & ((p - t < window) if window else (t >= 0)))
    s = torch.where(see[:, None], s, -math.inf)
    ds = (hd + 8) * U * torch.where(see[:, None], mag, 0.0).amax(2)
    if cap:
        ds = ds + (4 * cap * U if cap <= FAST_CAP else 8 * U * torch.where(see[:, None], s.abs(), 0.0).amax(2))
    lse = torch.logsumexp(s, 2)
    w = torch.exp(s - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
    # a value that nobody of the call sees may be anything
    vz = torch.where(see.any(0)[:, None, None], vv, 0.0)
    out = torch.einsum("mht,thd->mhd", w, vz)
    amount = torch.einsum("mht,thd->mhd", w, vz.abs())
    sums = (min(n, 16384) / 16 + n / PAGE + 16) * U
    weight = 0.0 if c.dtype == "f32" else 2.0 ** -11 + (2.0 ** -17 if cap and tc else 0.0)
    fi = torch.finfo(TYPES[c.dtype])
    tol = HALF[c.dtype] * out.abs() + fi.tiny * fi.eps / 2 + amount * (2 * ds + sums + weight)[..., None]
    cut = torch.einsum("mt,thd->mhd", see.double(), vz.abs()) * w.amax(2)[..., None]
    tol = tol + (2.0 ** -28 if tc else 2.0 ** -39) * cut
    # twice a weight's error is exp(2 ds) - 1 <= 4 ds only for ds <= 1/2; where scores are so large that theirs is
    # beyond 1/4, any weights are right that are none below 0 and sum to 1: an output lies among the values seen
    if (ds > 0.25).any():
        most = torch.where(see[:, :, None, None], vz.abs()[None], 0.0).amax(1) * (1 + 4 * HALF[c.dtype])
        tol = torch.where((ds > 0.25)[..., None], out.abs() + most, tol)
    return out, lse, tol, ds + sums + lse.abs().nan_to_num(0, 0, 0) * U


def uses_tc(c, new):
    """The prompt form of these sizes (16-bit rows from head_dim 128 up, or 512 rows of 64)."""
    return c.dtype != "f32" and (c.hd >= 128 or new * c.h // c.kv >= 512)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("far", [2.0 ** 19, 2.0 ** 22, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28, 1e12, 1e30])
def test_huge_scores(ctx, heads, dtype, far):
    """Finite scores whose fp32 steps are whole numbers: each row is its highest key's value.

    All queries lie along one direction, one key does so at full length: its score leads by half its size or more,
    so every other weight is 0 in any precision."""
    if dtype == "f16" and far > 1e10:
        return  # out of the type's reach
    n, m = 300, 150
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(22)
    u = torch.where(torch.rand((c.hd,), generator=g, device="cuda") < 0.5, -1.0, 1.0)
    length = math.sqrt(far / math.sqrt(c.hd))  # of a query, and of the key: score = length^2 sqrt(hd)
    k, v = c.random(n, g).float().clamp(-4, 4) * (length / 64), c.random(n, g)
    k[33] = length * u
    c.append([(k.to(TYPES[dtype]), v)])
    q = (length * u * torch.linspace(0.6, 2.1, m * c.h, device="cuda").view(m, c.h, 1)).to(TYPES[dtype])
    want = c.values(0)[1][33].repeat_interleave(c.h // c.kv, 0)
    # the one weight is an fp16 operand in the 16-bit types (half a step, 2^-11), its sum is not; then a product by the
    # page's scale, a reciprocal and its product, a step each, and the stored value
    tol = want.abs() * (HALF[dtype] + (0.0 if dtype == "f32" else 2.0 ** -11) + 4 * U) + 2.0 ** -25
    for rows in (slice(0, m), slice(m - 20, m)):
        out, lse = c.prefill(q[rows], [rows.stop - rows.start])
        near(out, want.expand(out.shape), tol.expand(out.shape), "prompt")
        assert torch.isfinite(lse).all()
    for row in range(0, m, 7):
        out, lse = c.decode(q[row:row + 1])
        near(out, want[None], tol[None], "token")
        assert torch.isfinite(lse).all()
    # lse: the score, whose products' sum may be cut at each of hd additions
    top = torch.einsum("mhd,hd->mh", q[-1:].double(), c.values(0)[0][33].repeat_interleave(c.h // c.kv, 0)) * c.hd ** -0.5
    near(lse if row == m - 1 else c.decode(q[-1:])[1], top, (c.hd + 24) * U * top.abs(), "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [127.0, 129.0, 1e3, 1e4, 1e5, 1e8, 3e38])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
def test_large_caps(ctx, heads, dtype, cap):
    """A cap far above the scores leaves them as they are; scores near it and above it are bent."""
    n, m = 300, 150
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(21)
    c.append([(c.random(n, g), c.random(n, g))])
    # ordinary scores, and (as far as the type holds the query) scores of the cap's size
    for size in {2.0, min(2.0 * cap, 3e3 if dtype == "f16" else 1e30)}:
        q = c.queries(m, g, size)
        for few in (False, True):  # 64 dims: few rows take the warp form, more the tcgen05 form
            rows = slice(m - 20, m) if few else slice(0, m)
            out, lse = c.prefill(q[rows], [20 if few else m], cap=cap)
            ro, rl, to, tl = exact(c, 0, q[rows], range(n - m, n)[rows], cap=cap, tc=uses_tc(c, 20 if few else m))
            near(out, ro, to, f"prompt, {size}")
            near(lse, rl, tl, f"lse of the prompt, {size}")
        out, lse = c.decode(q[m - 1:], cap=cap)
        ro, rl, to, tl = exact(c, 0, q[m - 1:], [n - 1], cap=cap)
        near(out, ro, to, f"token, {size}")
        near(lse, rl, tl, f"lse of the token, {size}")
    assert status(ctx) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [1e-20, 1e-38, 1e-42])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
def test_tiny_caps(ctx, heads, dtype, cap):
    """A cap whose reciprocal, or that times a score, is beyond fp32: all weights are the same, of scores of 0 too."""
    n, m = 100, 70
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(23)
    k, v = c.random(n, g), c.random(n, g)
    k[7] = 0
    k[64:96] = 0  # a page of zeros: its scale is 0
    c.append([(k, v)])
    q = c.queries(m, g, 300.0)
    q[::3] = 0
    ro, rl, to, tl = exact(c, 0, q, range(n - m, n), cap=cap, tc=True)
    for few in (False, True):
        rows = slice(m - 20, m) if few else slice(0, m)
        out, lse = c.prefill(q[rows], [20 if few else m], cap=cap)
        near(out, ro[rows], to[rows], "prompt")
        near(lse, rl[rows], tl[rows], "lse of the prompt")
    for row in (m - 1, m - 2):  # a query of zeros is among them
        out, lse = c.decode(q[row:row + 1], cap=cap, lens=[n - m + row + 1])
        near(out, ro[row:row + 1], to[row:row + 1], "token")
        near(lse, rl[row:row + 1], tl[row:row + 1], "lse of the token")
    assert status(ctx) == 0


def unlike(c, n, g, places, times, base):
    """Values of size `base`, and `times` that in the tokens of `places`."""
    v = base * torch.randn((n, c.kv, c.hd), generator=g, device="cuda")
    for a, b in places:
        v[a:b] *= times
    return v.to(TYPES[c.dtype])


# (dtype, size of the ordinary values, how much larger the others are); fp16 holds 2^-24 to 2^16
UNLIKE = [("f16", 2.0 ** -12, 2.0 ** 12), ("f16", 2.0 ** -14, 2.0 ** 24), ("f16", 2.0 ** -15, 2.0 ** 28),
          ("bf16", 1.0, 2.0 ** 20), ("bf16", 2.0 ** -20, 2.0 ** 27), ("bf16", 1e-4, 2.0 ** 30), ("bf16", 1e-9, 2.0 ** 60),
          ("bf16", 1e30, 2.0 ** -100), ("bf16", 1e-36, 1.0), ("f32", 1e-4, 2.0 ** 30)]


@pytest.mark.parametrize("dtype,base,times", UNLIKE)
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (3, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("places", [[(96, 128)], [(0, 32)], [(70, 71), (200, 201)], [(290, 300)]])
def test_values_of_unlike_size(ctx, heads, dtype, base, times, places):
    """Values far larger or smaller than a row's own, in pages that it does not see (later ones, or behind its window),
    in its own page, and in sight, where they decide."""
    n = 300
    c = Cache(ctx, heads, dtype, [n, 40])
    g = torch.Generator("cuda").manual_seed(24)
    c.append([(c.random(n, g), unlike(c, n, g, places, times, base)), (c.random(40, g), c.random(40, g))])
    for window, prefix, cap in ((0, 0, 0.0), (40, 0, 0.0), (33, 5, 20.0), (0, 100, 500.0)):
        q = c.queries(n + 40, g)
        pre = [prefix, min(40, prefix)] if prefix else None
        out, lse = c.prefill(q, [n, 40], window, pre, cap)
        tc = uses_tc(c, n)
        for i, (m, r) in enumerate(((n, 0), (40, n))):
            ro, rl, to, tl = exact(c, i, q[r:r + m], range(m), window, pre[i] if pre else 0, cap, tc)
            near(out[r:r + m], ro, to, f"window {window}, prefix {prefix}, cap {cap}")
            near(lse[r:r + m], rl, tl, f"lse, window {window}, prefix {prefix}, cap {cap}")
        out, lse = c.decode(q[[n - 1, n + 39]], window, pre, cap)
        for i, m in enumerate((n, 40)):
            ro, rl, to, tl = exact(c, i, q[[(n - 1, n + 39)[i]]], [m - 1], window, pre[i] if pre else 0, cap)
            near(out[i:i + 1], ro, to, "token")
            near(lse[i:i + 1], rl, tl, "lse of the token")
    assert status(ctx) == 0


@pytest.mark.parametrize("dtype,base,times", [("f16", 2.0 ** -14, 2.0 ** 24), ("bf16", 1.0, 2.0 ** 40)])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (10, 2, 256)])
def test_values_of_unlike_size_split(ctx, heads, dtype, base, times):
    """The same behind a long history that is split: parts whose scales are alike beside parts whose are not."""
    n, m = 3001, 140
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(25)
    c.append([(c.random(n, g), unlike(c, n, g, [(1000, 1032), (2900, 2901)], times, base))])
    q = c.queries(m, g)
    for window, prefix in ((0, 0), (1900, 0), (90, 0), (64, 999)):
        out, lse = c.prefill(q, [m], window, [prefix] if prefix else None)
        ro, rl, to, tl = exact(c, 0, q, range(n - m, n), window, prefix, tc=True)
        near(out, ro, to, f"window {window}, prefix {prefix}")
        near(lse, rl, tl, f"lse, window {window}, prefix {prefix}")
    again, _ = c.prefill(q, [m], 64, [999])
    assert torch.equal(out, again)


@pytest.mark.parametrize("heads,dtype", [((8, 2, 128), "bf16"), ((4, 1, 256), "f16"), ((8, 1, 64), "bf16")])
@pytest.mark.parametrize("times", [1.0, 2.0 ** 20, 2.0 ** 35])
def test_values_of_unlike_size_missing_page(ctx, heads, dtype, times):
    """A page that is not in the pool beside pages of unlike value size: rows in front of it are as before."""
    n = 300
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(26)
    c.append([(c.random(n, g), unlike(c, n, g, [(128, 160)], times, 2.0 ** -22 if dtype == "f16" else 1.0))])
    q = c.queries(n, g)
    good, _ = c.prefill(q, [n])
    c.table[0, 3] = c.pages
    out, lse = c.prefill(q, [n])
    assert status(ctx) == 32
    assert torch.equal(out[:96], good[:96]) and torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_foreign_value_scales(ctx):
    """Scales that no append makes, in arrays that a program filled itself: negative, and near both ends of fp32."""
    c = Cache(ctx, (8, 2, 128), "bf16", [200])
    g = torch.Generator("cuda").manual_seed(27)
    c.append([(c.random(200, g), c.random(200, g))])
    q = c.queries(200, g)
    good, lse = c.prefill(q, [200])
    keep = c.vs.clone()
    for f in (-1.0, 2.0 ** -100, 2.0 ** 119):
        c.vs.copy_(keep * f)
        out, l2 = c.prefill(q, [200])
        # exact products by a power of two, until fp32's subnormal numbers: 2^-100 is not near them
        near(out.double() / f, good.double(), good.double().abs() * 2.0 ** -7 + 2.0 ** -9 * good.double().abs().max(), f"{f}")
        near(l2, lse.double(), torch.full_like(lse, 1e-4).double(), f"lse, {f}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("cap", [0.0, 25.0, 300.0])
def test_non_finite_values(ctx, heads, dtype, cap):
    """A NaN or an infinity among the values makes the outputs that see its page NaN; the weights, and so lse, are the
    keys' and the query's alone, in every form and type.  Other rows and heads are as they would be without it."""
    n = 260
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(28)
    k, v = c.random(n, g), c.random(n, g)
    v[100, 1, 5], v[101, 1, 9] = math.nan, -math.inf  # page 3, the second KV head
    c.append([(k, v)])
    q = c.queries(n, g)
    second = torch.arange(c.h, device="cuda") >= c.h // 2
    for window in (0, 20, 1):
        at = torch.arange(n, device="cuda")
        sees = (at >= 96) & (at <= 127 + window - 1 if window else True)
        bad = sees[:, None] & second
        ro, rl, to, tl = exact(c, 0, q, range(n), window, 0, cap, uses_tc(c, n))
        clean = Cache(ctx, heads, dtype, [n])
        clean.append([(k, v.nan_to_num(0, 0, 0))])
        want, _, tol, _ = exact(clean, 0, q, range(n), window, 0, cap, uses_tc(c, n))
        for few in (False, True):
            rows = slice(n - 20, n) if few else slice(0, n)
            out, lse = c.prefill(q[rows], [20 if few else n], window, cap=cap)
            assert torch.equal(torch.isnan(out).all(2), bad[rows]) and torch.equal(torch.isnan(out).any(2), bad[rows])
            near(lse, rl[rows], tl[rows], f"lse, window {window}")
            ok = ~bad[rows]
            near(out[ok], want[rows][ok], tol[rows][ok], f"out, window {window}")
        for row in (n - 1, 130, 95):
            out, lse = c.decode(q[row:row + 1], window, cap=cap, lens=[row + 1])
            assert torch.equal(torch.isnan(out).all(2)[0], bad[row]) and torch.equal(torch.isnan(out).any(2)[0], bad[row])
            near(lse, rl[row:row + 1], tl[row:row + 1], f"lse of the token, window {window}")
    assert status(ctx) == 0


ALL_ONE = 70000  # an upper bound of new rows from which a history is not split


@pytest.mark.parametrize("heads,dtype,m", [((8, 1, 64), "f16", 64), ((2, 1, 128), "f16", 40), ((1, 1, 256), "f16", 40),
                                           ((2, 1, 128), "bf16", 40)])
def test_long_sums(ctx, heads, dtype, m):
    """Sums over 300,000 keys in one piece stay in the middle.

    Positive values and nearly equal weights, so that a sum that is cut at every addition falls behind all the time:
    by a step U at most in each of a run's 16,384 / 16 = 1024 additions.  Runs, and the sums of weights by page, are
    joined by rounding additions, half a step each.  What is rounded to 16 bits, weights and outputs, is right on
    average: its mean over the outputs is below a twentieth of the half step that each may be off by."""
    n = 300000
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(29)
    for i in range(0, n, 50000):
        c.append([(c.random(50000, g), (1 + torch.rand((50000, c.kv, c.hd), generator=g, device="cuda")).to(TYPES[dtype]))])
    q = c.queries(m, g, 0.02)
    out, lse = c.prefill(q, [m], max_new=ALL_ONE)
    k, v = c.values(0)
    s = torch.einsum("mhd,td->mht", q.double(), k[:, 0]) * c.hd ** -0.5
    t = torch.arange(n, device="cuda")
    s.masked_fill_(t > torch.arange(n - m, n, device="cuda")[:, None, None], -math.inf)
    ref = torch.einsum("mht,td->mhd", torch.softmax(s, 2), v[:, 0])
    off = (out.double() - ref) / ref
    sums = 1024 * U + n / PAGE * U / 2
    assert off.mean().abs() <= sums + (HALF[dtype] + 2.0 ** -11) / 20, f"{off.mean():.3g}"
    assert off.abs().max() <= sums + HALF[dtype] + 2.0 ** -11, f"{off.abs().max():.3g}"
    near(lse, torch.logsumexp(s, 2), torch.full_like(lse, sums + 64 * U).double() + (c.hd + 8) * U, "lse")


@pytest.mark.parametrize("heads,dtype", [((8, 1, 64), "f16"), ((6, 2, 128), "bf16"), ((2, 1, 256), "f16")])
@pytest.mark.parametrize("n", [16384, 16385, 16448, 33000, 49153])
def test_long_runs(ctx, heads, dtype, n):
    """Histories of whole and broken runs whose scores rise and fall from run to run."""
    m = 70
    c = Cache(ctx, heads, dtype, [ALL_ONE])
    g = torch.Generator("cuda").manual_seed(30)
    k, v = c.random(n, g), c.random(n, g)
    size = 1 + 2 * torch.sin(torch.arange(n, device="cuda") / 6000)[:, None, None]
    c.append([((k.float() * size).to(TYPES[dtype]), v)])
    q = c.queries(m, g, 3.0)
    for window, prefix, cap in ((0, 0, 0.0), (n - 20, 0, 30.0), (9000, 12000, 0.0)):
        out, lse = c.prefill(q, [m], window, [prefix] if prefix else None, cap, max_new=ALL_ONE)
        ro, rl, to, tl = exact(c, 0, q, range(n - m, n), window, prefix, cap, True)
        near(out, ro, to, f"window {window}, prefix {prefix}, cap {cap}")
        near(lse, rl, tl, f"lse, window {window}, prefix {prefix}, cap {cap}")
    assert status(ctx) == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("n,m", [(300, 150), (2500, 33), (6000, 3)])
def test_values_near_the_end(ctx, heads, dtype, n, m):
    """Values of 1e36: a sum of them with weights up to 1 is within fp32, with weights held larger it is not."""
    c = Cache(ctx, heads, dtype, [n])
    g = torch.Generator("cuda").manual_seed(32)
    v = (1e36 * torch.randn((n, c.kv, c.hd), generator=g, device="cuda")).to(TYPES[dtype])
    v[64:96] *= 2.0 ** -60  # the tcgen05 form's fp32 pipes too, where the page is walked
    c.append([(c.random(n, g), v)])
    q = c.queries(m, g)
    for window, cap in ((0, 0.0), (40, 20.0)):
        for few in (False, True):
            rows = slice(m - min(m, 20), m) if few else slice(0, m)
            out, lse = c.prefill(q[rows], [rows.stop - rows.start], window, cap=cap)
            ro, rl, to, tl = exact(c, 0, q[rows], range(n - m, n)[rows], window, 0, cap, uses_tc(c, rows.stop - rows.start))
            near(out, ro, to, f"prompt, window {window}")
            near(lse, rl, tl, f"lse of the prompt, window {window}")
        out, lse = c.decode(q[m - 1:], window, cap=cap)
        ro, rl, to, tl = exact(c, 0, q[m - 1:], [n - 1], window, 0, cap)
        near(out, ro, to, f"token, window {window}")
        near(lse, rl, tl, f"lse of the token, window {window}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1000], [1024, 1, 0, 517]])
def test_capacity_far_above_lengths(ctx, dtype, lens):
    """Full-width heads with a table and max_len of 32,768 positions, as a batch gives them, and a few short sequences."""
    c = Cache(ctx, (32, 16, 128), dtype, [max(1, n) for n in lens], pages=200)
    wide = torch.full((len(lens), 1024), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.pps] = c.table
    c.table, c.pps = wide, 1024
    c.c.s.pages_per_seq, c.c.s.d_table = 1024, wide.data_ptr()
    g = torch.Generator("cuda").manual_seed(31)
    c.append([(c.random(n, g), c.random(n, g)) for n in lens])
    new = [min(n, 33) for n in lens]
    for window, prefix in ((0, 0), (200, 0), (200, 4)):
        pre = [min(n, prefix) for n in lens] if prefix else None
        q = c.queries(len(lens), g)
        out, lse = c.decode(q, window, pre, max_len=32768)
        for i, n in enumerate(lens):
            if n:
                ro, rl, to, tl = exact(c, i, q[i:i + 1], [n - 1], window, pre[i] if pre else 0)
                near(out[i:i + 1], ro, to, f"token of {n}")
                near(lse[i:i + 1], rl, tl, f"lse of the token of {n}")
            else:
                assert (out[i] == 0).all() and torch.isneginf(lse[i]).all()
        q = c.queries(sum(new), g)
        out, lse = c.prefill(q, new, window, pre, max_len=32768)
        r = 0
        for i, (n, m) in enumerate(zip(lens, new)):
            if m:
                ro, rl, to, tl = exact(c, i, q[r:r + m], range(n - m, n), window, pre[i] if pre else 0, tc=uses_tc(c, max(new)))
                near(out[r:r + m], ro, to, f"chunk of {n}")
                near(lse[r:r + m], rl, tl, f"lse of the chunk of {n}")
            r += m
    assert status(ctx) == 0
