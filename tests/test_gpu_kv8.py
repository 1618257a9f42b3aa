"""The paged 8-bit KV cache (vrt_kv8_append, _read, _decode, _prefill) on a
B200 against plain implementations in 64 bits.

What a cache stands for is compared bit for bit: scale = fl32(max|x| / 127)
and codes rounded half to even are exactly defined, and code * scale is one
fp32 product.  Attention is compared over the values that the cache stands
for, within what its roundings can add up to (see `Ref.attend`)."""

import math

import numpy as np
import pytest

import vrt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE = vrt.KV8_PAGE
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# a stored value is within half a step of the computed one
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
I32 = dict(dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream's handle


def quantised(rows):
    """[n, kv, hd] rows -> the fp32 values that a cache of them stands for, as float64."""
    n, kv, hd = rows.shape
    x = torch.zeros((-(-n // PAGE) * PAGE, kv, hd), dtype=torch.float64, device=rows.device)
    x[:n] = rows.double()
    x = x.view(-1, PAGE, kv, hd)
    bad = ~torch.isfinite(x).all(dim=3).all(dim=1)
    s = (x.abs().amax((1, 3)) / 127).float()
    s[bad] = math.nan
    sd = s.double()[:, None, :, None]
    q = torch.where(sd > 0, torch.round(x / torch.where(sd > 0, sd, 1.0)).clamp(-127, 127), torch.zeros_like(x))
    y = (q * sd).float().double()
    return y.reshape(-1, kv, hd)[:n]


class Cache:
    """A cache over torch arrays whose pages are dealt out in random order; pages that nobody holds are full of
    garbage (codes of any value, NaN scales)."""

    def __init__(self, ctx, heads, dtype, capacity, seed=0, spare=5, pages=None):
        self.h, self.kv, self.hd = heads
        self.dtype, self.ctx = dtype, ctx
        g = torch.Generator().manual_seed(seed)
        per = [-(-c // PAGE) for c in capacity]
        self.pps, self.pages = max(per), pages or sum(per) + spare
        self.n = len(capacity)
        dt = TYPES[dtype]
        self.k = torch.randint(-128, 128, (self.pages, self.kv, PAGE, self.hd), dtype=torch.int8, device="cuda")
        self.v = torch.randint(-128, 128, (self.pages, self.kv, self.hd, PAGE), dtype=torch.int8, device="cuda")
        self.ks = torch.full((self.pages, self.kv), math.nan, device="cuda")
        self.vs = torch.full((self.pages, self.kv), math.nan, device="cuda")
        self.kt = torch.full((self.n, self.kv, PAGE, self.hd), math.nan, dtype=dt, device="cuda")
        self.vt = torch.full((self.n, self.kv, PAGE, self.hd), math.nan, dtype=dt, device="cuda")
        order = torch.randperm(self.pages, generator=g).int()
        table, at = torch.full((self.n, self.pps), -1, dtype=torch.int32), 0
        for i, p in enumerate(per):
            table[i, :p] = order[at:at + p]
            at += p
        self.table = table.cuda()
        self.c = vrt.Kv8Cache(ctx, self.kv, self.hd, self.pages, self.n, self.pps, dtype, k=self.k.data_ptr(),
                              v=self.v.data_ptr(), k_scale=self.ks.data_ptr(), v_scale=self.vs.data_ptr(),
                              k_tail=self.kt.data_ptr(), v_tail=self.vt.data_ptr(), table=self.table.data_ptr())
        self.rows = [(torch.zeros((0, self.kv, self.hd), dtype=dt, device="cuda"),) * 2 for _ in capacity]

    def random(self, n, g):
        x = torch.randn((n, self.kv, self.hd), generator=g, device="cuda")
        return (x * torch.exp(0.5 * torch.randn((n, 1, 1), generator=g, device="cuda"))).to(TYPES[self.dtype])

    def append(self, new):
        """new: per sequence a pair of rows (or None)."""
        e = torch.zeros((0, self.kv, self.hd), dtype=TYPES[self.dtype], device="cuda")
        new = [p or (e, e) for p in new]
        cu = np.cumsum([0] + [p[0].shape[0] for p in new])
        start = torch.tensor([r[0].shape[0] for r in self.rows], **I32)
        k, v = torch.cat([p[0] for p in new] + [e + 0]), torch.cat([p[1] for p in new])
        most = max(1, max(p[0].shape[0] for p in new))
        if k.shape[0]:
            cut = torch.tensor(cu, **I32)
            self.c.append(k.data_ptr(), v.data_ptr(), start.data_ptr(), self.n, cu=cut.data_ptr(), max_new=most,
                          stream=stream())
        self.rows = [(torch.cat([r[0], p[0]]), torch.cat([r[1], p[1]])) for r, p in zip(self.rows, new)]
        torch.cuda.synchronize()

    def lens(self):
        return [r[0].shape[0] for r in self.rows]

    def read(self, lo=None, hi=None):
        hi = hi or self.lens()
        lo = lo or [0] * self.n
        cu = np.cumsum([0] + [b - a for a, b in zip(lo, hi)])
        k = torch.full((int(cu[-1]) + 1, self.kv, self.hd), -7.0, device="cuda")
        v = torch.full_like(k, -7.0)
        st, cut = torch.tensor(lo, **I32), torch.tensor(cu, **I32)
        self.c.read(st.data_ptr(), self.n, k.data_ptr(), v.data_ptr(), cu=cut.data_ptr(),
                    max_rows=max(1, max(b - a for a, b in zip(lo, hi))), stream=stream())
        torch.cuda.synchronize()
        assert (k[-1] == -7).all() and (v[-1] == -7).all()  # rows behind the last
        return [(k[cu[i]:cu[i + 1]], v[cu[i]:cu[i + 1]]) for i in range(self.n)]

    def values(self, i):
        return quantised(self.rows[i][0]), quantised(self.rows[i][1])

    def expect(self, i, q, pos, window=0, prefix=0, cap=0.0, scale=None):
        """q [m, h, hd] of positions pos -> out, lse and their tolerances, in 64 bits.

        Tolerances: scores are sums of hd products in fp32 (each addition may be cut, a step 2^-23 of the sum of
        magnitudes), scaled, capped (tanh within 4 steps of the cap) and rounded; a weight exp(s) is then off by twice
        the largest score error, and by half an fp16 step where weights are fp16 operands (16-bit types), which are
        kept to 2^-39 of the largest weight, 1 (2^14 times them is held, and fp16 ends at 2^-25), or, where they are
        multiplied by their page's value scale, to 2^-28 of the largest with the largest scale (held times 2^3 while
        the largest weight is at most 2^12 above 1); sums over
        the keys add a step for each; the stored value half a step of its type (below the smallest normal number,
        2^-14 in fp16, a step is finfo.tiny * finfo.eps whatever the value: half of it is added)."""
        k, v = self.values(i)
        n, (m, h, hd) = k.shape[0], q.shape
        scale = hd ** -0.5 if scale is None else scale
        r = h // self.kv
        kk, vv = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
        s = torch.einsum("mhd,thd->mht", q.double(), kk) * scale
        mag = torch.einsum("mhd,thd->mht", q.double().abs(), kk.abs()) * abs(scale)
        if cap:
            s = cap * torch.tanh(s / cap)
        t = torch.arange(n, device="cuda")
        p = torch.as_tensor(pos, device="cuda")[:, None]
        see = (t < prefix) | ((t <= p) & ((p - t < window) if window else (t >= 0)))
        s = torch.where(see[:, None], s, -math.inf)
        mag = torch.where(see[:, None], mag, 0.0)
        lse = torch.logsumexp(s, 2) if n else torch.full((m, h), -math.inf, dtype=torch.float64, device="cuda")
        w = torch.exp(s - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
        vz = torch.where(see.any(0)[:, None, None], vv, 0.0)
        out = torch.einsum("mht,thd->mhd", w, vz)
        amount = torch.einsum("mht,thd->mhd", w, vz.abs())
        u = 2.0 ** -23
        ds = (hd + 8) * u * mag.amax(2) + 4 * cap * u if n else torch.zeros((m, h), dtype=torch.float64, device="cuda")
        weight = 0.0 if self.dtype == "f32" else 2.0 ** -11
        fi = torch.finfo(TYPES[self.dtype])
        tol = HALF[self.dtype] * out.abs() + fi.tiny * fi.eps / 2 + amount * (2 * ds + (n + 16) * u + weight)[..., None]
        if self.dtype == "f32":
            tol = tol + 2.0 ** -39 * torch.where(torch.isfinite(vz), vz.abs(), 0.0).sum(0)
        elif n:
            tol = tol + 2.0 ** -28 * n * vv.nan_to_num(0, 0, 0).abs().max()
        return out, lse, tol, ds + (n + 16) * u + lse.abs().nan_to_num(0, 0, 0) * u

    def workspace(self, new, most):
        b = self.c.workspace_bytes(self.h, self.n, new, most)
        return torch.full((max(b, 16),), 255, dtype=torch.uint8, device="cuda"), b

    def decode(self, q, window=0, prefix=None, cap=0.0, max_len=None, lens=None, scale=None):
        most = max_len or self.pps * PAGE
        ws, nb = self.workspace(1, most)
        out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
        ln = torch.tensor(lens or self.lens(), **I32)
        pre = torch.tensor(prefix, **I32) if prefix else None
        self.c.decode(q.data_ptr(), ln.data_ptr(), self.n, self.h, out.data_ptr(), max_len=most, window=window,
                      softcap=cap, scale=scale, prefix=pre.data_ptr() if prefix else None, lse=lse.data_ptr(),
                      workspace=ws.data_ptr(), workspace_bytes=nb, stream=stream())
        torch.cuda.synchronize()
        return out, lse

    def prefill(self, q, new, window=0, prefix=None, cap=0.0, max_len=None, max_new=None, scale=None):
        cu = torch.tensor(np.cumsum([0] + list(new)), **I32)
        most, mn = max_len or self.pps * PAGE, max_new or max(1, max(new))
        ws, nb = self.workspace(mn, most)
        out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda")
        ln = torch.tensor(self.lens(), **I32)
        pre = torch.tensor(prefix, **I32) if prefix else None
        self.c.prefill(q.data_ptr(), ln.data_ptr(), cu.data_ptr(), self.n, self.h, out.data_ptr(), max_new=mn,
                       max_len=most, window=window, softcap=cap, scale=scale, prefix=pre.data_ptr() if prefix else None,
                       lse=lse.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=nb, stream=stream())
        torch.cuda.synchronize()
        return out, lse

    def queries(self, n, g, size=2.0):
        return (size * torch.randn((n, self.h, self.hd), generator=g, device="cuda")).to(TYPES[self.dtype])


def status(ctx):
    import ctypes as C
    w = C.c_uint32()
    torch.cuda.synchronize()
    vrt.check(vrt.lib().vrt_pipeline_status(ctx.h, C.byref(w)))
    return w.value


def near(got, ref, tol, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), what
    ok = torch.isfinite(ref)
    over = ((got - ref).abs() - tol)[ok]
    assert over.numel() == 0 or over.max() <= 0, f"{what}: over by {over.max():.3g}, at most {tol[ok].max():.3g} allowed"


def fill(c, lens, seed=3):
    g = torch.Generator("cuda").manual_seed(seed)
    c.append([(c.random(n, g), c.random(n, g)) for n in lens])
    return g


HEADS = [(4, 1, 256), (32, 16, 128), (8, 2, 64)]


@pytest.fixture(autouse=True)
def clean_status(ctx):
    status(ctx)
    yield


# ---------------------------------------------------------------- append, read


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", HEADS)
def test_append_any_pieces(ctx, heads, dtype):
    """Sequences brought in pieces of many sizes stand for what they would in one piece, after each piece."""
    c = Cache(ctx, heads, dtype, [200, 70, 33, 1])
    g = torch.Generator("cuda").manual_seed(1)
    for piece in ([1, 33, 0, 1], [31, 1, 32, 0], [1, 1, 0, 0], [64, 0, 0, 0], [5, 30, 1, 0], [90, 4, 0, 0]):
        c.append([(c.random(n, g), c.random(n, g)) if n else None for n in piece])
        for i, (k, v) in enumerate(c.read()):
            rk, rv = c.values(i)
            assert torch.equal(k.double(), rk) and torch.equal(v.double(), rv), (piece, i)
    assert status(ctx) == 0
    lo = [7, 32, 31, 0]
    for i, (k, v) in enumerate(c.read(lo, [190, 69, 33, 1])):
        assert torch.equal(k.double(), c.values(i)[0][lo[i]:lo[i] + k.shape[0]])
        assert torch.equal(v.double(), c.values(i)[1][lo[i]:lo[i] + v.shape[0]])


def test_append_single_rows(ctx):
    """Token by token without offsets, rows inside wider packed rows, growing and equal scales."""
    c = Cache(ctx, (8, 2, 64), "bf16", [70, 70])
    g = torch.Generator("cuda").manual_seed(2)
    wide = torch.randn((70, 2, 8 + 4, 64), generator=g, device="cuda").to(torch.bfloat16)  # q | k | v
    for t in range(70):
        start = torch.tensor([t, t], **I32)
        row = wide[t].reshape(2, -1)
        c.c.append(row.data_ptr() + 2 * 8 * 64, row.data_ptr() + 2 * 10 * 64, start.data_ptr(), 2, row_stride=12 * 64,
                   stream=stream())
        torch.cuda.synchronize()
    for i in range(2):
        c.rows[i] = (wide[:, i, 8:10].contiguous(), wide[:, i, 10:12].contiguous())
    for i, (k, v) in enumerate(c.read()):
        rk, rv = c.values(i)
        assert torch.equal(k.double(), rk) and torch.equal(v.double(), rv)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_append_halves_and_extremes(ctx, hd):
    """Quotients on and next to a half, zeros, the smallest and largest numbers."""
    c = Cache(ctx, (1, 1, hd), "f32", [32 * 8])
    x = torch.zeros((32 * 8, 1, hd))
    f = x.view(8, 32, hd)
    f[0] = ((torch.arange(32 * hd).view(32, hd) % 255) - 127) + 0.5        # halves of a scale of 1
    f[0].clamp_(-126.5, 126.5)
    f[0, 0, 0] = 127.0
    f[1] = torch.nextafter(f[0], torch.tensor(math.inf))                    # just above them
    f[1, 0, 0] = 127.0
    f[2] = f[0] * (1 / 3)                                                   # a scale that is not a power of two
    f[4] = 1e-45 * torch.arange(32 * hd).view(32, hd) % 1e-42               # subnormal, scale 0 or the smallest
    f[5] = 3e38 * torch.linspace(-1, 1, 32 * hd).view(32, hd)
    f[6] = 1e-37 * torch.linspace(-1, 1, 32 * hd).view(32, hd)              # 1 / scale is not finite
    f[7, 5, 3] = -2.0                                                       # one value
    x = x.cuda()
    c.append([(x, x.flip(0).contiguous())])
    (k, v), = c.read()
    rk, rv = c.values(0)
    assert torch.equal(k.double(), rk) and torch.equal(v.double(), rv)


def test_append_non_finite(ctx):
    """A page and head with an infinity or NaN reads NaN, its neighbours do not; also when it comes later."""
    c = Cache(ctx, (2, 2, 64), "f16", [100])
    g = torch.Generator("cuda").manual_seed(4)
    k, v = c.random(100, g), c.random(100, g)
    k[40, 1, 3], v[70, 0, 9] = math.inf, math.nan
    c.append([(k[:35], v[:35])])
    c.append([(k[35:], v[35:])])
    (a, b), = c.read()
    rk, rv = c.values(0)
    assert torch.equal(torch.isnan(a.double()), torch.isnan(rk)) and torch.isnan(a[32:64, 1]).all() and torch.isfinite(a[:, 0]).all()
    assert torch.equal(torch.isnan(b.double()), torch.isnan(rv)) and torch.isnan(b[64:96, 0]).all()
    near(a, rk, torch.zeros_like(rk), "k")
    near(b, rv, torch.zeros_like(rv), "v")


# ------------------------------------------------------------------- decode

GROUPS = [(4, 1, 256), (32, 16, 128), (8, 2, 64), (3, 1, 64), (8, 1, 128), (10, 2, 128), (5, 5, 64), (16, 2, 256)]
LENS = [0, 1, 31, 32, 33, 64, 65, 200, 517, 1025]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", GROUPS)
@pytest.mark.parametrize("window,prefix,cap", [(0, 0, 0.0), (40, 0, 0.0), (33, 5, 20.0), (1, 0, 0.0)])
def test_decode(ctx, heads, dtype, window, prefix, cap):
    c = Cache(ctx, heads, dtype, [max(1, n) for n in LENS], seed=sum(heads))
    g = fill(c, LENS)
    q = c.queries(len(LENS), g)
    pre = [min(n, prefix + 7 * i) for i, n in enumerate(LENS)] if prefix else None
    out, lse = c.decode(q, window, pre, cap)
    for i, n in enumerate(LENS):
        ro, rl, to, tl = c.expect(i, q[i:i + 1], [n - 1], window, pre[i] if pre else 0, cap)
        near(out[i:i + 1], ro, to, f"out of length {n}")
        near(lse[i:i + 1], rl, tl, f"lse of length {n}")
    assert status(ctx) == 0


@pytest.mark.parametrize("heads,dtype,n", [((4, 1, 256), "f32", 9000), ((2, 1, 128), "bf16", 20011), ((8, 1, 64), "f16", 12345)])
def test_decode_long(ctx, heads, dtype, n):
    """One long sequence on few heads: the history is split over the GPU and joined."""
    c = Cache(ctx, heads, dtype, [n, 5])
    g = fill(c, [n, 5])
    q = c.queries(2, g, 4.0)
    out, lse = c.decode(q)
    for i, m in enumerate((n, 5)):
        ro, rl, to, tl = c.expect(i, q[i:i + 1], [m - 1])
        near(out[i:i + 1], ro, to, "out")
        near(lse[i:i + 1], rl, tl, "lse")
    again, _ = c.decode(q)
    assert torch.equal(out, again)  # sums are in one order


def test_decode_far_pages(ctx):
    """Pages behind the first 4 GiB of the pool."""
    pages = 36000  # 131,072 bytes of keys each: 4.7 GB
    c = Cache(ctx, (16, 16, 256), "bf16", [300, 64], pages=pages)
    table = torch.full((2, c.pps), -1, dtype=torch.int32)
    table[0, :10] = torch.arange(pages - 1, pages - 11, -1)
    table[1, :2] = torch.tensor([32767, 32768])
    c.table.copy_(table)
    g = fill(c, [300, 64])
    for i, (k, v) in enumerate(c.read()):
        rk, rv = c.values(i)
        assert torch.equal(k.double(), rk) and torch.equal(v.double(), rv)
    q = c.queries(2, g)
    out, _ = c.decode(q)
    for i, n in enumerate((300, 64)):
        ro, _, to, _ = c.expect(i, q[i:i + 1], [n - 1])
        near(out[i:i + 1], ro, to, "out")
    new = [120, 64]
    q = c.queries(sum(new), g)
    out, _ = c.prefill(q, new)
    ro, _, to, _ = c.expect(0, q[:120], range(180, 300))
    near(out[:120], ro, to, "prefill")


@pytest.mark.parametrize("dtype", TYPES)
def test_decode_extreme_scores(ctx, dtype):
    """One key far above the others, scores of hundreds, values of very unlike size by page."""
    c = Cache(ctx, (8, 2, 128), dtype, [700])
    g = torch.Generator("cuda").manual_seed(6)
    k, v = c.random(700, g), c.random(700, g)
    k[333] *= 20
    v[64:96] *= 200
    v[320:352] *= 0.01
    c.append([(k, v)])
    for size in (0.01, 1.0, 8.0):
        q = c.queries(1, g, size)
        out, lse = c.decode(q)
        ro, rl, to, tl = c.expect(0, q, [699])
        near(out, ro, to, f"out at {size}")
        near(lse, rl, tl, f"lse at {size}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,qs,ks", [(-0.2, 1.0, 1.0), (0.0, 1.0, 1.0), (0.1, 1e-3, 1e3), (0.1, 1e4, 1e-4), (1e3, 1e-2, 1e-2)])
def test_scales(ctx, dtype, scale, qs, ks):
    """Negative and zero score scales; small queries on large keys and the other way round."""
    c = Cache(ctx, (8, 2, 64), dtype, [300])
    g = torch.Generator("cuda").manual_seed(12)
    c.append([((c.random(300, g).float() * ks).to(TYPES[dtype]), c.random(300, g))])
    q = (c.queries(150, g).float() * qs).to(TYPES[dtype])
    for cap in (0.0, 5.0):
        out, lse = c.prefill(q, [150], cap=cap, scale=scale)
        ro, rl, to, tl = c.expect(0, q, range(150, 300), cap=cap, scale=scale)
        near(out, ro, to, "prompt")
        near(lse, rl, tl, "lse of the prompt")
        out, lse = c.decode(q[149:], cap=cap, scale=scale)
        near(out, ro[149:], to[149:], "token")
        near(lse, rl[149:], tl[149:], "lse of the token")


def test_far_magnitudes(ctx):
    """f32 rows near both ends of the type whose products are ordinary."""
    c = Cache(ctx, (4, 2, 128), "f32", [200])
    g = torch.Generator("cuda").manual_seed(13)
    for qs in (1e-35, 1e33):
        c.rows = [(c.rows[0][0][:0], c.rows[0][1][:0])]
        c.append([(c.random(200, g) / qs, c.random(200, g))])
        q = c.queries(100, g) * qs
        out, lse = c.prefill(q, [100])
        ro, rl, to, tl = c.expect(0, q, range(100, 200))
        near(out, ro, to, "prompt")
        out, lse = c.decode(q[99:])
        near(out, ro[99:], to[99:], "token")
        near(lse, rl[99:], tl[99:], "lse")


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_non_finite(ctx, dtype):
    """Non-finite keys and values outside the window leave no trace; in sight they make NaN."""
    c = Cache(ctx, (4, 2, 64), dtype, [160])
    g = torch.Generator("cuda").manual_seed(8)
    k, v = c.random(160, g), c.random(160, g)
    k[10], v[20], v[40] = math.inf, math.nan, -math.inf
    c.append([(k, v)])
    q = c.queries(1, g)
    out, lse = c.decode(q, window=90)
    ro, rl, to, tl = c.expect(0, q, [159], 90)
    assert torch.isfinite(ro).all()
    near(out, ro, to, "out")
    near(lse, rl, tl, "lse")
    assert torch.isnan(c.decode(q)[0]).all()
    q = c.queries(40, g)
    out, _ = c.prefill(q, [40], window=50)
    ro, _, to, _ = c.expect(0, q, range(120, 160), 50)
    assert torch.isfinite(ro).all()
    near(out, ro, to, "prefill")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", ["k", "v"])
def test_non_finite_in_sight(ctx, dtype, which):
    """One page and head with a NaN: the rows and heads that see the page give NaN, all others do not."""
    c = Cache(ctx, (4, 2, 64), dtype, [200])
    g = torch.Generator("cuda").manual_seed(9)
    k, v = c.random(200, g), c.random(200, g)
    (k if which == "k" else v)[100, 1, 5] = math.nan  # page 3, KV head 1: query heads 2 and 3
    c.append([(k, v)])
    q = c.queries(1, g)
    out, _ = c.decode(q)
    assert torch.isfinite(out[0, :2]).all() and torch.isnan(out[0, 2:]).all()
    q = c.queries(200, g)
    for window, cap in ((0, 0.0), (20, 0.0), (0, 25.0), (1, 25.0)):
        out, _ = c.prefill(q, [200], window=window, cap=cap)
        sees = torch.arange(200) >= 96
        if window:
            sees &= torch.arange(200) <= 127 + window - 1
        assert torch.equal(torch.isnan(out).all(2).cpu(), sees[:, None] & torch.tensor([False, False, True, True]))
        assert torch.equal(torch.isnan(out).any(2).cpu(), sees[:, None] & torch.tensor([False, False, True, True]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("window", [0, 1, 2])
@pytest.mark.parametrize("heads,value", [((8, 2, 64), math.nan), ((8, 2, 128), math.nan), ((8, 2, 64), math.inf), ((8, 2, 128), -math.inf)])
def test_non_finite_query(ctx, dtype, cap, window, heads, value):
    """A NaN or an infinity in a query gives NaN in its own token and head alone, whatever the key that it sees."""
    c = Cache(ctx, heads, dtype, [130])
    g = fill(c, [130])
    q = c.queries(130, g)
    q[17, 3, 5] = q[38, 0, 63] = q[127, 7, 0] = value
    bad = torch.zeros((130, 8), dtype=torch.bool, device="cuda")
    bad[17, 3] = bad[38, 0] = bad[127, 7] = True
    out, lse = c.prefill(q, [130], window=window, cap=cap)
    assert torch.equal(torch.isnan(out).all(2), bad) and torch.equal(torch.isnan(out).any(2), bad)
    assert torch.equal(torch.isnan(lse), bad)
    out, lse = c.decode(q[127:128], window=window, cap=cap)
    assert torch.equal(torch.isnan(out).all(2), bad[127:128]) and torch.equal(torch.isnan(out).any(2), bad[127:128])


@pytest.mark.parametrize("heads,dtype", [((8, 2, 128), "bf16"), ((4, 1, 256), "f16"), ((8, 1, 64), "bf16"), ((4, 2, 128), "f32")])
def test_prompt_without_a_page(ctx, heads, dtype):
    """A page that is not in the pool is left out of a prompt's attention; an upper bound of rows far above the rows."""
    c = Cache(ctx, heads, dtype, [600, 600])
    g = fill(c, [500, 450])
    q = c.queries(500, g)
    good, _ = c.prefill(q, [300, 200], max_new=600)
    assert status(ctx) == 0
    c.table[0, 5] = c.pages + 7
    out, lse = c.prefill(q, [300, 200], max_new=600)
    assert status(ctx) == 32
    assert torch.equal(out[300:], good[300:])
    r = c.h // c.kv
    k, v = c.values(0)
    keep = torch.ones(500, dtype=torch.bool, device="cuda")
    keep[160:192] = False
    t = torch.arange(500, device="cuda")
    see = keep & (t <= torch.arange(200, 500, device="cuda")[:, None])
    s = torch.einsum("mhd,thd->mht", q[:300].double(), k.repeat_interleave(r, 1)) * c.hd ** -0.5
    s = torch.where(see[:, None], s, -math.inf)
    ref = torch.einsum("mht,thd->mhd", torch.softmax(s, 2), v.repeat_interleave(r, 1))
    _, _, tol, tl = c.expect(0, q[:300], range(200, 500))
    # the weights' sum is smaller by what the page had: tolerances grow with it
    grow = torch.exp(torch.logsumexp(torch.einsum("mhd,thd->mht", q[:300].double(), k.repeat_interleave(r, 1)) * c.hd ** -0.5
                                     + torch.where((t <= torch.arange(200, 500, device="cuda")[:, None])[:, None], 0.0, -math.inf), 2)
                     - torch.logsumexp(s, 2))
    near(out[:300], ref, tol * grow[..., None] + HALF[dtype] * ref.abs(), "out")
    near(lse[:300], torch.logsumexp(s, 2), tl, "lse")


@pytest.mark.parametrize("dtype", TYPES)
def test_taken_back(ctx, dtype):
    """A sequence taken back within its last page, and to a multiple of a page, then grown on."""
    c = Cache(ctx, (4, 2, 64), dtype, [200])
    g = fill(c, [110])
    for keep in (100, 97, 96, 64):
        c.rows = [(c.rows[0][0][:keep], c.rows[0][1][:keep])]
        c.append([(c.random(20, g), c.random(20, g))])
        (k, v), = c.read()
        rk, rv = c.values(0)
        assert torch.equal(k.double(), rk) and torch.equal(v.double(), rv), keep


def test_out_of_range(ctx):
    """A page outside the pool is left out, a length beyond the table or max_len is cut, and the status says so."""
    c = Cache(ctx, (8, 2, 64), "f32", [128, 128, 128])
    g = fill(c, [128, 100, 128])
    q = c.queries(3, g)
    good, _ = c.decode(q)
    assert status(ctx) == 0
    keep = c.table.clone()
    c.table[0, 3], c.table[2, 0] = c.pages, -5
    out, _ = c.decode(q)
    assert status(ctx) == 32
    assert torch.equal(out[1], good[1])
    k, v = c.values(0)
    s = torch.einsum("hd,thd->ht", q[0].double(), k[:96].repeat_interleave(4, 1)) / 8
    ref = torch.einsum("ht,thd->hd", torch.softmax(s, 1), v[:96].repeat_interleave(4, 1))
    assert (out[0].double() - ref).abs().max() < 1e-4
    pf, _ = c.prefill(q, [1, 1, 1])
    assert status(ctx) == 32 and (pf - out).abs().max() < 1e-4
    c.table.copy_(keep)
    out, _ = c.decode(q, lens=[128, 100, 1000])  # longer than the row of the table: as long as the row
    assert status(ctx) == 32 and torch.equal(out, good)
    out, _ = c.decode(q, lens=[-3, 100, 128])
    assert status(ctx) == 32 and (out[0] == 0).all() and torch.equal(out[1:], good[1:])
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs, c.kt, c.vt)]
    x = torch.ones((3, 2, 64), device="cuda")
    start = torch.tensor([128, -1, 5000], **I32)
    c.c.append(x.data_ptr(), x.data_ptr(), start.data_ptr(), 3, stream=stream())
    assert status(ctx) == 32
    for a, b in zip(before, (c.k, c.v, c.ks, c.vs, c.kt, c.vt)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    c.c.read(start.data_ptr(), 3, x.data_ptr(), x.data_ptr(), stream=stream())
    assert status(ctx) == 32 and (x == 1).all()
    cu = torch.tensor([0, 1, 0, 9], **I32)  # falling, and more rows than max_new
    start = torch.tensor([64, 64, 64], **I32)
    x = torch.full((9, 2, 64), 3.0, device="cuda")
    c.c.read(start.data_ptr(), 3, x.data_ptr(), x.data_ptr(), cu=cu.data_ptr(), max_rows=2, stream=stream())
    assert status(ctx) == 32 and (x[2:] == 3).all()


# ------------------------------------------------------------------ prefill


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", GROUPS)
@pytest.mark.parametrize("window,prefix,cap", [(0, 0, 0.0), (40, 0, 0.0), (33, 5, 20.0), (1, 0, 0.0), (0, 70, 0.0)])
def test_prefill(ctx, heads, dtype, window, prefix, cap):
    lens, new = [1, 70, 33, 300, 40, 129, 513], [1, 70, 2, 131, 0, 128, 40]
    c = Cache(ctx, heads, dtype, lens, seed=sum(heads))
    g = fill(c, lens)
    q = c.queries(sum(new) + 3, g)
    pre = [min(n, prefix + 7 * i) for i, n in enumerate(lens)] if prefix else None
    out, lse = c.prefill(q, new, window, pre, cap)
    assert (out[sum(new):] == 9).all() and (lse[sum(new):] == 9).all()  # rows behind the last sequence
    r = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        if not m:
            continue
        ro, rl, to, tl = c.expect(i, q[r:r + m], range(n - m, n), window, pre[i] if pre else 0, cap)
        near(out[r:r + m], ro, to, f"out of {m} at {n}")
        near(lse[r:r + m], rl, tl, f"lse of {m} at {n}")
        r += m
    assert status(ctx) == 0


@pytest.mark.parametrize("heads,dtype,n,m", [((32, 16, 128), "bf16", 1500, 1500), ((4, 1, 256), "f32", 900, 900),
                                             ((8, 2, 64), "f16", 4100, 77), ((4, 1, 256), "bf16", 6000, 5),
                                             ((2, 1, 128), "f32", 5000, 33)])
def test_prefill_long(ctx, heads, dtype, n, m):
    c = Cache(ctx, heads, dtype, [n])
    g = fill(c, [n])
    q = c.queries(m, g, 3.0)
    out, lse = c.prefill(q, [m])
    ro, rl, to, tl = c.expect(0, q, range(n - m, n))
    near(out, ro, to, "out")
    near(lse, rl, tl, "lse")
    again, _ = c.prefill(q, [m])
    assert torch.equal(out, again)


def test_prefill_rows_without_keys(ctx):
    """More query rows than tokens: rows of positions before the first see nothing."""
    c = Cache(ctx, (8, 2, 64), "bf16", [64, 64])
    g = fill(c, [10, 20])
    q = c.queries(35, g)
    out, lse = c.prefill(q, [15, 20])
    assert (out[:5] == 0).all() and torch.isneginf(lse[:5]).all()
    ro, rl, to, tl = c.expect(0, q[5:15], range(10))
    near(out[5:15], ro, to, "out")
    ro, rl, to, tl = c.expect(1, q[15:], range(20))
    near(out[15:], ro, to, "out")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(ctx, dtype):
    """Queries inside packed rows, outputs inside wider rows whose rest stays."""
    c = Cache(ctx, (8, 2, 64), dtype, [100, 40])
    g = fill(c, [100, 40])
    for new in (None, [30, 40]):
        m = sum(new) if new else 2
        packed = torch.randn((m, 12 * 64), generator=g, device="cuda").to(TYPES[dtype])
        q = packed[:, :512].reshape(m, 8, 64).contiguous()
        want = (c.prefill(q, new) if new else c.decode(q))[0]
        wide = torch.full((m, 9 * 64), 5.0, device="cuda").to(TYPES[dtype])
        ws, nb = c.workspace(max(new) if new else 1, 128)
        ln = torch.tensor(c.lens(), **I32)
        more = dict(q_stride=768, out_stride=576, workspace=ws.data_ptr(), workspace_bytes=nb, stream=stream(), max_len=128)
        if new:
            cu = torch.tensor([0, 30, 70], **I32)
            c.c.prefill(packed.data_ptr(), ln.data_ptr(), cu.data_ptr(), 2, 8, wide.data_ptr(), max_new=40, **more)
        else:
            c.c.decode(packed.data_ptr(), ln.data_ptr(), 2, 8, wide.data_ptr(), **more)
        torch.cuda.synchronize()
        assert torch.equal(wide[:, :512].reshape(m, 8, 64), want) and (wide[:, 512:] == 5).all()


# ----------------------------------------------------------- used together


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_then_tokens(ctx, dtype):
    """A prompt in chunks, then token by token, as a server does; prompt and single-token attention agree."""
    c = Cache(ctx, (8, 2, 128), dtype, [150, 90])
    g = torch.Generator("cuda").manual_seed(11)
    for piece in ([40, 17], [33, 50]):
        c.append([(c.random(n, g), c.random(n, g)) for n in piece])
        q = c.queries(sum(piece), g)
        out, _ = c.prefill(q, piece, window=64)
        r = 0
        for i, m in enumerate(piece):
            n = c.lens()[i]
            ro, _, to, _ = c.expect(i, q[r:r + m], range(n - m, n), 64)
            near(out[r:r + m], ro, to, "chunk")
            r += m
    for _ in range(20):
        c.append([(c.random(1, g), c.random(1, g)) for _ in range(2)])
        q = c.queries(2, g)
        out, _ = c.decode(q, window=64)
        pf, _ = c.prefill(q, [1, 1], window=64)
        for i, n in enumerate(c.lens()):
            ro, _, to, _ = c.expect(i, q[i:i + 1], [n - 1], 64)
            near(out[i:i + 1], ro, to, "token")
            near(pf[i:i + 1], ro, to, "token as a prompt")


def test_captured_and_on_another_stream(ctx):
    """append + decode + prefill captured in a graph, replayed with lengths that changed on the device; two graphs
    with a workspace each."""
    c = Cache(ctx, (8, 2, 64), "bf16", [400, 400])
    g = fill(c, [250, 31])
    kv = c.random(2, g), c.random(2, g)
    q, out, out2 = c.queries(2, g), torch.zeros((2, 8, 64), dtype=torch.bfloat16, device="cuda"), None
    out2 = torch.zeros_like(out)
    start, lens = torch.tensor([250, 31], **I32), torch.tensor([251, 32], **I32)
    cu = torch.tensor([0, 1, 2], **I32)
    ws, nb = c.workspace(1, 416)
    ws2, nb2 = c.workspace(1, 416)

    def step(o, w, n, first):
        st = torch.cuda.current_stream().cuda_stream
        if first:
            c.c.append(kv[0].data_ptr(), kv[1].data_ptr(), start.data_ptr(), 2, stream=st)
            c.c.decode(q.data_ptr(), lens.data_ptr(), 2, 8, o.data_ptr(), max_len=416, workspace=w.data_ptr(),
                       workspace_bytes=n, stream=st)
        else:
            c.c.prefill(q.data_ptr(), lens.data_ptr(), cu.data_ptr(), 2, 8, o.data_ptr(), max_new=1, max_len=416,
                        workspace=w.data_ptr(), workspace_bytes=n, stream=st)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(out, ws, nb, True)
        step(out2, ws2, nb2, False)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        step(out, ws, nb, True)
    with torch.cuda.graph(g2):
        step(out2, ws2, nb2, False)
    for _ in range(3):
        kv[0].copy_(c.random(2, g)), kv[1].copy_(c.random(2, g)), q.copy_(c.queries(2, g))
        torch.cuda.synchronize()
        out.zero_(), out2.zero_()
        g1.replay(), g2.replay()
        torch.cuda.synchronize()
        c.rows = [(torch.cat([r[0], kv[0][i:i + 1]]), torch.cat([r[1], kv[1][i:i + 1]])) for i, r in enumerate(c.rows)]
        for i, n in enumerate(c.lens()):
            ro, _, to, _ = c.expect(i, q[i:i + 1], [n - 1])
            near(out[i:i + 1], ro, to, "captured decode")
            near(out2[i:i + 1], ro, to, "captured prefill")
        start += 1
        lens += 1


def test_workspace_too_small(ctx):
    c = Cache(ctx, (4, 1, 256), "bf16", [20000])
    q, ln = c.queries(1, fill(c, [100])), torch.tensor([100], **I32)
    need = c.c.workspace_bytes(4, 1, 1, 20000)
    if need:
        with pytest.raises(vrt.VrtError, match="workspace"):
            c.c.decode(q.data_ptr(), ln.data_ptr(), 1, 4, q.data_ptr(), max_len=20000, workspace=None, stream=stream())
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        with pytest.raises(vrt.VrtError, match="workspace"):
            c.c.decode(q.data_ptr(), ln.data_ptr(), 1, 4, q.data_ptr(), max_len=20000, workspace=ws.data_ptr(),
                       workspace_bytes=need - 1, stream=stream())


def test_no_sequences(ctx):
    c = Cache(ctx, (4, 1, 64), "f32", [32])
    p = c.k.data_ptr()
    c.c.append(p, p, p, 0, stream=stream())
    c.c.read(p, 0, p, p, stream=stream())
    c.c.decode(p, p, 0, 4, p, max_len=32, stream=stream())
    c.c.prefill(p, p, p, 0, 4, p, max_new=1, max_len=32, stream=stream())
    torch.cuda.synchronize()


def test_owned_arrays(ctx):
    """A cache whose arrays the binding allocates, without torch."""
    c = vrt.Kv8Cache(ctx, 2, 64, 6, 2, 3, "f32")
    c.set_table(np.array([[5, 0, 2], [1, 3, 4]]))
    with pytest.raises(vrt.VrtError, match="table"):
        c.set_table(np.zeros((3, 2)))
    x = np.random.default_rng(0).standard_normal((50, 2, 64)).astype(np.float32)
    dk, st, cu = ctx.upload(x), ctx.upload(np.zeros(2, np.int32)), ctx.upload(np.array([0, 40, 50], np.int32))
    ko, vo = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    c.append(dk, dk, st, 2, cu=cu, max_new=40)
    c.read(st, 2, ko, vo, cu=cu, max_rows=40)
    ctx.sync()
    t = torch.from_numpy(x)
    want = torch.cat([quantised(t[:40]), quantised(t[40:])]).numpy()
    for p in (ko, vo):
        assert np.array_equal(ctx.download(p, x.size).reshape(x.shape).astype(np.float64), want)
    c.close()
    for p in (dk, st, cu, ko, vo):
        ctx.free(p)
