"""Cases for the operators over the paged 8-bit KV cache: append, read, single-token and prompt attention.

The cache: pages of 32 tokens.  Keys are int8 [pages][kv_heads][32][head_dim], values int8
[pages][kv_heads][head_dim][32] (a page's tokens side by side), each with one fp32 scale per (page, KV head);
sequence i's page p is page table[i][p] of the pool.  A page's scale is max|x| / 127 over the rows it holds, a code
is x / scale rounded half to even.  The rows of a page that is not full yet are also kept as given ("tail"), so that
a page can be quantised again when rows join it.

Attention: s = scale * q.k, with a cap c > 0 replaced by c * tanh(s / c).  The query of position p sees key t < len if
t < prefix, or if t <= p and (no window, or p - t < window).  A query that sees nothing gives 0 and lse = -inf.
"""

import math
import os
import sys

import torch

own = False

PAGE = 32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# Head layouts (query heads, KV heads, head_dim) of the shapes this repository builds: 27B, 270M, and the small
# grouped one.
H27, H270, HGQA = (32, 16, 128), (4, 1, 256), (8, 2, 64)


def _case(name, op, heads, dtype, **more):
    h, kv, hd = heads
    case = {"name": name, "op": op, "heads": h, "kv_heads": kv, "head_dim": hd, "dtype": dtype, "count": 1,
            "longest": 0, "new": 1, "even": True, "window": 0, "cap": 0.0, "prefix": 0, "lse": False}
    case.update(more)
    return case


def listed():
    return [
        # a decode step of 32 conversations: one new key and value row for each, at unlike fills of the last page
        _case("append-step-32", "append", H27, "bf16", count=32, longest=2304, even=False),
        # a whole prompt written in one go
        _case("append-prompt-8192", "append", H27, "bf16", longest=0, new=8192),
        # a short conversation of the small model taken out of the cache (to move or to keep it)
        _case("read-512", "read", H270, "f32", longest=512),
        # four conversations read back
        _case("read-4x4096", "read", H27, "bf16", count=4, longest=4096, even=False),
        # one conversation of the small model on a sliding layer: latency
        _case("decode-1x512", "decode", H270, "f32", longest=512, window=512),
        # an ordinary serving step: 32 conversations around 2K
        _case("decode-32x2304", "decode", H27, "bf16", count=32, longest=2304, even=False),
        # long documents, capped scores
        _case("decode-8x32768", "decode", H27, "f16", count=8, longest=32768, even=False, cap=50.0, lse=True),
        # a sliding window that keeps the first tokens in sight, in the model's own fp32
        _case("decode-32x4096-window", "decode", H27, "f32", count=32, longest=4096, even=False, window=1024, prefix=4),
        # the shortest prompts: a greeting on the small model
        _case("prefill-17", "prefill", H270, "f32", longest=17, new=17),
        # chunks of three prompts behind their histories, sliding window, the model's own fp32
        _case("prefill-3x512-window", "prefill", H27, "f32", count=3, longest=4096, new=512, even=False, window=1024),
        # a prompt whose first part (an image's tokens) is seen by all its tokens, capped scores, grouped heads
        _case("prefill-2048-prefix", "prefill", HGQA, "f16", count=4, longest=2048, new=2048, even=False, cap=30.0,
              prefix=256, lse=True),
        # a long prompt
        _case("prefill-8192", "prefill", H27, "bf16", longest=8192, new=8192),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "prefill", "prefill"])
    heads = rng.choice([H27, H27, H270, HGQA, (16, 2, 128), (6, 2, 128), (8, 8, 64), (8, 4, 256)])
    c = _case("", op, heads, rng.choice(["f32", "f16", "bf16"]), even=rng.random() < 0.3)
    del c["name"]
    if op == "append":
        c["count"] = _log(rng, 1, 32)
        c["longest"] = rng.choice([0, _log(rng, 1, 4096)])
        c["new"] = rng.choice([1, _log(rng, 2, max(2, 8192 // c["count"]))])
    elif op == "read":
        c["count"] = _log(rng, 1, 16)
        c["longest"] = _log(rng, 1, 16384 // c["count"])
    else:
        if op == "decode":
            c["count"] = _log(rng, 1, 64)
            c["longest"] = _log(rng, 1, min(32768, 131072 // c["count"]))
        else:
            c["count"] = _log(rng, 1, 8)
            c["new"] = _log(rng, 2, 4096 // c["count"])
            c["longest"] = max(c["new"], _log(rng, 1, 8192 // c["count"]))
        c["window"] = rng.choice([0, 0, _log(rng, 1, 1024)])
        c["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
        c["prefix"] = rng.choice([0, 0, _log(rng, 1, 300)])
        c["lse"] = rng.random() < 0.5
    return c


def _lengths(case):
    """Host lists: tokens held in the end and new tokens among them, by sequence.  They belong to the case."""
    g = torch.Generator().manual_seed(case["count"] * 7919 + case["longest"] * 31 + case["new"])
    held, new = [], []
    for i in range(case["count"]):
        full = case["even"] or i == 0
        n = case["new"] if full else int(torch.randint(1, case["new"] + 1, (1,), generator=g))
        if case["op"] == "append":
            # tokens held before.  A call is made again on the same state, so the rows of the page that it starts in
            # must not be replaced by those of a later one: the call starts on a page, stays in one, or ends on one.
            start = case["longest"] if full else int(torch.randint(0, case["longest"] + 1, (1,), generator=g))
            if start % PAGE and start // PAGE != (start + n) // PAGE:
                n += -(start + n) % PAGE
            held.append(start + n)
        else:
            low = max(n, case["longest"] // 2)
            held.append(case["longest"] if full else int(torch.randint(low, max(low, case["longest"]) + 1, (1,), generator=g)))
        new.append(n)
    if case["op"] == "read":
        new = list(held)
    return held, new


def _rows(g, shape, dtype):
    """Normalised, rotated keys or values: a few strong channels, tokens of unlike size."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))
    x *= torch.exp(0.4 * torch.randn((1,) * (len(shape) - 1) + shape[-1:], generator=g, device="cuda"))
    return x.to(dtype)


def prepare(case, seed):
    held, new = _lengths(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed) + 1)
    dt, kv, hd, n = TYPES[case["dtype"]], case["kv_heads"], case["head_dim"], case["count"]
    per = [-(-h // PAGE) for h in held]
    pps, pages = max(per), sum(per) + 3
    table = torch.full((n, pps), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).int(), 0
    for i, p in enumerate(per):
        table[i, :p] = order[at:at + p]
        at += p
    before = [h - m if case["op"] == "append" else h for h, m in zip(held, new)]
    s = {"case": case, "held": held, "new": new, "table": table.cuda(), "pages": pages, "pages_per_seq": pps}
    s["k"] = torch.zeros((pages, kv, PAGE, hd), dtype=torch.int8, device="cuda")
    s["v"] = torch.zeros((pages, kv, hd, PAGE), dtype=torch.int8, device="cuda")
    s["k_scale"] = torch.zeros((pages, kv), device="cuda")
    s["v_scale"] = torch.zeros((pages, kv), device="cuda")
    s["k_tail"] = torch.zeros((n, kv, PAGE, hd), dtype=dt, device="cuda")
    s["v_tail"] = torch.zeros((n, kv, PAGE, hd), dtype=dt, device="cuda")
    for i, b in enumerate(before):  # what the sequences hold when the call is made
        p = -(-b // PAGE)
        if not p:
            continue
        ids = s["table"][i, :p].long()
        for name in ("k", "v"):
            x = _rows(g, (p * PAGE, kv, hd), dt).float()
            x[b:] = 0
            x = x.view(p, PAGE, kv, hd).transpose(1, 2)
            sc = x.abs().amax((2, 3)) / 127
            q = torch.round(x / sc.clamp_min(1e-30)[:, :, None, None]).to(torch.int8)
            s[name][ids] = q if name == "k" else q.transpose(2, 3)
            s[name + "_scale"][ids] = sc
            if b % PAGE:
                s[name + "_tail"][i, :, :b % PAGE] = x[-1, :, :b % PAGE].to(dt)
            del x, q
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    s["total"] = cu[-1]
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["len"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    s["start"] = torch.tensor([h - m for h, m in zip(held, new)], dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        s["k_new"], s["v_new"] = _rows(g, (cu[-1], kv, hd), dt), _rows(g, (cu[-1], kv, hd), dt)
    elif case["op"] != "read":
        s["q"] = 2 * _rows(g, (cu[-1], case["heads"], hd), dt)
        s["prefix"] = torch.tensor([min(h, case["prefix"] + (i if case["prefix"] else 0)) for i, h in enumerate(held)],
                                   dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ plain


def _places(s):
    """Sequence and position of every new token."""
    at = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"][1:], at, right=True)
    return seq, at - s["cu"][seq] + s["start"][seq]


def _plain_read(s):
    seq, pos = _places(s)
    page, slot = s["table"][seq, pos // PAGE].long(), (pos % PAGE).long()
    k = s["k"][page, :, slot].float() * s["k_scale"][page][:, :, None]
    v = s["v"][page, :, :, slot].float() * s["v_scale"][page][:, :, None]
    return k, v


def _plain_append(s):
    start, end = s["start"], s["len"]
    first, most = start // PAGE, max(-(-h // PAGE) - (h - m) // PAGE for h, m in zip(s["held"], s["new"]))
    block = first[:, None] + torch.arange(most, device="cuda", dtype=torch.int32)  # [count, most] pages touched
    live = block * PAGE < end[:, None]
    # pages past a sequence's end: its first page once more, with the same contents
    block = torch.where(live, block, first[:, None])
    pos = block[:, :, None] * PAGE + torch.arange(PAGE, device="cuda", dtype=torch.int32)
    rows = (s["cu"][:-1, None, None] + (pos - start[:, None, None]).clamp_min(0)).clamp_max(s["total"] - 1).long()
    old, inside = pos < start[:, None, None], pos < end[:, None, None]
    page = torch.gather(s["table"], 1, block.long()).long()
    last = live & (end[:, None] // PAGE == block) & (end % PAGE != 0)[:, None]
    for name in ("k", "v"):
        x = s[name + "_new"][rows]  # [count, most, PAGE, kv, hd]
        x = torch.where(old[..., None, None], s[name + "_tail"].transpose(1, 2)[:, None], x)
        x = torch.where(inside[..., None, None], x, torch.zeros_like(x)).transpose(2, 3)
        f = x.float()
        sc = (f.abs().amax((3, 4)).double() / 127).float()
        q = torch.round(f.double() / torch.where(sc > 0, sc, 1.0).double()[..., None, None]).clamp(-127, 127).to(torch.int8)
        s[name][page] = q if name == "k" else q.transpose(3, 4)
        s[name + "_scale"][page] = sc
        keep = (last[:, :, None] & inside).any(1)[:, None, :, None]
        s[name + "_tail"].copy_(torch.where(keep, (x * last[:, :, None, None, None]).sum(1, dtype=x.dtype), s[name + "_tail"]))
    return _plain_read(s)


def _plain_attention(s):
    c = s["case"]
    kv, hd, n = c["kv_heads"], c["head_dim"], c["count"]
    r, m, t = c["heads"] // kv, max(s["new"]), s["pages_per_seq"] * PAGE
    page = s["table"].clamp_min(0).long()
    k = (s["k"][page].float() * s["k_scale"][page][..., None, None]).transpose(1, 2).reshape(n, kv, t, hd)
    v = (s["v"][page].float() * s["v_scale"][page][..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, kv, t, hd)
    at = torch.arange(m, device="cuda", dtype=torch.int32)
    rows = (s["cu"][:-1, None] + at).clamp_max(s["total"] - 1).long()
    q = s["q"][rows].float().reshape(n, m, kv, r, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, r * m, hd)
    x = (torch.matmul(q, k.transpose(2, 3)) * hd ** -0.5).view(n, kv, r, m, t)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    pos = (s["start"][:, None] + at)[:, :, None]
    key = torch.arange(t, device="cuda", dtype=torch.int32)
    see = key <= pos
    if c["window"]:
        see = see & (pos - key < c["window"])
    see = (see | (key < s["prefix"][:, None, None])) & (key < s["len"][:, None, None])
    x = torch.where(see[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-1e30)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(n, kv, r * m, t), v).view(n, kv, r, m, hd) / total.clamp_min(1e-30)
    seq, p = _places(s)
    p = (p - s["start"][seq]).long()
    out = out.permute(0, 3, 1, 2, 4)[seq, p].reshape(s["total"], c["heads"], hd).to(s["q"].dtype)
    if not c["lse"]:
        return (out,)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)[seq, p].reshape(s["total"], c["heads"])
    return out, lse


# -------------------------------------------------------- the framework's

_context = None


def _handle(s):
    """The cache as the framework sees it, and the calls' workspace: made once, as a program keeps them."""
    global _context
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vortex-rt_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import vrt

    if _context is None:
        _context = vrt.Context(torch.cuda.current_device())
    c = s["case"]
    cache = vrt.Kv8Cache(_context, c["kv_heads"], c["head_dim"], s["pages"], c["count"], s["pages_per_seq"], c["dtype"],
                         k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_scale=s["k_scale"].data_ptr(),
                         v_scale=s["v_scale"].data_ptr(), k_tail=s["k_tail"].data_ptr(), v_tail=s["v_tail"].data_ptr(),
                         table=s["table"].data_ptr())
    s["cache"] = cache
    if c["op"] in ("decode", "prefill"):
        need = cache.workspace_bytes(c["heads"], c["count"], max(s["new"]), max(s["held"]))
        s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return cache


def _own_run(s):
    cache = s.get("cache") or _handle(s)
    c, n, stream = s["case"], s["case"]["count"], torch.cuda.current_stream().cuda_stream or 1
    if c["op"] in ("append", "read"):
        most = max(s["new"])
        if c["op"] == "append":
            cache.append(s["k_new"].data_ptr(), s["v_new"].data_ptr(), s["start"].data_ptr(), n, cu=s["cu"].data_ptr(),
                         max_new=most, stream=stream)
        k = torch.empty((s["total"], c["kv_heads"], c["head_dim"]), device="cuda")
        v = torch.empty_like(k)
        cache.read(s["start"].data_ptr(), n, k.data_ptr(), v.data_ptr(), cu=s["cu"].data_ptr(), max_rows=most,
                   stream=stream)
        return k, v
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], device="cuda") if c["lse"] else None
    more = dict(scale=c["head_dim"] ** -0.5, softcap=c["cap"], window=c["window"],
                prefix=s["prefix"].data_ptr() if c["prefix"] else None, lse=lse.data_ptr() if c["lse"] else None,
                workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), stream=stream)
    if c["op"] == "decode":
        cache.decode(s["q"].data_ptr(), s["len"].data_ptr(), n, c["heads"], out.data_ptr(), max_len=max(s["held"]), **more)
    else:
        cache.prefill(s["q"].data_ptr(), s["len"].data_ptr(), s["cu"].data_ptr(), n, c["heads"], out.data_ptr(),
                      max_new=max(s["new"]), max_len=max(s["held"]), **more)
    return (out, lse) if c["lse"] else (out,)


def run(s):
    if own:
        return _own_run(s)
    op = s["case"]["op"]
    return _plain_append(s) if op == "append" else _plain_read(s) if op == "read" else _plain_attention(s)


# ------------------------------------------------------------------- work


def _seen(c, held, new):
    """(query, key) pairs that the mask leaves, and the keys that some query sees."""
    pairs = keys = 0
    w = c["window"] or 1 << 60
    for i, (h, m) in enumerate(zip(held, new)):
        pre = min(h, c["prefix"] + (i if c["prefix"] else 0))
        for p in range(h - m, h):
            lo = max(0, p + 1 - w)
            pairs += (p + 1 - lo) + (pre if pre <= lo else max(0, pre - (p + 1)) + lo)
        lo = max(0, h - m + 1 - w)
        keys += h - lo + min(pre, lo)
    return pairs, keys


def work(case):
    held, new = _lengths(case)
    kv, hd, size = case["kv_heads"], case["head_dim"], SIZE[case["dtype"]]
    n = 2 * sum(new) * kv * hd  # elements of K and V
    if case["op"] == "append":  # rows in, codes held, their values out
        return {"bytes": n * (size + 1 + 4), "flops": 2 * n}
    if case["op"] == "read":
        return {"bytes": n * (1 + 4), "flops": n}
    pairs, keys = _seen(case, held, new)
    io = 2 * sum(new) * case["heads"] * hd * size
    return {"bytes": io + 2 * keys * kv * hd + 8 * kv * (keys // PAGE), "flops": 4 * pairs * case["heads"] * hd}


# ------------------------------------------------------------------ exact


def exact(case, seed):
    s = prepare(case, seed)
    held, new, kv, hd = s["held"], s["new"], case["kv_heads"], case["head_dim"]
    outs = []
    r = 0
    for i in range(case["count"]):
        h, m = held[i], new[i]
        ids = s["table"][i, :-(-h // PAGE)].long()
        if case["op"] == "append":
            pair = []
            first = (h - m) // PAGE * PAGE
            for name in ("k", "v"):
                x = torch.cat([s[name + "_tail"][i].double().transpose(0, 1)[:h - m - first],
                               s[name + "_new"][r:r + m].double()])
                y = torch.zeros((-(-x.shape[0] // PAGE) * PAGE, kv, hd), dtype=torch.float64, device="cuda")
                y[:x.shape[0]] = x
                y = y.view(-1, PAGE, kv, hd)
                step = y.abs().amax((1, 3), keepdim=True) / 127
                held_step = step.float().double()  # a scale is kept in 32 bits
                y = torch.round(y / torch.where(held_step > 0, held_step, 1.0)).clamp(-127, 127) * held_step
                pair.append(y.reshape(-1, kv, hd)[h - m - first:][:m])
            outs.append(pair)
            r += m
            continue
        k = (s["k"][ids].double() * s["k_scale"][ids].double()[:, :, None, None]).transpose(1, 2).reshape(-1, kv, hd)[:h]
        v = (s["v"][ids].double() * s["v_scale"][ids].double()[:, :, None, None]).permute(0, 3, 1, 2).reshape(-1, kv, hd)[:h]
        if case["op"] == "read":
            outs.append([k, v])
            continue
        group = case["heads"] // kv
        out = torch.zeros((m, case["heads"], hd), dtype=torch.float64, device="cuda")
        lse = torch.full((m, case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
        pre = int(s["prefix"][i])
        t = torch.arange(h, device="cuda")
        for a in range(0, m, 2048):
            b = min(m, a + 2048)
            p = torch.arange(h - m + a, h - m + b, device="cuda")[:, None]
            hidden = (t > p) | (p - t >= (case["window"] or h + 1))
            hidden &= t >= pre
            for j in range(case["heads"]):
                x = s["q"][r + a:r + b, j].double() @ k[:, j // group].T / math.sqrt(hd)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                x.masked_fill_(hidden, -math.inf)
                z = torch.logsumexp(x, 1)
                lse[a:b, j] = z
                out[a:b, j] = torch.exp(x - torch.where(z.isfinite(), z, 0.0)[:, None]) @ v[:, j // group]
        outs.append([out, lse])
        r += m
    cat = [torch.cat([o[j] for o in outs]) for j in range(2)]
    if case["op"] in ("decode", "prefill") and not case["lse"]:
        return (cat[0],)
    return tuple(cat)
