"""Refusals of the paged 8-bit KV cache calls (vrt_kv8_*): every bad argument
is turned away before a device is touched, with its own message.  No GPU: the
pointers are made up and the context is null, which a call finds out last."""

import pytest

import vrt

A = 1 << 20  # an aligned address that nothing reads


class NoContext:
    h = None


def cache(**kw):
    a = dict(kv_heads=2, head_dim=64, pages=8, max_seqs=4, pages_per_seq=3, dtype="bf16")
    arrays = dict(k=A, v=A, k_scale=A, v_scale=A, k_tail=A, v_tail=A, table=A)
    for k in list(kw):
        (arrays if k in arrays else a)[k] = kw[k]
    return vrt.Kv8Cache(NoContext(), **a, **arrays)


def call(c, what, **kw):
    if what == "append":
        a = dict(k=A, v=A, start=A, count=2, cu=A, max_new=3)
        a.update(kw)
        return c.append(a.pop("k"), a.pop("v"), a.pop("start"), a.pop("count"), **a)
    if what == "read":
        a = dict(start=A, count=2, k_out=A, v_out=A, cu=A, max_rows=3)
        a.update(kw)
        return c.read(a.pop("start"), a.pop("count"), a.pop("k_out"), a.pop("v_out"), **a)
    a = dict(q=A, lens=A, cu=A, count=2, heads=4, out=A, max_len=96, max_new=5, workspace=A, workspace_bytes=1 << 40)
    a.update(kw)
    pos = [a.pop("q"), a.pop("lens")] + ([a.pop("cu")] if what == "prefill" else [])
    if what == "decode":
        a.pop("cu"), a.pop("max_new")
    return getattr(c, what)(*pos, a.pop("count"), a.pop("heads"), a.pop("out"), **a)


ALL = ("append", "read", "decode", "prefill")


@pytest.mark.parametrize("what", ALL)
@pytest.mark.parametrize("kw,code,text", [
    (dict(head_dim=96), vrt.VRT_E_UNSUPPORTED, "head_dim"),
    (dict(kv_heads=0), vrt.VRT_E_INVALID, "kv_heads"),
    (dict(kv_heads=1025), vrt.VRT_E_INVALID, "kv_heads"),
    (dict(pages=0), vrt.VRT_E_INVALID, "pages"),
    (dict(max_seqs=0), vrt.VRT_E_INVALID, "max_seqs"),
    (dict(max_seqs=65536), vrt.VRT_E_INVALID, "max_seqs"),
    (dict(pages_per_seq=0), vrt.VRT_E_INVALID, "pages_per_seq"),
    (dict(pages_per_seq=1 << 26), vrt.VRT_E_INVALID, "pages_per_seq"),
    (dict(k=0), vrt.VRT_E_INVALID, "lacks an array"),
    (dict(table=0), vrt.VRT_E_INVALID, "lacks an array"),
    (dict(v=A + 8), vrt.VRT_E_INVALID, "aligned"),
    (dict(k_tail=A + 2), vrt.VRT_E_INVALID, "aligned"),
])
def test_bad_cache(what, kw, code, text):
    c = cache(**kw)
    with pytest.raises(vrt.VrtError, match=text) as e:
        call(c, what, **(dict(heads=max(1, c.s.kv_heads)) if what in ("decode", "prefill") else {}))
    assert e.value.code == code


@pytest.mark.parametrize("what,kw,text", [
    ("append", dict(k=0), "k is null"), ("append", dict(v=A + 4), "16-byte"), ("append", dict(start=None), "null"),
    ("append", dict(row_stride=120), "overlap"), ("append", dict(row_stride=132), "16-byte"),
    ("append", dict(count=5), "exceeds"), ("append", dict(max_new=0), "max_new"), ("append", dict(max_new=97), "max_new"),
    ("read", dict(k_out=0), "null"), ("read", dict(v_out=A + 4), "aligned"), ("read", dict(max_rows=97), "max_rows"),
    ("read", dict(count=5), "exceeds"),
    ("decode", dict(q=0), "q is null"), ("decode", dict(lens=None), "null"), ("decode", dict(out=A + 8), "16-byte"),
    ("decode", dict(heads=3), "query heads"), ("decode", dict(heads=0), "query heads"),
    ("decode", dict(heads=18), "query heads"), ("decode", dict(max_len=0), "max_len"),
    ("decode", dict(max_len=97), "max_len"), ("decode", dict(count=5), "exceeds"),
    ("decode", dict(scale=float("nan")), "scale"), ("decode", dict(scale=float("inf")), "scale"),
    ("decode", dict(softcap=-1.0), "softcap"), ("decode", dict(softcap=float("nan")), "softcap"),
    ("decode", dict(q_stride=252), "overlap"), ("decode", dict(out_stride=260), "16-byte"),
    ("prefill", dict(cu=None), "null"), ("prefill", dict(max_new=0), "max_new"), ("prefill", dict(max_new=97), "max_new"),
    ("prefill", dict(heads=18), "query heads"), ("prefill", dict(out=0), "out is null"),
])
def test_bad_call(what, kw, text):
    with pytest.raises(vrt.VrtError, match=text) as e:
        call(cache(), what, **kw)
    assert e.value.code == vrt.VRT_E_INVALID


@pytest.mark.parametrize("what", ALL)
def test_good_call_needs_a_context(what):
    with pytest.raises(vrt.VrtError, match="null context"):
        call(cache(), what)


def test_unknown_dtype():
    with pytest.raises(vrt.VrtError, match="dtype"):
        cache(dtype="f64")
    c = cache()
    c.s.dtype = 7
    with pytest.raises(vrt.VrtError, match="dtype"):
        call(c, "append")
