"""Host-side refusals of the paged cache's and the sampler's C entry points: every bad argument
returns its documented code before any device work."""
import ctypes

import pytest

from mdflash_b200 import _lib

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(258)


def _call(name, order, base, **change):
    args = dict(base, **change)
    return getattr(_lib.load(), name)(*[args[k] for k in order.split()])


TABLES = ("old new n table tstride maxp page free cap count kv cu slots pos maxt count_out ws wsb "
          "status stream")
TABLES_OK = dict(old=P, new=P, n=4, table=P, tstride=8, maxp=8, page=16, free=P, cap=64, count=P, kv=P,
                 cu=P, slots=P, pos=P, maxt=128, count_out=P, ws=P, wsb=4, status=P, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(old=None), -1), (dict(count_out=None), -1), (dict(slots=None), -1), (dict(n=0), -1),
    (dict(tstride=7), -1), (dict(maxp=0), -1), (dict(maxt=-1), -1), (dict(n=2049), -2),
    (dict(page=8), -2), (dict(page=24), -2), (dict(page=2048), -2), (dict(page=0), -2),
    (dict(maxt=1 << 31), -2), (dict(maxp=1 << 28, tstride=1 << 28), -2), (dict(ws=None), -7),
    (dict(wsb=2), -7), (dict(ws=ODD), -4)])
def test_page_tables_refusals(change, code):
    assert _call("ddt_page_tables", TABLES, TABLES_OK, **change) == code


WRITE = "qkv qs t hq hkv d qw kw eps rope slots q k v np page ps hs rs stream"
WRITE_OK = dict(qkv=P, qs=6144, t=4, hq=32, hkv=8, d=128, qw=P, kw=P, eps=1e-6, rope=P, slots=P, q=P,
                k=P, v=P, np=8, page=16, ps=16384, hs=2048, rs=128, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(qkv=None), -1), (dict(slots=None), -1), (dict(t=-1), -1), (dict(hq=0), -1), (dict(np=0), -1),
    (dict(qs=6143), -1), (dict(d=64), -2), (dict(page=17), -2), (dict(qs=6145), -4), (dict(rs=132), -4),
    (dict(qkv=ODD), -4), (dict(k=ODD), -4), (dict(t=0, qkv=None), 0)])
def test_paged_write_refusals(change, code):
    assert _call("ddt_paged_qk_norm_rope", WRITE, WRITE_OK, **change) == code


ATTN = ("q qt qh k v np page ps hs rs table tstride maxp cu kv n t maxn hq hkv d scale out ot oh ws wsb "
        "status stream")
ATTN_OK = dict(q=P, qt=4096, qh=128, k=P, v=P, np=8, page=16, ps=16384, hs=2048, rs=128, table=P,
               tstride=8, maxp=8, cu=P, kv=P, n=4, t=4, maxn=1, hq=32, hkv=8, d=128, scale=1.0, out=P,
               ot=4096, oh=128, ws=P, wsb=1 << 40, status=P, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(table=None), -1), (dict(out=None), -1), (dict(n=0), -1), (dict(t=-1), -1),
    (dict(hq=30), -1), (dict(tstride=7), -1), (dict(maxn=-1), -1), (dict(d=64), -2), (dict(page=48), -2),
    (dict(hq=1024), -2), (dict(n=4096), -2), (dict(t=1 << 31), -2), (dict(q=ODD), -4), (dict(qh=100), -4),
    (dict(ps=16385), -4), (dict(oh=129), -4), (dict(t=0, q=None), 0), (dict(maxn=0), 0)])
def test_paged_attention_refusals(change, code):
    assert _call("ddt_paged_attn", ATTN, ATTN_OK, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(limit=99_999), -1), (dict(limit=2_000_000_001), -1), (dict(first=-1), -1),
    (dict(status=None), -1), (dict(hq=30), -1), (dict(page=48), -2), (dict(q=ODD), -4),
    (dict(maxn=0), 0)])
def test_paged_attention_wait_check_refusals(change, code):
    order = ATTN.replace("stream", "first limit stream")
    assert _call("ddt_paged_attn_wait_check", order, dict(ATTN_OK, first=0, limit=10 ** 6), **change) == code


SAMPLE = "x dtype rows vocab rs u temp k p mp tok logp stream"
SAMPLE_OK = dict(x=P, dtype=1, rows=2, vocab=100, rs=100, u=P, temp=P, k=P, p=P, mp=P, tok=P, logp=P, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), -1), (dict(u=None), -1), (dict(temp=None), -1), (dict(tok=None), -1),
    (dict(rows=-1), -1), (dict(vocab=0), -1), (dict(rs=99), -1), (dict(dtype=3), -3),
    (dict(vocab=1 << 22, rs=1 << 22), -2), (dict(x=ctypes.c_void_p(257)), -4), (dict(rows=0, x=None), 0)])
def test_sample_refusals(change, code):
    assert _call("ddt_sample", SAMPLE, SAMPLE_OK, **change) == code


def test_binding_refuses_host_tensors_and_wrong_kinds():
    torch = pytest.importorskip("torch")
    from mdflash_b200 import kernels as K
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        K.page_tables(i, i, i.view(1, 1), i, i, 16, 4)
    with pytest.raises(ValueError, match="CUDA tensors"):
        K.paged_qk_norm_rope(i, i, i, i, i, i, i)
    with pytest.raises(ValueError, match="CUDA tensors"):
        K.paged_attention(i, i, i, i, i, i, 1)
    with pytest.raises(ValueError, match="CUDA tensors"):
        K.sample(i, i, i)
    with pytest.raises(TypeError):
        K.sample(None, i, i)
