"""Host-side checks of the attention operators that need no GPU: refusals of the C entry points before any HIP call, scratch
sizes, and the torch operators' schemas and shape-only forms."""
import ctypes

import pytest
import torch

P = 0x1000  # a pointer that is never followed


@pytest.fixture()
def cache(capi):
    def make(k=P, v=P, pages=4, page_size=16, strides=None, heads=2, d=64):
        s = strides or (heads * page_size * d, page_size * d, d)
        return ctypes.byref(capi.KvCache(k, v, pages, page_size, *s))
    return make


def test_kv_append_codes(capi, cache):
    def v(dtype=0, T=4, Hq=4, Hkv=2, D=64, rot=64, q=(P, 256, 64), k=(P, 128, 64), val=(P, 128, 64), table=P, rows=8, pos=P, slots=P,
          qo=(P, 256, 64), ko=(P, 128, 64), c=None):
        return capi.lib().fsw_validate_kv_append(dtype, T, Hq, Hkv, D, rot, *q, *k, *val, table, rows, pos, slots, *qo, *ko,
                                                 c or cache())
    assert v() == v(dtype=1) == v(rot=0, table=None, rows=0) == v(ko=(None, 0, 0)) == capi.OK
    assert v(T=0, q=(None, 0, 0), pos=None) == capi.OK
    assert v(dtype=2) == capi.E_DTYPE
    for kw in (dict(T=-1), dict(T=(1 << 20) + 1), dict(Hq=3), dict(Hkv=0), dict(Hq=2048, Hkv=1), dict(D=264), dict(D=0), dict(rot=66),
               dict(rot=-2), dict(rot=7), dict(rows=0), dict(rows=-1)):
        assert v(**kw) == capi.E_SHAPE, kw
    assert v(D=60) == capi.E_ALIGN
    for kw in (dict(q=(None, 256, 64)), dict(k=(None, 128, 64)), dict(val=(None, 128, 64)), dict(qo=(None, 256, 64)), dict(pos=None),
               dict(slots=None), dict(table=None), dict(c=cache(k=None)), dict(c=cache(v=None))):
        assert v(**kw) == capi.E_NULL, kw
    for kw in (dict(q=(P, -8, 64)), dict(qo=(P, 64, 64)), dict(qo=(P, 256, 32)), dict(qo=(P, 0, 64)), dict(ko=(P, 64, 64)),
               dict(c=cache(strides=(2048, 1024, 32))), dict(c=cache(strides=(32, 1024, 64)))):
        assert v(**kw) == capi.E_LD, kw
    for kw in (dict(q=(P + 8, 256, 64)), dict(q=(P, 260, 64)), dict(k=(P, 128, 60)), dict(table=P + 4), dict(pos=P + 2), dict(slots=P + 1),
               dict(c=cache(k=P + 8)), dict(c=cache(strides=(2052, 1024, 64)))):
        assert v(**kw) == capi.E_ALIGN, kw
    assert v(rot=12, table=P + 4) == capi.OK                   # single angles are read there
    assert v(q=(P, 0, 64), k=(P, 0, 0)) == capi.OK             # inputs may repeat rows
    assert v(qo=(P, 64, 256)) == capi.OK                       # head-major rows
    for c in (cache(pages=0), cache(page_size=0), cache(pages=1 << 20, page_size=1 << 11), cache(strides=(1 << 41, 1024, 64))):
        assert v(c=c) == capi.E_SHAPE
    # entry points return the same codes before any HIP call
    L = capi.lib()
    tail = (P, 8, P, P, P, 256, 64, P, 128, 64)
    assert L.fsw_kv_append(0, 4, 3, 2, 64, 64, 0, P, 256, 64, P, 128, 64, P, 128, 64, *tail, cache(), None) == capi.E_SHAPE
    assert L.fsw_kv_append(0, 0, 4, 2, 64, 64, 0, None, 0, 0, None, 0, 0, None, 0, 0, None, 0, None, None, None, 0, 0, None, 0, 0, None,
                           None) == capi.OK


def test_attn_decode_codes(capi, cache):
    def v(dtype=0, B=3, Hq=4, Hkv=2, D=64, q=(P, 256, 64), c=None, table=P, ld=4, lengths=P, max_len=64, scale=0.125, o=(P, 256, 64)):
        return capi.lib().fsw_validate_attn_decode(dtype, B, Hq, Hkv, D, *q, c or cache(), table, ld, lengths, max_len, scale, *o)
    assert v() == v(B=0, q=(None, 0, 0)) == v(max_len=0, table=None, ld=0) == capi.OK
    assert v(dtype=5) == capi.E_DTYPE
    for kw in (dict(B=-1), dict(B=65536), dict(max_len=-1), dict(max_len=(1 << 30) + 1), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-40), dict(Hq=5), dict(c=cache(pages=0))):
        assert v(**kw) == capi.E_SHAPE, kw
    for kw in (dict(q=(None, 256, 64)), dict(table=None), dict(lengths=None), dict(o=(None, 256, 64)), dict(c=cache(k=None))):
        assert v(**kw) == capi.E_NULL, kw
    assert v(ld=3) == v(max_len=65) == v(o=(P, 128, 64)) == capi.E_LD
    assert v(table=P + 2) == v(lengths=P + 1) == v(o=(P + 8, 256, 64)) == v(q=(P, 252, 64)) == capi.E_ALIGN
    L = capi.lib()
    assert L.fsw_attn_decode(0, 3, 4, 2, 64, P, 256, 64, cache(), P, 3, P, 64, 0.125, P, 256, 64, None, 0, None) == capi.E_LD
    need = L.fsw_attn_decode_workspace_bytes(0, 1, 4, 2, 64, 10000)
    assert need > 0
    wide = (P, 1000, P, 10000, 0.125, P, 256, 64)
    assert L.fsw_attn_decode(0, 1, 4, 2, 64, P, 256, 64, cache(), *wide, None, 0, None) == capi.E_WORKSPACE
    assert L.fsw_attn_decode(0, 1, 4, 2, 64, P, 256, 64, cache(), *wide, P, need - 1, None) == capi.E_WORKSPACE
    assert L.fsw_attn_decode(0, 1, 4, 2, 64, P, 256, 64, cache(), *wide, P + 4, need, None) == capi.E_ALIGN


def test_attn_decode_scratch(capi):
    ws = capi.lib().fsw_attn_decode_workspace_bytes
    assert ws(0, 0, 4, 2, 64, 1000) == ws(0, 4, 4, 2, 64, 0) == ws(7, 4, 4, 2, 64, 1000) == 0
    assert ws(0, 1024, 8, 8, 128, 100000) == 0                        # sequences enough: none is split
    assert ws(0, 128, 64, 8, 128, 2560) == 0 < ws(0, 128, 64, 8, 128, 2561)
    assert ws(0, 1, 32, 8, 128, 131072) % (32 * (128 + 2) * 4) == 0   # float32 sums, maximum and sum of each part and head
    for B, n in ((1, 1 << 30), (65535, 1 << 30), (7, 12345)):
        assert 0 <= ws(0, B, 1024, 1024, 256, n) < 1 << 42


def test_attn_prompt_codes(capi):
    def v(dtype=0, Tq=9, Tk=9, B=2, Hq=4, Hkv=2, D=64, q=(P, 256, 64), k=(P, 128, 64), val=(P, 128, 64), cu_q=P, cu_k=P, scale=0.125,
          o=(P, 256, 64)):
        return capi.lib().fsw_validate_attn_prompt(dtype, Tq, Tk, B, Hq, Hkv, D, *q, *k, *val, cu_q, cu_k, scale, *o)
    assert v() == v(Tq=0, q=(None, 0, 0)) == v(Tk=0, k=(None, 0, 0), val=(None, 0, 0)) == v(B=0) == v(Tk=1, k=(P, 0, 0)) == capi.OK
    assert v(dtype=-1) == capi.E_DTYPE
    for kw in (dict(Tq=-1), dict(Tk=-1), dict(Tq=(1 << 20) + 1), dict(B=-1), dict(scale=0.0), dict(scale=float("inf")), dict(Hkv=3),
               dict(k=(P, (1 << 21) + 8, 64)), dict(val=(P, 1 << 22, 64))):
        assert v(**kw) == capi.E_SHAPE, kw
    assert v(q=(None, 0, 0)) == v(cu_q=None) == v(cu_k=None) == v(k=(None, 0, 0)) == v(o=(None, 0, 0)) == capi.E_NULL
    assert v(k=(P, 0, 64)) == v(val=(P, 32, 64)) == v(o=(P, 192, 64)) == v(q=(P, 256, -64)) == capi.E_LD
    assert v(cu_q=P + 2) == v(k=(P + 4, 128, 64)) == v(D=12) == v(o=(P, 256, 68)) == capi.E_ALIGN
    assert capi.lib().fsw_attn_prompt(0, 9, 9, 2, 4, 3, 64, P, 256, 64, P, 128, 64, P, 128, 64, P, P, 0.125, P, 256, 64, None) == capi.E_SHAPE


def test_torch_operators_trace_without_a_gpu(ext):
    for name, dtype in (("bf16", torch.bfloat16), ("fp16", torch.float16)):
        t = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
        i = lambda *s: t(*s, dt=torch.int32)  # noqa: E731
        op = lambda n: getattr(torch.ops.ASMLLM, "%s_%s" % (n, name))  # noqa: E731
        caches = (t(5, 2, 16, 64), t(5, 2, 16, 64))
        q, k = op("kv_append")(t(7, 4, 64), t(7, 2, 64), t(7, 2, 64), t(9, 64, dt=torch.float32), i(7), i(7), *caches)
        assert q.shape == (7, 4, 64) and k.shape == (7, 2, 64) and q.dtype == dtype
        assert op("attn_decode")(t(3, 4, 64), *caches, i(3, 2), i(3), 32, 0.125).shape == (3, 4, 64)
        assert op("attn_prompt")(t(7, 4, 64), t(7, 2, 64), t(7, 2, 64), i(2), i(2), 0.125).shape == (7, 4, 64)
        with pytest.raises(RuntimeError):
            op("attn_decode")(t(3, 4, 64), *caches, i(3, 2), i(3), 33, 0.125)          # more keys than the table has pages for
        with pytest.raises(RuntimeError):
            op("attn_prompt")(t(7, 4, 64), t(7, 2, 64), t(7, 2, 32), i(2), i(2), 0.125)
        with pytest.raises(RuntimeError):
            op("kv_append")(t(7, 4, 64), t(7, 2, 64), t(7, 2, 64), t(9, 64, dt=torch.float32), t(7, dt=torch.int64), i(7), *caches)
        schema = op("kv_append").default._schema
        written = [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write]
        assert written == ["k_cache", "v_cache"]
    # on the CPU there is no implementation to fall back to
    with pytest.raises(RuntimeError, match="GPU"):
        ext.attn_prompt_bf16(*(torch.empty(7, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2)), torch.zeros(2, dtype=torch.int32),
                             torch.zeros(2, dtype=torch.int32), 0.125)
