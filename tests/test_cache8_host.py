"""Host-side checks of the cache in 8 bits, the shared prefix and the norms that need no GPU: refusals of the C entry points before any HIP
call, scratch sizes, the torch operators' schemas and shape-only forms, and the definition of the elements (oracle/cache8.py)."""
import ctypes

import pytest
import torch

from oracle import cache8

P = 0x1000  # a pointer that is never followed


@pytest.fixture()
def cache(capi):
    def make(k=P, v=P, ks=P, vs=P, pages=4, page_size=16, strides=(2048, 1024, 64), marks=(32, 16, 1)):
        return ctypes.byref(capi.KvCache8(k, v, ks, vs, pages, page_size, *strides, *marks))
    return make


def cache16(capi, pages=4, page_size=16):
    return ctypes.byref(capi.KvCache(P, P, pages, page_size, 2 * page_size * 64, page_size * 64, 64))


def test_kv_append8_codes(capi, cache):
    def v(dtype=0, T=4, Hq=4, Hkv=2, D=64, rot=64, q=(P, 256, 64), k=(P, 128, 64), val=(P, 128, 64), table=P, rows=8, pos=P, slots=P,
          qo=(P, 256, 64), ko=(P, 128, 64), vo=(P, 128, 64), c=None):
        return capi.lib().fsw_validate_kv_append8(dtype, T, Hq, Hkv, D, rot, *q, *k, *val, table, rows, pos, slots, *qo, *ko, *vo,
                                                  c or cache())
    none = (None, 0, 0)
    assert v() == v(dtype=1) == v(rot=0, table=None, rows=0) == v(ko=none) == v(vo=none) == v(T=0, q=none, pos=None) == capi.OK
    assert v(dtype=2) == capi.E_DTYPE
    for kw in (dict(T=-1), dict(T=(1 << 20) + 1), dict(Hq=3), dict(D=272), dict(rot=66), dict(rot=7), dict(rows=0)):
        assert v(**kw) == capi.E_SHAPE, kw
    assert v(D=72) == v(D=8) == v(D=60) == capi.E_ALIGN                  # 16 elements are a vector of the cache
    for kw in (dict(q=none), dict(k=none), dict(val=none), dict(qo=none), dict(pos=None), dict(slots=None), dict(table=None), dict(c=cache(k=None)),
               dict(c=cache(v=None)), dict(c=cache(ks=None)), dict(c=cache(vs=None))):
        assert v(**kw) == capi.E_NULL, kw
    for kw in (dict(qo=(P, 64, 64)), dict(ko=(P, 64, 64)), dict(vo=(P, 0, 64)), dict(c=cache(strides=(2048, 1024, 48))),
               dict(c=cache(strides=(64, 1024, 64))), dict(c=cache(marks=(32, 16, 0))), dict(c=cache(marks=(31, 16, 1))), dict(c=cache(marks=(32, 8, 1))),
               dict(c=cache(marks=(-32, 16, 1)))):
        assert v(**kw) == capi.E_LD, kw
    for kw in (dict(q=(P + 8, 256, 64)), dict(k=(P, 132, 64)), dict(table=P + 4), dict(c=cache(k=P + 8)), dict(c=cache(strides=(2056, 1024, 64)))):
        assert v(**kw) == capi.E_ALIGN, kw
    assert v(c=cache(marks=(1, 4, 8))) == v(c=cache(ks=P + 1, marks=(33, 16, 1))) == capi.OK      # scales anywhere, as long as they are apart
    for c in (cache(pages=0), cache(pages=1 << 20, page_size=1 << 11), cache(marks=(1 << 41, 16, 1))):
        assert v(c=c) == capi.E_SHAPE
    L = capi.lib()
    tail = (P, 8, P, P, P, 256, 64, P, 128, 64, P, 128, 64)
    assert L.fsw_kv_append8(0, 4, 3, 2, 64, 64, 0, P, 256, 64, P, 128, 64, P, 128, 64, *tail, cache(), None) == capi.E_SHAPE


@pytest.mark.parametrize("eight", [True, False])
def test_kv_read_codes(capi, cache, eight):
    fn, c16 = (capi.lib().fsw_validate_kv_read8, None) if eight else (capi.lib().fsw_validate_kv_read, cache16(capi))
    sound = cache() if eight else c16

    def v(dtype=0, T=9, B=3, Hkv=2, D=64, c=sound, table=P, ld=4, width=4, cu=P, k=(P, 128, 64), val=(P, 128, 64)):
        return fn(dtype, T, B, Hkv, D, c, table, ld, width, cu, *k, *val)
    none = (None, 0, 0)
    assert v() == v(T=0, k=none, cu=None) == v(B=0, c=None, table=None) == v(ld=0) == v(ld=9) == v(width=0, table=None) == capi.OK
    assert v(dtype=3) == capi.E_DTYPE
    for kw in (dict(T=-1), dict(T=(1 << 20) + 1), dict(B=-1), dict(B=65536), dict(width=-1), dict(Hkv=0)):
        assert v(**kw) == capi.E_SHAPE, kw
    for kw in (dict(k=none), dict(val=none), dict(cu=None), dict(table=None), dict(c=None)):
        assert v(**kw) == capi.E_NULL, kw
    assert v(ld=3) == v(k=(P, 64, 64)) == v(val=(P, 0, 64)) == capi.E_LD
    assert v(table=P + 2) == v(cu=P + 1) == v(k=(P + 8, 128, 64)) == v(D=68) == capi.E_ALIGN


def test_attn_decode8_codes_and_scratch(capi, cache):
    L = capi.lib()

    def v(dtype=0, B=3, Hq=4, Hkv=2, D=64, q=(P, 256, 64), c=None, table=P, ld=4, lengths=P, max_len=64, scale=0.125, o=(P, 256, 64)):
        return L.fsw_validate_attn_decode8(dtype, B, Hq, Hkv, D, *q, c or cache(), table, ld, lengths, max_len, scale, *o)
    assert v() == v(B=0, q=(None, 0, 0)) == v(max_len=0, table=None, ld=0) == v(ld=0) == capi.OK
    assert v(dtype=5) == capi.E_DTYPE
    for kw in (dict(B=65536), dict(max_len=-1), dict(max_len=(1 << 30) + 1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e-40),
               dict(scale=3e38), dict(Hq=5)):
        assert v(**kw) == capi.E_SHAPE, kw
    for kw in (dict(q=(None, 256, 64)), dict(table=None), dict(lengths=None), dict(o=(None, 256, 64)), dict(c=cache(vs=None))):
        assert v(**kw) == capi.E_NULL, kw
    assert v(ld=3) == v(max_len=65) == v(o=(P, 128, 64)) == capi.E_LD
    assert v(table=P + 2) == v(D=24) == v(q=(P, 252, 64)) == capi.E_ALIGN
    ws = L.fsw_attn_decode8_workspace_bytes
    assert ws(0, 0, 4, 2, 64, 1000) == ws(0, 4, 4, 2, 64, 0) == ws(7, 4, 4, 2, 64, 1000) == ws(0, 4, 4, 2, 72, 100000) == 0
    need = ws(0, 1, 4, 2, 64, 10000)
    assert need > 0 and need % (4 * (64 + 2) * 4) == 0
    wide = (P, 1000, P, 10000, 0.125, P, 256, 64)
    for work, size, code in ((None, 0, capi.E_WORKSPACE), (P, need - 1, capi.E_WORKSPACE), (P + 4, need, capi.E_ALIGN)):
        assert L.fsw_attn_decode8(0, 1, 4, 2, 64, P, 256, 64, cache(), *wide, work, size, None) == code


@pytest.mark.parametrize("eight", [True, False])
def test_attn_shared_codes_and_scratch(capi, cache, eight):
    L = capi.lib()
    s = "8" if eight else ""
    fn, call, ws = (getattr(L, n % s) for n in ("fsw_validate_attn_shared%s", "fsw_attn_shared%s", "fsw_attn_shared%s_workspace_bytes"))
    sound = cache() if eight else cache16(capi)

    def v(dtype=0, B=3, Hq=4, Hkv=2, D=64, q=(P, 256, 64), c=sound, prefix=P, plen=40, table=P, ld=4, lengths=P, max_len=64, scale=0.125, o=(P, 256, 64)):
        return fn(dtype, B, Hq, Hkv, D, *q, c, prefix, plen, table, ld, lengths, max_len, scale, *o)
    assert v() == v(plen=0, prefix=None) == v(max_len=0, table=None) == v(B=0) == capi.OK
    assert v(plen=0, max_len=0, c=None, prefix=None, table=None) == capi.OK
    assert v(dtype=2) == v(dtype=2, plen=-1) == capi.E_DTYPE
    for kw in (dict(plen=-1), dict(plen=(1 << 30) - 63), dict(plen=1 << 62, max_len=1 << 62), dict(B=65536), dict(scale=-1.0)):
        assert v(**kw) == capi.E_SHAPE, kw
    for kw in (dict(prefix=None), dict(c=None), dict(max_len=0, c=None), dict(lengths=None), dict(table=None)):
        assert v(**kw) == capi.E_NULL, kw
    assert v(ld=3) == capi.E_LD and v(prefix=P + 2) == v(table=P + 1) == capi.E_ALIGN
    assert ws(0, 3, 4, 2, 64, -1, 64) == ws(0, 0, 4, 2, 64, 40, 64) == ws(0, 3, 4, 2, 64, 0, 64) == ws(0, 3, 5, 2, 64, 40, 64) == 0
    need = ws(0, 3, 4, 2, 64, 40, 64)
    share = 3 * 4 * (64 + 2) * 4
    assert need % share == 0 and need >= share                                       # a share of the prefix; few own keys need none
    assert ws(0, 3, 4, 2, 64, 40, 2000) % share == 0 and ws(0, 3, 4, 2, 64, 40, 2000) >= need + 2 * share
    for work, size, code in ((None, 0, capi.E_WORKSPACE), (P, need - 1, capi.E_WORKSPACE), (P + 4, need, capi.E_ALIGN)):
        assert call(0, 3, 4, 2, 64, P, 256, 64, sound, P, 40, P, 4, P, 64, 0.125, P, 256, 64, work, size, None) == code
    for B, Hq, plen, n in ((1, 1024, 1 << 29, 1 << 29), (65535, 1024, 1 << 20, 100), (7, 14, 12345, 0), (200, 64, 8000, 1500)):
        assert 0 < ws(0, B, Hq, 1 if Hq == 1024 else 2, 128, plen, n) < 1 << 45


def test_add_norm_codes(capi):
    def v(dtype=0, M=3, D=64, x=(P, 64), y=(P, 64), gate=(P, 0), post=P, pre=P, scale=1.0, eps=1e-5, xo=(P, 64), h=(P, 64)):
        return capi.lib().fsw_validate_add_norm(dtype, M, D, *x, *y, *gate, post, pre, scale, eps, *xo, *h)
    none = (None, 0)
    assert v() == v(dtype=1) == v(M=0, x=none) == v(gate=none, post=None, pre=None) == v(gate=(P, 64)) == v(x=(P, 0)) == v(xo=none) == v(h=none) == capi.OK
    assert v(y=none, gate=none, post=None, xo=none) == v(D=32768, x=(P, 32768), y=(P, 32768), xo=(P, 32768), h=(P, 32768)) == capi.OK
    assert v(dtype=2) == capi.E_DTYPE
    for kw in (dict(M=-1), dict(M=(1 << 30) + 1), dict(D=0), dict(D=32776), dict(scale=float("inf")), dict(scale=float("nan")), dict(eps=0.0),
               dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=1e-39), dict(x=(P, (1 << 31) + 8))):
        assert v(**kw) == capi.E_SHAPE, kw
    for kw in (dict(x=none), dict(y=none), dict(y=none, gate=none, post=None), dict(y=none, gate=none, xo=none), dict(xo=none, h=none)):
        assert v(**kw) == capi.E_NULL, kw
    for kw in (dict(x=(P, -8)), dict(xo=(P, 56)), dict(h=(P, 0)), dict(gate=(P, 56))):
        assert v(**kw) == capi.E_LD, kw
    assert v(M=1, xo=(P, 0), h=(P, 8)) == capi.OK
    for kw in (dict(D=60), dict(x=(P + 8, 64)), dict(y=(P, 68)), dict(gate=(P + 2, 0)), dict(post=P + 2), dict(pre=P + 8), dict(h=(P + 4, 64))):
        assert v(**kw) == capi.E_ALIGN, kw
    assert capi.lib().fsw_add_norm(0, 3, 60, P, 64, P, 64, P, 0, P, P, 1.0, 1e-5, P, 64, P, 64, None) == capi.E_ALIGN


def test_torch_operators_trace_without_a_gpu(ext):
    for name, dtype in (("bf16", torch.bfloat16), ("fp16", torch.float16)):
        t = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
        i = lambda *s: t(*s, dt=torch.int32)  # noqa: E731
        op = lambda n: getattr(torch.ops.ASMLLM, "%s_%s" % (n, name))  # noqa: E731
        c16 = (t(5, 2, 16, 64), t(5, 2, 16, 64))
        c8 = tuple(t(5, 2, 16, 64, dt=torch.float8_e4m3fn) for _ in range(2)) + tuple(t(5, 2, 16, dt=torch.float8_e8m0fnu) for _ in range(2))
        outs = op("kv_append8")(t(7, 4, 64), t(7, 2, 64), t(7, 2, 64), t(9, 64, dt=torch.float32), i(7), i(7), *c8)
        assert [tuple(o.shape) for o in outs] == [(7, 4, 64), (7, 2, 64), (7, 2, 64)] and all(o.dtype == dtype for o in outs)
        for s, c in (("", c16), ("8", c8)):
            k, v = op("kv_read" + s)(*c, i(3, 2), i(4), 11)
            assert k.shape == v.shape == (11, 2, 64) and k.dtype == dtype
            assert op("attn_shared" + s)(t(3, 4, 64), *c, i(3), 40, i(3, 2), i(3), 32, 0.125).shape == (3, 4, 64)
            for bad in ((i(2), 40, i(3, 2), i(3), 32), (i(3), -1, i(3, 2), i(3), 32), (i(3), 40, i(3, 2), i(3), 33), (i(3, 1), 40, i(3, 2), i(3), 32)):
                with pytest.raises(RuntimeError):
                    op("attn_shared" + s)(t(3, 4, 64), *c, *bad, 0.125)
            for bad in ((i(3, 2), i(3), 11), (i(3, 2), i(4), -1), (i(6), i(4), 11)):
                with pytest.raises(RuntimeError):
                    op("kv_read" + s)(*c, *bad)
        assert op("attn_decode8")(t(3, 4, 64), *c8, i(3, 2), i(3), 32, 0.125).shape == (3, 4, 64)
        for bad in ((c16[0], c16[1], *c8[2:]), (*c8[:2], c8[2], c8[3][:, :1]), (*c8[:2], t(5, 2, 16, dt=torch.uint8), c8[3]),
                    (c8[0][:4], *c8[1:])):
            with pytest.raises(RuntimeError):
                op("attn_decode8")(t(3, 4, 64), *bad, i(3, 2), i(3), 32, 0.125)
        x, h = op("add_norm")(t(2, 3, 64), t(2, 3, 64), t(64), t(64), t(64), 0.5)
        assert x.shape == h.shape == (2, 3, 64) and op("rms_norm")(t(3, 64), t(64)).shape == (3, 64)
        with pytest.raises(RuntimeError):
            op("add_norm")(t(2, 64), t(2, 64), t(2, 32))
        schema = op("kv_append8").default._schema
        assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == ["k_cache", "v_cache", "k_scale", "v_scale"]
    with pytest.raises(RuntimeError, match="GPU"):
        ext.add_norm_bf16(torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, 64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="GPU"):
        ext.kv_read_bf16(*(torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16) for _ in range(2)), torch.zeros(1, 2, dtype=torch.int32),
                         torch.zeros(2, dtype=torch.int32), 3)


def test_ctypes_wrappers_refuse_what_the_c_abi_would_misread(capi):
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    kv = torch.zeros(5, 2, 16, 64, dtype=torch.uint8).view(e4)
    sc = torch.zeros(5, 2, 16, dtype=torch.uint8).view(e8)
    assert capi.kv_cache8(kv, kv, sc, sc).scale_page_stride == 32
    for bad, code in (((kv.view(torch.uint8), kv, sc, sc), capi.E_DTYPE), ((kv, kv, sc, sc.view(torch.uint8)), capi.E_DTYPE),
                      ((kv, kv, sc[:4], sc[:4]), capi.E_SHAPE), ((kv, kv[:, :1], sc, sc), capi.E_SHAPE),
                      ((kv, kv, sc, sc.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(e8)), capi.E_SHAPE)):
        with pytest.raises(capi.FswError) as e:
            capi.kv_cache8(*bad)
        assert e.value.code == code


def test_elements_of_the_oracle_are_those_of_the_type():
    codes = torch.arange(256, dtype=torch.uint8)
    assert torch.equal(cache8.held(codes, torch.tensor(127, dtype=torch.uint8)).nan_to_num(99.0), codes.view(torch.float8_e4m3fn).double().nan_to_num(99.0))
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(300, 32, generator=gen) * torch.logspace(-30, 30, 300)[:, None]
    code, scale = cache8.quantise(x, torch.bfloat16)
    top = x.double().abs().amax(-1)
    for row, s in zip(top.tolist(), scale.tolist()):
        assert row <= 448 * 2.0 ** (s - 127) and (s == 1 or row > 448 * 2.0 ** (s - 128))
    err = (cache8.held(code, scale) - x.double()).abs()
    assert (err <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * cache8.power(scale.long() - 127)[:, None])).all()
    assert torch.equal(code.view(torch.float8_e4m3fn), (x.double() / cache8.power(scale.long() - 127)[:, None]).float().to(torch.float8_e4m3fn))
