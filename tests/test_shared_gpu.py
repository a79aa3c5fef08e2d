"""Attention of single tokens over a prefix that a batch shares and their own keys, on the device, against the float64 restatement of
attention over both together (oracle/attention.py): both caches, all forms of the kernels, edges, invalid input, graphs."""
import pytest
import torch

from oracle import attention
from test_attention_gpu import BF, DEV, HF, NAN, angles, inside, int32, randn, untouched
from test_cache8_gpu import codes_of, paged8, rows_of

pytestmark = pytest.mark.gpu
INF = float("inf")


def setup(gen, prefix, lengths, Hkv, D, page, dtype, bits, **kw):
    """-> (cache on the device, its rows in float64, table, prefix pages). 16 bits: elements of the type, NaN where no key lies."""
    cache, table, pages = paged8(gen, lengths, Hkv, D, page, dtype, prefix=prefix, **kw)
    rows = rows_of(cache)
    if bits == 16:
        cache = [r.to(dtype).to(DEV) for r in rows]
    return cache, rows, table, pages


def reference(q, rows, pages, prefix, table, lengths, page, scale):
    """Every sequence's pages, the prefix's and its own, as one list of cells."""
    o, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // rows[0].shape[1]
    first = [torch.stack([r[int(pages[j // page]), :, j % page] for j in range(prefix)]) if prefix else r[0, :, 0][None][:0] for r in rows]
    for b, n in enumerate(lengths):
        k, v = (torch.cat([f] + [r[int(table[b, j // page]), :, j % page][None] for j in range(n)]) for f, r in zip(first, rows))
        for h in range(q.shape[1]):
            o[b, h:h + 1], mag[b, h:h + 1] = attention.attend(q[b, h:h + 1], k[:, h // group], v[:, h // group], scale, [prefix + n])
    return o, mag


def widened(table, most, page):
    width = -(-most // page)
    return torch.cat([table, table[:, -1:].expand(-1, max(0, width - table.shape[1]))], 1)


def check(capi, gen, prefix, lengths, Hq, Hkv, D, page, dtype, bits, max_len=None, q_scale=1.5, **kw):
    cache, rows, table, pages = setup(gen, prefix, lengths, Hkv, D, page, dtype, bits, **kw)
    B, most, scale = len(lengths), max_len if max_len is not None else max(lengths), D ** -0.5
    table = widened(table, most, page)
    q = randn(gen, B, Hq, D, dtype=dtype, scale=q_scale)
    out, wide = inside(torch.zeros(B, Hq, D, dtype=dtype))
    q_dev = inside(q)[0]
    capi.attn_shared(q_dev, cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), most, scale, out=out)
    ref, mag = reference(q, rows, pages, prefix, table, lengths, page, scale)
    err, tol = (out.cpu().double() - ref).abs(), attention.tolerance(ref, mag, dtype, True, prefix + most)
    assert (err <= tol).all(), (err - tol).max().item()
    assert untouched(wide, out.shape)
    return q_dev, cache, pages.to(DEV), table.to(DEV), most, scale


@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 130])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 64, 16), (8, 2, 128, 16), (3, 1, 80, 24), (5, 5, 128, 3), (6, 2, 96, 8), (2, 1, 256, 4)])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_shared(capi, prefix, Hq, Hkv, D, page, bits, dtype):
    """64 rows a workgroup. Lengths of own keys from none; pages that end inside a tile and pages of any size."""
    gen = torch.Generator().manual_seed(prefix * 7 + D)
    check(capi, gen, prefix, [1, 0, 17, 33, 5], Hq, Hkv, D, page, dtype, bits)


@pytest.mark.parametrize("B,Hq,Hkv,D,page,prefix", [
    (17, 5, 1, 128, 16, 200),      # 85 rows: 128 a workgroup, three waves with rows
    (33, 8, 2, 64, 8, 333),        # 132 rows of 64 channels: two of them
    (40, 8, 1, 128, 32, 500),      # 320 rows
    (70, 4, 1, 112, 64, 129),
    (20, 16, 1, 256, 16, 190),     # 256 channels
    (9, 16, 1, 256, 2, 70),
    (40, 8, 1, 128, 5, 300)])      # pages that a load's rows do not fit
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_shared_by_many_rows(capi, B, Hq, Hkv, D, page, prefix, bits, dtype):
    gen = torch.Generator().manual_seed(B + D)
    check(capi, gen, prefix, [(7 * b) % 40 for b in range(B)], Hq, Hkv, D, page, dtype, bits)


def joined(q, rows, pages, prefix, table, lengths, page, scale):
    """reference() for one key-value head and many rows: a sequence's heads in one product, the prefix gathered once."""
    o, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    at = torch.arange(prefix)
    first = [r[pages[at // page].long(), 0, at % page] for r in rows]
    for b, n in enumerate(lengths):
        own = torch.arange(n)
        k, v = (torch.cat([f, r[table[b, own // page].long(), 0, own % page]]) for f, r in zip(first, rows))
        w = torch.softmax(q[b].double() @ k.T * scale, -1)
        o[b], mag[b] = w @ v, w @ v.abs()
    return o, mag


@pytest.mark.parametrize("D", [112, 128, 256])
@pytest.mark.parametrize("bits,dtype,infinities", [(8, BF, False), (8, HF, False), (16, BF, False), (16, HF, False), (16, BF, True), (16, HF, True)])
def test_shared_by_thousands_of_rows(capi, bits, dtype, D, infinities):
    """256 rows a workgroup (128 of 256 channels), the last with 192 (64) of them, in several shares, the last of which ends inside a tile."""
    gen = torch.Generator().manual_seed(D + bits)
    B, Hq, page, prefix = 99, 64, 16, 4000
    lengths = [(7 * b) % 23 for b in range(B)]
    cache, rows, table, pages = setup(gen, prefix, lengths, 1, D, page, dtype, bits)
    if infinities:
        for key, channel, value in ((2000, 3, INF), (3999, 4, -INF), (0, 5, NAN), (77, 6, INF), (3998, 6, -INF)):
            rows[1][int(pages[key // page]), 0, key % page, channel] = value
        cache = [r.to(dtype).to(DEV) for r in rows]
    q = randn(gen, B, Hq, D, dtype=dtype, scale=1.5)
    out, wide = inside(torch.zeros(B, Hq, D, dtype=dtype))
    capi.attn_shared(q.to(DEV), cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), max(lengths), D ** -0.5, out=out)
    ref, mag = joined(q, rows, pages, prefix, table, lengths, page, D ** -0.5)
    got, finite = out.cpu().double(), torch.isfinite(ref)
    assert ((got - ref).abs() <= attention.tolerance(ref, mag, dtype, True, prefix + 23))[finite].all()
    assert torch.equal(got[~finite].nan_to_num(7.0, INF, -INF), ref[~finite].nan_to_num(7.0, INF, -INF)) and finite.all() == (not infinities)
    assert untouched(wide, out.shape)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("prefix,lengths,max_len", [(4000, [3, 0], 2000), (2500, [700, 1, 130], None), (70, [0, 0, 0], 0), (300, [1], 1)])
def test_shared_in_many_shares(capi, prefix, lengths, max_len, bits):
    """Long prefixes of few rows, own keys in several shares, none at all."""
    gen = torch.Generator().manual_seed(prefix)
    check(capi, gen, prefix, lengths, 4, 2, 128, 16, BF, bits, max_len)
    check(capi, gen, prefix, lengths, 2, 1, 64, 24, HF, bits, max_len)


@pytest.mark.parametrize("bits", [8, 16])
def test_without_a_prefix_it_is_the_decode(capi, bits):
    gen = torch.Generator().manual_seed(4)
    cache, _, table, pages = setup(gen, 0, [40, 0, 700], 2, 64, 16, BF, bits)
    q = randn(gen, 3, 4, 64).to(DEV)
    args = (table.to(DEV), int32([40, 0, 700]), 700, 0.125)
    want = capi.attn_decode8(q, cache, *args) if bits == 8 else capi.attn_decode(q, *cache, *args)
    assert torch.equal(capi.attn_shared(q, cache, pages.to(DEV), 0, *args), want)


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("bits", [8, 16])
def test_what_lies_in_no_page_is_nan(capi, bits, page):
    gen = torch.Generator().manual_seed(6)
    prefix, lengths = 150, [20, 33, 40, 7]
    q, cache, pages, table, most, scale = check(capi, gen, prefix, lengths, 4, 2, 64, page, BF, bits, max_len=60)
    args = (int32(lengths), most, scale)
    good = capi.attn_shared(q, cache, pages, prefix, table, *args)
    bad = table.clone()
    bad[1, 0], bad[2, 1] = -1, cache[0].shape[0]
    out = capi.attn_shared(q, cache, pages, prefix, bad, int32([20, 33, 40, most + 1]), most, scale)
    assert torch.equal(out[0], good[0]) and torch.isnan(out[1:]).all()
    out = capi.attn_shared(q, cache, pages, prefix, table, int32([20, -1, 40, 7]), most, scale)
    assert torch.equal(out[[0, 2, 3]], good[[0, 2, 3]]) and torch.isnan(out[1]).all()
    wrong = torch.cat([pages, int32([1 << 30])])
    assert torch.equal(capi.attn_shared(q, cache, wrong, prefix, table, *args), good)          # behind the prefix's pages
    wrong[-(-prefix // page) - 1] = 1 << 30
    assert torch.isnan(capi.attn_shared(q, cache, wrong, prefix, table, *args)).all()
    wrong[-(-prefix // page) - 1], wrong[0] = pages[-1], -1
    assert torch.isnan(capi.attn_shared(q, cache, wrong, prefix, table, *args)).all()


@pytest.mark.parametrize("B,Hq,Hkv,D,page,prefix", [(3, 4, 2, 64, 16, 100), (40, 8, 1, 128, 32, 500), (17, 5, 1, 128, 16, 3000), (3, 2, 2, 96, 5, 100),
                                                    (5, 2, 1, 256, 64, 70)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinities_in_a_prefix(capi, B, Hq, Hkv, D, page, prefix, dtype):
    """What the weighted sum gives, in every sequence: the infinity, NaN where both signs or a NaN are among the values."""
    gen = torch.Generator().manual_seed(D + prefix)
    lengths = [(5 * b) % 30 for b in range(B)]
    cache, rows, table, pages = setup(gen, prefix, lengths, Hkv, D, page, dtype, 16)
    for key, channel, value in ((prefix // 2, 3, INF), (prefix - 1, 4, -INF), (0, 5, NAN), (prefix // 3, 6, INF), (prefix - 2, 6, -INF),
                                (1, D - 1, INF), (prefix - 3, D - 1, INF)):
        rows[1][int(pages[key // page]), 0, key % page, channel] = value
    cache = [r.to(dtype).to(DEV) for r in rows]
    q = randn(gen, B, Hq, D, dtype=dtype)
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), max(lengths), D ** -0.5).cpu().double()
    ref, mag = reference(q, rows, pages, prefix, table, lengths, page, D ** -0.5)
    finite = torch.isfinite(ref)
    assert ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, True, prefix + 30))[finite].all()
    assert torch.equal(out[~finite].nan_to_num(7.0, INF, -INF), ref[~finite].nan_to_num(7.0, INF, -INF)) and not finite[:, 0, 3].any()


@pytest.mark.parametrize("B,Hq,Hkv,D,page,prefix", [(3, 4, 2, 64, 16, 150), (3, 4, 2, 80, 5, 150), (40, 16, 2, 128, 32, 500), (20, 16, 2, 256, 16, 190)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_what_is_no_number_in_a_prefix_of_8_bits(capi, B, Hq, Hkv, D, page, prefix, dtype):
    """An element, or a row's scale: NaN in its channel, or in all, of the heads that read it, in every sequence. A scale of 2^-127 is a number."""
    gen = torch.Generator().manual_seed(D + prefix)
    lengths = [(5 * b) % 30 for b in range(B)]
    cache, rows, table, pages = setup(gen, prefix, lengths, Hkv, D, page, dtype, 8)
    args = (pages.to(DEV), prefix, table.to(DEV), int32(lengths), max(lengths), D ** -0.5)
    q = randn(gen, B, Hq, D, dtype=dtype)
    for which, value, key, channel in ((1, 127, 7, 3), (1, 255, prefix - 1, D - 1), (0, 127, 20, 7), (3, 255, 66, None), (2, 255, 0, None), (3, 0, 9, None), (2, 0, 9, None)):
        raw = cache[which].view(torch.uint8)
        at = (int(pages[key // page]), Hkv - 1, key % page) + (() if channel is None else (channel,))
        kept = int(raw[at])
        raw[at] = value
        ref, mag = reference(q, rows_of(cache), pages, prefix, table, lengths, page, D ** -0.5)
        out = capi.attn_shared(q.to(DEV), cache, *args).cpu().double()
        finite = torch.isfinite(ref)
        assert ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, True, prefix + 30))[finite].all()
        assert torch.isnan(out[~finite]).all() and finite[:, 0].all() and finite.all() == (value == 0)
        raw[at] = kept


@pytest.mark.parametrize("lengths", [[20, 0, 33], [300, 0, 700]])  # own keys in one share, whose workgroup ends the work, and in several
@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinities_on_both_sides(capi, lengths, dtype):
    gen = torch.Generator().manual_seed(len(lengths) + lengths[0])
    prefix, page, D = 200, 16, 64
    cache, rows, table, pages = setup(gen, prefix, lengths, 1, D, page, dtype, 16)
    for key, channel, value in ((7, 0, INF), (199, 1, -INF), (60, 2, INF)):
        rows[1][int(pages[key // page]), 0, key % page, channel] = value
    for key, channel, value in ((5, 0, INF), (19, 1, INF), (0, 3, -INF), (11, 4, NAN)):
        rows[1][int(table[0, key // page]), 0, key % page, channel] = value
    cache = [r.to(dtype).to(DEV) for r in rows]
    q = randn(gen, 3, 4, D, dtype=dtype)
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), max(lengths), D ** -0.5).cpu().double()
    ref, mag = reference(q, rows, pages, prefix, table, lengths, page, D ** -0.5)
    finite = torch.isfinite(ref)
    assert ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, True, prefix + max(lengths)))[finite].all()
    assert torch.equal(out[~finite].nan_to_num(7.0, INF, -INF), ref[~finite].nan_to_num(7.0, INF, -INF))
    assert torch.equal((~finite).sum(-1), torch.tensor([[5] * 4, [3] * 4, [3] * 4]))


@pytest.mark.parametrize("bits", [8, 16])
def test_one_side_outweighs_the_other(capi, bits):
    """Scores of the prefix far above or below the own keys': the join keeps what weighs."""
    gen = torch.Generator().manual_seed(8)
    for q_scale in (0.0, 60.0):
        check(capi, gen, 200, [1, 40, 90], 4, 2, 128, 16, BF, bits, q_scale=q_scale)
        check(capi, gen, 200, [1, 40, 90], 4, 2, 128, 16, HF, bits, q_scale=q_scale)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [1.2e-38, 2.0e-38, 1e-30])
def test_scales_that_leave_all_weights_alike(capi, bits, dtype, scale):
    """Scores times the scale are nothing: means over prefix and own keys, none of which is lost whatever the units of the maximum."""
    gen = torch.Generator().manual_seed(bits)
    prefix, lengths = 150, [100, 0, 700]
    cache, rows, table, pages = setup(gen, prefix, lengths, 2, 64, 16, dtype, bits)
    q = randn(gen, 3, 4, 64, dtype=dtype)
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), 700, scale)
    ref, mag = reference(q, rows, pages, prefix, table, lengths, 16, scale)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, dtype, True, prefix + 700)).all()


@pytest.mark.parametrize("kw", [dict(token_major=True), dict(wide_scales=True), dict(token_major=True, wide_scales=True)])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 64, 16), (6, 3, 128, 8), (4, 2, 80, 5), (4, 4, 256, 16)])
def test_caches_in_any_order(capi, Hq, Hkv, D, page, kw):
    gen = torch.Generator().manual_seed(D)
    check(capi, gen, 150, [1, 0, 40], Hq, Hkv, D, page, BF, 8, **kw)
    cache, rows, table, pages = setup(gen, 150, [1, 0, 40], Hkv, D, page, HF, 16, **kw)
    cache = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in cache]
    q = randn(gen, 1, Hq, D, dtype=HF).expand(3, -1, -1)                                # one query for all
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), 150, table.to(DEV), int32([1, 0, 40]), 40, 0.1)
    ref, mag = reference(q, rows, pages, 150, table, [1, 0, 40], page, 0.1)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, HF, True, 190)).all()


@pytest.mark.parametrize("dtype,size", [(BF, 3.0e38), (HF, 65504.0)])
def test_values_as_large_as_the_type_has(capi, dtype, size):
    gen = torch.Generator().manual_seed(9)
    prefix, lengths = 700, [100, 3]
    cache, rows, table, pages = setup(gen, prefix, lengths, 1, 64, 16, dtype, 16)
    rows = (rows[0], torch.where(torch.isnan(rows[1]), rows[1], torch.full_like(rows[1], size)))
    cache = [r.to(dtype).to(DEV) for r in rows]
    q = randn(gen, 2, 4, 64, dtype=dtype)
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), 100, 0.125).cpu().double()
    assert torch.isfinite(out).all() and ((out - size).abs() <= 2.0 ** -6 * size).all()


def test_workspace_and_refusals(capi):
    gen = torch.Generator().manual_seed(1)
    cache, _, table, pages = setup(gen, 100, [5, 7], 2, 64, 16, BF, 8)
    q, pages, table, lengths = randn(gen, 2, 4, 64).to(DEV), pages.to(DEV), table.to(DEV), int32([5, 7])
    need = capi.lib().fsw_attn_shared8_workspace_bytes(0, 2, 4, 2, 64, 100, 7)
    want = capi.attn_shared(q, cache, pages, 100, table, lengths, 7, 0.125)
    # room for no more than it asks for, uninitialised
    wide = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(capi.attn_shared(q, cache, pages, 100, table, lengths, 7, 0.125, workspace=wide[:need]), want)
    assert (wide[need:] == 255).all()
    for bad, code in ((dict(workspace=wide[:need - 16]), capi.E_WORKSPACE), (dict(out=torch.empty(2, 4, 32, dtype=BF, device=DEV)), capi.E_SHAPE)):
        with pytest.raises(capi.FswError) as e:
            capi.attn_shared(q, cache, pages, 100, table, lengths, 7, 0.125, **bad)
        assert e.value.code == code
    for args in ((pages, 113), (pages[:1], 17)):
        with pytest.raises(capi.FswError) as e:
            capi.attn_shared(q, cache, *args, table, lengths, 7, 0.125)
        assert e.value.code == capi.E_LD
    with pytest.raises(capi.FswError) as e:
        capi.attn_shared(q, [cache[0].view(torch.uint8), *cache[1:]], pages, 100, table, lengths, 7, 0.125)
    assert e.value.code == capi.E_DTYPE
    with pytest.raises(capi.FswError) as e:
        capi.attn_shared(q, [*cache[:3], cache[3][:, :1]], pages, 100, table, lengths, 7, 0.125)
    assert e.value.code == capi.E_SHAPE


@pytest.mark.parametrize("bits", [8, 16])
def test_scratch_may_hold_anything(capi, bits):
    """Sequences of one share of own keys beside longer ones, NaN all over the scratch; one row of pages for all."""
    gen = torch.Generator().manual_seed(11)
    lengths = [5, 700, 0, 64, 300, 128]
    cache, rows, table, pages = setup(gen, 1000, [700], 2, 64, 16, BF, bits)
    q, table = randn(gen, 6, 8, 64), table.expand(6, -1)
    L = capi.lib()
    need = (L.fsw_attn_shared8_workspace_bytes if bits == 8 else L.fsw_attn_shared_workspace_bytes)(0, 6, 8, 2, 64, 1000, 700)
    scratch = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), 1000, table[:1].to(DEV).expand(6, -1), int32(lengths), 700, 0.125, workspace=scratch)
    ref, mag = reference(q, rows, pages, 1000, table, lengths, 16, 0.125)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, BF, True, 1700)).all()


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype,name", [(BF, "bf16"), (HF, "fp16")])
def test_torch_operators_equal_the_c_entry_points(capi, ext, dtype, name):
    gen = torch.Generator().manual_seed(21)
    op = lambda n: getattr(ext, "%s_%s" % (n, name))  # noqa: E731
    ops = lambda n: getattr(torch.ops.ASMLLM, "%s_%s" % (n, name))  # noqa: E731
    q, k, v = (randn(gen, 50, h, 64, dtype=dtype).to(DEV) for h in (4, 2, 2))
    table, at = angles(gen, 50, 64).to(DEV), int32(list(range(50)))
    a, b = (paged8(gen, [64], 2, 64, 16, dtype)[0] for _ in range(2))
    for x, y in zip(a, b):
        y.view(torch.uint8).copy_(x.view(torch.uint8))
    got = op("kv_append8")(q, k, v, table, at, at, *a, interleaved=True)
    want = capi.kv_append8(q, k, v, table, at, at, b, True)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(x, y) for x, y in zip(codes_of(a), codes_of(b)))
    assert all(torch.equal(x, y) for x, y in zip(ops("kv_append8")(q, k, v, table, at, at, *b, True), want))
    pages, lengths, cu = int32([[0, 1, 2, 3], [3, 2, 1, 0]]), int32([50, 3]), int32([0, 20, 23])
    sixteen = [torch.randn(4, 2, 16, 64, generator=gen).to(dtype).to(DEV) for _ in range(2)]
    for cache, s in ((a, "8"), (sixteen, "")):
        for f in (op, ops):
            got = f("kv_read" + s)(*cache, pages, cu, 25)
            assert all(torch.equal(x, y) for x, y in zip(got, capi.kv_read(cache, pages, cu, 25, dtype)))
            got = f("attn_shared" + s)(q[:2], *cache, int32([2, 0]), 19, pages, lengths, 50, 0.125)
            assert torch.equal(got, capi.attn_shared(q[:2], cache, int32([2, 0]), 19, pages, lengths, 50, 0.125))
    for f in (op, ops):
        assert torch.equal(f("attn_decode8")(q[:2], *a, pages, lengths, 50, 0.125), capi.attn_decode8(q[:2], a, pages, lengths, 50, 0.125))
    empty = q[:0]
    assert op("attn_decode8")(empty, *a, pages[:0], lengths[:0], 50, 0.125).shape == (0, 4, 64)
    assert op("attn_shared8")(empty, *a, int32([2, 0]), 19, pages[:0], lengths[:0], 50, 0.125).shape == (0, 4, 64)
    assert op("kv_append8")(empty, k[:0], v[:0], table, at[:0], at[:0], *a)[2].shape == (0, 2, 64)
    other = ext.attn_decode8_bf16 if dtype == HF else ext.attn_decode8_fp16
    with pytest.raises(RuntimeError, match="type"):
        other(q[:2], *a, pages, lengths, 50, 0.125)
    with pytest.raises(RuntimeError, match="type"):
        op("attn_decode8")(q[:2], *a[:2], a[2].view(torch.uint8), a[3], pages, lengths, 50, 0.125)


@pytest.mark.parametrize("bits", [8, 16])
def test_a_step_replays_from_a_hip_graph(ext, bits):
    """Append, attention behind a prefix and over own keys, norm: captured once, with inputs, slots and lengths that change; two graphs of one
    program alternate. Another stream's work goes on beside."""
    gen = torch.Generator().manual_seed(22)
    B, Hq, Hkv, D, page, most, prefix = 3, 8, 2, 128, 16, 300, 200
    lens = [100, 0, 260]
    cache, _, block, pages = setup(gen, prefix, [most] * B, Hkv, D, page, BF, bits)
    block, pages, table = block.to(DEV), pages.to(DEV), angles(gen, prefix + most, D).to(DEV)
    weight = randn(gen, Hq * D).to(DEV)

    def make():
        return dict(q=randn(gen, B, Hq, D).to(DEV), k=randn(gen, B, Hkv, D).to(DEV), v=randn(gen, B, Hkv, D).to(DEV),
                    positions=int32([0] * B), lengths=int32([1] * B), slots=int32([0] * B))

    def place(st, step):
        n = [x + step for x in lens]
        st["positions"].copy_(int32([prefix + x for x in n]))
        st["lengths"].copy_(int32([x + 1 for x in n]))
        st["slots"].copy_(int32([int(block[b, x // page]) * page + x % page for b, x in enumerate(n)]))
        for name in "qkv":
            st[name].copy_(randn(gen, *st[name].shape).to(DEV))

    def run(st, caches):
        s = "8" if bits == 8 else ""
        qr = getattr(ext, "kv_append%s_bf16" % s)(st["q"], st["k"], st["v"], table, st["positions"], st["slots"], *caches)[0]
        o = getattr(ext, "attn_shared%s_bf16" % s)(qr, *caches, pages, prefix, block, st["lengths"], most, D ** -0.5).view(B, -1)
        return ext.add_norm_bf16(st["q"].view(B, -1), o, None, weight, weight, 0.5)

    sts = [make(), make()]
    for st in sts:
        place(st, 0)
        run(st, cache)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for st in sts:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(st, cache))
    side = torch.cuda.Stream()
    for step in range(1, 6):
        for st, graph, out in zip(sts, graphs, outs):
            place(st, step)
            copies = [c.clone() if bits == 16 else c.view(torch.uint8).clone().view(c.dtype) for c in cache]
            eager = run(st, copies)
            torch.cuda.synchronize()
            for o in out:
                o.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                busy = torch.randn(512, 512, device=DEV) @ torch.randn(512, 512, device=DEV)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager)), "replay %d" % step
            assert all(torch.equal(x, y) for x, y in zip(codes_of(cache), codes_of(copies)))
            del busy


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_operators_under_torch_compile_fullgraph(ext, backend):
    """A function of the operators traces whole, with the caches it writes, and gives what the operators give."""
    import torch._dynamo
    torch._dynamo.reset()
    gen = torch.Generator().manual_seed(31)
    ops, D, page, prefix = torch.ops.ASMLLM, 64, 16, 50
    cache, rows, block, pages = setup(gen, prefix, [40, 40], 2, D, page, BF, 8)
    sixteen = [r.to(BF).to(DEV) for r in rows]
    block, pages, table, weight = block.to(DEV), pages.to(DEV), angles(gen, 100, D).to(DEV), randn(gen, 4 * D).to(DEV)
    at = [0, 7]
    slots = int32([int(block[b, x // page]) * page + x % page for b, x in enumerate(at)])
    where, lengths, cu = int32([prefix + x for x in at]), int32([x + 1 for x in at]), int32([0, 1, 9])

    def step(q, k, v, a, b, a_s, b_s, c, d):
        qr, ka, va = ops.kv_append8_bf16(q, k, v, table, where, slots, a, b, a_s, b_s, False)
        o = ops.attn_shared8_bf16(qr, a, b, a_s, b_s, pages, prefix, block, lengths, 40, 0.125)
        p = ops.attn_shared_bf16(qr, c, d, pages, prefix, block, lengths, 40, 0.125)
        o = o + p + ops.attn_decode8_bf16(qr, a, b, a_s, b_s, block, lengths, 40, 0.125)
        x, y = ops.add_norm_bf16(q.flatten(1), o.flatten(1), None, weight, weight, 0.5)
        return (x, y, ops.rms_norm_bf16(y, weight), ka, va, *ops.kv_read8_bf16(a, b, a_s, b_s, block, cu, 9), *ops.kv_read_bf16(c, d, block, cu, 9))

    q, k, v = (randn(gen, 2, h, D).to(DEV) for h in (4, 2, 2))
    copy = lambda c: [x.view(torch.uint8).clone().view(x.dtype) for x in c]  # noqa: E731
    ones, others = copy(cache), copy(cache)
    want = step(q, k, v, *ones, *sixteen)
    got = torch.compile(step, fullgraph=True, backend=backend)(q, k, v, *others, *sixteen)
    assert len(want) == len(got) and all(torch.equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(x, y) for x, y in zip(codes_of(others), codes_of(ones)))
    assert not torch.equal(codes_of(cache)[0], codes_of(ones)[0])


def test_calls_on_other_streams_at_once(capi):
    """Scratch is each call's own: two streams' calls give what they give one after the other."""
    gen = torch.Generator().manual_seed(30)
    cache, _, table, pages = setup(gen, 2000, [40, 300], 2, 128, 16, BF, 16)
    pages, table, lengths = pages.to(DEV), table.to(DEV), int32([40, 300])
    qs = [randn(gen, 2, 8, 128).to(DEV) for _ in range(6)]
    want = [capi.attn_shared(q, cache, pages, 2000, table, lengths, 300, 0.1) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(capi.attn_shared(q, cache, pages, 2000, table, lengths, 300, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
