"""The cache in 8 bits on the device: the append (elements and scales exactly those of the definition in float64, oracle/cache8.py), the
packed rows read back, and the attention of single tokens over it, against the float64 restatement (oracle/attention.py) of what the
elements and scales stand for. Tolerances are derived there; outputs lie inside wider buffers of NaN."""
import pytest
import torch

from oracle import attention, cache8
from test_attention_gpu import BF, DEV, HF, NAN, angles, inside, int32, randn, starts, untouched

pytestmark = pytest.mark.gpu
E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def new_cache(pages, Hkv, page, D, code=127, scale=255, token_major=False, wide_scales=False):
    """(k, v, k_scale, v_scale) on the device, filled with one byte each (NaN, unless said otherwise), in either order of tokens and heads."""
    shape = (pages, page, Hkv) if token_major else (pages, Hkv, page)
    kv = [torch.full((*shape, D), code, dtype=torch.uint8, device=DEV).view(E4) for _ in range(2)]
    sc = [torch.full((*shape, 3 if wide_scales else 1), scale, dtype=torch.uint8, device=DEV)[..., 0].view(E8) for _ in range(2)]
    return [c.transpose(1, 2) if token_major else c for c in kv + sc]


def codes_of(cache):
    return [c.view(torch.uint8).cpu() for c in cache]


# ---------------------------------------------------------------------------------------------- append

def check_append(capi, qkv, Hq, Hkv, rot, interleaved, page, dtype, slots, positions, table, pages, token_major=False, **outs):
    T, _, D = qkv.shape
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    cache = new_cache(pages, Hkv, page, D, 1, 2, token_major, wide_scales=token_major)
    q_out, wide_q = inside(torch.zeros_like(q))
    k_out, wide_k = inside(torch.zeros_like(k))
    v_out, wide_v = inside(torch.zeros_like(v))
    dev = qkv.to(DEV).split([Hq, Hkv, Hkv], 1)
    capi.kv_append8(*dev, table.to(DEV), int32(positions.tolist()), int32(slots.tolist()), cache, interleaved, q_out, k_out, v_out)
    ref_q = attention.rotate(q, table, positions, interleaved)
    assert ((q_out.cpu().double() - ref_q).abs() <= attention.rotate_tolerance(q, ref_q, dtype)).all()
    assert untouched(wide_q, q.shape) and untouched(wide_k, k.shape) and untouched(wide_v, v.shape)
    want = [torch.full((pages, Hkv, page, D), 1, dtype=torch.uint8) for _ in range(2)] + \
           [torch.full((pages, Hkv, page), 2, dtype=torch.uint8) for _ in range(2)]
    for i, (rows, got) in enumerate(((attention.rotate(k, table, positions, interleaved), k_out), (v.double(), v_out))):
        code, scale = cache8.quantise(rows, dtype)
        # rotated NaN has no sign to speak of
        assert torch.equal(got.cpu().nan_to_num(7.0), cache8.held(code, scale).to(dtype).nan_to_num(7.0))
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                want[i][slot // page, :, slot % page] = code[t]
                want[i + 2][slot // page, :, slot % page] = scale[t]
    got = codes_of(cache)
    for i in range(2):
        a, b = got[i], want[i]
        assert torch.equal(torch.where(a % 128 == 127, 127, a), torch.where(b % 128 == 127, 127, b))
        assert torch.equal(got[i + 2], want[i + 2])


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,interleaved,page", [
    (1, 1, 1, 16, 16, False, 1), (1, 32, 8, 128, 128, False, 16), (5, 4, 2, 64, 64, True, 3), (7, 6, 3, 80, 48, False, 8),
    (33, 8, 1, 96, 48, True, 24), (19, 5, 5, 128, 64, False, 16), (130, 3, 1, 256, 256, False, 64), (3, 2, 2, 112, 112, True, 5),
    (9, 2, 1, 32, 6, False, 16), (9, 2, 1, 32, 10, True, 16), (17, 7, 7, 16, 0, False, 4), (300, 40, 8, 128, 128, True, 32),
    (2, 1024, 1, 16, 16, False, 2), (11, 3, 3, 48, 34, False, 16), (4, 2, 2, 240, 8, True, 16)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_append(capi, T, Hq, Hkv, D, rot, interleaved, page, dtype):
    gen = torch.Generator().manual_seed(T * 1000 + D)
    qkv = randn(gen, T, Hq + 2 * Hkv, D, dtype=dtype) * torch.tensor([0.01, 1.0, 30.0])[torch.randint(3, (T, 1, 1), generator=gen)].to(dtype)
    table, positions = angles(gen, T + 7, rot), torch.randperm(T + 7, generator=gen)[:T]
    pages = T // page + 3
    slots = torch.randperm(pages * page, generator=gen)[:T]
    if T > 4:
        slots[T // 2], slots[0] = -1, pages * page          # outside the cache: appended nowhere
    check_append(capi, qkv, Hq, Hkv, rot, interleaved, page, dtype, slots, positions, table, pages, token_major=T % 2 == 1)


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,page", [(21, 6, 2, 80, 40, 8), (9, 4, 4, 112, 56, 16), (5, 2, 1, 32, 24, 3), (3, 1, 1, 256, 248, 16), (70, 3, 1, 16, 8, 16)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_of_halves_that_are_multiples_of_four(capi, T, Hq, Hkv, D, rot, page, dtype):
    gen = torch.Generator().manual_seed(T + D)
    qkv = randn(gen, T, Hq + 2 * Hkv, D, dtype=dtype)
    table, positions, pages = angles(gen, T + 7, rot), torch.randperm(T + 7, generator=gen)[:T], T // page + 2
    check_append(capi, qkv, Hq, Hkv, rot, False, page, dtype, torch.randperm(pages * page, generator=gen)[:T], positions, table, pages, token_major=T % 2 == 1)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_rows_at_the_edges_of_the_types(capi, dtype):
    """Zeros of both signs, the smallest and the largest numbers, largest elements next to 448 scales, ties, infinities and NaN among the others."""
    D, big, small = 64, torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    tiny = 2.0 ** (-133 if dtype == BF else -24)
    gen = torch.Generator().manual_seed(5)
    rows = [torch.zeros(D), -torch.zeros(D), torch.full((D,), tiny), torch.full((D,), -small)]
    rows += [torch.full((D,), big), torch.linspace(-1, 1, D) * big]
    for top in (448.0, 450.0 if dtype == BF else 448.25, 447.0, 1.75, 1.7578125, 224.0):
        x = torch.randn(D, generator=gen) * top / 4
        x[3] = top
        rows.append(x.clamp(-top, top))
    ties = torch.tensor([17.0, 19.0, 21.0, 23.0, 25.0, 1.0625, 1.1875, 2.0 ** -7 * 1.5, 2.0 ** -10, 2.0 ** -10 * 3])   # halfway between two elements
    rows.append(torch.cat([torch.tensor([448.0]), ties, -ties, torch.zeros(D - 21)]))
    for bad in (float("inf"), -float("inf"), NAN):
        x = torch.randn(D, generator=gen)
        x[5], x[6] = bad, 3.0
        rows.append(x)
    rows += [torch.full((D,), NAN), torch.full((D,), float("inf")), torch.cat([torch.tensor([100.0]), torch.full((D - 1,), 2.0 ** -6)])]
    x = torch.stack(rows).to(dtype)
    T = x.shape[0]
    for rot, interleaved in ((0, False), (D, False), (D, True)):
        table = torch.cat([torch.full((2, rot // 2), 0.75), torch.full((2, rot // 2), -0.625)], 1) if rot else torch.zeros(2, 0)
        qkv = torch.stack([torch.zeros_like(x), x, x], 1)
        check_append(capi, qkv, 1, 1, rot, interleaved, 8, dtype, torch.arange(T), torch.ones(T, dtype=torch.int64), table, T // 8 + 1)


def test_append_positions_outside_the_table(capi):
    gen = torch.Generator().manual_seed(3)
    qkv = randn(gen, 3, 4, 64).to(DEV)
    q, k, v = qkv.split([2, 1, 1], 1)
    cache = new_cache(1, 1, 16, 64, 0, 0)
    q_out, k_out, v_out = capi.kv_append8(q, k, v, angles(gen, 5, 32).to(DEV), int32([-1, 5, 4]), int32([0, 1, 2]), cache)
    assert torch.isnan(q_out[:2, :, :32]).all() and torch.isnan(k_out[:2, :, :32]).all() and not torch.isnan(q_out[2]).any()
    code, scale = cache8.quantise(k[:2, :, 32:].cpu().double(), BF)          # the others keep their elements and decide the scale
    got = codes_of(cache)
    assert torch.equal(got[0][0, 0, :2, 32:], code[:, 0]) and (got[0][0, 0, :2, :32] % 128 == 127).all()
    assert torch.equal(got[2][0, 0, :2], scale[:, 0]) and not torch.isnan(v_out).any()


@pytest.mark.parametrize("rot,interleaved", [(64, False), (64, True), (24, False), (10, False), (14, True)])
def test_append_in_place_and_without_rows(capi, rot, interleaved):
    gen = torch.Generator().manual_seed(rot)
    q, k, v = (randn(gen, 37, h, 64).to(DEV) for h in (6, 2, 2))
    args = (angles(gen, 37, rot).to(DEV), int32(list(range(37))), int32(list(range(37))))
    a, b, c = (new_cache(3, 2, 16, 64, 0, 0) for _ in range(3))
    want = capi.kv_append8(q, k, v, *args, a, interleaved)
    assert capi.kv_append8(q, k, v, *args, b, interleaved, None, False, False)[1:] == (None, None)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    capi.kv_append8(q2, k2, v2, *args, c, interleaved, q2, k2, v2)
    assert all(torch.equal(x, y) for x, y in zip(want, (q2, k2, v2)))
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(codes_of(a), codes_of(b), codes_of(c)))


# ---------------------------------------------------------------------------------------------- caches of sequences

def paged8(gen, lengths, Hkv, D, page, dtype, spare=3, prefix=0, **kw):
    """A cache with the sequences' pages in random order; what no key lies in is NaN. -> (cache on the device, table, pages of a prefix)"""
    used, shared = [-(-n // page) for n in lengths], -(-prefix // page)
    pages = sum(used) + shared + spare
    cache = new_cache(pages, Hkv, page, D, **kw)
    order = torch.randperm(pages, generator=gen).tolist()
    width, at, table = max(used + [1]), shared, []
    host = [c.view(torch.uint8) for c in cache]
    where = [(j, order[:shared]) for j in range(prefix)]
    for n, u in zip(lengths, used):
        mine = order[at:at + u]
        at += u
        where += [(j, mine) for j in range(n)]
        table.append(mine + [order[-1]] * (width - u))
    if where:
        page_of = torch.tensor([mine[j // page] for j, mine in where], device=DEV)
        place = torch.tensor([j % page for j, _ in where], device=DEV)
        for i in range(2):
            code, scale = cache8.quantise(randn(gen, len(where), Hkv, D, dtype=dtype).double(), dtype)
            host[i][page_of, :, place] = code.to(DEV)
            host[i + 2][page_of, :, place] = scale.to(DEV)
    return cache, torch.tensor(table, dtype=torch.int32), torch.tensor(order[:shared], dtype=torch.int32)


def rows_of(cache):
    """Keys and values of all cells, float64 [pages, Hkv, page, D]."""
    k, v, ks, vs = codes_of(cache)
    return cache8.held(k, ks), cache8.held(v, vs)


# ---------------------------------------------------------------------------------------------- read

@pytest.mark.parametrize("Hkv,D,page", [(2, 64, 16), (1, 128, 5), (8, 128, 64), (3, 80, 24), (4, 256, 1), (130, 16, 8)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bits", [8, 16])
def test_read(capi, Hkv, D, page, dtype, bits):
    gen = torch.Generator().manual_seed(Hkv * 100 + D)
    lengths = [1, 0, 17, 64, 0, 0, 130, 3]
    cache, table, _ = paged8(gen, lengths, Hkv, D, page, dtype, token_major=Hkv % 2 == 0)
    rows = rows_of(cache)
    if bits == 16:
        cache = [r.to(dtype).to(DEV) for r in rows]
    T, cu = sum(lengths) + 5, starts(lengths)
    outs = [inside(torch.zeros(T, Hkv, D, dtype=dtype)) for _ in range(2)]
    capi.kv_read(cache, table.to(DEV), int32(cu), T, dtype, outs[0][0], outs[1][0])
    for (got, wide), cells in zip(outs, rows):
        want = torch.cat([cells[int(table[b, j // page]), :, j % page][None] for b, n in enumerate(lengths) for j in range(n)]
                         + [torch.zeros(5, Hkv, D, dtype=torch.float64)]).to(dtype)
        assert torch.equal(got.cpu(), want) and untouched(wide, got.shape)


@pytest.mark.parametrize("bits", [8, 16])
def test_read_of_many_sequences_and_of_none(capi, bits):
    gen = torch.Generator().manual_seed(1)
    lengths = [0, 1, 3] * 1500
    cache, table, _ = paged8(gen, lengths, 1, 16, 2, BF)
    rows = rows_of(cache)
    if bits == 16:
        cache = [r.to(BF).to(DEV) for r in rows]
    k, v = capi.kv_read(cache, table.to(DEV), int32(starts(lengths)), sum(lengths), BF)
    for got, cells in ((k, rows[0]), (v, rows[1])):
        want = torch.stack([cells[int(table[b, j // 2]), :, j % 2] for b, n in enumerate(lengths) for j in range(n)]).to(BF)
        assert torch.equal(got.cpu(), want)
    k, v = capi.kv_read(cache, table[:0].to(DEV), int32([0]), 7, BF)
    assert not k.any() and not v.any()
    assert capi.kv_read(cache, table[:1].to(DEV), int32([0, 0]), 0, BF)[0].shape == (0, 1, 16)


@pytest.mark.parametrize("bits", [8, 16])
def test_read_answers_what_is_in_no_page_with_nan(capi, bits):
    gen = torch.Generator().manual_seed(2)
    cache, table, _ = paged8(gen, [40, 40, 40], 2, 64, 16, BF)
    if bits == 16:
        cache = [r.to(BF).to(DEV) for r in rows_of(cache)]
    good = capi.kv_read(cache, table.to(DEV), int32([0, 40, 80, 120]), 120, BF)
    table[1, 1], table[2, 0] = -1, cache[0].shape[0]
    wide = torch.full((3, 6), 1 << 30, dtype=torch.int32)
    wide[:, :3] = table
    k, v = capi.kv_read(cache, wide.to(DEV)[:, :3], int32([0, 40, 80, 140]), 140, BF)          # the last has more tokens than its row has pages
    for got, want in ((k, good[0]), (v, good[1])):
        assert torch.equal(got[:56], want[:56]) and torch.isnan(got[56:72]).all() and torch.equal(got[72:80], want[72:80])
        assert torch.isnan(got[80:96]).all() and torch.equal(got[96:120], want[96:120]) and torch.isnan(got[128:]).all()
    # offsets that ascend from nowhere stay in the arrays
    for bad in ([5, 1000, 90, 120], [-5, 40, 1 << 30, 3], [0, 80, 20, 10], [-(1 << 31), 0, 0, (1 << 31) - 1]):
        capi.kv_read(cache, wide.to(DEV)[:, :3], int32(bad), 120, BF)
    # one row of pages for all
    k, _ = capi.kv_read(cache, table[:1].to(DEV).expand(2, -1), int32([0, 40, 80]), 80, BF)
    assert torch.equal(k[:40], k[40:]) and torch.equal(k[:40], good[0][:40])


# ---------------------------------------------------------------------------------------------- decode

def check_decode8(capi, gen, lengths, Hq, Hkv, D, page, dtype, max_len=None, **kw):
    cache, table, _ = paged8(gen, lengths, Hkv, D, page, dtype, **kw)
    q = randn(gen, len(lengths), Hq, D, dtype=dtype, scale=1.5)
    out, wide = inside(torch.zeros(len(lengths), Hq, D, dtype=dtype))
    max_len = max_len or max(lengths)
    width = -(-max_len // page)
    if width > table.shape[1]:
        table = torch.cat([table, table[:, -1:].expand(-1, width - table.shape[1])], 1)
    q_dev = inside(q)[0]
    capi.attn_decode8(q_dev, cache, table.to(DEV), int32(lengths), max_len, D ** -0.5, out=out)
    ref, mag = attention.decode(q, *rows_of(cache), table, lengths, D ** -0.5)
    err, tol = (out.cpu().double() - ref).abs(), attention.tolerance(ref, mag, dtype, False, max(lengths))
    assert (err <= tol).all(), (err - tol).max().item()
    assert untouched(wide, out.shape)
    return q_dev, cache, table


@pytest.mark.parametrize("Hq,Hkv,D,page", [
    (1, 1, 16, 1), (4, 2, 64, 16), (8, 2, 128, 16), (3, 1, 80, 24), (5, 5, 128, 3), (16, 1, 128, 32), (17, 1, 64, 8),
    (40, 2, 96, 16), (4, 4, 256, 16), (6, 2, 144, 7), (2, 1, 208, 64), (33, 1, 256, 48)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode8(capi, Hq, Hkv, D, page, dtype):
    gen = torch.Generator().manual_seed(Hq * 100 + D)
    check_decode8(capi, gen, [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 130], Hq, Hkv, D, page, dtype, token_major=Hq % 2 == 0)


@pytest.mark.parametrize("token_major,wide", [(False, True), (True, False), (True, True)])
def test_decode8_scales_in_any_order(capi, token_major, wide):
    gen = torch.Generator().manual_seed(17)
    check_decode8(capi, gen, [70, 33, 200], 4, 2, 128, 16, BF, token_major=token_major, wide_scales=wide)


@pytest.mark.parametrize("lengths,max_len", [([700], None), ([1], 5000), ([0, 300], 4000), ([255, 256, 257, 511, 512, 513, 1], 520),
                                             ([1030, 3], 1031), ([9000, 600], None)])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 128, 16), (2, 2, 64, 5), (18, 1, 256, 32)])
def test_decode8_joined_parts(capi, lengths, max_len, Hq, Hkv, D, page):
    gen = torch.Generator().manual_seed(len(lengths) + D)
    most = max_len or max(lengths)
    if most > 768:
        assert capi.lib().fsw_attn_decode8_workspace_bytes(0, len(lengths), Hq, Hkv, D, most) > 0
    check_decode8(capi, gen, lengths, Hq, Hkv, D, page, BF, max_len=max_len)


@pytest.mark.parametrize("Hq,Hkv,D,page", [(6, 6, 128, 16), (20, 10, 64, 5), (17, 1, 128, 3), (16, 8, 256, 32), (5, 5, 80, 24)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode8_of_many_sequences(capi, Hq, Hkv, D, page, dtype):
    gen = torch.Generator().manual_seed(Hq + D)
    check_decode8(capi, gen, [1, 0, 17, 64, 65, 130] * (1 + 512 // (6 * Hkv)), Hq, Hkv, D, page, dtype)


@pytest.mark.parametrize("page,max_len", [(16, 40), (5, 40), (16, 2000)])
def test_decode8_answers_invalid_sequences_with_nan(capi, page, max_len):
    gen = torch.Generator().manual_seed(10)
    lengths = [20, 33, 40, 7, 12]
    q, cache, table = check_decode8(capi, gen, lengths, 4, 2, 64, page, BF, max_len=max_len)
    good = capi.attn_decode8(q, cache, table.to(DEV), int32(lengths), max_len, 0.125)
    table[2, 1] = cache[0].shape[0]
    table[3, 0] = -1
    table[0, -(-20 // page):] = 1 << 30       # not among the pages of its 20 keys
    out = capi.attn_decode8(q, cache, table.to(DEV), int32([20, max_len + 1, 40, 7, -5]), max_len, 0.125)
    assert torch.equal(out[0], good[0]) and torch.isnan(out[1:]).all()


@pytest.mark.parametrize("Hq,Hkv,D,page,most", [(4, 2, 128, 16, None), (3, 1, 80, 5, None), (40, 40, 64, 16, None), (4, 2, 256, 32, 3000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode8_numbers_that_are_none(capi, Hq, Hkv, D, page, most, dtype):
    """A NaN among the values: NaN in its channel, one among the keys, or a scale of 255, all of the heads that read it; others as before."""
    gen = torch.Generator().manual_seed(D)
    lengths = [40, 300, 17, 65, 33, 80, 5] * 2
    cache, table, _ = paged8(gen, lengths, Hkv, D, page, dtype)
    q = randn(gen, len(lengths), Hq, D, dtype=dtype).to(DEV)
    most = most or max(lengths)
    table = torch.cat([table, table[:, -1:].expand(-1, max(0, -(-most // page) - table.shape[1]))], 1)
    args = (table.to(DEV), int32(lengths), most, D ** -0.5)
    clean = capi.attn_decode8(q, cache, *args)
    raw, group = [c.view(torch.uint8) for c in cache], Hq // Hkv
    for seq, (which, value, channel) in enumerate(((1, 127, 3), (1, 255, D - 1), (0, 127, 7), (3, 255, None), (2, 255, None))):
        n = lengths[seq] * 2 // 3
        cell = raw[which][int(table[seq, n // page]), 0, n % page]
        if channel is None:
            cell.fill_(value)
        else:
            cell[channel] = value
    out = capi.attn_decode8(q, cache, *args)
    want = clean.clone()
    want[0, :group, 3] = want[1, :group, D - 1] = NAN
    want[2:5, :group] = NAN
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [16, 9])
def test_decode8_scales_far_apart(capi, dtype, page):
    """Values from the smallest to the largest that a row may have, and keys of which one outweighs all others."""
    gen = torch.Generator().manual_seed(page)
    D, n, Hkv = 64, 130, 2
    for spread in ((-126, -100), (60, 118) if dtype == BF else (-20, 8), (-8, -6)):
        cache, table, _ = paged8(gen, [n, 70], Hkv, D, page, dtype)
        raw = cache[3].view(torch.uint8)
        raw.copy_(torch.where(raw == 255, raw, torch.randint(spread[0] + 127, spread[1] + 128, raw.shape, generator=gen).to(torch.uint8).to(DEV)))
        q = randn(gen, 2, 4, D, dtype=dtype, scale=6.0)
        out = capi.attn_decode8(q.to(DEV), cache, table.to(DEV), int32([n, 70]), n, 0.5)
        ref, mag = attention.decode(q, *rows_of(cache), table, [n, 70], 0.5)
        # A weight times its scale is held in two bf16 numbers, whose smallest step is 2^-133: off by at most half of it, times an element of up to
        # 448, for each of n keys, in units in which the largest weight, and so their sum, is 2^-(8 + log2 n) = 2^-16 at least. Beside that the
        # outputs' own steps, halved.
        small = n * 448 * 2.0 ** -134 * 2.0 ** 16
        tol = attention.U[dtype] * ref.abs() + 2 * 2.0 ** -12 * mag + small + (2.0 ** -25 if dtype == HF else 2.0 ** -134)
        assert ((out.cpu().double() - ref).abs() <= tol).all(), spread


def test_cache8_offsets_beyond_32_bits(capi):
    gen = torch.Generator().manual_seed(12)
    D, page, Hkv = 128, 64, 8
    pages = (1 << 32) // (Hkv * page * D) + 9
    cache = [torch.empty(pages, Hkv, page, D, dtype=torch.uint8, device=DEV).view(E4) for _ in range(2)] + \
            [torch.empty(pages, Hkv, page, dtype=torch.uint8, device=DEV).view(E8) for _ in range(2)]
    mine, n = [pages - 1, 0, pages - 2, 3], 4 * page - 5
    kv = [randn(gen, n, Hkv, D) for _ in range(2)]
    slots = int32([mine[j // page] * page + j % page for j in range(n)])
    none = torch.zeros(1, 0, device=DEV)
    _, k, v = capi.kv_append8(torch.zeros(n, 16, D, dtype=BF, device=DEV), *(x.to(DEV) for x in kv), none, int32([0] * n), slots, cache)
    table = int32([mine])
    q = randn(gen, 1, 16, D)
    got = capi.kv_read(cache, table, int32([0, n]), n, BF)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    ref, mag = attention.prompt(q, k, v, [0, 1], [0, n], D ** -0.5)
    tol = attention.tolerance(ref, mag, BF, True, n)
    assert ((capi.attn_decode8(q.to(DEV), cache, table, int32([n]), n, D ** -0.5).cpu().double() - ref).abs() <= tol).all()
    own = int32([mine[2:]])
    out = capi.attn_shared(q.to(DEV), cache, int32(mine[:2]), 2 * page, own, int32([n - 2 * page]), 2 * page, D ** -0.5)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
