"""The attention operators on the device against their plain float64 restatement (oracle/attention.py): the rotation with the
append to a paged cache, attention of single tokens over it, and causal attention of packed prompts, through the C ABI and
the torch operators. Tolerances are derived there; outputs lie inside wider buffers of NaN."""
import pytest
import torch

from oracle import attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
NAN = float("nan")


def randn(gen, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def inside(x, fill=NAN, extra=8):
    """x on the device as a view of a wider buffer; -> (view, buffer)"""
    wide = torch.full((x.shape[0] + 1, x.shape[1] + 1, x.shape[2] + extra), fill, dtype=x.dtype, device=DEV)
    view = wide[:x.shape[0], :x.shape[1], :x.shape[2]]
    view.copy_(x)
    return view, wide


def untouched(wide, shape):
    keep = torch.ones(wide.shape, dtype=torch.bool)
    keep[:shape[0], :shape[1], :shape[2]] = False
    return bool(torch.isnan(wide.cpu()[keep]).all())


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def angles(gen, rows, rot):
    a = torch.rand(rows, rot // 2, generator=gen, dtype=torch.float64) * 6.28
    return torch.cat([a.cos(), a.sin()], 1).float()


# ---------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("T,Hq,Hkv,D,rot,interleaved,page", [
    (1, 1, 1, 8, 8, False, 1), (1, 32, 8, 128, 128, False, 16), (5, 4, 2, 64, 64, True, 3), (7, 6, 3, 80, 40, False, 8),
    (33, 8, 1, 96, 48, True, 24), (19, 5, 5, 128, 64, False, 16), (130, 3, 1, 256, 256, False, 64), (3, 2, 2, 72, 72, True, 5),
    (9, 2, 1, 24, 6, False, 16), (9, 2, 1, 24, 10, True, 16), (17, 7, 7, 16, 0, False, 4), (300, 40, 8, 128, 128, True, 32),
    (2, 1024, 1, 8, 8, False, 2)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_append(capi, T, Hq, Hkv, D, rot, interleaved, page, dtype):
    gen = torch.Generator().manual_seed(T * 1000 + D)
    qkv = randn(gen, T, Hq + 2 * Hkv, D, dtype=dtype)
    q, k, v = (t.contiguous() for t in qkv.split([Hq, Hkv, Hkv], 1))
    rows = T + 7
    table = angles(gen, rows, rot)
    positions = torch.randperm(rows, generator=gen)[:T]
    pages = T // page + 3
    slots = torch.randperm(pages * page, generator=gen)[:T]
    slots[T // 2] = -1 if T > 2 else slots[T // 2]        # a padding token: rotated, not appended
    if T > 4:
        slots[1] = pages * page                            # and one slot past the cache
    qkv_dev = qkv.to(DEV)
    caches = [torch.full((pages, Hkv, page, D), NAN, dtype=dtype, device=DEV) for _ in range(2)]
    q_out, q_wide = inside(torch.zeros(T, Hq, D, dtype=dtype))
    k_out, k_wide = inside(torch.zeros(T, Hkv, D, dtype=dtype))
    capi.kv_append(qkv_dev[:, :Hq], qkv_dev[:, Hq:Hq + Hkv], qkv_dev[:, Hq + Hkv:], table.to(DEV), int32(positions.tolist()),
                   int32(slots.tolist()), caches[0], caches[1], interleaved, q_out=q_out, k_out=k_out)
    want_q, want_k = (attention.rotate(x, table, positions, interleaved) for x in (q, k))
    for got, want, src, wide in ((q_out, want_q, q, q_wide), (k_out, want_k, k, k_wide)):
        assert ((got.cpu().double() - want).abs() <= attention.rotate_tolerance(src, want, dtype)).all()
        assert torch.equal(got.cpu()[..., rot:], src[..., rot:]) and untouched(wide, got.shape)
    seen = torch.zeros(pages * page, dtype=torch.bool)
    flat = [c.cpu().transpose(1, 2).reshape(pages * page, Hkv, D) for c in caches]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            seen[s] = True
            assert torch.equal(flat[0][s], k_out.cpu()[t]) and torch.equal(flat[1][s], v[t])
    assert torch.isnan(flat[0][~seen]).all() and torch.isnan(flat[1][~seen]).all()


def test_append_in_place_and_without_rotated_keys(capi):
    """Qout = Q, Kout = NULL, a cache whose tokens lie outside its heads, on another stream."""
    gen = torch.Generator().manual_seed(5)
    T, Hq, Hkv, D = 21, 6, 2, 64
    qkv = randn(gen, T, Hq + 2 * Hkv, D).to(DEV)
    table, positions = angles(gen, 64, 64).to(DEV), int32(list(range(11, 11 + T)))
    caches = [torch.zeros(4, 8, Hkv, D, dtype=BF, device=DEV).transpose(1, 2) for _ in range(2)]
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    want = attention.rotate(q, table, positions, False)
    want_k = attention.rotate(k, table, positions, False)
    src = qkv.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        L, c = capi.lib(), capi.kv_cache(*caches)
        row = lambda t: (t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
        slots = int32(list(range(T)))
        assert L.fsw_kv_append(0, T, Hq, Hkv, D, 64, 0, *row(q), *row(k), *row(v), table.data_ptr(), 64, positions.data_ptr(),
                               slots.data_ptr(), *row(q), None, 0, 0, c, stream.cuda_stream) == capi.OK
    stream.synchronize()
    assert ((q.cpu().double() - want).abs() <= attention.rotate_tolerance(src, want, BF)).all()
    assert torch.equal(qkv[:, Hq:], src[:, Hq:])
    rows = caches[0].cpu().transpose(1, 2).reshape(32, Hkv, D)[:T].double()
    assert ((rows - want_k).abs() <= attention.rotate_tolerance(src, want_k, BF)).all()
    assert torch.equal(caches[1].cpu().transpose(1, 2).reshape(32, Hkv, D)[:T], v.cpu())


def test_append_positions_outside_the_table(capi, ext):
    gen = torch.Generator().manual_seed(6)
    q, k, v = (randn(gen, 4, h, 32).to(DEV) for h in (2, 1, 1))
    caches = [torch.zeros(2, 1, 4, 32, dtype=BF, device=DEV) for _ in range(2)]
    table = angles(gen, 8, 16).to(DEV)
    q_out, k_out = ext.kv_append_bf16(q, k, v, table, int32([7, 8, -1, 0]), int32([0, 1, 2, 3]), *caches)
    for t, bad in enumerate([False, True, True, False]):
        for x in (q_out, k_out):
            assert bool(torch.isnan(x[t, :, :16]).all()) == bad and bool(torch.isnan(x[t, :, :16]).any()) == bad
        assert torch.equal(q_out[t, :, 16:], q[t, :, 16:])
    # a table of rows that are no vectors long, from an odd row on
    odd = angles(gen, 9, 6).to(DEV)[1:]
    q_out, _ = ext.kv_append_bf16(q, k, v, odd, int32([0, 1, 2, 3]), int32([0, 1, 2, 3]), *caches, True)
    want = attention.rotate(q, odd, torch.arange(4), True)
    assert ((q_out.cpu().double() - want).abs() <= attention.rotate_tolerance(q, want, BF)).all()


# ---------------------------------------------------------------------------------------------- decode

def paged(gen, lengths, Hkv, D, page, dtype, spare=3, holes=NAN, token_major=False):
    """Caches with the sequences' pages in random order; what no key lies in holds `holes`. -> (k, v, table)"""
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + spare
    shape = (pages, page, Hkv, D) if token_major else (pages, Hkv, page, D)
    caches = [torch.full(shape, holes, dtype=dtype) for _ in range(2)]
    views = [c.transpose(1, 2) if token_major else c for c in caches]
    order = torch.randperm(pages, generator=gen).tolist()
    width = max(used + [1])
    table, at = [], 0
    for n, u in zip(lengths, used):
        mine = order[at:at + u]
        at += u
        for j in range(n):
            for c in views:
                c[mine[j // page], :, j % page] = randn(gen, Hkv, D, dtype=dtype)
        table.append(mine + [order[-1]] * (width - u))
    devs = [c.to(DEV) for c in caches]
    return [c.transpose(1, 2) if token_major else c for c in devs], torch.tensor(table, dtype=torch.int32)


def check_decode(capi, gen, lengths, Hq, Hkv, D, page, dtype, max_len=None, **kw):
    caches, table = paged(gen, lengths, Hkv, D, page, dtype, **kw)
    q = randn(gen, len(lengths), Hq, D, dtype=dtype, scale=1.5)
    scale = D ** -0.5
    out, wide = inside(torch.zeros(len(lengths), Hq, D, dtype=dtype))
    max_len = max_len or max(lengths)
    width = -(-max_len // page)
    if width > table.shape[1]:
        table = torch.cat([table, table[:, -1:].expand(-1, width - table.shape[1])], 1)
    q_dev = inside(q)[0]
    capi.attn_decode(q_dev, *caches, table.to(DEV), int32(lengths), max_len, scale, out=out)
    ref, mag = attention.decode(q, *caches, table, lengths, scale)
    err = (out.cpu().double() - ref).abs()
    tol = attention.tolerance(ref, mag, dtype, False, max(lengths))
    assert (err <= tol).all(), (err - tol).max().item()
    assert untouched(wide, out.shape)
    return q_dev, caches, table


@pytest.mark.parametrize("Hq,Hkv,D,page", [
    (1, 1, 8, 1), (4, 2, 64, 16), (8, 2, 128, 16), (3, 1, 80, 24), (5, 5, 128, 3), (16, 1, 128, 32), (17, 1, 64, 8),
    (40, 2, 96, 16), (4, 4, 256, 16), (6, 2, 136, 7), (2, 1, 200, 64), (33, 1, 256, 48)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode(capi, Hq, Hkv, D, page, dtype):
    gen = torch.Generator().manual_seed(Hq * 100 + D)
    check_decode(capi, gen, [1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 130], Hq, Hkv, D, page, dtype, token_major=Hq % 2 == 0)


@pytest.mark.parametrize("lengths,max_len", [([700], None), ([1], 5000), ([0, 300], 4000), ([255, 256, 257, 511, 512, 513, 1], 520),
                                             ([1030, 3], 1031)])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 128, 16), (2, 2, 64, 5), (18, 1, 256, 32)])
def test_decode_joined_parts(capi, lengths, max_len, Hq, Hkv, D, page):
    """Few sequences: their keys are shared by several workgroups whose sums are joined; the host's bound is met or far off."""
    gen = torch.Generator().manual_seed(len(lengths) + D)
    most = max_len or max(lengths)
    if most > 600:
        assert capi.lib().fsw_attn_decode_workspace_bytes(0, len(lengths), Hq, Hkv, D, most) > 0
    check_decode(capi, gen, lengths, Hq, Hkv, D, page, BF, max_len=max_len)


@pytest.mark.parametrize("Hq,Hkv,D,page", [(6, 6, 128, 16), (20, 10, 64, 5), (17, 1, 128, 3), (16, 8, 256, 32), (5, 5, 80, 24)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_of_many_sequences(capi, Hq, Hkv, D, page, dtype):
    """128 (sequence, key-value head) items and more: workgroups of four waves."""
    gen = torch.Generator().manual_seed(Hq + D)
    lengths = [1, 0, 17, 64, 65, 130] * (1 + 128 // (6 * Hkv))
    check_decode(capi, gen, lengths, Hq, Hkv, D, page, dtype)


@pytest.mark.parametrize("Hq,Hkv,D,page", [(128, 128, 16, 16), (160, 130, 8, 7)])
def test_decode_joined_parts_of_many_items(capi, Hq, Hkv, D, page):
    gen = torch.Generator().manual_seed(Hq)
    Hq = Hkv if Hq % Hkv else Hq
    assert capi.lib().fsw_attn_decode_workspace_bytes(0, 2, Hq, Hkv, D, 2600) > 0
    check_decode(capi, gen, [2600, 1030], Hq, Hkv, D, page, BF)


@pytest.mark.parametrize("holes", [float("inf"), float("-inf"), NAN, torch.finfo(BF).min])
def test_decode_ignores_what_lies_behind_a_length(capi, holes):
    gen = torch.Generator().manual_seed(9)
    check_decode(capi, gen, [1, 70, 300, 16, 5], 4, 2, 128, 32, BF, holes=holes)
    check_decode(capi, gen, [1, 70, 300, 16, 5], 4, 2, 64, 9, BF, holes=holes)


@pytest.mark.parametrize("page,max_len", [(16, 40), (5, 40), (16, 2000)])
def test_decode_answers_invalid_sequences_with_nan(capi, page, max_len):
    gen = torch.Generator().manual_seed(10)
    lengths = [20, 33, 40, 7, 12]
    q, caches, table = check_decode(capi, gen, lengths, 4, 2, 64, page, BF, max_len=max_len)
    good = capi.attn_decode(q, *caches, table.to(DEV), int32(lengths), max_len, 0.125)
    table[2, 1] = caches[0].shape[0]
    table[3, 0] = -1
    table[0, -(-20 // page):] = 1 << 30       # not among the pages of its 20 keys
    out = capi.attn_decode(q, *caches, table.to(DEV), int32([20, max_len + 1, 40, 7, -5]), max_len, 0.125)
    assert torch.equal(out[0], good[0])
    assert torch.isnan(out[1:]).all()


def test_decode_scores_far_apart(capi):
    """Scores that grow along the sequence by more than fp32 exponents hold, one key that outweighs all others at either end,
    and equal scores: the running maximum moves at every tile, once, and never."""
    gen = torch.Generator().manual_seed(11)
    D, n, page = 64, 600, 16
    k = torch.zeros(n, D)
    for q_scale, ramp in ((40.0, torch.linspace(-8, 8, n)), (40.0, torch.linspace(8, -8, n)), (1.0, torch.zeros(n))):
        k[:, 0] = ramp
        v = randn(gen, n, D)
        q = torch.zeros(1, 1, D)
        q[..., 0] = q_scale
        q = q.to(BF)
        pages = -(-n // page)
        caches = [torch.zeros(pages * page, D, dtype=BF) for _ in range(2)]
        caches[0][:n], caches[1][:n] = k.to(BF), v
        devs = [c.view(pages, 1, page, D).to(DEV) for c in caches]
        table = torch.arange(pages, dtype=torch.int32).view(1, -1)
        for scale in (1.0, 0.125):
            out = capi.attn_decode(q.to(DEV), *devs, table.to(DEV), int32([n]), n, scale)
            ref, mag = attention.decode(q, *devs, table, [n], scale)
            assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, BF, False, n)).all()


def test_decode_offsets_beyond_32_bits(capi):
    """A cache of more than 2^32 elements: keys in its first and last pages."""
    gen = torch.Generator().manual_seed(12)
    D, page, Hkv = 128, 64, 8
    pages = (1 << 32) // (Hkv * page * D) + 9
    caches = [torch.empty(pages, Hkv, page, D, dtype=BF, device=DEV) for _ in range(2)]
    mine = [pages - 1, 0, pages - 2, 3]
    n = 4 * page - 5
    for c in caches:
        for p in mine:
            c[p] = randn(gen, Hkv, page, D).to(DEV)
    table = torch.tensor([mine], dtype=torch.int32)
    q = randn(gen, 1, 16, D)
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32([n]), n, D ** -0.5)
    few = [c[mine].cpu() for c in caches]
    ref, mag = attention.decode(q, *few, torch.arange(4).view(1, -1), [n], D ** -0.5)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, BF, False, n)).all()
    # and an append to the last slot but one
    qkv = [randn(gen, 1, h, D).to(DEV) for h in (16, Hkv, Hkv)]
    slot = pages * page - 2
    q_out, k_out = capi.kv_append(*qkv, angles(gen, 4, D).to(DEV), int32([2]), int32([slot]), *caches)
    assert torch.equal(caches[0][-1, :, page - 2], k_out[0]) and torch.equal(caches[1][-1, :, page - 2], qkv[2][0])


# ---------------------------------------------------------------------------------------------- prompts

def starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def check_prompt(capi, gen, nq, nk, Hq, Hkv, D, dtype, behind=0, scale=None, q_scale=1.5):
    cu_q, cu_k = starts(nq), starts(nk)
    Tq, Tk = cu_q[-1] + behind, cu_k[-1]
    q = randn(gen, Tq, Hq, D, dtype=dtype, scale=q_scale)
    kv = randn(gen, max(Tk, 1), 2 * Hkv, D, dtype=dtype)[:Tk]
    scale = scale or D ** -0.5
    out, wide = inside(torch.full((Tq, Hq, D), NAN, dtype=dtype))
    kv_dev = kv.to(DEV)
    capi.attn_prompt(inside(q)[0], kv_dev[:, :Hkv], kv_dev[:, Hkv:], int32(cu_q), int32(cu_k), scale, out=out)
    ref, mag = attention.prompt(q, kv[:, :Hkv], kv[:, Hkv:], cu_q, cu_k, scale)
    err = (out.cpu().double() - ref).abs()
    tol = attention.tolerance(ref, mag, dtype, True, max(nk))
    assert (err <= tol).all(), (err - tol).max().item()
    assert untouched(wide, out.shape)


@pytest.mark.parametrize("Hq,Hkv,D", [(1, 1, 8), (4, 2, 64), (2, 2, 128), (8, 1, 128), (3, 1, 80), (5, 1, 96), (2, 1, 256), (3, 3, 136),
                                      (20, 1, 64), (130, 1, 16)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt(capi, Hq, Hkv, D, dtype):
    gen = torch.Generator().manual_seed(Hq * 100 + D)
    lengths = [1, 2, 31, 32, 33, 64, 0, 65, 127, 1, 130] if Hq < 20 else [1, 3, 0, 70]
    check_prompt(capi, gen, lengths, lengths, Hq, Hkv, D, dtype, behind=3)


@pytest.mark.parametrize("lengths", [[1], [63], [257], [300, 1, 300], [513], [128] * 5])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_of_several_tiles(capi, lengths, D):
    gen = torch.Generator().manual_seed(sum(lengths) + D)
    check_prompt(capi, gen, lengths, lengths, 2, 1, D, BF if len(lengths) % 2 else HF)


def test_prompt_of_many_sequences(capi):
    """More sequences than one look at 64 offsets finds, empty ones among them."""
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 5, (4200,), generator=gen).tolist()
    lengths[0], lengths[-1], lengths[64], lengths[2000] = 0, 2, 140, 0
    check_prompt(capi, gen, lengths, lengths, 2, 2, 16, BF, behind=1)


@pytest.mark.parametrize("nq,nk", [([5, 1, 40], [70, 200, 40]), ([70, 3], [5, 0]), ([130, 64, 1], [64, 130, 1]), ([300], [1]),
                                   ([1, 1, 1], [1, 129, 0])])
def test_prompt_with_other_numbers_of_keys(capi, nq, nk):
    """Ends aligned: a query that stands before the first key sees none and gives zeros."""
    gen = torch.Generator().manual_seed(sum(nq))
    check_prompt(capi, gen, nq, nk, 4, 2, 64, BF)
    check_prompt(capi, gen, nq, nk, 3, 1, 128, HF)


def test_prompt_is_not_touched_by_other_sequences(capi):
    """NaN and infinities in one sequence stay in it, and a row is not touched by keys that come after it in other tiles."""
    gen = torch.Generator().manual_seed(4)
    lengths = [70, 40, 129]
    cu = starts(lengths)
    q, k, v = (randn(gen, cu[-1], h, 64) for h in (4, 2, 2))
    clean = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32(cu), int32(cu), 0.125)
    for bad in (NAN, float("inf"), float("-inf")):
        k2, v2 = k.clone(), v.clone()
        k2[cu[1]:cu[2]], v2[cu[1]:cu[2]] = bad, bad
        k2[cu[2] + 128:], v2[cu[2] + 128:] = bad, bad
        out = capi.attn_prompt(q.to(DEV), k2.to(DEV), v2.to(DEV), int32(cu), int32(cu), 0.125)
        assert torch.equal(out[:cu[1]], clean[:cu[1]])
        assert torch.equal(out[cu[2]:cu[2] + 128], clean[cu[2]:cu[2] + 128])
        assert torch.isnan(out[cu[2] + 128:]).all()


@pytest.mark.parametrize("Hq,Hkv,D,n", [(2, 1, 64, 90), (4, 4, 128, 70), (3, 1, 256, 40), (16, 2, 72, 130), (8, 1, 128, 1500)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_rows_are_not_touched_by_later_values(capi, Hq, Hkv, D, n, dtype):
    """An infinity or NaN in a later token's value or key does not reach the rows before it, in the same tile either; the rows that
    see it get what the weighted sum gives."""
    gen = torch.Generator().manual_seed(n + D)
    q, k, v = (randn(gen, n, h, D, dtype=dtype) for h in (Hq, Hkv, Hkv))
    cu = int32([0, n])
    clean = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), cu, cu, D ** -0.5).cpu()
    at, late = n // 2, n - 2
    v2 = v.clone()
    v2[at, :, 3], v2[at, :, 4], v2[late, :, 3], v2[late, :, 5] = float("inf"), float("-inf"), float("-inf"), NAN
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v2.to(DEV), cu, cu, D ** -0.5).cpu()
    assert torch.equal(out[:at], clean[:at])
    keep = [c for c in range(D) if c not in (3, 4, 5)]
    assert torch.equal(out[..., keep], clean[..., keep])
    assert torch.equal(out[:late, :, 5], clean[:late, :, 5]) and torch.isnan(out[late:, :, 5]).all()
    assert (out[at:late, :, 3] == float("inf")).all() and torch.isnan(out[late:, :, 3]).all()
    assert (out[at:, :, 4] == float("-inf")).all()
    k2 = k.clone()
    k2[at] = NAN
    out = capi.attn_prompt(q.to(DEV), k2.to(DEV), v.to(DEV), cu, cu, D ** -0.5).cpu()
    assert torch.equal(out[:at], clean[:at]) and torch.isnan(out[at:]).all()


def test_prompt_scores_far_apart(capi):
    gen = torch.Generator().manual_seed(12)
    n, D = 400, 64
    for sign in (1, -1, 0):
        q, k, v = torch.zeros(n, 1, D), torch.zeros(n, 1, D), randn(gen, n, 1, D)
        q[..., 0], k[:, 0, 0] = 40.0, sign * torch.linspace(-8, 8, n)
        q, k = q.to(BF), k.to(BF)
        out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32([0, n]), int32([0, n]), 1.0)
        ref, mag = attention.prompt(q, k, v, [0, n], [0, n], 1.0)
        assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, BF, True, n)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("high", [0, 3, 4, 9, 14, 17, 40, 63, 70, 130])
def test_one_key_far_above_the_others(capi, dtype, high):
    """A key whose score lies 2^30 above all others, wherever it stands in a tile: the running maximum has to be its score, or the
    weights of fp16 overflow. Prompts and single tokens."""
    gen = torch.Generator().manual_seed(high)
    n, D, page = 140, 64, 16
    q, k, v = torch.zeros(n, 2, D), torch.zeros(n, 1, D), randn(gen, n, 1, D, dtype=dtype)
    q[..., 0], k[:, 0, 0], k[high, 0, 0] = 4.0, -2.5, 2.5
    q, k = q.to(dtype), k.to(dtype)
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32([0, n]), int32([0, n]), 1.0)
    ref, mag = attention.prompt(q, k, v, [0, n], [0, n], 1.0)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, dtype, True, n)).all()
    pages = -(-n // page)
    caches = [torch.zeros(pages * page, D, dtype=dtype) for _ in range(2)]
    caches[0][:n], caches[1][:n] = k[:, 0], v[:, 0]
    devs = [c.view(pages, 1, page, D).to(DEV) for c in caches]
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    out = capi.attn_decode(q[:1].to(DEV), *devs, table.to(DEV), int32([n]), n, 1.0)
    ref, mag = attention.decode(q[:1], *devs, table, [n], 1.0)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, dtype, False, n)).all()


def test_prompt_rows_in_other_orders(capi):
    """Head-major rows, a query stride of its own, one key-value head of a wider row."""
    gen = torch.Generator().manual_seed(13)
    n, D = 150, 64
    q = randn(gen, 4, n, D).to(DEV).transpose(0, 1)
    k = randn(gen, 2, n, D).to(DEV).transpose(0, 1)
    v = randn(gen, n, 3, D).to(DEV)[:, 1:]
    out = torch.empty(4, n, D, dtype=BF, device=DEV).transpose(0, 1)
    cu = int32([0, 50, n])
    capi.attn_prompt(q, k, v, cu, cu, 0.1, out=out)
    assert torch.equal(out, capi.attn_prompt(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu, 0.1))


def test_offsets_out_of_range_stay_in_the_arrays(capi):
    """Offsets below zero, past the rows, or descending: the call ends and writes nothing outside (values are unspecified)."""
    gen = torch.Generator().manual_seed(14)
    q, k, v = (randn(gen, 90, h, 64).to(DEV) for h in (2, 1, 1))
    for bad in ([0, 1000, 90], [-5, 40, 1 << 30], [0, 80, 20], [50, 60, 70], [-(1 << 31), 0, (1 << 31) - 1]):
        out, wide = inside(torch.zeros(90, 2, 64, dtype=BF))
        capi.attn_prompt(q, k, v, int32(bad), int32(bad), 0.125, out=out)
        capi.attn_prompt(q, k, v, int32([0, 40, 90]), int32(bad), 0.125, out=out)
        assert untouched(wide, out.shape)


# ---------------------------------------------------------------------------------------------- together

def layer_step(m, q, k, v, table, positions, slots, caches, block_table, lengths, max_len, scale):
    qr, _ = m.kv_append_bf16(q, k, v, table, positions, slots, *caches)
    return m.attn_decode_bf16(qr, *caches, block_table, lengths, max_len, scale)


def test_prompt_then_single_tokens_equal_the_whole_prompt(ext):
    """A prompt's keys appended, then token after token decoded from the cache: what the prompt operator gives for the
    whole sequence, within both sides' roundings."""
    gen = torch.Generator().manual_seed(20)
    T, first, Hq, Hkv, D, page = 90, 77, 8, 2, 128, 16
    q, k, v = (randn(gen, T, h, D).to(DEV) for h in (Hq, Hkv, Hkv))
    table = angles(gen, T, D).to(DEV)
    caches = [torch.full((7, Hkv, page, D), NAN, dtype=BF, device=DEV) for _ in range(2)]
    pages = [3, 5, 0, 6, 1, 2]
    block_table = int32([pages])
    slot = lambda t: pages[t // page] * page + t % page  # noqa: E731
    everything = int32(list(range(T)))
    qr, kr = ext.kv_append_bf16(q[:first], k[:first], v[:first], table, everything[:first],
                                int32([slot(t) for t in range(first)]), *caches)
    cu = int32([0, first])
    parts = [ext.attn_prompt_bf16(qr, kr, v[:first], cu, cu, D ** -0.5)]
    for t in range(first, T):
        parts.append(layer_step(ext, q[t:t + 1], k[t:t + 1], v[t:t + 1], table, int32([t]), int32([slot(t)]), caches, block_table,
                                int32([t + 1]), T, D ** -0.5))
    got = torch.cat(parts).cpu().double()
    scratch = [torch.zeros(6, Hkv, page, D, dtype=BF, device=DEV) for _ in range(2)]
    qr, kr = ext.kv_append_bf16(q, k, v, table, everything, everything, *scratch)
    ref, mag = attention.prompt(qr, kr, v, [0, T], [0, T], D ** -0.5)
    assert ((got - ref).abs() <= attention.tolerance(ref, mag, BF, True, T)).all()


def test_torch_operators_equal_the_c_entry_points(capi, ext):
    gen = torch.Generator().manual_seed(21)
    for dtype, name in ((BF, "bf16"), (HF, "fp16")):
        q, k, v = (randn(gen, 50, h, 64, dtype=dtype).to(DEV) for h in (4, 2, 2))
        table, positions, slots = angles(gen, 50, 64).to(DEV), int32(list(range(50))), int32(list(range(50)))
        a = [torch.zeros(4, 2, 16, 64, dtype=dtype, device=DEV) for _ in range(2)]
        b = [torch.zeros_like(c) for c in a]
        got = getattr(ext, "kv_append_" + name)(q, k, v, table, positions, slots, *a, interleaved=True)
        want = capi.kv_append(q, k, v, table, positions, slots, *b, True)
        assert all(torch.equal(x, y) for x, y in zip(list(got) + a, list(want) + b))
        cu = int32([0, 20, 50])
        assert torch.equal(getattr(ext, "attn_prompt_" + name)(q, k, v, cu, cu, 0.125), capi.attn_prompt(q, k, v, cu, cu, 0.125))
        op = getattr(torch.ops.ASMLLM, "attn_prompt_" + name)
        assert torch.equal(op(q, k, v, cu, cu, 0.125), capi.attn_prompt(q, k, v, cu, cu, 0.125))
        pages, lengths = int32([[0, 1, 2, 3]]), int32([50])
        assert torch.equal(getattr(ext, "attn_decode_" + name)(q[:1], *a, pages, lengths, 50, 0.125),
                           capi.attn_decode(q[:1], *b, pages, lengths, 50, 0.125))
        out = ext.attn_decode_bf16 if dtype == HF else ext.attn_decode_fp16
        with pytest.raises(RuntimeError, match="type"):
            out(q[:1], *a, pages, lengths, 50, 0.125)
    empty = q[:0]
    assert ext.attn_decode_fp16(empty, *a, pages[:0], lengths[:0], 50, 0.125).shape == (0, 4, 64)
    assert ext.attn_prompt_fp16(empty, k[:0], v[:0], int32([0]), int32([0]), 0.125).shape == (0, 4, 64)


def test_a_decode_step_replays_from_a_hip_graph(ext):
    """Append and attention captured once, with split keys; lengths, slots and inputs change between replays."""
    gen = torch.Generator().manual_seed(22)
    B, Hq, Hkv, D, page, most = 2, 8, 2, 128, 16, 1200
    lens = [700, 260]
    caches, block = paged(gen, [most, most], Hkv, D, page, BF, holes=0.0)
    block = block.to(DEV)
    table = angles(gen, most, D).to(DEV)
    q, k, v = (randn(gen, B, h, D).to(DEV) for h in (Hq, Hkv, Hkv))
    positions, lengths, slots = int32([0, 0]), int32([1, 1]), int32([0, 0])

    def place(step):
        n = [x + step for x in lens]
        positions.copy_(int32(n))
        lengths.copy_(int32([x + 1 for x in n]))
        slots.copy_(int32([int(block[b, x // page]) * page + x % page for b, x in enumerate(n)]))

    args = (table, positions, slots, caches, block, lengths, most, D ** -0.5)
    place(0)
    layer_step(ext, q, k, v, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer_step(ext, q, k, v, *args)
    for step in range(1, 5):
        place(step)
        q.copy_(randn(gen, B, Hq, D).to(DEV))
        k.copy_(randn(gen, B, Hkv, D).to(DEV))
        before = [c.clone() for c in caches]
        eager = layer_step(ext, q, k, v, table, positions, slots, before, block, lengths, most, D ** -0.5)
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), "replay %d" % step
        assert all(torch.equal(x, y) for x, y in zip(before, caches))
