"""The attention operators where values and weights come to the edges of their types: infinities and NaN that are seen, weights
far below the largest, sums beyond fp32. Against the definition in float64 (oracle/attention.py), which answers these too."""
import pytest
import torch

from oracle import attention
from test_attention_gpu import BF, DEV, HF, int32, paged, randn

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def agrees(out, ref, mag, dtype, weights_rounded, keys):
    """Finite where the definition is, within the tolerance; the same infinities and NaN elsewhere."""
    out, finite = out.cpu().double(), torch.isfinite(ref)
    tol = attention.tolerance(ref, mag, dtype, weights_rounded, keys)
    return bool(((out - ref).abs() <= tol)[finite].all()) and torch.equal(out[~finite].nan_to_num(7.0, INF, -INF),
                                                                          ref[~finite].nan_to_num(7.0, INF, -INF))


def put(cache, table, page, seq, key, channel, value):
    cache[int(table[seq, key // page]), :, key % page, channel] = value


@pytest.mark.parametrize("lengths,max_len,Hq,Hkv,D,page", [
    ([40, 1, 17, 300], None, 4, 2, 64, 16),        # one share, sixteen waves
    ([40, 1, 17, 300], None, 3, 1, 80, 5),         # pages that 16 keys do not fit
    ([40, 1, 17, 300], None, 17, 1, 128, 32),      # two tiles of heads
    ([40, 2, 33], None, 4, 4, 256, 16),
    ([1300, 40, 700], None, 4, 2, 128, 16),        # shares that are joined
    ([1300, 40, 700], None, 2, 1, 256, 7),
    ([9000, 600], None, 2, 1, 64, 64),             # more than eight of them
    ([70, 1, 130], None, 64, 64, 64, 16),
    ([70, 1, 33, 130] * 3, None, 64, 64, 64, 16),  # many items: four waves
    ([70, 1, 130], None, 200, 200, 128, 9)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_infinities_that_are_seen(capi, lengths, max_len, Hq, Hkv, D, page, dtype):
    """What the weighted sum gives: the infinity, NaN where both signs or a NaN are seen; other channels and sequences as before."""
    gen = torch.Generator().manual_seed(sum(lengths) + D)
    caches, table = paged(gen, lengths, Hkv, D, page, dtype)
    q = randn(gen, len(lengths), Hq, D, dtype=dtype, scale=1.5)
    most, scale = max_len or max(lengths), D ** -0.5
    args = (table.to(DEV), int32(lengths), most, scale)
    clean = capi.attn_decode(q.to(DEV), *caches, *args)
    v = caches[1].clone()
    for seq in (0, len(lengths) - 1):
        n = lengths[seq]
        put(v, table, page, seq, n // 2, 3, INF)
        put(v, table, page, seq, n - 1, 4, -INF)
        put(v, table, page, seq, 0, 5, NAN)
        put(v, table, page, seq, n // 3, 6, INF)
        put(v, table, page, seq, n - 2, 6, -INF)
        put(v, table, page, seq, n // 4, D - 1, INF)
        put(v, table, page, seq, n // 4 + 1, D - 1, INF)
    out = capi.attn_decode(q.to(DEV), caches[0], v, *args)
    ref, mag = attention.decode(q, caches[0], v, table, lengths, scale)
    assert (ref[0, :, 3] == INF).all() and torch.isnan(ref[0, :, 6]).all()
    assert agrees(out, ref, mag, dtype, False, most)
    assert torch.equal(out[1:-1], clean[1:-1])


@pytest.mark.parametrize("n,page", [(81, 16), (90, 9), (4097, 16)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_infinity_of_a_key_that_weighs_little(capi, n, page, dtype):
    """A key whose score lies 2^288 below the others' weighs more than nothing, also where it has a share to itself."""
    D, pages = 64, -(-n // page)
    gen = torch.Generator().manual_seed(n)
    k, v = torch.zeros(pages * page, D), randn(gen, pages * page, D, dtype=dtype)
    k[n - 1, 0] = -10.0
    v[n - 1, 2] = -INF
    q = torch.zeros(1, 1, D)
    q[..., 0] = 20.0
    q = q.to(dtype)
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    caches = [c.to(dtype).view(pages, 1, page, D).to(DEV) for c in (k, v)]
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32([n]), n, 1.0)
    ref, mag = attention.decode(q, *caches, table, [n], 1.0)
    assert ref[0, 0, 2] == -INF and agrees(out, ref, mag, dtype, False, n)


def one_above_the_others(gen, n, D, bits, dtype):
    """q [1, 2, D], k and v [n, D]: at scale 1 a key's weight is 2^bits times that of each of the others, wherever it stands (here: first).
    Channel 0 of the values is one everywhere, channel 1 one but for that key's zero, so that its sum is what the others weigh."""
    k, v = torch.zeros(n, D), randn(gen, n, D, dtype=dtype)
    k[:, 0], k[0, 0] = -bits * 0.6931472 / 4, bits * 0.6931472 / 4
    v[:, :2], v[0, 1] = 1.0, 0.0
    q = torch.zeros(1, 2, D)
    q[..., 0] = 2.0
    return q.to(dtype), k.to(dtype), v


@pytest.mark.parametrize("bits", [12.0, 20.4, 24.4, 24.8, 25.1, 30.0])
@pytest.mark.parametrize("n,D,page", [(131071, 64, 64), (40000, 128, 9)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_many_small_weights_beside_a_large_one(capi, n, D, page, bits, dtype):
    """A long context whose first key outweighs each of the others by far, but not all of them together: no weight may be lost, and the
    sum that normalises has to be the sum of the weights that were used."""
    gen = torch.Generator().manual_seed(n)
    q, k, v = one_above_the_others(gen, n, D, bits, dtype)
    pages = -(-n // page)
    caches = [torch.cat([c, c.new_zeros(pages * page - n, D)]).view(pages, 1, page, D) for c in (k, v)]
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    out = capi.attn_decode(q.to(DEV), *(c.to(DEV) for c in caches), table.to(DEV), int32([n]), n, 1.0).cpu().double()
    for h in range(2):
        ref, mag = attention.attend(q[:, h], k, v, 1.0, [n])
        assert ((out[:, h] - ref).abs() <= attention.tolerance(ref, mag, dtype, False, n)).all()


@pytest.mark.parametrize("bits", [20.4, 24.8, 25.1, 30.0])
@pytest.mark.parametrize("page", [64, 9])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_many_small_weights_in_one_share(capi, page, bits, dtype):
    """The same where sequences are so many that none is split: a wave takes a quarter of the keys beside the large one."""
    n, D, B = 131071, 16, 8192
    gen = torch.Generator().manual_seed(n)
    q, k, v = one_above_the_others(gen, n, D, bits, dtype)
    pages = -(-n // page)
    caches = [torch.cat([c, c.new_zeros(pages * page - n, D)]).view(pages, 1, page, D).to(DEV) for c in (k, v)]
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(B, 1)
    lengths = torch.full((B,), 1, dtype=torch.int32, device=DEV)
    lengths[5] = n
    assert capi.lib().fsw_attn_decode_workspace_bytes(0, B, 2, 1, D, n) == 0
    out = capi.attn_decode(q.to(DEV).repeat(B, 1, 1), *caches, table, lengths, n, 1.0).cpu().double()
    for h in range(2):
        ref, mag = attention.attend(q[:, h], k, v, 1.0, [n])
        assert ((out[5, h] - ref[0]).abs() <= attention.tolerance(ref, mag, dtype, False, n)[0]).all()
    assert torch.equal(out[:5], v[0].double().expand(5, 2, D)) and torch.equal(out[6:], v[0].double().expand(B - 6, 2, D))


@pytest.mark.parametrize("bits", [12.0, 20.4, 24.8, 25.1, 30.0])
@pytest.mark.parametrize("nq,D", [(1, 64), (3, 128), (2, 256)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_many_small_weights_beside_a_large_one(capi, nq, D, bits, dtype):
    """The last rows of a long prompt, whose first key outweighs each of the others by far. Weights are rounded once, to u of their size. fp16 has
    none below 2^-24; a kernel that lets a weight reach 2^15 where the running maximum's is at least 2^11 loses at most 2^-25 / 2^11 of each."""
    n = 131071
    gen = torch.Generator().manual_seed(n)
    q, k, v = one_above_the_others(gen, n, D, bits, dtype)
    q = q.repeat(nq, 1, 1)
    out = capi.attn_prompt(q.to(DEV), k.to(DEV).view(n, 1, D), v.to(DEV).view(n, 1, D), int32([0, nq]), int32([0, n]), 1.0).cpu().double()
    u = attention.U[dtype]
    for i in range(nq):
        ref, mag = attention.attend(q[i, :1], k, v, 1.0, [n - nq + 1 + i])
        tol = u * ref.abs() + 2 * (2.0 ** -12 + u) * mag + 2.0 ** -24
        if dtype == HF:
            tol += n * 2.0 ** -36 * v.abs().max()
        for h in range(2):
            assert ((out[i, h] - ref[0]).abs() <= tol[0]).all()


def huge(x, dtype, size):
    """x of the order of one, scaled to the largest finite values there are (fp16: 60000)."""
    return (x.float().clamp(-1, 1) * (size if dtype == BF else 60000.0)).to(dtype)


@pytest.mark.parametrize("size", [3.3e38, 1e37])
@pytest.mark.parametrize("n,Hq,Hkv,D,page,max_len", [(40, 2, 1, 64, 16, None), (700, 4, 2, 128, 9, None), (9000, 2, 1, 64, 64, None),
                                                     (2600, 130, 130, 8, 16, None), (300, 2, 1, 256, 16, 20000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_values_as_large_as_the_type_has(capi, n, Hq, Hkv, D, page, max_len, dtype, size):
    """A mean of finite values is finite, whatever their size and number."""
    gen = torch.Generator().manual_seed(n)
    caches, table = paged(gen, [n], Hkv, D, page, dtype)
    most = max_len or n
    table = torch.cat([table, table[:, :1].expand(1, -(-most // page) - table.shape[1])], 1)
    v = caches[1].cpu()
    v = huge(torch.where(torch.isnan(v), v, v.abs() + 0.5), dtype, size)  # of one sign: nothing cancels
    q = randn(gen, 1, Hq, D, dtype=dtype)
    out = capi.attn_decode(q.to(DEV), caches[0], v.to(DEV), table.to(DEV), int32([n]), most, 0.3).cpu().double()
    ref, mag = attention.decode(q, caches[0], v, table, [n], 0.3)
    assert torch.isfinite(ref).all() and ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, False, n)).all()


@pytest.mark.parametrize("size", [3.3e38, 1e37])
@pytest.mark.parametrize("n,Hq,Hkv,D", [(40, 2, 1, 64), (300, 4, 2, 128), (130, 2, 1, 256), (700, 1, 1, 16)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_values_as_large_as_the_type_has(capi, n, Hq, Hkv, D, dtype, size):
    gen = torch.Generator().manual_seed(n)
    q, k, v = (randn(gen, n, h, D, dtype=dtype) for h in (Hq, Hkv, Hkv))
    v = huge(v.abs() + 0.5, dtype, size)
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32([0, n]), int32([0, n]), 0.3).cpu().double()
    ref, mag = attention.prompt(q, k, v, [0, n], [0, n], 0.3)
    assert torch.isfinite(ref).all() and ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, True, n)).all()


@pytest.mark.parametrize("size", [1e-33, 1e-30])
def test_values_as_small_as_bf16_has(capi, size):
    """What keeps large values finite costs small ones little: sums are off by less than 2^-149 (fp32's smallest) over the largest weight, which is
    at least 2^-8 over twice the number of keys the launch counts with."""
    gen = torch.Generator().manual_seed(1)
    n, D = 500, 64
    q, k, v = (randn(gen, n, 1, D) for _ in range(3))
    v = (v.float() * size).to(BF)
    least = n * 2.0 ** -149 * 2 ** 8 * 2 * n
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32([0, n]), int32([0, n]), 0.1).cpu().double()
    ref, mag = attention.prompt(q, k, v, [0, n], [0, n], 0.1)
    assert ((out - ref).abs() <= 2.0 ** -8 * ref.abs() + 2 * (2.0 ** -12 + 2.0 ** -8) * mag + least).all()
    caches = [torch.cat([c, c.new_zeros(12, 1, D)]).view(32, 16, 1, D).transpose(1, 2).to(DEV) for c in (k, v)]
    table = torch.arange(32, dtype=torch.int32).view(1, -1)
    out = capi.attn_decode(q[:1].to(DEV), *caches, table.to(DEV), int32([n]), n, 0.1).cpu().double()
    ref, mag = attention.decode(q[:1], *caches, table, [n], 0.1)
    assert ((out - ref).abs() <= 2.0 ** -8 * ref.abs() + 2 * 2.0 ** -12 * mag + least).all()


@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -125, 2.0 ** -120])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_smallest_scales_weigh_all_keys_alike(capi, dtype, scale):
    gen = torch.Generator().manual_seed(2)
    n, D = 200, 64
    q, k, v = (randn(gen, n, 1, D, dtype=dtype) for _ in range(3))
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32([0, n]), int32([0, n]), scale).cpu().double()
    ref, mag = attention.prompt(q, k, v, [0, n], [0, n], scale)
    assert ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, True, n)).all()
    caches = [torch.cat([c, c.new_zeros(8, 1, D)]).view(13, 16, 1, D).transpose(1, 2).to(DEV) for c in (k, v)]
    table = torch.arange(13, dtype=torch.int32).view(1, -1)
    out = capi.attn_decode(q[:1].to(DEV), *caches, table.to(DEV), int32([n]), n, scale).cpu().double()
    ref, mag = attention.decode(q[:1], *caches, table, [n], scale)
    assert ((out - ref).abs() <= attention.tolerance(ref, mag, dtype, False, n)).all()
