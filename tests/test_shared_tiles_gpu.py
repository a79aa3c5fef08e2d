"""Attention behind a shared prefix, on the device, where shares of the prefix have several tiles of 64 keys (every form of the kernel: tiles alternate between
two buffers, the maximum moves on, a tile ends with the prefix), and where the join adds them whatever the own keys are; against the definition in float64.
test_shared_plan_host.py checks that the plan gives these calls that. Tolerances are those of oracle/attention.py."""
import pytest
import torch

from oracle import attention
from test_attention_gpu import BF, DEV, HF, NAN, inside, int32, randn, untouched
from test_cache8_gpu import paged8, rows_of
from test_shared_gpu import widened
from test_shared_plan_host import JOINED, ODD_TILES, ODD_TILES_OF_8, TILES, check_tiles

pytestmark = pytest.mark.gpu
INF = float("inf")
BOTH = [(bits, dtype) for bits in (8, 16) for dtype in (BF, HF)]


def setup(gen, prefix, lengths, Hkv, D, page, dtype, bits, growth=0, odd=()):
    """-> (cache on the device, its cells in float64, table, the prefix's pages). growth: keys of later tiles are up to 2^growth times as large. odd: (key,
    channel, value) among the prefix's values; in 8 bits all are NaN, which is what there is of them."""
    cache, table, pages = paged8(gen, lengths, Hkv, D, page, dtype, prefix=prefix)
    j = torch.arange(prefix)
    at, place = pages[j // page].long().to(DEV), (j % page).to(DEV)
    if growth:
        exponents = cache[2].view(torch.uint8)
        exponents[at, :, place] += (j // 64 % (growth + 1)).to(torch.uint8).to(DEV)[:, None]
    if bits == 8:
        for key, channel, _ in odd:
            cache[1].view(torch.uint8)[int(at[key]), 0, int(place[key]), channel] = 127
    rows = rows_of(cache)
    if bits == 16:
        for key, channel, value in odd:
            rows[1][int(at[key]), 0, int(place[key]), channel] = value
        cache = [r.to(dtype).to(DEV) for r in rows]
    return cache, rows, table, pages


def reference(q, rows, pages, prefix, table, lengths, page, scale):
    """Outputs and weighted sums of magnitudes, a key-value head at a time: the scores of the prefix in one product, own keys sequence by sequence."""
    o, mag = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    Hkv, j = rows[0].shape[1], torch.arange(prefix)
    group = q.shape[1] // Hkv
    for h in range(Hkv):
        heads = slice(h * group, (h + 1) * group)
        k, v = (r[pages[j // page].long(), h, j % page] for r in rows)
        qs = q[:, heads].double()
        first = (qs.reshape(-1, q.shape[2]) @ k.T).view(len(lengths), group, prefix)
        for b, n in enumerate(lengths):
            own = torch.arange(n)
            k_own, v_own = (r[table[b, own // page].long(), h, own % page] for r in rows)
            w = torch.softmax(torch.cat([first[b], qs[b] @ k_own.T], 1) * scale, 1)
            both = torch.cat([v, v_own])
            o[b, heads], mag[b, heads] = w @ both, w @ both.abs()
    return o, mag


def check(capi, seed, B, Hq, Hkv, D, page, prefix, bits, dtype, lengths, max_len=None, growth=0, odd=(), scratch=False):
    gen = torch.Generator().manual_seed(seed)
    cache, rows, table, pages = setup(gen, prefix, lengths, Hkv, D, page, dtype, bits, growth, odd)
    most, scale = max(lengths) if max_len is None else max_len, D ** -0.5
    table = widened(table, most, page)
    q = randn(gen, B, Hq, D, dtype=dtype, scale=1.5)
    out, wide = inside(torch.zeros(B, Hq, D, dtype=dtype))
    workspace = None
    if scratch:  # NaN all over it
        L = capi.lib()
        need = (L.fsw_attn_shared8_workspace_bytes if bits == 8 else L.fsw_attn_shared_workspace_bytes)(0, B, Hq, Hkv, D, prefix, most)
        workspace = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    q_dev, own = q.to(DEV), int32(lengths)
    capi.attn_shared(q_dev, cache, pages.to(DEV), prefix, table.to(DEV), own, most, scale, out=out, workspace=workspace)
    ref, mag = reference(q, rows, pages, prefix, table, lengths, page, scale)
    got, finite = out.cpu().double(), torch.isfinite(ref)
    # scores of keys 2^growth times as large carry that much more of their products' roundings, which is the 2^-12 there
    tol = attention.tolerance(ref, mag, dtype, True, prefix + most) + 2 * (2 ** growth - 1) * 2.0 ** -12 * mag
    assert ((got - ref).abs() <= tol)[finite].all(), ((got - ref).abs() - tol)[finite].max().item()
    assert torch.equal(got[~finite].nan_to_num(7.0, INF, -INF), ref[~finite].nan_to_num(7.0, INF, -INF)) and finite.all() == (not odd)
    assert untouched(wide, out.shape)
    return q_dev, cache, pages.to(DEV), table.to(DEV), own, most, scale, out


@pytest.mark.parametrize("bits,dtype", BOTH)
@pytest.mark.parametrize("case", TILES + ODD_TILES, ids=str)
def test_tiles_one_after_another(capi, case, bits, dtype):
    """The maximum moves on from tile to tile."""
    check_tiles(capi, bits, *case)
    check(capi, case[5] + case[3], *case[:6], bits, dtype, [(7 * b) % 23 for b in range(case[0])], growth=3)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", ODD_TILES_OF_8, ids=str)
def test_tiles_of_8_bits_one_after_another(capi, case, dtype):
    check_tiles(capi, 8, *case)
    check(capi, case[5] + case[3], *case[:6], 8, dtype, [(7 * b) % 23 for b in range(case[0])], growth=3)


@pytest.mark.parametrize("bits,dtype", BOTH)
@pytest.mark.parametrize("case", [TILES[i] for i in (0, 3, 5, 8, 11, 12, 13)] + [ODD_TILES[i] for i in (0, 4, 6)] + ODD_TILES_OF_8[:1], ids=str)
def test_infinities_in_later_tiles(capi, case, bits, dtype):
    prefix, D = case[5], case[3]
    odd = [(70, 3, INF), (prefix - 1, 4, -INF), (prefix - 2, 5, NAN), (prefix // 2, 6, INF), (prefix - 70, 6, -INF), (127, D - 1, INF)]
    check(capi, prefix + D + 1, *case[:6], bits, dtype, [(5 * b) % 30 for b in range(case[0])], odd=odd)


@pytest.mark.parametrize("bits,dtype", BOTH)
@pytest.mark.parametrize("case", JOINED, ids=str)
def test_shares_that_the_join_adds(capi, case, bits, dtype):
    """Own keys none, in one share, in several: each joined with all of the prefix's shares; then lengths and pages that are none of the cache's."""
    B, Hq, Hkv, D, page, prefix, most = case[:7]
    lengths = {1: [most], 2: [0, most], 3: [0, 5, most]}[B]
    q, cache, pages, table, own, most, scale, good = check(capi, prefix + D, B, Hq, Hkv, D, page, prefix, bits, dtype, lengths, most, scratch=True)
    if B == 1:
        check(capi, prefix + D, B, Hq, Hkv, D, page, prefix, bits, dtype, [0], most, scratch=True)
    for bad in (-1, most + 1):
        wrong = own.clone()
        wrong[0] = bad
        out = capi.attn_shared(q, cache, pages, prefix, table, wrong, most, scale)
        assert torch.isnan(out[0]).all() and torch.equal(out[1:], good[1:])
    wrong = table.clone()
    wrong[B - 1, (most - 1) // page] = cache[0].shape[0]
    out = capi.attn_shared(q, cache, pages, prefix, wrong, own, most, scale)
    assert torch.isnan(out[B - 1]).all() and torch.equal(out[:B - 1], good[:B - 1])
    wrong = pages.clone()
    wrong[(prefix - 1) // page] = -1
    assert torch.isnan(capi.attn_shared(q, cache, wrong, prefix, table, own, most, scale)).all()


@pytest.mark.parametrize("bits", [8, 16])
def test_more_rows_than_a_prefix_has_tiles_for_replay_from_a_graph(capi, bits):
    """Shares of several tiles and own keys in several, captured once and replayed over other queries, with eager calls between."""
    B, Hq, Hkv, D, page, prefix = TILES[10][:6]
    gen = torch.Generator().manual_seed(bits)
    lengths = [(37 * b) % 700 for b in range(B)]
    cache, _, table, pages = setup(gen, prefix, lengths, Hkv, D, page, BF, bits)
    q, table, pages, own = randn(gen, B, Hq, D).to(DEV), table.to(DEV), pages.to(DEV), int32(lengths)
    run = lambda x: capi.attn_shared(x, cache, pages, prefix, table, own, max(lengths), D ** -0.5)  # noqa: E731
    run(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(q)
    for step in range(4):
        q.copy_(randn(gen, B, Hq, D))
        want = run(q)
        torch.cuda.synchronize()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
