"""Every form of the attention kernels against oracle/attention.py: prompts with 64 and with 128 rows a workgroup at every width, single tokens
whose keys lie in few and in many joined shares; and the operators inside compiled functions."""
import pytest
import torch

from oracle import attention
from test_attention_gpu import BF, DEV, HF, angles, inside, int32, randn, starts, untouched

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")

# Hq, Hkv, D of launches of 128 rows a workgroup with few tokens: many heads instead
WIDE = [(128, 64, 128), (96, 96, 128), (256, 32, 128), (144, 144, 64), (300, 100, 40), (64, 32, 256), (160, 32, 256), (80, 80, 80), (48, 48, 136)]
RAGGED = [1, 33, 65, 129, 0, 2, 130, 64, 127]


def sampled(Hq, Hkv):
    """Three key-value heads and their query heads."""
    kv = sorted({0, Hkv // 2, Hkv - 1})
    return kv, [h * (Hq // Hkv) + g for h in kv for g in range(Hq // Hkv)]


def check(capi, nq, nk, Hq, Hkv, D, dtype, rows, behind=0):
    gen = torch.Generator().manual_seed(Hq * 1000 + D + sum(nk))
    cu_q, cu_k = starts(nq), starts(nk)
    Tq, Tk = cu_q[-1] + behind, cu_k[-1]
    assert capi.lib().fsw_attn_prompt_rows(0, Tq, len(nq), Hq, Hkv, D) == rows
    q = randn(gen, Tq, Hq, D, dtype=dtype, scale=1.5)
    kv = randn(gen, max(Tk, 1), 2 * Hkv, D, dtype=dtype)[:Tk]
    out, wide = inside(torch.full((Tq, Hq, D), NAN, dtype=dtype))
    dev = kv.to(DEV)
    capi.attn_prompt(q.to(DEV), dev[:, :Hkv], dev[:, Hkv:], int32(cu_q), int32(cu_k), D ** -0.5, out=out)
    some, heads = sampled(Hq, Hkv)
    ref, mag = attention.prompt(q[:, heads], kv[:, some], kv[:, [Hkv + h for h in some]], cu_q, cu_k, D ** -0.5)
    err = (out[:, heads].cpu().double() - ref).abs()
    assert (err <= attention.tolerance(ref, mag, dtype, True, max(nk))).all()
    assert not torch.isnan(out).any() and untouched(wide, out.shape)


@pytest.mark.parametrize("Hq,Hkv,D", WIDE)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_of_128_rows(capi, Hq, Hkv, D, dtype):
    check(capi, RAGGED, RAGGED, Hq, Hkv, D, dtype, 128, behind=3)


@pytest.mark.parametrize("Hq,Hkv,D", [(64, 64, 128), (96, 48, 64), (32, 16, 256), (128, 16, 80), (32, 16, 200)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_of_128_rows_and_long_walks(capi, Hq, Hkv, D, dtype):
    check(capi, [1500, 130, 1], [1500, 130, 1], Hq, Hkv, D, dtype, 128)


@pytest.mark.parametrize("Hq,Hkv,D", [(128, 64, 128), (256, 64, 64), (64, 32, 256)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_of_128_rows_with_other_numbers_of_keys(capi, Hq, Hkv, D, dtype):
    check(capi, [130, 64, 1, 200, 5, 33, 70], [64, 130, 1, 500, 0, 1, 333], Hq, Hkv, D, dtype, 128)


@pytest.mark.parametrize("Hq,Hkv,D,rows", [(128, 64, 128, 128), (256, 64, 64, 128), (64, 32, 256, 128), (4, 2, 64, 64), (4, 2, 128, 64),
                                           (4, 2, 256, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_infinities_and_later_keys(capi, Hq, Hkv, D, rows, dtype):
    """Infinities and NaN in values and keys reach the rows that see them, as the weighted sum has it, and no others."""
    gen = torch.Generator().manual_seed(D + rows)
    n = 700
    assert capi.lib().fsw_attn_prompt_rows(0, n, 1, Hq, Hkv, D) == rows
    q, k, v = (randn(gen, n, h, D, dtype=dtype).to(DEV) for h in (Hq, Hkv, Hkv))
    cu = int32([0, n])
    clean = capi.attn_prompt(q, k, v, cu, cu, D ** -0.5)
    for at, late in ((n // 2, n - 2), (5, 64), (127, 128)):
        v2 = v.clone()
        v2[at, :, 3], v2[at, :, 4], v2[late, :, 3], v2[late, :, D - 1] = INF, -INF, -INF, NAN
        out = capi.attn_prompt(q, k, v2, cu, cu, D ** -0.5)
        want = clean.clone()
        want[at:, :, 3], want[late:, :, 3], want[at:, :, 4], want[late:, :, D - 1] = INF, NAN, -INF, NAN
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(7.0, INF, -INF), want.nan_to_num(7.0, INF, -INF))
        k2 = k.clone()
        k2[late] = NAN
        out = capi.attn_prompt(q, k2, v, cu, cu, D ** -0.5)
        assert torch.equal(out[:late], clean[:late]) and torch.isnan(out[late:]).all()


# ---------------------------------------------------------------------------------------------- joined shares

def decode_case(gen, lengths, Hq, Hkv, D, page, dtype, max_len):
    """Queries, keys and values [tokens, Hkv, D] of each sequence, caches with pages in random order (NaN where no key lies) and their table."""
    used = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(used) + 2, generator=gen)
    caches = [torch.full((len(order), page, Hkv, D), NAN, dtype=dtype) for _ in range(2)]
    table = torch.zeros(len(lengths), -(-max_len // page), dtype=torch.int32)
    rows, at = [], 0
    for b, (n, u) in enumerate(zip(lengths, used)):
        mine = order[at:at + u]
        table[b, :u] = mine
        at += u
        kv = [randn(gen, n, Hkv, D, dtype=dtype) for _ in range(2)]
        j = torch.arange(n)
        for c, x in zip(caches, kv):
            c[mine[j // page], j % page] = x
        rows.append(kv)
    return randn(gen, len(lengths), Hq, D, dtype=dtype, scale=1.5), rows, [c.transpose(1, 2).to(DEV) for c in caches], table


def parts(capi, B, Hq, Hkv, D, max_len):
    """Shares of a sequence's keys, by the scratch for their sums, maxima and totals."""
    return capi.lib().fsw_attn_decode_workspace_bytes(0, B, Hq, Hkv, D, max_len) // (B * Hq * (D + 2) * 4)


def check_shares(out, q, rows, lengths, scale, dtype, most, seqs=None):
    group = q.shape[1] // rows[0][0].shape[1]
    for b in seqs if seqs is not None else range(len(lengths)):
        for h in range(q.shape[1]):
            ref, mag = attention.attend(q[b, h:h + 1], rows[b][0][:, h // group], rows[b][1][:, h // group], scale, [lengths[b]])
            assert ((out[b, h].cpu().double() - ref[0]).abs() <= attention.tolerance(ref, mag, dtype, False, most)[0]).all(), (b, h)


@pytest.mark.parametrize("lengths", [[5000], [20000, 4100, 513, 0], [4608, 4609, 512, 1, 8191]])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 64, 16), (2, 1, 80, 24), (4, 1, 128, 64), (2, 2, 256, 16), (3, 1, 128, 7)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_of_more_than_eight_shares(capi, lengths, Hq, Hkv, D, page, dtype):
    gen = torch.Generator().manual_seed(sum(lengths) + D)
    most = max(lengths)
    assert parts(capi, len(lengths), Hq, Hkv, D, most) > 8
    q, rows, caches, table = decode_case(gen, lengths, Hq, Hkv, D, page, dtype, most)
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32(lengths), most, D ** -0.5)
    check_shares(out, q, rows, lengths, D ** -0.5, dtype, most)


@pytest.mark.parametrize("lengths,most", [([2000, 1025, 7, 1024], 2000), ([4000, 100], 4096)])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 64, 16), (2, 1, 128, 24), (2, 2, 256, 16)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_of_up_to_eight_shares(capi, lengths, most, Hq, Hkv, D, page, dtype):
    gen = torch.Generator().manual_seed(sum(lengths) + D)
    assert 1 < parts(capi, len(lengths), Hq, Hkv, D, most) <= 8
    q, rows, caches, table = decode_case(gen, lengths, Hq, Hkv, D, page, dtype, most)
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32(lengths), most, D ** -0.5)
    check_shares(out, q, rows, lengths, D ** -0.5, dtype, most)


@pytest.mark.parametrize("Hq,Hkv,D,page,most", [(2, 1, 16, 16, 12000), (16, 8, 64, 7, 30000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_of_many_items_and_a_far_bound(capi, Hq, Hkv, D, page, most, dtype):
    """Many sequences, one of which is as long as the bound: workgroups of four waves, and more than eight shares to join."""
    gen = torch.Generator().manual_seed(most)
    B = 130 // Hkv + 1
    lengths = [17] * B
    lengths[3], lengths[5], lengths[7], lengths[-1] = most, 1024, 1025, 0
    assert B * Hkv >= 128 and parts(capi, B, Hq, Hkv, D, most) > 8
    q, rows, caches, table = decode_case(gen, lengths, Hq, Hkv, D, page, dtype, most)
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32(lengths), most, D ** -0.5)
    check_shares(out, q, rows, lengths, D ** -0.5, dtype, most, [0, 3, 5, 7, B - 1])


@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_bad_pages_in_joined_shares(capi, page, dtype):
    """A page outside the cache, in whichever share, gives NaN for its sequence and leaves the others."""
    gen = torch.Generator().manual_seed(8)
    lengths = [6000, 5999, 4097, 700]
    q, _, caches, table = decode_case(gen, lengths, 4, 2, 64, page, dtype, 6000)
    good = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32(lengths), 6000, 0.125)
    assert torch.isfinite(good).all()
    bad = table.clone()
    bad[0, 5990 // page] = caches[0].shape[0]
    bad[2, 4096 // page] = -1
    bad[3, 0] = 1 << 30
    out = capi.attn_decode(q.to(DEV), *caches, bad.to(DEV), int32(lengths), 6000, 0.125)
    assert torch.isnan(out[[0, 2, 3]]).all() and torch.equal(out[1], good[1])
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32([6001, 5999, -1, 700]), 6000, 0.125)
    assert torch.isnan(out[[0, 2]]).all() and torch.equal(out[[1, 3]], good[[1, 3]])


# ---------------------------------------------------------------------------------------------- compiled functions

def step(q, k, v, cos_sin, positions, slots, k_cache, v_cache, block_table, lengths, cu):
    ops = torch.ops.ASMLLM
    q, k = ops.kv_append_bf16(q, k, v, cos_sin, positions, slots, k_cache, v_cache)
    before = k_cache.sum(dtype=torch.float32) + v_cache[0].sum(dtype=torch.float32)  # read behind the write
    return ops.attn_decode_bf16(q, k_cache, v_cache, block_table, lengths, 64, 0.125), ops.attn_prompt_bf16(q, k, v, cu, cu, 0.125), before


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_attention_operators_under_torch_compile_fullgraph(ext, backend):
    """The append's writes to the caches, declared in its schema, are kept and ordered: what reads the caches behind it sees them."""
    import torch._dynamo
    torch._dynamo.reset()
    gen = torch.Generator().manual_seed(9)
    B, D, page = 5, 64, 16
    q, k, v = (randn(gen, B, h, D).to(DEV) for h in (4, 2, 2))
    caches = [randn(gen, 20, 2, page, D).to(DEV) for _ in range(2)]
    table = torch.randperm(20, generator=gen).int().view(B, 4).to(DEV)
    at = [0, 15, 16, 40, 63]
    slots = int32([int(table[b, t // page]) * page + t % page for b, t in enumerate(at)])
    args = (angles(gen, 64, D).to(DEV), int32(at), slots)
    rest = (table, int32([t + 1 for t in at]), int32([0, 2, B]))
    eager_caches, compiled_caches = [c.clone() for c in caches], [c.clone() for c in caches]
    want = step(q, k, v, *args, *eager_caches, *rest)
    try:
        compiled = torch.compile(step, fullgraph=True, backend=backend)
        got = compiled(q, k, v, *args, *compiled_caches, *rest)
    except Exception as e:  # noqa: BLE001
        if backend == "inductor" and "ASMLLM" not in str(e) and "fullgraph" not in str(e).lower():
            pytest.skip("the inductor backend does not run in this environment: %s" % (str(e).splitlines() or ["?"])[0][:200])
        raise
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and abs(got[2].item() - want[2].item()) < 1.0
    assert all(torch.equal(x, y) for x, y in zip(eager_caches, compiled_caches))
    assert not any(torch.equal(x, y) for x, y in zip(caches, compiled_caches))
    # other inputs through the same compiled function
    q2 = (q * 0.5).contiguous()
    assert torch.equal(compiled(q2, k, v, *args, *compiled_caches, *rest)[0], step(q2, k, v, *args, *eager_caches, *rest)[0])


def test_the_dispatcher_calls_the_kernels_in_both_types(capi):
    gen = torch.Generator().manual_seed(10)
    for dtype, name in ((BF, "bf16"), (HF, "fp16")):
        lengths = [300, 1]
        q, _, caches, table = decode_case(gen, lengths, 4, 2, 64, 16, dtype, 300)
        args = (q.to(DEV), *caches, table.to(DEV), int32(lengths), 300, 0.125)
        assert torch.equal(getattr(torch.ops.ASMLLM, "attn_decode_" + name)(*args), capi.attn_decode(*args))
        k, v = (randn(gen, 2, 2, 64, dtype=dtype).to(DEV) for _ in range(2))
        a, b = ([torch.zeros_like(c) for c in caches] for _ in range(2))
        rest = (angles(gen, 4, 64).to(DEV), int32([3, 1]), int32([17, 5]))
        got = getattr(torch.ops.ASMLLM, "kv_append_" + name)(args[0], k, v, *rest, *a, True)
        want = capi.kv_append(args[0], k, v, *rest, *b, True)
        assert all(torch.equal(x, y) for x, y in zip(list(got) + a, list(want) + b))


@pytest.mark.parametrize("Hq,Hkv,D,page", [(64, 64, 128, 16), (160, 80, 64, 16), (66, 66, 80, 5), (72, 72, 256, 16), (64, 64, 136, 24), (1024, 64, 16, 7)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decode_of_more_than_512_items(capi, Hq, Hkv, D, page, dtype):
    """Workgroups of four waves whose sequences are whole."""
    gen = torch.Generator().manual_seed(Hq + D)
    lengths = [1, 0, 17, 64, 65, 130, 300, 33, 257]
    assert len(lengths) * Hkv > 512 and parts(capi, len(lengths), Hq, Hkv, D, 300) == 0
    q, rows, caches, table = decode_case(gen, lengths, Hq, Hkv, D, page, dtype, 300)
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32(lengths), 300, D ** -0.5)
    some, heads = sampled(Hq, Hkv)
    check_shares(out[:, heads], q[:, heads], [[x[:, some] for x in kv] for kv in rows], lengths, D ** -0.5, dtype, 300)


@pytest.mark.parametrize("B,Hkv", [(16, 8), (43, 6), (64, 8), (65, 8)])
@pytest.mark.parametrize("most", [64, 65, 512, 513, 2560, 2561])
def test_decode_on_both_sides_of_the_rules(capi, B, Hkv, most):
    """Numbers of items and bounds where the workgroups and the shares change."""
    gen = torch.Generator().manual_seed(B + most)
    lengths = [3] * B
    lengths[0], lengths[1], lengths[B - 1] = most, most - 1, 0
    q, rows, caches, table = decode_case(gen, lengths, Hkv, Hkv, 16, 16, BF, most)
    out = capi.attn_decode(q.to(DEV), *caches, table.to(DEV), int32(lengths), most, 0.25)
    check_shares(out, q, rows, lengths, 0.25, BF, most, [0, 1, 2, B - 1])
