"""The attention operators at the limits of what they accept, against oracle/attention.py."""
import pytest
import torch

from oracle import attention
from test_attention_gpu import BF, DEV, HF, angles, int32, paged, randn, starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H", [(65535, 320), (65535, 256)])
def test_prompt_of_most_sequences_and_many_heads(capi, B, H):
    """More (sequence, key-value head) pairs than a launch has workgroups of 256 threads along one dimension; nearly all are empty."""
    gen = torch.Generator().manual_seed(H)
    D, at = 8, {0: 3, 1: 1, 40000: 70, B - 1: 5}
    lengths = torch.zeros(B, dtype=torch.int64)
    for b, n in at.items():
        lengths[b] = n
    cu = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
    T = int(cu[-1])
    q, k, v = (randn(gen, T, H, D) for _ in range(3))
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), cu.int().to(DEV), cu.int().to(DEV), 0.35)
    some = [0, 1, 100, H - 1]
    seqs = starts(list(at.values()))
    ref, mag = attention.prompt(q[:, some], k[:, some], v[:, some], seqs, seqs, 0.35)
    assert ((out[:, some].cpu().double() - ref).abs() <= attention.tolerance(ref, mag, BF, True, 70)).all()


@pytest.mark.parametrize("lengths", [[70, 1, 64, 33], [1100, 3]])
def test_decode_of_sequences_that_share_their_pages(capi, ext, lengths):
    """A block table made by expand(): one row for all sequences, lengths of their own."""
    gen = torch.Generator().manual_seed(5)
    caches, table = paged(gen, [max(lengths)], 2, 64, 16, BF)
    q, B = randn(gen, len(lengths), 4, 64), len(lengths)
    args = (q.to(DEV), *caches, table.to(DEV).expand(B, -1), int32(lengths), max(lengths), 0.125)
    want = capi.attn_decode(*args[:3], table.to(DEV).repeat(B, 1), *args[4:])
    for got in (capi.attn_decode(*args), ext.attn_decode_bf16(*args), torch.ops.ASMLLM.attn_decode_bf16(*args)):
        assert torch.equal(got, want)
    ref, mag = attention.decode(q, *caches, table.expand(B, -1), lengths, 0.125)
    assert ((want.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, BF, False, max(lengths))).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_without_rotated_keys(capi, dtype):
    """k_out=False: the caches and the queries as with them, nothing else."""
    gen = torch.Generator().manual_seed(6)
    T, D = 9, 64
    q, k, v = (randn(gen, T, h, D, dtype=dtype).to(DEV) for h in (4, 2, 2))
    args = (angles(gen, T, D).to(DEV), int32(list(range(T))), int32(list(range(T))))
    a, b = ([torch.zeros(2, 2, 8, D, dtype=dtype, device=DEV) for _ in range(2)] for _ in range(2))
    want, _ = capi.kv_append(q, k, v, *args, *a)
    got, none = capi.kv_append(q, k, v, *args, *b, k_out=False)
    assert none is None and torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(a, b))
