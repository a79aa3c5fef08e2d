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
