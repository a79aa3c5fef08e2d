"""The bookkeeping of decoder_layer.py's paged cache with a shared prefix and with 8 bits, which needs no GPU."""
import pytest
import torch

import decoder_layer


def new(eight=False, prefix=32, page=16):
    return decoder_layer.PagedCache(3, 37, 2, 16, page, torch.bfloat16, "cpu", eight, prefix)


def test_a_prefix_has_pages_of_its_own_and_comes_first():
    cache = new()
    positions, slots = cache.prefix_slots()
    taken = set(slots.tolist())
    assert positions.tolist() == list(range(32)) and len(taken) == 32
    for counts in ([5, 0, 16], [1, 37, 1]):
        before = list(cache.lengths)
        positions, slots = cache.grow(counts)
        assert positions.tolist() == [32 + t for b, n in enumerate(counts) for t in range(before[b], before[b] + n)]
        assert not taken & set(slots.tolist())
        taken |= set(slots.tolist())
    whole, (own, lengths, _) = cache.whole_table(), cache.table()
    assert torch.equal(whole[:, 2:], own) and whole[:, :2].tolist() == [cache.prefix_pages] * 3 and lengths.tolist() == [6, 37, 17]


def test_a_prefix_fills_its_pages():
    with pytest.raises(ValueError, match="33"):
        new(prefix=33)


def test_eight_bits_are_elements_and_scales():
    cache = new(eight=True)
    assert [a.dtype for a in cache.arrays] == [torch.float8_e4m3fn] * 2 + [torch.float8_e8m0fnu] * 2
    assert cache.arrays[2].shape == cache.k.shape[:3] and [a is b for a, b in zip(cache.arrays, (cache.k, cache.v))] == [True, True]
    assert len(new().arrays) == 2


def test_prompts_behind_a_prefix_are_not_taken_without_it():
    layer = decoder_layer.DecoderLayer.__new__(decoder_layer.DecoderLayer)
    with pytest.raises(ValueError, match="prefix"):
        layer.prefill(torch.zeros(5, 16), [2, 3, 0], new())
