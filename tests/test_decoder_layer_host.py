"""The bookkeeping of decoder_layer.py's paged cache, which needs no GPU."""
import pytest
import torch

import decoder_layer


def new(seqs=3, longest=37, page=16):
    return decoder_layer.PagedCache(seqs, longest, 2, 8, page, torch.bfloat16, "cpu")


def test_tokens_have_slots_of_their_own_and_tables_that_lead_to_them():
    cache, seen = new(), set()
    for counts in ([5, 0, 16], [1, 1, 1], [31, 36, 0], [0, 0, 20]):
        before = list(cache.lengths)
        positions, slots = cache.grow(counts)
        table, lengths, longest = cache.table()
        want = [(b, t) for b, n in enumerate(counts) for t in range(before[b], before[b] + n)]
        assert positions.tolist() == [t for _, t in want] and lengths.tolist() == cache.lengths and longest == max(cache.lengths)
        for (b, t), slot in zip(want, slots.tolist()):
            assert slot == int(table[b, t // 16]) * 16 + t % 16 and slot not in seen
            seen.add(slot)
    assert cache.lengths == [37, 37, 37] and len(seen) == 111


def test_a_sequence_grows_no_longer_than_the_cache_was_made_for():
    """Behind it there are no angles, and its row of the table ends: refused before anything has changed."""
    cache = new()
    cache.grow([37, 1, 0])
    state = (list(cache.lengths), list(cache.free), [list(p) for p in cache.pages])
    for counts in ([1, 0, 0], [0, 37, 0], [0, 0, 38], [0, 1, 1000]):
        with pytest.raises(ValueError, match="37"):
            cache.grow(counts)
        assert state == (cache.lengths, cache.free, cache.pages)
    cache.grow([0, 36, 37])


def test_prompts_are_of_sequences_that_have_no_tokens():
    """prefill attends within the rows that it is given: a sequence that has tokens in the cache would lose them."""
    layer, cache = decoder_layer.DecoderLayer.__new__(decoder_layer.DecoderLayer), new()
    cache.grow([3, 0, 0])
    with pytest.raises(ValueError, match="sequence 0"):
        layer.prefill(torch.zeros(5, 16), [2, 3, 0], cache)
    assert cache.lengths == [3, 0, 0]
