"""What a refused call leaves of decoder_layer.py's paged cache: the tokens that it had. The operators are stand-ins, so no GPU is needed."""
import pytest
import torch

import decoder_layer


class Refused(RuntimeError):
    pass


def layer_that_fails_at(name):
    """A layer whose operator `name` refuses its call; the others return rows of the right sizes."""
    layer = decoder_layer.DecoderLayer.__new__(decoder_layer.DecoderLayer)
    layer.heads, layer.kv_heads, layer.channels, layer.sandwich, layer.cos_sin = 4, 2, 16, False, torch.zeros(69, 16)
    layer.w_qkv, layer.w_out, layer.w13, layer.w2 = (torch.zeros(n, 64) for n in (128, 64, 8, 64))

    def stand_in(op, result):
        def call(*args):
            if op == name:
                raise Refused(op)
            return result(*args)
        setattr(layer, op, call)

    stand_in("project", lambda h, w: h.new_zeros(h.shape[0], w.shape[0]))
    for op in ("append", "append8"):
        stand_in(op, lambda q, k, v, *rest: (q, k) if len(rest) == 5 else (q, k, v))
    for op in ("read", "read8"):
        stand_in(op, lambda *args: [torch.zeros(args[-1], 2, 16)] * 2)
    for op in ("prompt", "decode", "decode8", "shared", "shared8"):
        stand_in(op, lambda q, *rest: torch.zeros_like(q))
    stand_in("mlp", lambda h, *weights: h)
    return layer


def new(prefix, eight=False):
    return decoder_layer.PagedCache(3, 37, 2, 16, 16, torch.bfloat16, "cpu", eight, prefix)


def state(cache):
    return list(cache.lengths), sorted(cache.free), [list(p) for p in cache.pages]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("prefix", [0, 32])
@pytest.mark.parametrize("name", ["project", "append", "read", "prompt", "decode", "mlp", None])
def test_a_refused_call_leaves_the_tokens_that_were_there(name, prefix, eight):
    cache, s = new(prefix, eight), "8" if eight else ""
    name = {"append": "append" + s, "read": "read" + s, "decode": ("shared" if prefix else "decode") + s}.get(name, name)
    cache.grow([0, 16, 5])
    before = state(cache)
    layer = layer_that_fails_at(name)
    calls = {"step": lambda: layer.step(torch.zeros(3, 64), cache), "extend": lambda: layer.extend(torch.zeros(30, 64), [12, 1, 17], cache)}
    if not prefix:
        calls["prefill"] = lambda: layer.prefill(torch.zeros(20, 64), [20, 0, 0], cache)
    reached = {"step": ("project", "append" + s, ("shared" if prefix else "decode") + s, "mlp"), "extend": ("project", "append" + s, "read" + s, "prompt", "mlp"),
               "prefill": ("project", "append" + s, "prompt", "mlp")}
    for what, call in calls.items():
        if name in reached[what]:
            with pytest.raises(Refused):
                call()
            assert state(cache) == before, what
            cache.grow([0, 21, 1])  # the places that were given back are handed out again, once
            taken = [p for own in cache.pages for p in own] + cache.free + cache.prefix_pages
            assert sorted(taken) == list(range(len(taken)))
            cache = new(prefix, eight)
            cache.grow([0, 16, 5])
    if name is None:
        layer.extend(torch.zeros(30, 64), [12, 1, 17], cache)
        layer.step(torch.zeros(3, 64), cache)
        assert cache.lengths == [13, 18, 23]


def test_more_cached_rows_than_a_call_takes_are_refused_before_the_cache_grows(monkeypatch):
    """The prefix is packed once for every sequence: 3 x 32 tokens and 51 of their own."""
    cache, layer = new(32), layer_that_fails_at("append")
    cache.grow([0, 16, 5])
    before = state(cache)
    monkeypatch.setattr(decoder_layer, "MOST_ROWS", 146)
    with pytest.raises(ValueError, match="147"):
        layer.extend(torch.zeros(30, 64), [12, 1, 17], cache)
    assert state(cache) == before
    monkeypatch.setattr(decoder_layer, "MOST_ROWS", 147)
    layer_that_fails_at(None).extend(torch.zeros(30, 64), [12, 1, 17], cache)
    assert cache.lengths == [12, 17, 22]


@pytest.mark.parametrize("prefix", [0, 32])
def test_no_rows_are_an_answer_of_no_rows(prefix):
    """Prompts in more parts than the longest has tokens: some parts have none."""
    cache, layer = new(prefix), layer_that_fails_at(None)
    cache.grow([0, 16, 5])
    assert layer.extend(torch.zeros(0, 64), [0, 0, 0], cache).shape == (0, 64)
    if not prefix:
        assert layer.prefill(torch.zeros(0, 64), [0, 0, 0], cache).shape == (0, 64)
    assert cache.lengths == [0, 16, 5]


@pytest.mark.parametrize("turns", [0, -1])
def test_prompts_come_in_parts(turns):
    """Without any, tokens would be decoded behind nothing."""
    with pytest.raises(ValueError, match="part"):
        decoder_layer.run(turns=turns)


def test_positions_behind_a_prefix_have_angles():
    """The cache was made for 37 tokens behind 32, the layer for 40 in a row: refused, not NaN."""
    cache, layer = new(32), layer_that_fails_at(None)
    layer.cos_sin = torch.zeros(40, 16)
    layer.extend(torch.zeros(7, 64), [7, 0, 0], cache)
    before = state(cache)
    assert layer.step(torch.zeros(3, 64), cache).shape == (3, 64)
    with pytest.raises(ValueError, match="made for 40"):
        layer.step(torch.zeros(3, 64), cache)
    with pytest.raises(ValueError, match="made for 40"):
        layer.extend(torch.zeros(9, 64), [0, 0, 9], cache)
    assert cache.lengths == [8, 1, 1] and before[0] == [7, 0, 0]
    layer.cos_sin = torch.zeros(31, 16)
    with pytest.raises(ValueError, match="made for 31"):
        layer.prefill_shared(torch.zeros(32, 64), new(32))
