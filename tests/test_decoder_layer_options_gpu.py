"""decoder_layer.py with a cache of 8 bits, a shared prefix, prompts in parts and norms around both blocks: tokens decoded one by one against the
same tokens inside whole prompts. Both sides round at the same places and see the same keys and values (those that the cache holds), but a projection of
other shapes sums in another order: a dozen roundings of terms of the outputs' size may differ, and in 8 bits an element of a key or a value may be
the next one, 2^-3 of it. Such an element's row is one of many in the weighted mean and one channel of many in a score, so that it moves less than half of its own change; outputs reach
four times their root mean square."""
import pytest
import torch

import decoder_layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,u", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d,ff,heads,kv_heads,prompts,steps,page,prefix,turns,sandwich", [
    (1024, 2816, 16, 4, (37, 5, 130), 9, 16, 0, 1, False), (1024, 2816, 16, 4, (37, 5, 130), 5, 16, 208, 1, True),
    (512, 1032, 4, 4, (3, 64, 63), 3, 24, 0, 3, False), (640, 1024, 8, 1, (200, 1), 5, 8, 72, 2, True)])
def test_decoded_tokens_equal_whole_prompts(d, ff, heads, kv_heads, prompts, steps, page, prefix, turns, sandwich, eight, dtype, u):
    worst = decoder_layer.run(d, ff, heads, kv_heads, prompts, steps, page, dtype, eight=eight, prefix=prefix, turns=turns, sandwich=sandwich)
    assert worst <= 4 * (12 * u + (2.0 ** -4 if eight else 0.0))
