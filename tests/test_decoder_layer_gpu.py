"""The decoder layer of decoder_layer.py: tokens decoded one by one through the paged cache against the same tokens inside
whole prompts. Both sides round at the same places: weights of the prompt's softmax (u = 2^-8 in bf16, 2^-11 in fp16, relative to sums of at most
the values' size), the attention output, both projections' inputs and the layer's two sums, each u of terms of the
outputs' size, a dozen roundings of either side that may all differ; outputs reach four times their root mean square."""
import pytest
import torch

import decoder_layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,u", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("d,ff,heads,kv_heads,prompts,steps,page", [
    (1024, 2816, 16, 4, (37, 5, 130), 9, 16), (512, 1032, 4, 4, (1, 64, 63), 3, 24), (640, 1024, 8, 1, (200,), 5, 8)])
def test_decoded_tokens_equal_whole_prompts(d, ff, heads, kv_heads, prompts, steps, page, dtype, u):
    assert decoder_layer.run(d, ff, heads, kv_heads, prompts, steps, page, dtype) <= 4 * 12 * u
