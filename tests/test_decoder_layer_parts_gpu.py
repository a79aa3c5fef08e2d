"""decoder_layer.py with prompts in more parts than they have tokens: parts without rows pass through every operator. Tolerance as for prompts of fewer
parts: a dozen roundings of terms of the outputs' size, which reach four times their root mean square."""
import pytest
import torch

import decoder_layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,u", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("prefix,sandwich", [(0, False), (32, True)])
def test_parts_without_rows(prefix, sandwich, dtype, u):
    assert decoder_layer.run(512, 1032, 4, 2, (3, 1), 2, 16, dtype, prefix=prefix, turns=7, sandwich=sandwich) <= 48 * u
