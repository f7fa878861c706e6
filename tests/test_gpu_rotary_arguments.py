"""rotary_embedding: first positions that are numbers."""
import numpy as np
import pytest
import torch

import flash_attention_v100 as fa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [1.5, 2 ** 63, -2 ** 63 - 1, 2 ** 64 + 5, float("0.25"), "5"])
@pytest.mark.parametrize("inplace", [False, True])
def test_no_whole_number_of_64_bits(device, bad, inplace):
    x, f = torch.randn(1, 4, 2, 8, device=device), fa.rotary_frequencies(8, device=device)[0]
    with pytest.raises(ValueError, match="whole number"):
        fa.rotary_embedding(x, inv_freq=f, positions=bad, inplace=inplace)


@pytest.mark.parametrize("first", [7, np.int64(7), np.int32(7), np.array(7), 7.0], ids=lambda x: type(x).__name__)
def test_whole_numbers_of_any_type(device, first):
    x, f = torch.randn(1, 4, 2, 8, device=device), fa.rotary_frequencies(8, device=device)[0]
    want = fa.rotary_embedding(x, inv_freq=f, positions=torch.arange(7, 11, device=device))
    assert torch.equal(fa.rotary_embedding(x, inv_freq=f, positions=first), want)
    assert torch.equal(fa.rotary_embedding(x.clone(), inv_freq=f, positions=first, inplace=True), want)
