"""Arguments of attention under rules at the ends of their ranges."""
import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100.ops.rules import check_rules


@pytest.mark.parametrize("cap", [1e-46, 1e-60, 5e-324, 0.0, -1.0, float("nan"), float("inf"), 1e30])
def test_caps_that_32_bits_do_not_hold(cap):
    q = torch.zeros(1, 4, 1, 8)
    with pytest.raises(ValueError, match="positive and finite"):
        check_rules(q, q, cap, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-46, 5e-324])
def test_a_cap_too_small_is_no_missing_cap(device, cap):
    q = torch.randn(1, 8, 1, 64, device=device).half()
    for more in ({}, dict(key_ranges=fa.build_key_ranges(8, 8, device=device))):
        with pytest.raises(ValueError, match="positive and finite"):
            fa.flash_attention_v100_with_rules(q, q, q, score_cap=cap, **more)
