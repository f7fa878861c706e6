"""build_key_ranges: numbers of any kind mean the same in the native form, in the general one and when a plan is built anew."""
import numpy as np
import pytest
import torch

import flash_attention_v100 as fa


@pytest.mark.parametrize("bad,error", [(3.0, TypeError), ("3", TypeError), ([3], TypeError), (2 ** 31, ValueError), (2 ** 32 + 5, ValueError),
                                       (-2 ** 31 - 5, ValueError), (np.float32(2), TypeError), (np.int64(2 ** 40), ValueError)])
def test_offsets_that_are_no_whole_numbers_of_32_bits(bad, error):
    for more in ({}, dict(rows=torch.zeros(1, 4, 2, dtype=torch.int32))):
        with pytest.raises(error, match="query_offsets"):
            fa.build_key_ranges(4, 8, query_offsets=bad, device="cuda:0", **more)


@pytest.mark.parametrize("sizes", [dict(seq_q=2 ** 32 + 8, seq_k=4), dict(seq_q=8, seq_k=2 ** 31), dict(seq_q=1, seq_k=1, batch=2 ** 32 + 1)])
def test_sizes_beyond_32_bits(sizes):
    with pytest.raises(ValueError, match="below 2"):
        fa.build_key_ranges(**sizes, device="cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [5, np.int64(5), np.int32(5), np.array(5), np.uint8(5)], ids=lambda o: type(o).__name__)
def test_offsets_of_any_integer_type(device, offset):
    lengths = torch.tensor([7], device=device)                       # (64 bits: the general form)
    first = fa.build_key_ranges(3, 50, causal=True, query_offsets=offset, device=device)
    general = fa.build_key_ranges(3, 50, causal=True, key_lengths=lengths, query_offsets=offset)
    anew = fa.build_key_ranges(3, 50, causal=True, query_offsets=2, device=device)
    fa.build_key_ranges(3, 50, causal=True, query_offsets=offset, out=anew)
    by_hand = fa.build_key_ranges(3, 50, rows=torch.tensor([[[0, 6], [0, 7], [0, 8]]], device=device), query_offsets=offset)
    for r, ends in ((first, [6, 7, 8]), (general, [6, 7, 7]), (anew, [6, 7, 8]), (by_hand, [6, 7, 8])):
        assert r.end.tolist() == [ends] and r.positions.tolist() == [[5, 6, 7]]
