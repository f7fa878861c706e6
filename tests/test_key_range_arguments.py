"""build_key_ranges: numbers of any kind mean the same in the native form, in the general one and when a plan is built anew."""
import numpy as np
import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100.ops.rules import check_rules
from test_gpu_key_ranges import build, check


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


def _by_hand(device, entries, dtype=torch.int32):
    return fa.KeyRanges(torch.zeros(entries, dtype=dtype, device=device), torch.zeros(2, 300, dtype=torch.int32, device=device), 2, 300, 300)


def test_a_plan_made_by_hand_is_measured():
    q = torch.zeros(2, 300, 1, 8)
    need = 2 * 384 * 2 + 2 * 3 * 4 + 2 * 24 * 2 + 2 * 3 * 2 + 2 * (3 + 2 + 3) + 4
    check_rules(q, q, None, None, _by_hand("cpu", need))
    for bad in (_by_hand("cpu", need - 1), _by_hand("cpu", 0), _by_hand("cpu", need, torch.int64)):
        with pytest.raises(ValueError, match="come from build_key_ranges"):
            check_rules(q, q, None, None, bad)


@pytest.mark.gpu
def test_a_plan_made_by_hand_is_refused(device):
    """Both ways to use it: an attention call, in the native form first, and a build that would write it."""
    q = torch.zeros(2, 300, 1, 64, device=device).half()
    bad = _by_hand(device, 100)
    with pytest.raises(ValueError, match="come from build_key_ranges"):
        fa.flash_attention_v100_with_rules(q, q, q, key_ranges=bad)
    with pytest.raises(ValueError, match="come from build_key_ranges"):
        fa.build_key_ranges(300, 300, batch=2, device=device, out=bad)
    good = fa.build_key_ranges(300, 300, batch=2, device=device)
    good.positions = good.positions[:1]
    with pytest.raises(ValueError, match="positions"):
        fa.build_key_ranges(300, 300, batch=2, device=device, out=good)


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


@pytest.mark.gpu
@pytest.mark.parametrize("mask", [dict(causal=True), dict(), dict(window=4), dict(window=40), dict(causal=True, window=4), dict(causal=True, prefixes=[3, 0, 50])], ids=str)
def test_more_queries_than_a_cache_has_keys(device, mask):
    """Rows before the first key: by the mask's rule as any other row, with positions below 0."""
    lengths, Nq, Nk = [2, 20, 0], 20, 60
    host = dict(mask, lengths=lengths, starts=[n - Nq for n in lengths])
    r = build(Nq, Nk, 3, host, device)
    check(r, Nq, Nk, 3, host)
    assert r.positions.tolist() == [[n - Nq + i for i in range(Nq)] for n in lengths]
