"""One new token, or a few, for many requests: more (request, K/V head) pairs than blocks, so that a block goes from one to the next."""
import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100.testing import TOLERANCE
from rules_helpers import attention64, rel, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Nq,H,Hkv,D", [(300, 1, 2, 2, 64), (300, 1, 4, 2, 64), (160, 4, 6, 2, 64), (260, 1, 2, 2, 128), (160, 2, 12, 2, 128)])
def test_blocks_that_go_from_request_to_request(device, B, Nq, H, Hkv, D):
    """Requests of one key, of one block and of many, next to one another, the scores' size another for each: every one against the
    formula, and the same bits fifty times.  A row weighed with its neighbour's maximum would be off by powers of two."""
    dtype, Nk = torch.float16, 1000
    lengths = [(1, 900, 5, 128, 130, 0, 1000, 17)[b % 8] for b in range(B)]
    starts = [max(n - Nq, 0) for n in lengths]
    g = torch.Generator().manual_seed(7)
    q = torch.randn(B, Nq, H, D, generator=g) * torch.tensor([0.1, 4.0, 1.0])[torch.arange(B) % 3].view(B, 1, 1, 1)
    k, v = torch.randn(B, Nk, Hkv, D, generator=g), torch.randn(B, Nk, Hkv, D, generator=g)
    q, k, v = (t.to(dtype).to(device) for t in (q, k, v))
    counts = torch.tensor(lengths, dtype=torch.int32, device=device)
    r = fa.build_key_ranges(Nq, Nk, batch=B, causal=True, key_lengths=counts, query_offsets=torch.tensor(starts, dtype=torch.int32, device=device))
    see = torch.stack([visible(Nq, Nk, b, causal=True, lengths=lengths, starts=starts) for b in range(B)])
    at = torch.arange(Nq) + torch.tensor(starts).view(B, 1)
    want = attention64(q, k, v, see, at, D ** -0.5, 30.0)
    with torch.no_grad():
        call = lambda: fa.flash_attention_v100_with_rules(q, k, v, score_cap=30.0, key_ranges=r, return_softmax_lse=True)
        o, lse = call()
        for b in range(B):
            some = see[b].any(dim=1).to(device)
            assert rel(o[b][some], want[0][b][some]) <= TOLERANCE[dtype] and (o[b][~some] == 0).all(), b
            # 30 tanh is off by 30 * 2^-22, a score of at most 20 and the sum's logarithm by 16 * 2^-24 of it
            assert ((lse[b] - want[1][b])[:, some].abs() <= 3e-5).all() and (lse[b][:, ~some] == float("-inf")).all(), b
        for _ in range(50):
            again = call()
            assert torch.equal(again[0], o) and torch.equal(again[1], lse)


@pytest.mark.parametrize("B,Nk,H,Hkv,D", [(6, 4096, 8, 8, 128), (4, 3000, 8, 2, 64), (3, 700, 4, 1, 80)])
@pytest.mark.parametrize("cap", [None, 30.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_outputs_are_rounded_once(device, dtype, B, Nk, H, Hkv, D, cap):
    """Nearly every output is the formula's, rounded.  Before that rounding it is off by what scores (30 * 2^-22 under the cap) and
    sums in 32 bits are: 1e-5 of it, a fiftieth of the least distance of two fp16 numbers, so that one in fifty may be the
    neighbour.  (Probabilities rounded to 16 bits would be off by 2^-12 each, which moves one in three.)"""
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(B, n, h, D, generator=g).to(dtype).to(device) for n, h in ((1, H), (Nk, Hkv), (Nk, Hkv)))
    lengths = [Nk - 31 * b for b in range(B)]
    counts = torch.tensor(lengths, dtype=torch.int32, device=device)
    r = fa.build_key_ranges(1, Nk, batch=B, causal=True, key_lengths=counts, query_offsets=counts - 1)
    see = torch.stack([visible(1, Nk, b, lengths=lengths) for b in range(B)])
    want = attention64(q, k, v, see, torch.zeros(B, 1), D ** -0.5, cap)[0].to(dtype)
    with torch.no_grad():
        o = fa.flash_attention_v100_with_rules(q, k, v, score_cap=cap, key_ranges=r)
    assert (o != want).float().mean().item() <= 0.05
