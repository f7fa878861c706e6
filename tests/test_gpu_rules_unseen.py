"""Bits of a forward under rules do not depend on what lies where nobody looks: unwritten ends of caches, queries that see nothing."""
import pytest
import torch

import flash_attention_v100 as fa

pytestmark = pytest.mark.gpu
# what unwritten memory may hold: numbers far above the scores of the call, of both signs, and no numbers
FILLS = [0.0, 3.0, -60000.0, float("nan"), float("inf")]


def _normal(B, N, H, D, dtype, device, seed, std):
    return (torch.randn(B, N, H, D, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(device)


def _same_bits(call, changes):
    first = None
    with torch.no_grad():
        for change in changes:
            change()
            o, lse = call()
            first = first or (o, lse)
            assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


RULES = {"cap": (6.0, False), "slopes": (None, True), "both": (6.0, True)}


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("Nq,H,Hkv,D", [(1, 4, 2, 64), (7, 4, 2, 128), (20, 2, 2, 64), (33, 3, 1, 128), (300, 2, 1, 64), (700, 4, 4, 128), (300, 4, 2, 80)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
def test_unwritten_ends_of_caches(device, dtype, Nq, H, Hkv, D, rule):
    """Scores of a tenth of the cap, so that what is behind a cache would change how the cap's tanh is taken, or when a row's
    sums are scaled anew."""
    cap, slopes = RULES[rule]
    slopes = torch.linspace(0.01, 0.2, H, device=device) if slopes else None
    lengths = [Nq + 5, 1500, 128 * 7 + 3, 0, max(Nq - 4, 1)]
    B, Nk = len(lengths), 1500
    q, k, v = (_normal(B, n, h, D, dtype, device, s, x) for n, h, s, x in ((Nq, H, 0, 0.3), (Nk, Hkv, 1, 1.0), (Nk, Hkv, 2, 1.0)))
    counts = torch.tensor(lengths, dtype=torch.int32, device=device)
    for window in (None, 150):
        r = fa.build_key_ranges(Nq, Nk, batch=B, causal=True, window=window, key_lengths=counts, query_offsets=counts - Nq)

        def fill(x):
            for b, n in enumerate(lengths):
                k[b, n:], v[b, n:] = x, x

        _same_bits(lambda: fa.flash_attention_v100_with_rules(q, k, v, score_cap=cap, distance_slopes=slopes, key_ranges=r, return_softmax_lse=True),
                   [lambda x=x: fill(x) for x in FILLS])


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("N,D", [(12, 64), (40, 128), (300, 64), (1000, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_queries_that_see_nothing(device, dtype, N, D, rule):
    """Padding behind the last document, between the rows of a tile's others: its queries, keys and values may be anything."""
    cap, slopes = RULES[rule]
    slopes = torch.linspace(0.01, 0.2, 2, device=device) if slopes else None
    q, k, v = (_normal(2, N, 2, D, dtype, device, s, x) for s, x in ((0, 0.3), (1, 1.0), (2, 1.0)))
    ends = [N - 9, N // 2 - 3]
    r = fa.build_key_ranges(N, N, batch=2, causal=True, document_offsets=torch.tensor([[0, min(11, e), e] for e in ends], dtype=torch.int32, device=device))

    def fill(x):
        for b, e in enumerate(ends):
            q[b, e:], k[b, e:], v[b, e:] = x, x, x

    _same_bits(lambda: fa.flash_attention_v100_with_rules(q, k, v, score_cap=cap, distance_slopes=slopes, key_ranges=r, return_softmax_lse=True),
               [lambda x=x: fill(x) for x in FILLS])
