"""build_key_ranges against the definition, pair by pair."""
import pytest
import torch

import flash_attention_v100 as fa
from rules_helpers import visible

pytestmark = pytest.mark.gpu

CASES = {
    # Nq, Nk, batch, arguments on the host
    "plain": (5, 9, 2, {}),
    "one": (1, 1, 1, dict(causal=True)),
    "causal": (300, 300, 2, dict(causal=True)),
    "causal-short": (300, 40, 1, dict(causal=True)),
    "window": (257, 257, 1, dict(causal=True, window=100)),
    "window-both": (257, 300, 1, dict(window=100)),
    "window-one": (130, 130, 1, dict(causal=True, window=1)),
    "documents": (400, 400, 2, dict(causal=True, offsets=[[0, 0, 13, 13, 200, 390], [5, 5, 5, 5, 5, 5]])),
    "documents-shared": (400, 400, 2, dict(offsets=[0, 129, 256, 400])),
    "documents-window": (400, 400, 1, dict(causal=True, window=50, offsets=[[0, 129, 131, 400]])),
    "documents-beyond": (40, 40, 1, dict(offsets=[[30, 60, 90]])),
    "prefix": (300, 300, 2, dict(causal=True, offsets=[[0, 140, 300], [0, 10, 11]], prefixes=[[20, 1000], [0, 3]])),
    "prefix-shared": (300, 300, 2, dict(causal=True, offsets=[0, 140, 300], prefixes=[20, 200])),
    "prefix-alone": (200, 200, 2, dict(causal=True, prefixes=[150, 0])),
    "lengths": (130, 200, 3, dict(lengths=[0, 200, 77])),
    "cache": (1, 500, 4, dict(causal=True, lengths=[1, 500, 129, 128], starts=[0, 499, 128, 127])),
    "cache-window": (3, 500, 2, dict(causal=True, window=64, lengths=[3, 500], starts=[0, 497])),
    "start": (10, 50, 1, dict(causal=True, starts=40)),
    "before": (10, 50, 1, dict(causal=True, starts=-4)),
    "long": (5000, 5000, 1, dict(causal=True, offsets=[[0, 1, 3000, 4999, 5000]])),
}


def build(Nq, Nk, batch, host, device, index=torch.int32, **more):
    t = lambda x: None if x is None else torch.tensor(x, dtype=index, device=device)
    starts = host.get("starts", 0)
    return fa.build_key_ranges(Nq, Nk, batch=batch, causal=host.get("causal", False), window=host.get("window"),
                               document_offsets=t(host.get("offsets")), prefix_lengths=t(host.get("prefixes")), key_lengths=t(host.get("lengths")),
                               query_offsets=t(starts) if isinstance(starts, list) else starts, device=device, **more)


def check(r, Nq, Nk, batch, host):
    j = torch.arange(Nk)
    first, end = r.first.cpu(), r.end.cpu()
    for b in range(batch):
        got = (j >= first[b].unsqueeze(1)) & (j < end[b].unsqueeze(1))
        want = visible(Nq, Nk, b, **host)
        assert torch.equal(got, want), b
        none = ~want.any(dim=1)
        assert (first[b][none] == 0).all() and (end[b][none] == 0).all()
        # what the kernels skip by
        hull = r.plan.cpu()
        nq, nk = -(-Nq // 128), -(-Nk // 128)
        tiles = hull[r.batch * nq * 256:][:r.batch * nq * 4].view(r.batch, nq, 4)[b]
        parts = hull[r.batch * nq * 260:][:r.batch * nq * 16].view(r.batch, nq * 8, 2)[b]
        keys = hull[r.batch * nq * 276:][:r.batch * nk * 2].view(r.batch, nk, 2)[b]
        for rows, got_hull in [(128, tiles[:, :2]), (16, parts)]:
            for n in range(nq * 128 // rows):
                seen = want[n * rows:(n + 1) * rows].any(dim=0).nonzero()
                want_hull = [int(seen.min()), int(seen.max()) + 1] if len(seen) else [0, 0]
                assert got_hull[n].tolist() == want_hull, (b, rows, n)
        for n in range(nq):
            some = want[n * 128:(n + 1) * 128].any(dim=1)
            f, e = first[b][n * 128:(n + 1) * 128][some], end[b][n * 128:(n + 1) * 128][some]
            assert tiles[n, 2:].tolist() == ([int(f.max()), int(e.min())] if some.any() else [0, 2 ** 31 - 1])
        for n in range(nk):
            meets = ((tiles[:, 0] < n * 128 + 128) & (tiles[:, 1] > n * 128)).nonzero()
            assert keys[n].tolist() == ([int(meets.min()), int(meets.max()) + 1] if len(meets) else [0, 0]), (b, n)
        # the orders: every tile once, those that meet most first
        at = r.batch * (nq * 276 + nk * 2)
        for count, cost in ((nq, lambda t: -(-int(tiles[t, 1]) // 128) - int(tiles[t, 0]) // 128),
                            ((nq + 1) // 2, lambda p: _pair_cost(tiles[2 * p:2 * p + 2])), (nk, lambda n: int(keys[n, 1] - keys[n, 0]))):
            order = hull[at + b * count:at + (b + 1) * count].tolist()
            at += r.batch * count
            assert sorted(order) == list(range(count))
            costs = [cost(i) for i in order]
            if nq > 1 and max(nq, nk) <= 512:
                assert costs == sorted(costs, reverse=True), (b, costs)


def _pair_cost(tiles):
    some = tiles[tiles[:, 1] > 0]
    return -(-int(some[:, 1].max()) // 128) - int(some[:, 0].min()) // 128 if len(some) else 0


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["int32", "int64"])
@pytest.mark.parametrize("case", CASES)
def test_ranges_are_the_definitions(device, case, index):
    Nq, Nk, batch, host = CASES[case]
    check(build(Nq, Nk, batch, host, device, index), Nq, Nk, batch, host)


def test_positions_count_from_the_document(device):
    r = build(12, 12, 2, dict(offsets=[[0, 0, 5, 9], [2, 4, 10, 12]]), device)
    assert r.positions.tolist() == [[0, 1, 2, 3, 4, 0, 1, 2, 3, 0, 0, 0], [0, 0, 0, 1, 0, 1, 2, 3, 4, 5, 0, 1]]
    r = build(3, 50, 2, dict(causal=True, starts=[7, 20]), device)
    assert r.positions.tolist() == [[7, 8, 9], [20, 21, 22]]


def test_rows_given_by_hand_are_clipped(device):
    rows = torch.tensor([[[0, 3], [-5, 2], [4, 99], [7, 7], [9, 2], [20, 30]]], dtype=torch.int32, device=device)
    r = fa.build_key_ranges(6, 10, rows=rows)
    assert r.first.tolist() == [[0, 0, 4, 0, 0, 0]] and r.end.tolist() == [[3, 2, 10, 0, 0, 0]]
    r = fa.build_key_ranges(6, 10, rows=rows.flip(2).flip(2).transpose(1, 2).contiguous().transpose(1, 2).long(), query_offsets=3)
    assert r.end.tolist() == [[3, 2, 10, 0, 0, 0]] and r.positions.tolist() == [[3, 4, 5, 6, 7, 8]]


def test_extreme_lengths_saturate(device):
    top = 2 ** 31 - 1
    r = build(3, 50, 1, dict(causal=True, lengths=[top], starts=[top]), device)
    assert r.end.tolist() == [[50, 50, 50]] and r.first.tolist() == [[0, 0, 0]]
    r = build(3, 50, 1, dict(causal=True, lengths=[-top], starts=[-top]), device)
    assert r.end.tolist() == [[0, 0, 0]]
    r = fa.build_key_ranges(3, 50, causal=True, window=top, device=device)
    assert r.first.tolist() == [[0, 0, 0]] and r.end.tolist() == [[1, 2, 3]]


@pytest.mark.parametrize("sizes", [(0, 0, 0), (2, 0, 5), (0, 4, 4), (1, 4, 0)])
def test_nothing_to_build(device, sizes):
    B, Nq, Nk = sizes
    r = fa.build_key_ranges(Nq, Nk, batch=B, causal=True, device=device)
    assert r.first.shape == (B, Nq) and (r.end <= Nk).all()


def test_built_anew_in_a_graph(device):
    """A captured build reads the lengths as they are at each replay."""
    lengths = torch.tensor([5, 300], dtype=torch.int32, device=device)
    r = fa.build_key_ranges(1, 400, batch=2, key_lengths=lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert fa.build_key_ranges(1, 400, batch=2, key_lengths=lengths, out=r) is r
    for new in ([1, 400], [0, 129]):
        lengths.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        check(r, 1, 400, 2, dict(lengths=new))
    with pytest.raises(ValueError, match="out is for"):
        fa.build_key_ranges(1, 401, batch=2, key_lengths=lengths, out=r)


def test_on_another_stream(device):
    lengths = torch.tensor([77], dtype=torch.int32, device=device)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        r = fa.build_key_ranges(200, 200, causal=True, key_lengths=lengths)
    side.synchronize()
    check(r, 200, 200, 1, dict(causal=True, lengths=[77]))


def test_lengths_beyond_32_bits_mean_all(device):
    r = fa.build_key_ranges(3, 50, key_lengths=torch.tensor([2 ** 40], device=device))
    assert r.end.tolist() == [[50, 50, 50]]
    r = fa.build_key_ranges(2, 50, rows=torch.tensor([[[3, 2 ** 33], [-2 ** 33, 7]]], device=device))
    assert r.first.tolist() == [[3, 0]] and r.end.tolist() == [[50, 7]]


def test_more_tiles_than_are_put_in_order(device):
    """Beyond 512 tiles the lists come from another launch and the orders are the tiles' own."""
    N, w = 66000, 700
    r = fa.build_key_ranges(N, N, causal=True, window=w, device=device)
    t = torch.arange(N)
    assert torch.equal(r.first[0].cpu(), (t - w + 1).clamp(min=0).int()) and torch.equal(r.end[0].cpu(), (t + 1).int())
    n = -(-N // 128)
    plan = r.plan.cpu()
    keys = plan[n * 276:][:2 * n].view(n, 2)
    first = torch.arange(n)
    last = ((first * 128 + 127 + w - 1).clamp(max=N - 1)) // 128
    assert torch.equal(keys, torch.stack([first, last + 1], dim=1).int())
    at = n * 278
    assert sorted(plan[at:at + n].tolist()) == list(range(n)) and sorted(plan[at + n:at + n + (n + 1) // 2].tolist()) == list(range((n + 1) // 2))
    assert sorted(plan[at + n + (n + 1) // 2:at + 2 * n + (n + 1) // 2].tolist()) == list(range(n))
