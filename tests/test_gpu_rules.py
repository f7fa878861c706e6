"""flash_attention_v100_with_rules against its definition in 64 bits: outputs, log-sum-exps and every gradient, at the tolerances
of the package's other attention calls (relative L2 2e-3 for fp16 and bf16, 1e-5 for fp32)."""
import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100.testing import TOLERANCE
from rules_helpers import attention64, rel, rotary64, visible

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(B, Nq, Nk, H, Hkv, D, dtype, device, std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, d = (torch.randn(B, n, h, D, generator=g) for n, h in ((Nq, H), (Nk, Hkv), (Nk, Hkv), (Nq, H)))
    return [(t * s).to(dtype).to(device) for t, s in ((q, std), (k, 1.0), (v, 1.0), (d, 1.0))]


def _ranges(Nq, Nk, B, host, device):
    t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=device)
    starts = host.get("starts", 0)
    r = fa.build_key_ranges(Nq, Nk, batch=B, causal=host.get("causal", False), window=host.get("window"), document_offsets=t(host.get("offsets")),
                            prefix_lengths=t(host.get("prefixes")), key_lengths=t(host.get("lengths")),
                            query_offsets=t(starts) if isinstance(starts, list) else starts, device=device)
    see = torch.stack([visible(Nq, Nk, b, **host) for b in range(B)])
    at = torch.stack([torch.arange(Nq) + (starts[b] if isinstance(starts, list) else starts) for b in range(B)])
    return r, see, at


def _slopes(H, device):
    return (2.0 ** (-8.0 * torch.arange(1, H + 1) / H)).to(device)


def _check(got, want, dtype, names):
    for n, a, w in zip(names, got, want):
        assert torch.equal(torch.isfinite(a).cpu(), torch.isfinite(w).cpu()), n
        fine = torch.isfinite(w)
        assert rel(a[fine], w[fine]) <= TOLERANCE[dtype], (n, rel(a[fine], w[fine]))


def _step(q, k, v, g, **rules):
    for t in (q, k, v):
        t.requires_grad_(True)
    o, lse = fa.flash_attention_v100_with_rules(q, k, v, return_softmax_lse=True, **rules)
    grads = torch.autograd.grad(o, (q, k, v), g)
    return (o.detach(), lse.detach()) + grads


MASKS = {
    "none": (200, 300, 2, {}),
    "causal": (333, 333, 1, dict(causal=True)),
    "one": (1, 1, 2, dict(causal=True)),
    "documents": (400, 400, 2, dict(causal=True, offsets=[[0, 1, 130, 131, 390], [7, 7, 7, 300, 400]])),
    "documents-full": (300, 300, 1, dict(offsets=[[0, 100, 250]])),
    "prefix": (300, 300, 2, dict(causal=True, offsets=[[0, 140, 300], [0, 10, 200]], prefixes=[[20, 1000], [0, 190]])),
    "window": (400, 400, 1, dict(causal=True, window=77)),
    "window-both": (270, 270, 1, dict(window=33)),
    "lengths": (130, 200, 3, dict(lengths=[0, 200, 77])),
    "cache": (5, 700, 3, dict(causal=True, lengths=[5, 700, 260], starts=[0, 695, 255])),
    "far-window": (3, 900, 2, dict(causal=True, window=100, lengths=[900, 850], starts=[897, 847])),
}


@pytest.mark.parametrize("rule", ["ranges", "cap", "slopes", "both"])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("dtype,H,Hkv,D", [("bf16", 4, 2, 64), ("bf16", 2, 2, 128), ("fp16", 4, 1, 64), ("fp16", 3, 3, 80), ("fp32", 2, 1, 64), ("bf16", 2, 1, 33)])
def test_step(device, dtype, H, Hkv, D, mask, rule):
    Nq, Nk, B, host = MASKS[mask]
    t = TYPES[dtype]
    q, k, v, g = _inputs(B, Nq, Nk, H, Hkv, D, t, device, std=2.0)
    ranges, see, at = _ranges(Nq, Nk, B, host, device)
    cap = 5.0 if rule in ("cap", "both") else None
    slopes = _slopes(H, device) if rule in ("slopes", "both") else None
    want = attention64(q, k, v, see, at, D ** -0.5, cap, slopes, grad=g)
    got = _step(q, k, v, g, score_cap=cap, distance_slopes=slopes, key_ranges=ranges)
    _check(got, want, t, ("o", "lse", "dq", "dk", "dv"))
    with torch.no_grad():
        o, lse = fa.flash_attention_v100_with_rules(q, k, v, score_cap=cap, distance_slopes=slopes, key_ranges=ranges, return_softmax_lse=True)
    _check((o, lse), want, t, ("o", "lse"))
    # rows and keys that see nothing or that nobody sees: zeros, not small numbers
    rows, keys = ~see.any(dim=2), ~see.any(dim=1)
    assert (got[0].cpu()[rows] == 0).all() and (got[2].cpu()[rows] == 0).all()
    assert (got[3].cpu()[keys] == 0).all() and (got[4].cpu()[keys] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.01, 1.0, 30.0, 1e4])
@pytest.mark.parametrize("std", [0.01, 3.0, 40.0])
def test_caps_and_scores_of_any_size(device, dtype, cap, std):
    """Scores from thousandths of a cap to hundreds of it.  Scores of a spread s give outputs whose distance from the formula
    grows with s times the score's rounding (2^-24 of a sum of D products whose terms are below 4 s): at most 1e-6 (1 + s)."""
    t = TYPES[dtype]
    q, k, v, g = _inputs(1, 200, 200, 2, 2, 64, t, device, std=std)
    ranges, see, at = _ranges(200, 200, 1, dict(causal=True), device)
    want = attention64(q, k, v, see, at, 0.125, cap, None, grad=g)
    got = _step(q, k, v, g, scale=0.125, score_cap=cap, key_ranges=ranges)
    for n, a, w in zip(("o", "lse", "dv"), (got[0], got[1], got[4]), (want[0], want[1], want[4])):
        assert rel(a, w) <= TOLERANCE[t] + 1e-6 * (1 + std), (n, rel(a, w))
    # dQ and dK: in a saturated score (1 - tanh^2) is the difference of 1 and a number rounded to 2^-24; what is left has that
    # absolute error, so gradients far below the scale |dO| |V| |K| are compared on that scale
    for n, a, w, x in (("dq", got[2], want[2], k), ("dk", got[3], want[3], q)):
        scale = 0.125 * 64 * x.double().abs().max().item()
        assert (a.double() - w).norm() <= (TOLERANCE[t] + 1e-6 * (1 + std)) * w.norm() + 2.0 ** -20 * scale * w.numel() ** 0.5, n


@pytest.mark.parametrize("dtype,H,Hkv,D", [("fp32", 2, 2, 128), ("fp32", 4, 2, 32), ("fp32", 2, 1, 20), ("fp32", 2, 2, 96), ("fp32", 3, 3, 33), ("fp32", 2, 2, 1),
                                           ("fp16", 2, 1, 100), ("bf16", 2, 2, 9)])
@pytest.mark.parametrize("layout", ["plain", "heads-first", "odd-addresses"])
def test_cuda_core_tiles(device, dtype, H, Hkv, D, layout):
    """Every width of tile, rows that can and cannot be copied 16 bytes at a time, K/V heads that several query heads read."""
    t = TYPES[dtype]
    host = dict(causal=True, offsets=[[0, 33, 190, 300]], prefixes=[[0, 40, 200]])
    q, k, v, g = _inputs(1, 310, 310, H, Hkv, D, t, device)
    if layout == "heads-first":
        q, k, v, g = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, g))
    if layout == "odd-addresses":
        q, k, v, g = (torch.cat([x[..., :1], x], dim=3)[..., 1:] for x in (q, k, v, g))
    ranges, see, at = _ranges(310, 310, 1, host, device)
    want = attention64(q, k, v, see, at, D ** -0.5, 4.0, _slopes(H, device), grad=g)
    got = _step(q, k, v, g, score_cap=4.0, distance_slopes=_slopes(H, device), key_ranges=ranges)
    _check(got, want, t, ("o", "lse", "dq", "dk", "dv"))


@pytest.mark.parametrize("H,Hkv,D", [(2, 1, 64), (2, 2, 128)])
def test_cuda_core_tiles_of_long_rows(device, H, Hkv, D):
    """More tiles of queries than a warp looks through at once, most of which a key tile's window leaves out."""
    N = 4500
    for host in (dict(causal=True, window=150), dict(causal=True, offsets=[[0, 100, 2300, 4490]])):
        q, k, v, g = _inputs(1, N, N, H, Hkv, D, torch.float32, device)
        ranges, see, at = _ranges(N, N, 1, host, device)
        want = attention64(q, k, v, see, at, D ** -0.5, None, None, grad=g)
        _check(_step(q, k, v, g, key_ranges=ranges), want, torch.float32, ("o", "lse", "dq", "dk", "dv"))


def test_cuda_core_tiles_rows_of_any_order(device):
    """Rows that see the first keys or the last ones, in turn: a key tile's list of query tiles has holes."""
    rows = torch.zeros(1, 700, 2, dtype=torch.int32)
    i = torch.arange(700)
    rows[0, :, 0] = torch.where(i // 64 % 3 == 0, 5, 600)
    rows[0, :, 1] = torch.where(i // 64 % 3 == 0, 90, 641)
    rows[0, i // 64 % 3 == 2] = 0
    r = fa.build_key_ranges(700, 650, batch=1, rows=rows.to(device))
    j = torch.arange(650)
    see = (j >= rows[..., :1]) & (j < rows[..., 1:])
    q, k, v, g = _inputs(1, 700, 650, 2, 1, 64, torch.float32, device)
    want = attention64(q, k, v, see, torch.arange(700).expand(1, 700), 0.125, 5.0, None, grad=g)
    _check(_step(q, k, v, g, score_cap=5.0, key_ranges=r), want, torch.float32, ("o", "lse", "dq", "dk", "dv"))


@pytest.mark.parametrize("dtype,Nq", [("bf16", 1), ("bf16", 40), ("fp32", 40)])
def test_caches_beyond_32_bits(device, dtype, Nq):
    """More than 2^31 elements of K and V, positions beyond 2^24: the last keys alone give the same."""
    N, n, t = 17_000_000, 2000, TYPES[dtype]
    k, v = (torch.zeros(1, N, 1, 128, device=device, dtype=t) for _ in range(2))
    q, ks, vs, g = _inputs(1, Nq, n, 2, 1, 128, t, device)
    k[:, -n:], v[:, -n:] = ks, vs
    host = dict(causal=True, window=700, starts=n - Nq)
    see, at = visible(Nq, n, 0, **host).unsqueeze(0), (torch.arange(Nq) + n - Nq).unsqueeze(0)
    slopes = _slopes(2, device)
    want = attention64(q, ks, vs, see, at, 0.1, 20.0, slopes, grad=g)
    r = fa.build_key_ranges(Nq, N, causal=True, window=700, query_offsets=N - Nq, device=device)
    with torch.no_grad():
        o, lse = fa.flash_attention_v100_with_rules(q, k, v, scale=0.1, score_cap=20.0, distance_slopes=slopes, key_ranges=r, return_softmax_lse=True)
    _check((o, lse), want, t, ("o", "lse"))
    o, lse, dq, dk, dv = _step(q, k, v, g, scale=0.1, score_cap=20.0, distance_slopes=slopes, key_ranges=r)
    _check((o, lse, dq, dk[:, -n:], dv[:, -n:]), want, t, ("o", "lse", "dq", "dk", "dv"))
    assert not dk[:, :-n].any() and not dv[:, :-n].any()


@pytest.mark.parametrize("dtype,B,Nq,Nk,H,Hkv,D", [("bf16", 1, 17, 16000, 2, 2, 128), ("fp16", 1, 300, 9000, 2, 2, 64), ("bf16", 2, 40, 6000, 4, 2, 80), ("fp16", 3, 33, 5000, 3, 1, 128)])
@pytest.mark.parametrize("window", [None, 3100])
def test_few_queries_on_long_caches(device, dtype, B, Nq, Nk, H, Hkv, D, window):
    """Rows whose keys are cut into many ranges, parts of which, or all, hold nothing for a request with few keys."""
    t = TYPES[dtype]
    lengths = [Nk, 200, 0][:B]
    host = dict(causal=True, window=window, lengths=lengths, starts=[max(n - Nq, 0) for n in lengths])
    q, k, v, _ = _inputs(B, Nq, Nk, H, Hkv, D, t, device)
    ranges, see, at = _ranges(Nq, Nk, B, host, device)
    for cap, slopes in ((None, None), (6.0, _slopes(H, device))):
        want = attention64(q, k, v, see, at, D ** -0.5, cap, slopes)
        with torch.no_grad():
            got = fa.flash_attention_v100_with_rules(q, k, v, score_cap=cap, distance_slopes=slopes, key_ranges=ranges, return_softmax_lse=True)
            again = fa.flash_attention_v100_with_rules(q, k, v, score_cap=cap, distance_slopes=slopes, key_ranges=ranges)
        _check(got, want, t, ("o", "lse"))
        assert torch.equal(got[0], again)
        assert (got[0].cpu()[~see.any(dim=2)] == 0).all()


@pytest.mark.parametrize("H,Hkv", [(3, 1), (10, 2), (7, 1), (100, 1)])
def test_forward_bits_do_not_depend_on_what_memory_held(device, H, Hkv):
    """Groups of heads that do not divide a tile: the same bits after other kernels have used shared memory."""
    q, k, v, _ = _inputs(1, 33, 3000, H, Hkv, 128, torch.float16, device)
    r = fa.build_key_ranges(33, 3000, causal=True, query_offsets=2967, device=device)
    other = [t * 50 for t in _inputs(1, 300, 900, 8, 8, 128, torch.float16, device)[:3]]
    first = None
    with torch.no_grad():
        for _ in range(40):
            o = fa.flash_attention_v100_with_rules(q, k, v, score_cap=6.0, distance_slopes=_slopes(H, device), key_ranges=r, return_softmax_lse=True)
            first = first or o
            assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
            fa.flash_attention_v100(*other)


def test_without_ranges_the_calls_own_masks(device):
    """causal, key_lengths and the alignment build the ranges of the call; without any rule the result is the plain call's."""
    q, k, v, g = _inputs(2, 100, 260, 4, 2, 64, torch.bfloat16, device)
    for mask, host in [(dict(), {}), (dict(causal=True), dict(causal=True)), (dict(causal=True, causal_alignment="bottom_right"), dict(causal=True, starts=160)),
                       (dict(key_lengths=torch.tensor([260, 31], device=device)), dict(lengths=[260, 31])),
                       (dict(causal=True, key_lengths=torch.tensor([90, 31], device=device)), dict(causal=True, lengths=[90, 31]))]:
        see = torch.stack([visible(100, 260, b, **host) for b in range(2)])
        at = (torch.arange(100) + host.get("starts", 0)).expand(2, 100)
        slopes = _slopes(4, device)
        want = attention64(q, k, v, see, at, 0.125, 9.0, slopes, grad=g)
        _check(_step(q, k, v, g, score_cap=9.0, distance_slopes=slopes, **mask), want, torch.bfloat16, ("o", "lse", "dq", "dk", "dv"))
        plain = fa.flash_attention_v100(q, k, v, return_softmax_lse=True, **mask)
        ruled = fa.flash_attention_v100_with_rules(q, k, v, return_softmax_lse=True, **mask)
        assert rel(ruled[0], plain[0]) <= 2 * TOLERANCE[torch.bfloat16] and rel(ruled[1], plain[1]) <= 1e-5


def test_one_plan_for_any_batch(device):
    q, k, v, g = _inputs(3, 150, 150, 2, 2, 64, torch.float16, device)
    host = dict(causal=True, offsets=[0, 60, 150])
    r = fa.build_key_ranges(150, 150, causal=True, document_offsets=torch.tensor([0, 60, 150], dtype=torch.int32, device=device))
    see = torch.stack([visible(150, 150, b, **host) for b in range(3)])
    want = attention64(q, k, v, see, torch.arange(150).expand(3, 150), 0.125, None, _slopes(2, device), grad=g)
    _check(_step(q, k, v, g, distance_slopes=_slopes(2, device), key_ranges=r), want, torch.float16, ("o", "lse", "dq", "dk", "dv"))


def test_rows_of_any_order(device):
    """Ranges given by hand: neither sorted nor overlapping, whole tiles that see nothing among them."""
    g0 = torch.Generator().manual_seed(5)
    first = torch.randint(0, 500, (2, 600), generator=g0)
    rows = torch.stack([first, first + torch.randint(0, 120, (2, 600), generator=g0)], dim=2)
    rows[0, 128:256] = 0
    rows[1, :, 1] = rows[1, :, 1].clamp(max=300)
    rows[1, 400:] = torch.tensor([250, 251])
    r = fa.build_key_ranges(600, 512, batch=2, rows=rows.to(torch.int32).to(device))
    j = torch.arange(512)
    see = (j >= rows[..., :1]) & (j < rows[..., 1:])
    for dtype, D in ((torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)):
        q, k, v, g = _inputs(2, 600, 512, 2, 1, D, dtype, device)
        want = attention64(q, k, v, see, torch.arange(600).expand(2, 600), D ** -0.5, 8.0, None, grad=g)
        _check(_step(q, k, v, g, score_cap=8.0, key_ranges=r), want, dtype, ("o", "lse", "dq", "dk", "dv"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Nq,H,Hkv,D", [(1, 8, 8, 64), (1, 32, 4, 128), (1, 6, 2, 80), (4, 8, 2, 128), (130, 4, 1, 64), (300, 2, 2, 128)])
def test_caches_of_ragged_lengths(device, dtype, Nq, H, Hkv, D):
    """New tokens at the end of caches, what lies behind each cache unwritten memory."""
    t = TYPES[dtype]
    lengths = [Nq, 1500, 128 + Nq, 777, 1024]
    B, Nk = len(lengths), 1500
    q, k, v, _ = _inputs(B, Nq, Nk, H, Hkv, D, t, device, std=2.0)
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        k2[b, n:], v2[b, n:] = float("nan"), float("inf")
    starts = [n - Nq for n in lengths]
    for window in (None, 200):
        ranges, see, at = _ranges(Nq, Nk, B, dict(causal=True, window=window, lengths=lengths, starts=starts), device)
        slopes = _slopes(H, device)
        want = attention64(q, k, v, see, at, D ** -0.5, 20.0, slopes)
        with torch.no_grad():
            got = fa.flash_attention_v100_with_rules(q, k2, v2, score_cap=20.0, distance_slopes=slopes, key_ranges=ranges, return_softmax_lse=True)
        _check(got, want, t, ("o", "lse"))


def test_bit_reproducible_and_on_another_stream(device):
    q, k, v, g = _inputs(2, 500, 500, 4, 2, 128, torch.bfloat16, device)
    ranges, _, _ = _ranges(500, 500, 2, dict(causal=True, offsets=[[0, 200, 500], [0, 1, 480]]), device)
    rules = dict(score_cap=10.0, distance_slopes=_slopes(4, device), key_ranges=ranges)
    a = _step(q, k, v, g, **rules)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        b = _step(q, k, v, g, **rules)
    side.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_views(device):
    """Slices of a fused projection, unaligned rows, a head dimension that is not contiguous, an expanded gradient."""
    ranges, see, at = _ranges(200, 200, 2, dict(causal=True, offsets=[[0, 90, 200], [0, 10, 150]]), device)
    qkv = torch.randn(2, 200, 8, 64, device=device).bfloat16()
    g = torch.randn(2, 200, 4, 64, device=device).bfloat16()
    views = {
        "fused": (qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]),
        "odd": tuple(torch.randn(2, 200, h, 65, device=device).bfloat16()[..., 1:] for h in (4, 2, 2)),
        "permuted": tuple(torch.randn(2, 64, h, 200, device=device).bfloat16().permute(0, 3, 2, 1) for h in (4, 2, 2)),
    }
    for name, (q, k, v) in views.items():
        q, k, v = (x.detach() for x in (q, k, v))
        want = attention64(q, k, v, see, at, 0.125, 7.0, None, grad=g)
        _check(_step(q, k, v, g, score_cap=7.0, key_ranges=ranges), want, torch.bfloat16, ("o", "lse", "dq", "dk", "dv"))
    q = views["fused"][0].detach().requires_grad_(True)
    o = fa.flash_attention_v100_with_rules(q, k, v, score_cap=7.0, key_ranges=ranges)
    d, = torch.autograd.grad(o.float().sum(), q)
    one = torch.ones_like(g)
    want = attention64(q.detach(), k, v, see, at, 0.125, 7.0, None, grad=one)
    assert rel(d, want[2]) <= TOLERANCE[torch.bfloat16] * 2       # (dO = 1: dP - delta cancels to a tenth of its terms)


def test_no_keys_and_no_queries(device):
    x = lambda n: torch.randn(2, n, 2, 64, device=device).half().requires_grad_(True)
    q, k, v = x(5), x(0), x(0)
    o, lse = fa.flash_attention_v100_with_rules(q, k, v, score_cap=3.0, return_softmax_lse=True)
    assert (o == 0).all() and (lse == float("-inf")).all()
    o.sum().backward()
    assert (q.grad == 0).all() and k.grad.shape == k.shape
    q, k, v = x(0), x(5), x(5)
    o = fa.flash_attention_v100_with_rules(q, k, v, causal=True, score_cap=3.0)
    o.sum().backward()
    assert o.shape == (2, 0, 2, 64) and (k.grad == 0).all() and (v.grad == 0).all()


def test_refusals(device):
    q = torch.zeros(2, 8, 4, 64, device=device).half()
    r = fa.build_key_ranges(8, 8, causal=True, device=device)
    call = fa.flash_attention_v100_with_rules
    for match, f in [
        ("positive", lambda: call(q, q, q, score_cap=0.0)), ("positive", lambda: call(q, q, q, score_cap=float("inf"))),
        ("shape", lambda: call(q, q, q, distance_slopes=torch.ones(3, device=device))),
        ("same device", lambda: call(q, q, q, distance_slopes=torch.ones(4))),
        ("no gradient", lambda: call(q, q, q, distance_slopes=torch.ones(4, device=device, requires_grad=True))),
        ("cannot be combined", lambda: call(q, q, q, causal=True, key_ranges=r)),
        ("cannot be combined", lambda: call(q, q, q, key_lengths=torch.ones(2, device=device), key_ranges=r)),
        ("are for", lambda: call(q, q[:, :4], q[:, :4], key_ranges=r)),
        ("are for", lambda: call(q, q, q, key_ranges=fa.build_key_ranges(8, 8, batch=3, device=device))),
        ("maximum 128", lambda: call(*(torch.zeros(1, 4, 1, 136, device=device).half(),) * 3, score_cap=1.0)),
    ]:
        with pytest.raises(ValueError, match=match):
            f()
    with pytest.raises(TypeError):
        call(q, q, q, key_ranges=torch.zeros(2, 8, 2, device=device))


def test_ranges_changed_behind_the_forward_are_noticed(device):
    q, k, v, g = _inputs(1, 64, 64, 1, 1, 64, torch.float16, device)
    r = fa.build_key_ranges(64, 64, causal=True, device=device)
    q.requires_grad_(True)
    o = fa.flash_attention_v100_with_rules(q, k, v, key_ranges=r)
    fa.build_key_ranges(64, 64, window=3, device=device, out=r)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(g)


def test_a_packed_training_step(device):
    """The operators together: ranges of packed documents, q and k turned by the positions within them, attention over the
    ranges, gradients back to q, k and v; every document as if it were alone."""
    B, N, H, Hkv, D = 2, 300, 4, 2, 64
    q, k, v, g = _inputs(B, N, N, H, Hkv, D, torch.bfloat16, device)
    offsets = [[0, 100, 260, 300], [0, 17, 17, 250]]
    r, see, at = _ranges(N, N, B, dict(causal=True, offsets=offsets), device)
    f = fa.rotary_frequencies(D, device=device)[0]
    for t in (q, k, v):
        t.requires_grad_(True)
    qr, kr = fa.rotary_embedding(q, k, inv_freq=f, positions=r.positions)
    o = fa.flash_attention_v100_with_rules(qr, kr, v, score_cap=30.0, key_ranges=r)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), g)
    within = r.positions
    with torch.no_grad():
        q64, k64 = (rotary64(t, within, f, False) for t in (q, k))
        want = attention64(q64, k64, v, see, at, D ** -0.5, 30.0, None, grad=g)
        want = (want[0], rotary64(want[2], within, f, False, inverse=True), rotary64(want[3], within, f, False, inverse=True), want[4])
    # q and k are rounded to bf16 once more on the way, and so are their gradients: 2^-8 / sqrt(3) each, independent
    for n, a, w in zip(("o", "dq", "dk", "dv"), (o, dq, dk, dv), want):
        assert rel(a, w) <= 4 * 2.0 ** -8 / 3 ** 0.5, (n, rel(a, w))


def test_a_decoding_step_in_a_graph(device):
    """Ranges, rotary and attention of one new token, captured once and replayed as the caches grow."""
    B, Nk, H, Hkv, D = 3, 600, 8, 2, 128
    q, k, v, _ = _inputs(B, 1, Nk, H, Hkv, D, torch.bfloat16, device)
    f = fa.rotary_frequencies(D, device=device)[0]
    lengths = torch.tensor([1, 130, 599], dtype=torch.int32, device=device)
    slopes = _slopes(H, device)

    def step(r=None):
        r = fa.build_key_ranges(1, Nk, batch=B, causal=True, key_lengths=lengths, query_offsets=lengths - 1, out=r)
        qr = fa.rotary_embedding(q, inv_freq=f, positions=r.positions)
        return r, fa.flash_attention_v100_with_rules(qr, k, v, score_cap=25.0, distance_slopes=slopes, key_ranges=r)

    with torch.no_grad():
        r, _ = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, o = step(r)
        for new in ([1, 130, 599], [2, 131, 600], [300, 128, 5]):
            lengths.copy_(torch.tensor(new, dtype=torch.int32))
            graph.replay()
            see = torch.stack([visible(1, Nk, b, causal=True, lengths=new, starts=[n - 1 for n in new]) for b in range(B)])
            at = torch.tensor(new).view(B, 1) - 1
            qr = rotary64(q, at.to(device), f, False).to(torch.bfloat16)
            want = attention64(qr, k, v, see, at, D ** -0.5, 25.0, slopes)[0]
            assert rel(o, want) <= 2 * TOLERANCE[torch.bfloat16]      # (q's rounding may fall on the other side)


@pytest.mark.parametrize("wants", ["qkv", "k", "none"])
@pytest.mark.parametrize("dtype", TYPES)
def test_native_and_general_forms_agree(device, dtype, wants):
    """The native operator and the Python one: same bits, also under a mode that watches operators."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    t = TYPES[dtype]
    base = _inputs(2, 90, 90, 4, 2, 64, t, device)
    offsets = torch.tensor([[0, 40, 90], [0, 0, 77]], dtype=torch.int32, device=device)
    f = fa.rotary_frequencies(64, device=device)[0]
    slopes = _slopes(4, device).float()
    got = []
    for native in (True, False):
        q, k, v, g = (x.clone().requires_grad_(n in wants) for x, n in zip(base, "qkvg"))

        def step():
            r = fa.build_key_ranges(90, 90, batch=2, causal=True, document_offsets=offsets)
            turned = fa.rotary_embedding(q, k, inv_freq=f, positions=r.positions, attention_factor=1.5)
            o, lse = fa.flash_attention_v100_with_rules(*turned, v, score_cap=9.0, distance_slopes=slopes, key_ranges=r, return_softmax_lse=True)
            return r, turned, o, lse

        if native:
            r, turned, o, lse = step()
        else:
            with Watch():
                r, turned, o, lse = step()
        if wants != "none":
            o.backward(g)
        assert o.requires_grad == (wants != "none") and not lse.requires_grad
        got.append([r.first, r.end, r.positions, turned[0], turned[1], o, lse, q.grad, k.grad, v.grad])
    for a, b in zip(*got):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


def test_a_changed_operand_is_noticed(device):
    q, k, v, g = _inputs(1, 64, 64, 1, 1, 64, torch.float16, device)
    r = fa.build_key_ranges(64, 64, causal=True, device=device)
    q.requires_grad_(True)
    o = fa.flash_attention_v100_with_rules(q, k, v, key_ranges=r)
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(g)


def test_gradient_of_a_gradient_is_refused(device):
    q, k, v, g = _inputs(1, 64, 64, 1, 1, 64, torch.float16, device)
    r = fa.build_key_ranges(64, 64, causal=True, device=device)
    q.requires_grad_(True)
    o = fa.flash_attention_v100_with_rules(q, k, v, key_ranges=r)
    d, = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), q)


def test_a_long_window_of_many_tiles(device):
    """More tiles than the plan puts in order: every row against its own few keys, in 64 bits."""
    N, w, D = 66000, 200, 64
    q, k, v, g = _inputs(1, N, N, 1, 1, D, torch.bfloat16, device)
    r = fa.build_key_ranges(N, N, causal=True, window=w, device=device)
    o, lse, dq, dk, dv = _step(q, k, v, g, score_cap=6.0, key_ranges=r)
    pad = lambda t: torch.nn.functional.pad(t[0, :, 0].double(), (0, 0, w - 1, 0)).unfold(0, w, 1)      # (N, D, w): a row's keys
    for rows in (slice(0, 3000), slice(30000, 33000), slice(63000, 66000)):
        x = torch.einsum("nd,ndw->nw", q[0, rows, 0].detach().double(), pad(k.detach())[rows]) * D ** -0.5
        t = torch.tanh(x / 6.0)
        at = torch.arange(N, device=device)[rows]
        x = (6.0 * t).masked_fill(at.view(-1, 1) - (w - 1) + torch.arange(w, device=device) < 0, float("-inf"))
        p = torch.softmax(x, dim=1)
        vw, go = pad(v.detach())[rows], g[0, rows, 0].double()
        want = torch.einsum("nw,ndw->nd", p, vw)
        dp = torch.einsum("nd,ndw->nw", go, vw)
        ds = p * (dp - (p * dp).sum(dim=1, keepdim=True)) * (1 - t * t) * D ** -0.5
        assert rel(o[0, rows, 0], want) <= TOLERANCE[torch.bfloat16] and rel(lse[0, 0, rows], torch.logsumexp(x, dim=1)) <= TOLERANCE[torch.bfloat16]
        assert rel(dq[0, rows, 0], torch.einsum("nw,ndw->nd", ds, pad(k.detach())[rows])) <= TOLERANCE[torch.bfloat16]
        # a key's gradients come from the rows behind it: those whose rows all lie in the slice
        n = rows.stop - rows.start - w + 1
        i = torch.arange(n, device=device).view(-1, 1) + torch.arange(w, device=device)                 # rows that see key n
        j = w - 1 - torch.arange(w, device=device)                                                      # ... at this place of theirs
        assert rel(dv[0, rows.start:rows.start + n, 0], torch.einsum("nw,nwd->nd", p[i, j], go[i])) <= TOLERANCE[torch.bfloat16]
        assert rel(dk[0, rows.start:rows.start + n, 0], torch.einsum("nw,nwd->nd", ds[i, j], q[0, rows, 0].detach().double()[i])) <= TOLERANCE[torch.bfloat16]


@pytest.mark.parametrize("dtype,H,Hkv,D", [("bf16", 4, 2, 64), ("fp16", 2, 2, 128), ("fp32", 2, 1, 64)])
def test_a_training_step_in_a_graph(device, dtype, H, Hkv, D):
    """Ranges, rotary, attention and all gradients, captured once, replayed on new documents and new inputs."""
    t = TYPES[dtype]
    N = 260
    q, k, v, g = (x.requires_grad_(n < 3) for n, x in enumerate(_inputs(1, N, N, H, Hkv, D, t, device)))
    f = fa.rotary_frequencies(D, device=device)[0]
    offsets = torch.tensor([0, 100, N], dtype=torch.int32, device=device)

    def step(r=None):
        r = fa.build_key_ranges(N, N, causal=True, document_offsets=offsets, out=r)
        qr, kr = fa.rotary_embedding(q, k, inv_freq=f, positions=r.positions)
        o = fa.flash_attention_v100_with_rules(qr, kr, v, score_cap=12.0, key_ranges=r)
        return r, (o,) + torch.autograd.grad(o, (q, k, v), g)

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        r, _ = step()
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, got = step(r)
    for seed, cuts in ((3, [0, 30, 200]), (4, [0, 259, 260])):
        with torch.no_grad():
            for x, y in zip((q, k, v, g), _inputs(1, N, N, H, Hkv, D, t, device, seed=seed)):
                x.copy_(y)
        offsets.copy_(torch.tensor(cuts, dtype=torch.int32))
        graph.replay()
        _, want = step()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_two_streams_at_once(device):
    """Calls on two streams share nothing: a split forward and a backward beside each other, many times."""
    q, k, v, g = _inputs(2, 300, 300, 4, 2, 64, torch.bfloat16, device)
    r, _, _ = _ranges(300, 300, 2, dict(causal=True, offsets=[[0, 90, 300], [0, 1, 250]]), device)
    q1, k1, v1, _ = _inputs(3, 1, 1200, 8, 2, 128, torch.float16, device)
    r1, _, _ = _ranges(1, 1200, 3, dict(lengths=[1200, 7, 600]), device)
    decode = lambda: fa.flash_attention_v100_with_rules(q1, k1, v1, score_cap=5.0, key_ranges=r1)
    train = lambda: _step(q, k, v, g, score_cap=5.0, key_ranges=r)
    want = (decode(),) + train()
    a, b = torch.cuda.Stream(device), torch.cuda.Stream(device)
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream(device))
    outs = []
    for _ in range(10):
        with torch.cuda.stream(a):
            x = decode()
        with torch.cuda.stream(b):
            y = train()
        outs.append((x,) + y)
    torch.cuda.synchronize()
    for got in outs:
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("Nq,H,Hkv", [(1, 48, 1), (1, 17, 1), (3, 40, 2), (16, 1, 1), (17, 1, 1), (2, 8, 1), (9, 2, 1), (200, 12, 1)])
def test_groups_of_any_size(device, Nq, H, Hkv):
    """Rows of a K/V head on either side of what a decoding block takes (16), groups that do not divide a tile."""
    lengths = [700, 130]
    host = dict(causal=True, lengths=lengths, starts=[max(n - Nq, 0) for n in lengths])
    for dtype, D in ((torch.bfloat16, 128), (torch.float16, 72)):
        q, k, v, _ = _inputs(2, Nq, 700, H, Hkv, D, dtype, device, std=2.0)
        r, see, at = _ranges(Nq, 700, 2, host, device)
        want = attention64(q, k, v, see, at, D ** -0.5, 10.0, _slopes(H, device))
        with torch.no_grad():
            got = fa.flash_attention_v100_with_rules(q, k, v, score_cap=10.0, distance_slopes=_slopes(H, device), key_ranges=r, return_softmax_lse=True)
        _check(got, want, dtype, ("o", "lse"))
