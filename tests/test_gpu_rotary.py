"""rotary_embedding against complex numbers in 64 bits.

An output u cos - w sin of values to fp32's rounding: the cosine and sine are off by 2^-23 (2 units of 2^-24), the products and
their sum by 2^-24 each, together at most 2^-22 (|u| + |w|) times the factor; then half a step of the type."""
import pytest
import torch

import flash_attention_v100 as fa
from rules_helpers import rotary64

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _close(got, x, want, dtype, factor=1.0):
    half_step = torch.finfo(dtype).eps / 2
    size = x.double().abs().amax(dim=-1, keepdim=True) * 2 * factor
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0                   # half a step of fp16's smallest numbers
    assert ((got.double() - want).abs() <= want.abs() * half_step + size * 2.0 ** -22 * (1 + half_step) + tiny).all()


def _inputs(B, N, H, Hkv, D, dtype, device):
    g = torch.Generator().manual_seed(B * 1000 + N)
    return [torch.randn(B, N, h, D, generator=g).to(dtype).to(device) for h in (H, Hkv, H, Hkv)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("B,N,H,Hkv,D,rotary", [(2, 37, 4, 2, 64, 64), (1, 1, 1, 1, 128, 128), (3, 5, 3, 1, 80, 32), (2, 9, 2, 2, 33, 10),
                                                (1, 7, 2, 1, 24, 12), (2, 130, 5, 1, 128, 2), (1, 3, 1, 1, 2, 2), (2, 6, 2, 1, 16, 0)])
def test_turned_and_turned_back(device, dtype, interleaved, B, N, H, Hkv, D, rotary):
    t = TYPES[dtype]
    q, k, gq, gk = _inputs(B, N, H, Hkv, D, t, device)
    f = fa.rotary_frequencies(rotary, device=device)[0] if rotary else torch.empty(0, dtype=torch.float64, device=device)
    at = torch.randint(0, 5000, (B, N), generator=torch.Generator().manual_seed(3), dtype=torch.int32).to(device)
    q.requires_grad_(True)
    k.requires_grad_(True)
    y = fa.rotary_embedding(q, k, inv_freq=f, positions=at, interleaved=interleaved, attention_factor=1.25)
    d = torch.autograd.grad(y, (q, k), (gq, gk))
    for got, x, inverse in zip(y + d, (q, k, gq, gk), (False, False, True, True)):
        x = x.detach()
        _close(got.detach(), x, rotary64(x, at, f, interleaved, 1.25, inverse), t, 1.25)
        assert torch.equal(got.detach()[..., 2 * f.shape[0]:], x[..., 2 * f.shape[0]:])
    with torch.no_grad():
        z = fa.rotary_embedding(q, k, inv_freq=f, positions=at, interleaved=interleaved, attention_factor=1.25)
        w = fa.rotary_embedding(k, inv_freq=f, positions=at.long(), interleaved=interleaved, attention_factor=1.25)
        assert torch.equal(z[0], y[0]) and torch.equal(z[1], y[1]) and torch.equal(w, y[1])
        q2, k2 = q.clone(), k.clone()
        u = fa.rotary_embedding(q2, k2, inv_freq=f, positions=at, interleaved=interleaved, attention_factor=1.25, inplace=True)
        assert u[0] is q2 and u[1] is k2 and torch.equal(q2, y[0]) and torch.equal(k2, y[1])


@pytest.mark.parametrize("far", [0, -3, 10 ** 6, 2 ** 31 - 10, 10 ** 12])
def test_far_positions(device, far):
    """Angles of far positions are reduced in 64 bits: a position times a frequency is off by 2^-53 of itself, 10^12 turns by
    1.1e-4 and 2^31 by 2.4e-7."""
    x = _inputs(2, 6, 2, 1, 64, torch.float32, device)[0]
    f = fa.rotary_frequencies(64, device=device)[0]
    at = far + torch.arange(6, device=device)
    slack = (abs(far) * 2.0 ** -52) * x.double().abs().amax(dim=-1, keepdim=True) * 2
    for positions in (at, far, at.expand(1, 6), at.expand(2, 6)):
        got = fa.rotary_embedding(x, inv_freq=f, positions=positions).double()
        want = rotary64(x, at.expand(2, 6), f, False)
        assert ((got - want).abs() <= want.abs() * 2.0 ** -24 + x.double().abs().amax(dim=-1, keepdim=True) * 2.0 ** -21 + slack).all()


def test_views_and_broadcasts(device):
    """Slices of a fused projection, a head dimension that is not contiguous, an expanded gradient, a part of a cache."""
    f = fa.rotary_frequencies(64, device=device)[0]
    qkv = torch.randn(2, 9, 6, 64, device=device).bfloat16()
    q, k = qkv[:, :, :3], qkv[:, :, 3:5]
    a = fa.rotary_embedding(q, k, inv_freq=f)
    b = fa.rotary_embedding(q.contiguous(), k.contiguous(), inv_freq=f)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.randn(2, 9, 3, 66, device=device).bfloat16()[..., 1:65]                # rows that are not 16-byte aligned
    assert torch.equal(fa.rotary_embedding(odd, inv_freq=f), fa.rotary_embedding(odd.contiguous(), inv_freq=f))
    turned = torch.randn(2, 64, 3, 9, device=device).bfloat16().permute(0, 3, 2, 1)
    assert torch.equal(fa.rotary_embedding(turned, inv_freq=f), fa.rotary_embedding(turned.contiguous(), inv_freq=f))
    x = turned.detach().requires_grad_(True)
    d, = torch.autograd.grad(fa.rotary_embedding(x, inv_freq=f).float().sum(), x)
    ones = torch.ones(2, 9, 3, 64, device=device).bfloat16()
    _close(d, ones, rotary64(ones, torch.arange(9, device=device).expand(2, 9), f, False, inverse=True), torch.bfloat16)
    cache = torch.randn(2, 100, 3, 64, device=device).bfloat16()
    want = cache.clone()
    want[:, 40:49] = fa.rotary_embedding(cache[:, 40:49], inv_freq=f, positions=40)
    fa.rotary_embedding(cache[:, 40:49], inv_freq=f, positions=40, inplace=True)
    assert torch.equal(cache, want)
    only_k = torch.randn(2, 9, 2, 64, device=device).bfloat16().requires_grad_(True)
    y = fa.rotary_embedding(q, only_k, inv_freq=f)
    y[1].sum().backward()
    assert only_k.grad is not None and not qkv.requires_grad


@pytest.mark.parametrize("shape", [(0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)])
def test_empty(device, shape):
    f = fa.rotary_frequencies(64, device=device)[0]
    x = torch.randn(*shape, device=device)
    assert fa.rotary_embedding(x, inv_freq=f).shape == shape
    k = torch.randn(shape[0], shape[1], 1, 64, device=device)
    y = fa.rotary_embedding(x, k, inv_freq=f)
    assert torch.equal(y[1], fa.rotary_embedding(k, inv_freq=f)) and y[0].shape == shape


def test_refusals(device):
    x = torch.zeros(1, 4, 2, 64, device=device)
    f = fa.rotary_frequencies(64, device=device)[0]
    for match, call in [
        ("must match", lambda: fa.rotary_embedding(x, x[:, :3], inv_freq=f)),
        ("must match", lambda: fa.rotary_embedding(x, x.half(), inv_freq=f)),
        ("at most", lambda: fa.rotary_embedding(x[..., :32], inv_freq=f)),
        ("maximum 128", lambda: fa.rotary_embedding(torch.zeros(1, 4, 2, 130, device=device), inv_freq=f)),
        ("same device", lambda: fa.rotary_embedding(x, inv_freq=f.cpu())),
        ("detach", lambda: fa.rotary_embedding(x, inv_freq=f.clone().requires_grad_(True))),
        ("expected", lambda: fa.rotary_embedding(x, inv_freq=f, positions=torch.zeros(2, 4, dtype=torch.int32, device=device))),
        ("int32 or int64", lambda: fa.rotary_embedding(x, inv_freq=f, positions=torch.zeros(4, device=device))),
        ("without gradients", lambda: fa.rotary_embedding(x.clone().requires_grad_(True), inv_freq=f, inplace=True)),
        ("rows of their own", lambda: fa.rotary_embedding(x[:, :1].expand(1, 4, 2, 64), inv_freq=f, inplace=True)),
        ("share memory", lambda: fa.rotary_embedding(x, x, inv_freq=f, inplace=True)),
        ("Unsupported dtype", lambda: fa.rotary_embedding(x.double(), inv_freq=f)),
    ]:
        with pytest.raises(ValueError, match=match):
            call()


def test_in_a_graph_and_on_another_stream(device):
    x = torch.randn(2, 5, 3, 64, device=device).bfloat16()
    at = torch.arange(5, dtype=torch.int32, device=device)
    f = fa.rotary_frequencies(64, device=device)[0]
    fa.rotary_embedding(x, inv_freq=f, positions=at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fa.rotary_embedding(x, inv_freq=f, positions=at)
    at += 100
    graph.replay()
    assert torch.equal(y, fa.rotary_embedding(x, inv_freq=f, positions=100))
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        z = fa.rotary_embedding(x, inv_freq=f, positions=at)
    side.synchronize()
    assert torch.equal(y, z)


def test_a_leaf_changed_behind_the_forward_is_noticed(device):
    """Positions written anew between forward and backward would turn the gradients by other angles."""
    x = torch.randn(1, 4, 1, 64, device=device, requires_grad=True)
    lengths = torch.tensor([4], dtype=torch.int32, device=device)
    r = fa.build_key_ranges(4, 4, key_lengths=lengths)
    y = fa.rotary_embedding(x, inv_freq=fa.rotary_frequencies(64, device=device)[0], positions=r.positions)
    fa.build_key_ranges(4, 4, key_lengths=lengths, query_offsets=3, out=r)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
