"""EnhancedMultiHeadAttention as a language model's layer: rotary positions, a score cap, distances, key ranges."""
import copy

import pytest
import torch

import flash_attention_v100 as fa
from rules_helpers import attention64, rel, rotary64, visible

E, H = 128, 2
SLOPES = torch.tensor([0.5, 0.0625])


def _layer(**kw):
    torch.manual_seed(1)
    return fa.EnhancedMultiHeadAttention(E, H, **kw)


def test_state_dict_and_refusals():
    layer = _layer(rotary_base=10000.0, score_cap=30.0, distance_slopes=SLOPES)
    assert set(layer.state_dict()) == set(_layer().state_dict())
    copy.deepcopy(layer)
    for kw in (dict(rotary_dim=8), dict(rotary_base=1e4, rotary_dim=7), dict(rotary_base=1e4, rotary_dim=66), dict(distance_slopes=torch.ones(3))):
        with pytest.raises(ValueError):
            _layer(**kw)
    x = torch.zeros(2, 4, E)
    with pytest.raises(ValueError, match="mask tensors or dropout"):
        _layer(score_cap=3.0)(x, attn_mask=torch.zeros(4, 4))
    with pytest.raises(ValueError, match="as many keys"):
        _layer(rotary_base=1e4)(x, torch.zeros(2, 5, E))
    with pytest.raises(ValueError, match="positions are for"):
        _layer()(x, positions=3)


@pytest.mark.gpu
@pytest.mark.parametrize("rotary_dim", [None, 32, 0])
@pytest.mark.parametrize("cap,slopes", [(None, None), (5.0, None), (5.0, SLOPES)])
def test_a_packed_step(device, rotary_dim, cap, slopes):
    """Every document as if it were alone, parameters' gradients included.  Weights and activations are rounded to bf16 at eight
    places between the input and a projection's gradient, half a step each: rel 2^-8 / sqrt(3) a place, independent."""
    B, N = 2, 150
    offsets = [[0, 60, 150], [0, 5, 120]]
    layer = _layer(rotary_base=None if rotary_dim == 0 else 500.0, rotary_dim=rotary_dim or None, score_cap=cap, distance_slopes=slopes).to(device).bfloat16()
    x = torch.randn(B, N, E, generator=torch.Generator().manual_seed(2)).bfloat16().to(device)
    r = fa.build_key_ranges(N, N, batch=B, causal=True, document_offsets=torch.tensor(offsets, dtype=torch.int32, device=device))
    out, weights = layer(x, key_ranges=r)
    assert weights is None
    w = torch.randn_like(out)
    out.backward(w)

    P = {n: p.detach().double().requires_grad_(True) for n, p in layer.named_parameters()}
    lin = lambda t, n: t @ P[n + ".weight"].T + P[n + ".bias"]
    q, k, v = (lin(x.double(), n).view(B, N, H, E // H) for n in ("q_proj", "k_proj", "v_proj"))
    if rotary_dim != 0:
        f = fa.rotary_frequencies(rotary_dim or E // H, 500.0, device=device)[0]
        q, k = (rotary64(t, r.positions, f, False) for t in (q, k))
    see = torch.stack([visible(N, N, b, causal=True, offsets=offsets) for b in range(B)]).to(device)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * (E // H) ** -0.5
    if cap is not None:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        at = torch.arange(N, device=device)
        s = s - slopes.to(device).double().view(1, H, 1, 1) * (at.view(-1, 1) - at).abs()
    s = s.masked_fill(~see.unsqueeze(1), float("-inf"))
    some = see.any(dim=2).view(B, 1, N, 1)
    p = torch.where(some, torch.softmax(torch.where(some, s, torch.zeros_like(s)), dim=3), torch.zeros_like(s))
    want = lin(torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, N, E), "out_proj")
    want.backward(w.double())
    bound = 8 * 2.0 ** -8 / 3 ** 0.5
    assert rel(out, want.detach()) <= bound
    for n, t in layer.named_parameters():
        if n == "k_proj.bias":
            continue                       # (no effect on a softmax but through the cap: what is computed is what rounding leaves)
        assert rel(t.grad, P[n].grad) <= bound, (n, rel(t.grad, P[n].grad))


@pytest.mark.gpu
def test_causal_layer_with_a_cap_and_positions(device):
    layer = _layer(rotary_base=1e4, score_cap=20.0).to(device).half().eval()
    x = torch.randn(1, 40, E, device=device).half()
    with torch.no_grad():
        a = layer(x, is_causal=True)[0]
        b = layer(x, is_causal=True, positions=1000)[0]          # a shift of all positions turns q and k alike
        c = layer(x, key_ranges=fa.build_key_ranges(40, 40, causal=True, device=device))[0]
        d = _layer(rotary_base=1e4, score_cap=20.0, batch_first=False).to(device).half().eval()(x.transpose(0, 1), is_causal=True)[0]
    assert rel(a, b) <= 4 * 2.0 ** -11 and torch.equal(a, c) and torch.equal(a, d.transpose(0, 1))
