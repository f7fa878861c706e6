"""What a layer keeps between calls: frequencies and slopes, good for any mode and as they are now."""
import pytest
import torch

import flash_attention_v100 as fa

SLOPES = torch.tensor([0.5, 0.0625])


def _layer(**kw):
    torch.manual_seed(1)
    return fa.EnhancedMultiHeadAttention(128, 2, rotary_base=1e4, score_cap=20.0, distance_slopes=SLOPES, **kw)


def test_tables_made_in_inference_mode_serve_training():
    layer = _layer()
    with torch.inference_mode():
        built_there = _layer()
        for n in ("frequencies", "slopes"):
            for x in (layer, built_there):
                assert not x._table(n, torch.device("cpu")).is_inference()
    for n in ("frequencies", "slopes"):
        assert not layer._table(n, torch.device("cpu")).is_inference()


def test_tables_follow_what_they_were_made_of():
    import copy
    layer, cpu = _layer(), torch.device("cpu")
    for x in (layer, copy.deepcopy(layer)):
        t = x._table("frequencies", cpu)
        assert torch.equal(x._table("slopes", cpu), SLOPES) and x._table("frequencies", cpu) is t
        x.distance_slopes = torch.tensor([0.25, 0.125])
        assert x._table("slopes", cpu).tolist() == [0.25, 0.125]
        x.distance_slopes.mul_(2)
        assert x._table("slopes", cpu).tolist() == [0.5, 0.25]
        x.rotary = (32, 500.0)
        assert torch.equal(x._table("frequencies", cpu), fa.rotary_frequencies(32, 500.0)[0])
        x.distance_slopes = None
        assert x._table("slopes", cpu) is None


def test_a_layer_pickled_before_there_were_rules():
    import io
    layer = fa.EnhancedMultiHeadAttention(128, 2)
    for name in ("score_cap", "rotary", "distance_slopes", "_tables"):
        del layer.__dict__[name]
    f = io.BytesIO()
    torch.save(layer, f)
    f.seek(0)
    old = torch.load(f, weights_only=False)
    with pytest.raises(ValueError, match="CUDA"):            # (what any layer says on the CPU)
        old(torch.zeros(1, 4, 128))


@pytest.mark.gpu
def test_slopes_assigned_anew_are_seen(device):
    x = torch.randn(1, 40, 128, generator=torch.Generator().manual_seed(0)).half().to(device)
    new = torch.tensor([0.25, 0.125])
    layer, fresh = _layer().to(device).half(), _layer().to(device).half()
    with torch.no_grad():
        before = layer(x, is_causal=True)[0]
        layer.distance_slopes = new
        fresh.distance_slopes = new.clone()
        after = layer(x, is_causal=True)[0]
        assert torch.equal(after, fresh(x, is_causal=True)[0]) and not torch.equal(after, before)
        layer.distance_slopes.copy_(SLOPES)
        assert torch.equal(layer(x, is_causal=True)[0], before)


@pytest.mark.gpu
def test_an_evaluation_before_training(device):
    """The first pass under inference_mode, then a training step: as if there had been no first pass."""
    x = torch.randn(2, 40, 128, generator=torch.Generator().manual_seed(0)).bfloat16().to(device)
    r = fa.build_key_ranges(40, 40, causal=True, device=device)
    grads = []
    for first in (True, False):
        layer = _layer().to(device).bfloat16()
        if first:
            with torch.inference_mode():
                layer.eval()(x, key_ranges=r)
            layer.train()
        layer(x, key_ranges=r)[0].float().square().sum().backward()
        grads.append([p.grad for p in layer.parameters()])
    for a, b in zip(*grads):
        assert torch.equal(a, b)
