"""Gradients of gradients: rotary positions have them, attention under rules refuses them, in the native form and in the general one."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import flash_attention_v100 as fa
from flash_attention_v100.ops import sequence_parallel as sp
from flash_attention_v100.utils import last_derivative
from ring_helpers import OracleBlockKernels, run_ring
from rules_helpers import rel, rotary64


class Watch(TorchDispatchMode):
    """A mode that watches operators: the native forms leave such calls to the general ones."""

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class Square(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y):
        ctx.save_for_backward(x)
        return x * x

    @staticmethod
    @last_derivative
    def backward(ctx, g):
        x, = ctx.saved_tensors
        return 2 * x * g, None


def test_a_last_derivative_is_no_constant():
    x = torch.tensor([1.0, 2.0], requires_grad=True)
    for g in (torch.ones(2), torch.ones(2, requires_grad=True)):
        d, = torch.autograd.grad(Square.apply(x, None), x, g, create_graph=True)
        assert torch.equal(d, 2 * x) and d.requires_grad
        with torch.no_grad():
            d.mul_(1.0)                                   # clipping, for instance
        loss = d.sum() + x.square().sum()
        for ask in (lambda: torch.autograd.grad(loss, x, retain_graph=True), loss.backward):
            with pytest.raises(RuntimeError, match="second derivative"):
                ask()
    d, = torch.autograd.grad(Square.apply(x, None).sum(), x)
    assert torch.equal(d, 2 * x) and not d.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False], ids=["native", "general"])
@pytest.mark.parametrize("weight_wants", [False, True])
def test_attention_under_rules_refuses(device, native, weight_wants):
    """The ordinary part of a loss beside a penalty on the gradient: the penalty's part is not dropped."""
    g = torch.Generator().manual_seed(0)
    q, k, v, w = (torch.randn(1, 64, 2, 64, generator=g).half().to(device) for _ in range(4))
    for t in (q, k, v):
        t.requires_grad_(True)
    w.requires_grad_(weight_wants)
    r = fa.build_key_ranges(64, 64, causal=True, device=device)

    def penalised(create):
        o = fa.flash_attention_v100_with_rules(q, k, v, score_cap=9.0, key_ranges=r)
        return o, torch.autograd.grad(o, (q, k, v), w, create_graph=create)

    def step():
        o, plain = penalised(False)
        o, d = penalised(True)
        for a, b in zip(d, plain):
            assert torch.equal(a, b) and a.requires_grad and not b.requires_grad
        for a, x in zip(d, (q, k, v)):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(o.float().sum() + a.float().square().sum(), x, retain_graph=True)
        o.float().sum().backward()                       # a first derivative alone is as it was
        assert q.grad is not None

    if native:
        step()
    else:
        with Watch():
            step()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False], ids=["native", "general"])
@pytest.mark.parametrize("interleaved,factor", [(False, 1.0), (True, 1.25)])
@pytest.mark.parametrize("both", [True, False])
def test_rotary_has_any_derivative(device, native, interleaved, factor, both):
    """sum(y^3 a) and a penalty on its gradient, against complex numbers in 64 bits.  Every turn rounds fp32 values by 2^-24 a
    product and the tables by 2^-22: below 1e-5 through the four turns that the second derivative takes."""
    g = torch.Generator().manual_seed(1)
    base = [torch.randn(2, 9, h, 32, generator=g).to(device) for h in (3, 1)]
    weights = [torch.randn(t.shape, generator=g).to(device) for t in base]
    f = fa.rotary_frequencies(24, device=device)[0]
    at = torch.randint(0, 500, (2, 9), generator=g).to(device)
    n = 2 if both else 1

    def losses(turn, xs, ws):
        ys = turn(xs)
        d = torch.autograd.grad(sum((y ** 3 * w).sum() for y, w in zip(ys, ws)), xs, create_graph=True)
        loss = sum((y * w).sum() for y, w in zip(ys, ws)) + sum((e * e * w).sum() for e, w in zip(d, ws))
        return list(d) + list(torch.autograd.grad(loss, xs))

    def kernels(xs):
        out = fa.rotary_embedding(*xs, inv_freq=f, positions=at, interleaved=interleaved, attention_factor=factor)
        return out if both else (out,)

    xs = [t.clone().requires_grad_(True) for t in base[:n]]
    if native:
        got = losses(kernels, xs, weights)
    else:
        with Watch():
            got = losses(kernels, xs, weights)
    xs = [t.double().requires_grad_(True) for t in base[:n]]
    want = losses(lambda xs: [rotary64(x, at, f, interleaved, factor) for x in xs], xs, [w.double() for w in weights])
    for a, b in zip(got, want):
        assert rel(a, b.detach()) <= 1e-5, rel(a, b.detach())


@pytest.mark.gpu
def test_one_of_two_rotary_gradients(device):
    """Only k's output is used, and only k's gradient is asked for: with and without a graph."""
    q, k = (torch.randn(1, 5, 2, 16, device=device, requires_grad=True) for _ in range(2))
    f = fa.rotary_frequencies(16, device=device)[0]
    _, kr = fa.rotary_embedding(q, k, inv_freq=f)
    w = torch.randn_like(kr, requires_grad=True)
    d, = torch.autograd.grad(kr, k, w, create_graph=True)
    dq, = torch.autograd.grad(kr, q, w, retain_graph=True, allow_unused=True)
    assert dq is None or not dq.any()
    back, = torch.autograd.grad(d, w, torch.ones_like(d))
    want = rotary64(torch.ones_like(k), torch.arange(5, device=device).view(1, 5), f, False)
    assert rel(back, want) <= 1e-6


def test_a_ring_refuses():
    def rank(ring):
        q, k, v = (torch.randn(1, 8, 2, 16, generator=torch.Generator().manual_seed(ring.rank), requires_grad=True) for _ in range(3))
        o = sp.flash_attention_v100_sequence_parallel(q, k, v, causal=True, ring=ring, kernels=OracleBlockKernels)
        d = torch.autograd.grad(o.sum(), (q, k, v), create_graph=True)
        for g, x in zip(d, (q, k, v)):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(g.square().sum() + x.square().sum(), x, retain_graph=True)
        return True

    assert all(run_ring(2, rank))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["native", "watched", "bias", "dropout", "fp32"])
def test_plain_attention_refuses(device, form):
    g = torch.Generator().manual_seed(0)
    t = torch.float32 if form == "fp32" else torch.bfloat16
    q, k, v, w = (torch.randn(1, 70, 2, 64, generator=g).to(t).to(device) for _ in range(4))
    for x in (q, k, v):
        x.requires_grad_(True)
    bias = torch.zeros(1, 2, 70, 70, device=device, requires_grad=True) if form == "bias" else None

    def step():
        inputs = (q, k, v) + ((bias,) if bias is not None else ())
        stream = dict(dropout_p=0.2, dropout_stream=(1, 0)) if form == "dropout" else {}
        call = lambda: fa.flash_attention_v100(q, k, v, causal=True, bias=bias, **stream)
        plain = torch.autograd.grad(call(), inputs, w)
        o = call()
        d = torch.autograd.grad(o, inputs, w, create_graph=True)
        for a, b, x in zip(d, plain, inputs):
            assert torch.equal(a, b)
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(o.float().sum() + a.float().square().sum(), x, retain_graph=True)

    if form == "watched":
        with Watch():
            step()
    else:
        step()


@pytest.mark.gpu
def test_a_layer_with_padding_refuses(device):
    layer = fa.EnhancedMultiHeadAttention(128, 2).to(device).bfloat16()
    x = torch.randn(2, 30, 128, device=device).bfloat16().requires_grad_(True)
    mask = torch.zeros(2, 30, dtype=torch.bool, device=device)
    mask[0, 20:] = True
    out = layer(x, key_padding_mask=mask)[0]
    d = torch.autograd.grad(out.float().sum(), [x, *layer.k_proj.parameters()], create_graph=True)
    for a in d:
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(a.float().square().sum() + x.float().sum(), x, retain_graph=True)
