"""The oracle of the operators with rules, and their refusals: no GPU."""
import ctypes

import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100.kernels import _cabi
from rules_helpers import attention64, rotary64, visible


@pytest.mark.parametrize("cap,slopes", [(None, None), (2.0, None), (None, [0.5, 0.1]), (1.5, [0.25, 0.0])])
def test_gradients_of_the_oracle_are_differences(cap, slopes):
    """Central differences of the output's product with a weight: h^2 |f'''| / 6 + 2^-53 |f| / h with h = 1e-5 and
    values of a few units stays below 1e-8."""
    g = torch.Generator().manual_seed(0)
    q, k, v, w = (torch.randn(1, 5, n, 4, generator=g, dtype=torch.float64) for n in (2, 1, 1, 2))
    see = visible(5, 5, 0, causal=True, offsets=[[0, 3, 4]]).unsqueeze(0)
    at = torch.arange(5).unsqueeze(0)
    f = lambda: (attention64(q, k, v, see, at, 0.7, cap, slopes)[0] * w).sum().item()
    grads = attention64(q, k, v, see, at, 0.7, cap, slopes, grad=w)[2:]
    for t, d in zip((q, k, v), grads):
        for e in range(0, t.numel(), 3):
            old = t.view(-1)[e].item()
            t.view(-1)[e] = old + 1e-5
            up = f()
            t.view(-1)[e] = old - 1e-5
            down = f()
            t.view(-1)[e] = old
            assert abs((up - down) / 2e-5 - d.reshape(-1)[e].item()) < 1e-8


def test_rotary_oracle_turns_back():
    x = torch.randn(2, 3, 2, 10, dtype=torch.float64)
    at, f = torch.tensor([[0, 5, 9], [100000, 3, 7]]), torch.tensor([1.0, 0.01, 0.3], dtype=torch.float64)
    for interleaved in (False, True):
        back = rotary64(rotary64(x, at, f, interleaved), at, f, interleaved, inverse=True)
        assert (back - x).abs().max() < 1e-13
    assert torch.equal(rotary64(x, at * 0, f, True), x)


def test_frequencies():
    f, a = fa.rotary_frequencies(8)
    assert f.dtype == torch.float64 and a == 1.0 and f[0] == 1.0 and abs(f[1] - 0.1) < 1e-15
    assert torch.equal(fa.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4)
    n, _ = fa.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert n[0] == f[0] and abs(n[3] / f[3] - 0.25) < 1e-12            # the highest stays, the lowest is a quarter
    p, a = fa.rotary_frequencies(64, scaling="by_parts", factor=4.0, original_length=4096)
    f = fa.rotary_frequencies(64)[0]
    turns = 4096 * f / (2 * torch.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and torch.allclose(p[turns <= 1], f[turns <= 1] / 4, rtol=1e-15)
    assert ((p <= f) & (p >= f / 4 * (1 - 1e-15))).all() and abs(a - 1.1386294361119891) < 1e-12
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.0),
                dict(rotary_dim=2, scaling="ntk", factor=2.0), dict(rotary_dim=8, scaling="by_parts", factor=2.0)):
        with pytest.raises(ValueError):
            fa.rotary_frequencies(**bad)


def test_ranges_are_refused_before_any_launch():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(ValueError, match="window"):
        fa.build_key_ranges(4, 4, window=0, device="cuda:0")
    with pytest.raises(ValueError, match="negative"):
        fa.build_key_ranges(-1, 4, device="cuda:0")
    with pytest.raises(ValueError, match="prefix_lengths are defined"):
        fa.build_key_ranges(4, 4, prefix_lengths=i32(1))
    with pytest.raises(ValueError, match="prefix_lengths are defined"):
        fa.build_key_ranges(4, 4, causal=True, window=2, prefix_lengths=i32(1))
    with pytest.raises(ValueError, match="rows are the ranges"):
        fa.build_key_ranges(4, 4, causal=True, rows=i32(1, 4, 2))
    with pytest.raises(ValueError, match="CUDA device"):
        fa.build_key_ranges(4, 4, key_lengths=i32(1))
    with pytest.raises(ValueError, match="two boundaries"):
        fa.build_key_ranges(4, 4, document_offsets=i32(1), device="cuda:0")
    with pytest.raises(ValueError, match="must be on"):
        fa.build_key_ranges(4, 4, document_offsets=i32(3), device="cuda:0")
    with pytest.raises(ValueError, match="int32 or int64"):
        fa.build_key_ranges(4, 4, key_lengths=torch.zeros(1), device="cuda:0")


def test_rotary_is_refused_before_any_launch():
    x = torch.zeros(1, 4, 2, 8)
    f = torch.ones(4, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        fa.rotary_embedding(x, inv_freq=f)
    with pytest.raises(ValueError, match="4-dimensional"):
        fa.rotary_embedding(x[0], inv_freq=f)
    with pytest.raises(TypeError):
        fa.rotary_embedding(1, inv_freq=f)


def test_rules_are_refused_before_any_launch():
    x = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError, match="requires CUDA tensors"):
        fa.flash_attention_v100_with_rules(x, x, x, score_cap=10.0)
    with pytest.raises(ValueError, match="4-dimensional"):
        fa.flash_attention_v100_with_rules(x[0], x, x)


def _params():
    p = _cabi.Params()
    p.struct_bytes = ctypes.sizeof(_cabi.Params)
    p.B, p.Nq, p.Nk, p.H, p.Hkv, p.D, p.scale = 1, 16, 16, 4, 2, 64, 0.125
    for n in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        setattr(p, n, _cabi.Tensor4(256, 64 * 4 * 16, 64 * 4, 64))
    p.lse = 256
    return p


@pytest.mark.parametrize("field,value", [("causal", 1), ("kv_lengths", 256), ("dropout_p", 0.5), ("d_scores", 256),
                                         ("causal_shift", 3), ("rng_heads", 8), ("bias", _cabi.Tensor4(256, 0, 0, 0))])
def test_masks_of_a_call_with_rules_are_the_plans(field, value):
    lib, p = _cabi.load(), _params()
    r = _cabi.RuleParams(ctypes.sizeof(_cabi.RuleParams), 256, 1, 0.0, None)
    setattr(p, field, value)
    for rc in (lib.fa_b200_fwd_with_rules(ctypes.byref(p), ctypes.byref(r), None, 0), lib.fa_b200_bwd_with_rules(ctypes.byref(p), ctypes.byref(r))):
        assert rc == _cabi.FA_EINVAL and b"of its own" in lib.fa_b200_last_error()


@pytest.mark.parametrize("rule,code,word", [
    (dict(struct_bytes=8), _cabi.FA_EINVAL, b"struct_bytes"), (dict(plan=None), _cabi.FA_EINVAL, b"null"),
    (dict(plan=8), _cabi.FA_EALIGN, b"aligned"), (dict(plan_batch=3), _cabi.FA_EINVAL, b"batch"),
    (dict(score_cap=-1.0), _cabi.FA_EINVAL, b"score_cap"), (dict(score_cap=float("nan")), _cabi.FA_EINVAL, b"score_cap"),
    (dict(score_cap=float("inf")), _cabi.FA_EINVAL, b"score_cap"), (dict(score_cap=1e-40), _cabi.FA_EINVAL, b"too large")])
def test_bad_rules_are_refused_before_any_cuda_call(rule, code, word):
    lib, p = _cabi.load(), _params()
    r = _cabi.RuleParams(ctypes.sizeof(_cabi.RuleParams), 256, 1, 0.0, None)
    for n, x in rule.items():
        setattr(r, n, x)
    assert lib.fa_b200_fwd_with_rules(ctypes.byref(p), ctypes.byref(r), None, 0) == code and word in lib.fa_b200_last_error()
    assert lib.fa_b200_bwd_with_rules(ctypes.byref(p), ctypes.byref(r)) == code
    assert lib.fa_b200_fwd_with_rules(ctypes.byref(p), None, None, 0) == _cabi.FA_EINVAL


@pytest.mark.parametrize("change,code", [
    (dict(struct_bytes=8), _cabi.FA_EINVAL), (dict(B=-1), _cabi.FA_EINVAL), (dict(window=-1), _cabi.FA_EINVAL), (dict(plan=None), _cabi.FA_EINVAL),
    (dict(plan=8), _cabi.FA_EALIGN), (dict(plan_bytes=16), _cabi.FA_EWORKSPACE), (dict(document_offsets=256), _cabi.FA_EINVAL),
    (dict(prefix_lengths=256), _cabi.FA_EINVAL), (dict(B=70000), _cabi.FA_EUNSUPPORTED), (dict(Nq=2 ** 31 - 1), _cabi.FA_EUNSUPPORTED)])
def test_bad_range_parameters_are_refused_before_any_cuda_call(change, code):
    lib = _cabi.load()
    p = _cabi.RangesParams()
    p.struct_bytes, p.plan, p.plan_bytes, p.B, p.Nq, p.Nk = ctypes.sizeof(_cabi.RangesParams), 256, 1 << 20, 2, 100, 100
    for n, x in change.items():
        setattr(p, n, x)
    assert lib.fa_b200_key_ranges(ctypes.byref(p)) == code
    assert lib.fa_b200_key_ranges(None) == _cabi.FA_EINVAL
    assert lib.fa_b200_key_ranges_bytes(-1, 4, 4) == 0
    # rows, 128-row hulls, 16-row hulls, key tiles, three orders, origins
    assert lib.fa_b200_key_ranges_bytes(2, 129, 300) == 4 * (2 * 256 * 2 + 2 * 2 * 4 + 2 * 16 * 2 + 2 * 3 * 2 + 2 * (2 + 1 + 3) + 4)


@pytest.mark.parametrize("change,code", [
    (dict(struct_bytes=8), _cabi.FA_EINVAL), (dict(D=130), _cabi.FA_EUNSUPPORTED), (dict(half=33), _cabi.FA_EINVAL), (dict(N=-1), _cabi.FA_EINVAL),
    (dict(dtype=9), _cabi.FA_EINVAL), (dict(inv_freq=None), _cabi.FA_EINVAL), (dict(factor=float("nan")), _cabi.FA_EINVAL)])
def test_bad_rotary_parameters_are_refused_before_any_cuda_call(change, code):
    lib = _cabi.load()
    p = _cabi.RotaryParams()
    p.struct_bytes, p.B, p.N, p.D, p.half, p.factor, p.inv_freq = ctypes.sizeof(_cabi.RotaryParams), 1, 4, 64, 32, 1.0, 256
    p.x[0], p.y[0], p.heads[0] = _cabi.Tensor4(256, 512, 128, 64), _cabi.Tensor4(256, 512, 128, 64), 2
    for n, x in change.items():
        setattr(p, n, x)
    assert lib.fa_b200_rotary(ctypes.byref(p)) == code
    assert lib.fa_b200_rotary(None) == _cabi.FA_EINVAL
