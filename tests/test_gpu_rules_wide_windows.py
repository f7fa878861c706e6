"""Windows as wide as 32 bits hold: a few queries on a long cache are divided as without a window, and give the same."""
import ctypes

import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100.kernels import _cabi
from flash_attention_v100.testing import TOLERANCE
from rules_helpers import attention64, rel, visible

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("Nq,Nk,H,Hkv", [(17, 16000, 2, 2), (300, 9000, 2, 2), (40, 6000, 4, 2), (700, 8892, 32, 8)])
@pytest.mark.parametrize("cap", [0.0, 6.0])
def test_scratch_of_a_hint_beyond_all_keys(device, Nq, Nk, H, Hkv, cap):
    lib, p = _cabi.load(), _cabi.Params()
    p.struct_bytes = ctypes.sizeof(_cabi.Params)
    p.B, p.Nq, p.Nk, p.H, p.Hkv, p.D, p.scale, p.dtype, p.device = 1, Nq, Nk, H, Hkv, 128, 0.1, _cabi.FA_B200_BF16, device.index
    for n in ("q", "k", "v", "o"):
        setattr(p, n, _cabi.Tensor4(256, 128 * 32 * 16000, 128 * 32, 128))
    p.lse = 256
    sizes = []
    for hint in (0, Nk, MOST - 1000, MOST):
        r = _cabi.RuleParams(ctypes.sizeof(_cabi.RuleParams), 256, 1, cap, None, hint)
        sizes.append(lib.fa_b200_fwd_rules_workspace_bytes(ctypes.byref(p), ctypes.byref(r)))
    assert sizes[0] > 0 and sizes == sizes[:1] * 4


@pytest.mark.parametrize("causal,window", [(True, MOST), (False, MOST), (False, 2 ** 30), (True, MOST - 200)])
def test_few_queries_under_a_wide_window(device, causal, window):
    Nq, Nk, H, D = 17, 6000, 2, 128
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, n, H, D, generator=g).bfloat16().to(device) for n in (Nq, Nk, Nk))
    call = lambda w: fa.flash_attention_v100_with_rules(q, k, v, score_cap=6.0, return_softmax_lse=True, key_ranges=fa.build_key_ranges(
        Nq, Nk, causal=causal, window=w, query_offsets=Nk - Nq, device=device))
    o, lse = call(window)
    plain = call(None)
    assert torch.equal(o, plain[0]) and torch.equal(lse, plain[1])
    see = visible(Nq, Nk, 0, causal=causal, window=window, starts=Nk - Nq).unsqueeze(0)
    want = attention64(q, k, v, see, (torch.arange(Nq) + Nk - Nq).unsqueeze(0), D ** -0.5, 6.0)
    assert rel(o, want[0]) <= TOLERANCE[torch.bfloat16] and rel(lse, want[1]) <= TOLERANCE[torch.bfloat16]
