"""The plain split forward, groups of heads that do not divide a tile: the same bits after other kernels have used shared memory."""
import pytest
import torch

import flash_attention_v100 as fa

pytestmark = pytest.mark.gpu


def _normal(B, N, H, D, dtype, device, seed, std=1.0):
    return (torch.randn(B, N, H, D, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(device)


@pytest.mark.parametrize("Nq,Nk,H,Hkv,D", [(33, 3000, 3, 1, 128), (33, 3000, 10, 2, 64), (17, 5000, 7, 1, 128), (20, 4000, 100, 1, 64), (1, 4000, 3, 1, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_bits_do_not_depend_on_what_shared_memory_held(device, dtype, Nq, Nk, H, Hkv, D):
    q, k, v = _normal(1, Nq, H, D, dtype, device, 0), _normal(1, Nk, Hkv, D, dtype, device, 1), _normal(1, Nk, Hkv, D, dtype, device, 2)
    others = [[_normal(1, 300, 8, 128, dtype, device, s, std) for s in (3, 4, 5)] for std in (50.0, 1.0, 0.0)]
    first = None
    with torch.no_grad():
        for n in range(40):
            o = fa.flash_attention_v100(q, k, v, causal=True, causal_alignment="bottom_right", return_softmax_lse=True)
            first = first or o
            assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1]), n
            fa.flash_attention_v100(*others[n % 3])
