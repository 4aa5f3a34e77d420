"""eve_amd.attention at the ends of its sizes and strides, on the GPU."""
import pytest
import torch

import eve_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_parts_of_tensors_with_odd_strides(dtype):
    wide = torch.randn(2, 5, 3, 9, device=DEV, dtype=dtype)
    none, some = wide[:, :0, :, :8].detach().requires_grad_(True), wide[..., :8].detach().requires_grad_(True)
    out = eve_amd.attention(none, some, some)  # no queries
    assert out.shape == none.shape
    for t, g in zip((none, some), torch.autograd.grad(out, (none, some), torch.empty_like(out))):
        assert g.shape == t.shape and float(g.abs().sum()) == 0.0
    out = eve_amd.attention(some, none, none)  # no keys
    assert out.shape == some.shape and float(out.abs().sum()) == 0.0
    for t, g in zip((none, some), torch.autograd.grad(out, (none, some), torch.ones_like(out))):
        assert g.shape == t.shape and float(g.abs().sum()) == 0.0
