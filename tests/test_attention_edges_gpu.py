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


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,Nk", [(40, 200), (70, 333), (2, 2000)])
@pytest.mark.parametrize("power", [-96, -60, 60, 96])
def test_the_smallest_and_largest_scales(power, Nq, Nk, dtype):
    """scale 2^n with queries of 2^-(n / 2) and keys of as much: the same scores, and the same results up to the powers of two."""
    B, H, D = 66 if Nk == 200 else 3, 2, 64
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(B, n, H, D, generator=g).to(dtype).to(DEV) for n in (Nq, Nk, Nk, Nq))
    mask = (torch.rand(B, Nk, generator=g) < 0.7).to(DEV)
    results = []
    for n in (0, power):
        f = 2.0 ** (-n // 2)
        parts = [t.detach().requires_grad_(True) for t in (q * f, k * f, v)]
        out = eve_amd.attention(*parts, mask, scale=2.0 ** (n - 3))
        dq, dk, dv = torch.autograd.grad(out, parts, do)
        results.append((out.detach(), dq * f, dk * f, dv))
    for a, b in zip(*results):
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b)
    if power < 0:  # every score is next to nothing: the mean of the visible values, and no gradient to speak of
        parts = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = eve_amd.attention(*parts, mask, scale=2.0 ** power)
        for t in (out, *torch.autograd.grad(out, parts, do)):
            assert bool(torch.isfinite(t).all())
