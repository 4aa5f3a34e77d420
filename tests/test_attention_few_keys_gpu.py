"""bf16: a sample that sees few keys keeps the digits of its gradients however many masked keys stand beside them."""
import pytest
import torch

import eve_amd
from tests.attn_few_keys import few_key_gradients

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def _mask(B, Nk, counts, where, g):
    mask = torch.zeros(B, Nk, dtype=torch.bool)
    for b in range(B):
        n = counts[b % len(counts)]
        if where == "front":
            mask[b, :n] = True
        elif where == "end":
            mask[b, Nk - n:] = True
        else:
            mask[b, torch.randperm(Nk, generator=g)[:n]] = True
    return mask


@pytest.mark.parametrize("where", ["front", "end", "anywhere"])
@pytest.mark.parametrize("low", [False, True])
@pytest.mark.parametrize("B,Nq,Nk,H,D", [
    (66, 40, 200, 2, 64), (66, 70, 256, 2, 16), (66, 1, 130, 2, 40),      # a head a workgroup
    (3, 100, 333, 2, 64), (3, 40, 1001, 2, 112), (3, 200, 130, 1, 128),   # a kernel for dq, one for dk and dv
    (3, 2, 4099, 2, 64), (2, 1, 9000, 1, 128),                            # keys split over workgroups
    (4, 90, 64, 2, 64), (4, 90, 64, 2, 96)])
def test_gradients_of_few_visible_keys(B, Nq, Nk, H, D, where, low):
    """`low`: scores far below zero, next to masked keys (whose score would be zero)."""
    g = torch.Generator().manual_seed(B + Nk + D)
    q, k, v, do = (torch.randn(*s, generator=g) for s in ((B, Nq, H, D), (B, Nk, H, D), (B, Nk, H, D), (B, Nq, H, D)))
    if low:
        q, k = q - 4.0, k + 4.0
    q, k, v, do = (t.to(BF16).to(DEV) for t in (q, k, v, do))
    mask = _mask(B, Nk, (2, 1, 3, 5, 17, 64), where, g).to(DEV)
    parts = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(eve_amd.attention(*parts, mask), parts, do)
    want = few_key_gradients(q, k, v, do, mask, D ** -0.5)
    for name, got in (("dq", dq), ("dk", dk)):
        val, tol = want[name]
        err = (got.detach().cpu().double() - val).abs()
        assert torch.isfinite(got).all() and bool((err <= 1.02 * tol + 1e-30).all()), (name, float((err / (tol + 1e-30)).max()))


def test_padding_does_not_change_what_few_keys_give():
    """The same keys alone, and in front of masked ones: both within the bound, and as near to each other."""
    B, Nq, n, H, D = 70, 40, 5, 2, 64
    g = torch.Generator().manual_seed(4)
    q, k, v, do = (torch.randn(B, m, H, D, generator=g).to(BF16).to(DEV) for m in (Nq, n, n, Nq))
    want = few_key_gradients(q, k, v, do, None, D ** -0.5)
    for Nk in (n, 100, 237, 700):
        kk, vv = (torch.cat([t, torch.full((B, Nk - n, H, D), float("nan"), dtype=BF16, device=DEV)], 1) for t in (k, v))
        mask = (torch.arange(Nk, device=DEV) < n).expand(B, Nk)
        parts = [t.detach().requires_grad_(True) for t in (q, kk, vv)]
        dq, dk, dv = torch.autograd.grad(eve_amd.attention(*parts, mask), parts, do)
        assert float(dk[:, n:].abs().sum()) == 0.0 and float(dv[:, n:].abs().sum()) == 0.0
        for name, got in (("dq", dq), ("dk", dk[:, :n])):
            val, tol = want[name]
            assert bool(((got.detach().cpu().double() - val).abs() <= 1.02 * tol + 1e-30).all()), (Nk, name)
