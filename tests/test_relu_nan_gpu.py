"""relu of NaN is NaN, in every kernel that applies it: the fused linear product's and the expert FFNs'."""
import pytest
import torch

import eve_amd
from eve_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32

# one size for each kernel the forward of the linear product may take: up to 4 rows, a shared contraction, general tiles of 64
# and 128, streamed tiles
SIZES = [(3, 100, 33), (40, 1024, 200), (400, 64, 504), (9000, 515, 777), (9000, 200, 776), (8000, 136, 1288)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_linear(rows, K, N, dtype):
    g = torch.Generator().manual_seed(rows + N)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    x, w, gamma, residual = r(rows, K), r(N, K) * K ** -0.5, r(N), r(rows, N)
    x[rows // 2, K - 1] = float("nan")
    bias = r(N)
    bias[N // 3] = float("nan")
    bad = torch.zeros(rows, N, dtype=torch.bool, device=DEV)
    bad[rows // 2] = True
    bad[:, N // 3] = True
    y = eve_amd.fused_linear(x, w, bias, activation="relu", gamma=gamma, residual=residual)
    assert torch.equal(torch.isnan(y), bad)
    p = [t.requires_grad_(True) for t in (x, w, bias, gamma)]
    y2 = eve_amd.fused_linear(x, w, bias, activation="relu", gamma=gamma, residual=residual)
    assert torch.equal(torch.isnan(y2), bad)
    dy = torch.ones_like(y2)
    _, _, db, dg = torch.autograd.grad(y2, p, dy)
    # relu(NaN) is a NaN term of every column's dgamma; the gradient passes a NaN as it does in torch, so dbias stays a number
    assert bool(torch.isnan(dg).all()) and bool(torch.isfinite(db).all())
    counted = float(db[N // 3]) / float(gamma.detach()[N // 3])
    assert abs(counted - rows) <= rows * (2 * 2 ** -8 if dtype == BF16 else rows * 2 ** -23), counted


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_expert_ffn(dtype):
    G, R, M, I = 4, 70, 64, 128
    g = torch.Generator().manual_seed(2)
    r = lambda *s, m=0.1: (torch.randn(*s, generator=g) * m).to(dtype).to(DEV)
    x, w1, b1, w2, b2 = r(G, R, M, m=1.0), r(G, I, M), r(G, I), r(G, M, I), r(G, M)
    x[2, 5, 7] = float("nan")
    rows = torch.full((G,), R, dtype=torch.int32, device=DEV)
    _, a, y = ops.ffn_fwd(x, w1, b1, w2, b2, rows, ops.ACTS["relu"])
    bad = torch.zeros(G, R, 1, dtype=torch.bool, device=DEV)
    bad[2, 5] = True
    assert torch.equal(torch.isnan(a), bad.expand_as(a)) and torch.equal(torch.isnan(y), bad.expand_as(y))
