"""Infinities and NaN in places that are seen: they show where the formula has them, and nowhere else."""
import pytest
import torch

import eve_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32

# each way through the kernels: (B, Nq, Nk, H, Hkv, D, dtype)
WAYS = [(66, 40, 200, 4, 2, 64, BF16), (3, 90, 333, 4, 2, 64, BF16), (3, 90, 333, 4, 2, 128, BF16), (2, 40, 20, 4, 2, 64, BF16),
        (2, 1, 3001, 4, 2, 64, BF16), (3, 90, 333, 4, 2, 64, F32), (2, 1, 3001, 4, 2, 128, F32)]


def _make(B, Nq, Nk, H, Hkv, D, dtype):
    g = torch.Generator().manual_seed(B + Nk)
    shapes = ((B, Nq, H, D), (B, Nk, Hkv, D), (B, Nk, Hkv, D), (B, Nq, H, D))
    return [torch.randn(*s, generator=g).to(dtype).to(DEV) for s in shapes]


def _grads(q, k, v, do, mask):
    parts = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*parts, mask)
    return (out.detach(), *torch.autograd.grad(out, parts, do))


@pytest.mark.parametrize("way", WAYS, ids=lambda w: "x".join(map(str, w[:6])) + str(w[6])[6:])
@pytest.mark.parametrize("few", [False, True])
def test_a_nan_key_spoils_its_heads_gradients_whole(way, few):
    """The row maximum, sum and so every probability of the heads that read it are NaN; the other sample and heads are as ever."""
    B, Nq, Nk, H, Hkv, D, dtype = way
    q, k, v, do = _make(*way)
    mask = torch.ones(B, Nk, dtype=torch.bool, device=DEV)
    mask[:, (6 if few else Nk - 2):] = False
    clean = _grads(q, k, v, do, mask)
    k[1, 4, 1, 3] = float("nan")
    out, dq, dk, dv = _grads(q, k, v, do, mask)
    mine = slice(H // Hkv, 2 * H // Hkv)
    seen = mask[1]
    assert bool(torch.isnan(out[1][:, mine]).all()) and bool(torch.isnan(dq[1][:, mine]).all())
    assert bool(torch.isnan(dk[1, seen, 1]).all()), "dk"
    assert bool(torch.isnan(dv[1, seen, 1]).all()), "dv"
    assert float(dk[1, ~seen].abs().sum()) == 0.0 and float(dv[1, ~seen].abs().sum()) == 0.0
    for got, want in zip((out, dq, dk, dv), clean):
        heads = mine if got.shape[2] == H else slice(1, 2)
        a, b = got.clone(), want.clone()
        a[1][:, heads], b[1][:, heads] = 0, 0
        assert torch.equal(a, b)


@pytest.mark.parametrize("way", WAYS, ids=lambda w: "x".join(map(str, w[:6])) + str(w[6])[6:])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_gradient_that_is_no_number_stays_in_its_column_of_dv(way, bad):
    """dv_jd = sum_i p_ij do_id: only column d.  ds of that row is no number, so its dq and all of the head's dk are none."""
    B, Nq, Nk, H, Hkv, D, dtype = way
    q, k, v, do = _make(*way)
    mask = torch.ones(B, Nk, dtype=torch.bool, device=DEV)
    mask[:, Nk - 2:] = False
    clean = _grads(q, k, v, do, mask)
    do[1, Nq - 1, 2, 5] = bad  # query head 2 reads key head 1
    _, dq, dk, dv = _grads(q, k, v, do, mask)
    assert not bool(torch.isfinite(dq[1, Nq - 1, 2]).any()) and not bool(torch.isfinite(dk[1, :Nk - 2, 1]).any())
    gone = torch.zeros(D, dtype=torch.bool, device=DEV)
    gone[5] = True
    assert not bool(torch.isfinite(dv[1, :Nk - 2, 1][:, gone]).any())
    assert torch.equal(dv[1, :, 1][:, ~gone], clean[3][1, :, 1][:, ~gone])
    assert torch.equal(dv[:, :, 0], clean[3][:, :, 0]) and torch.equal(dk[:, :, 0], clean[2][:, :, 0])


@pytest.mark.parametrize("way", WAYS, ids=lambda w: "x".join(map(str, w[:6])) + str(w[6])[6:])
def test_rows_whose_visible_scores_are_all_minus_infinity(way):
    """exp(-inf - max) with max = -inf is NaN; keys of score -inf beside others take no part; no visible key at all gives zeros."""
    B, Nq, Nk, H, Hkv, D, dtype = way
    q, k, v, do = _make(*way)
    q = q.abs() + 0.1
    mask = torch.ones(B, Nk, dtype=torch.bool, device=DEV)
    mask[:, Nk - 2:] = False
    half = Nk // 2
    some = k.clone()
    some[:, :half] = float("-inf")
    got = eve_amd.attention(q, some, v, mask)
    later = mask.clone()
    later[:, :half] = False
    want = eve_amd.attention(q, k, v, later)
    eps = 4 * 2.0 ** -8 if dtype == BF16 else Nk * 2.0 ** -22  # tiles fall otherwise: each result is rounded p's and its own rounding off
    assert bool(((got - want).float().abs() <= eps * (1 + v.float().abs().amax())).all())
    k[1, :, 1] = float("-inf")
    mask[0] = False
    out, dq, dk, dv = _grads(q, k, v, do, mask)
    mine = slice(H // Hkv, 2 * H // Hkv)
    assert bool(torch.isnan(out[1][:, mine]).all()), "out"
    assert bool(torch.isnan(dq[1][:, mine]).all()), "dq"
    assert bool(torch.isnan(dk[1, :Nk - 2, 1]).all()) and bool(torch.isnan(dv[1, :Nk - 2, 1]).all()), "dk, dv"
    assert bool(torch.isfinite(out[1][:, :H // Hkv]).all())
    for t in (out[0], dq[0], dk[0], dv[0], dk[1, Nk - 2:], dv[1, Nk - 2:]):
        assert float(t.abs().sum()) == 0.0
