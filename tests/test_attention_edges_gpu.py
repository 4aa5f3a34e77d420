"""eve_amd.attention at the ends of its sizes and strides, on the GPU."""
import pytest
import torch

import eve_amd
from eve_amd import ops
from tests.attn_reference import assert_within, attention64

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


def _far(B, N, H, D, dtype, seed):
    """[B, N, H, D] whose rows lie 2^22 elements apart, the furthest that are read in place, and samples and heads side by side."""
    step = 1 << 22
    g = torch.Generator().manual_seed(seed)
    values = torch.randn(B, N, H, D, generator=g).to(dtype).to(DEV)
    store = torch.empty((N - 1) * step + B * H * D, dtype=dtype, device=DEV)
    view = torch.as_strided(store, (B, N, H, D), (H * D, step, D, 1))
    view.copy_(values)
    return view, values


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,D,dtype", [(1, 600, 600, 2, 2, 64, BF16), (1, 70, 600, 4, 2, 128, BF16), (1, 3, 1030, 2, 1, 64, BF16),
                                                  (1, 600, 300, 1, 1, 40, F32), (64, 200, 256, 2, 2, 64, BF16)])
def test_rows_far_apart(B, Nq, Nk, H, Hkv, D, dtype):
    """Read where they lie (no copy): offsets of tiles pass 2^31 elements, or 2^31 bytes for the backward of whole heads."""
    (q, q0), (k, k0), (v, v0) = (_far(B, n, h, D, dtype, s) for s, (n, h) in enumerate(((Nq, H), (Nk, Hkv), (Nk, Hkv))))
    assert all(ops.attn_readable(t) is t for t in (q, k, v))
    do = torch.randn(B, Nq, H, D, generator=torch.Generator().manual_seed(7)).to(dtype).to(DEV)
    mask = (torch.rand(B, Nk, generator=torch.Generator().manual_seed(8)) < 0.8).to(DEV)
    results = []
    for parts in ((q, k, v), (q0, k0, v0)):
        parts = [t.detach().requires_grad_(True) for t in parts]
        out = eve_amd.attention(*parts, mask)
        results.append((out.detach(), *torch.autograd.grad(out, parts, do)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    some = slice(0, 2)
    assert_within(dict(zip(("out", "dq", "dk", "dv"), [t[some] for t in results[0]])),
                  attention64(q0[some], k0[some], v0[some], mask[some], dout=do[some]), "far rows")


@pytest.mark.parametrize("B,Nq,Nk,H,D,dtype", [(2, 2100, 2200, 16, 16, F32), (48, 20, 4300, 16, 8, BF16), (32, 70, 4300, 16, 8, BF16),
                                              (48, 20, 2200, 16, 72, BF16), (8, 500, 2200, 16, 72, BF16)])
@pytest.mark.parametrize("kind", ["holes", "head"])
def test_masks_of_more_tiles_than_are_held_at_a_time(B, Nq, Nk, H, D, dtype, kind):
    """Heads enough that a workgroup walks all keys: the words of the mask are made anew after 64 tiles.  Some heads are compared."""
    g = torch.Generator().manual_seed(Nk + D)
    q, k, v, do = (torch.randn(B, n, H, D, generator=g).to(dtype).to(DEV) for n in (Nq, Nk, Nk, Nq))
    if kind == "holes":
        mask = (torch.rand(B, Nk, generator=g) < 0.6).to(DEV)
    else:
        mask = torch.arange(Nk, device=DEV)[None] >= torch.linspace(0, Nk, B, device=DEV).long()[:, None]
    parts = [t.requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*parts, mask)
    grads = torch.autograd.grad(out, parts, do)
    for b, h in ((0, 0), (B // 2, 3), (B - 2, H - 1), (B - 1, 1)):
        at = slice(b, b + 1), slice(None), slice(h, h + 1)
        res = attention64(q[at], k[at], v[at], mask[b:b + 1], dout=do[at])
        assert_within(dict(zip(("out", "dq", "dk", "dv"), [t[at] for t in (out, *grads)])), res, f"sample {b}, head {h}")


def _calls():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)
    x, w = r(2, 5, 16), r(24, 16)
    qkv = r(2, 9, 3, 2, 16)
    return {"attention": (lambda t: eve_amd.attention(*t.unbind(2)), qkv), "self_attention": (eve_amd.self_attention, qkv),
            "fused_linear": (lambda t: eve_amd.fused_linear(t, w, activation="gelu"), x)}


@pytest.mark.parametrize("name", ["attention", "self_attention", "fused_linear"])
def test_second_derivatives_and_forward_mode_are_refused(name):
    fn, x = _calls()[name]
    x = x.requires_grad_(True)
    dx, = torch.autograd.grad(fn(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), torch.no_grad():
        dual = fwad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):
            fn(dual)
