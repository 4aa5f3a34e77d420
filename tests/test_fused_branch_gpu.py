"""The bf16 attention branch of a layer on the library's kernels, by what the branch adds and by the gradients of its parameters,
against the formula in 64 bits."""
import pytest
import torch

from eve_amd import encoder as enc
from eve_amd.encoder import MultiwayTransformerEncoder, MultiwayTransformerEnocderLayer

DEV = "cuda:0"
BF16, U = torch.bfloat16, 2.0 ** -8  # half a step of a rounding


class _Rounds(torch.autograd.Function):
    """A rounding of the value, of the gradient, or of both, as a relative error anywhere up to half a step."""

    @staticmethod
    def forward(ctx, x, g, value, grad):
        ctx.g, ctx.grad = g, grad
        return x * (1 + U * (2 * torch.rand(x.shape, generator=g, dtype=x.dtype) - 1)) if value else x.clone()

    @staticmethod
    def backward(ctx, d):
        return (d * (1 + U * (2 * torch.rand(d.shape, generator=ctx.g, dtype=d.dtype) - 1)) if ctx.grad else d), None, None, None


def _branch64(x, residual, p, heads, mask, row_scale, g=None):
    """residual + row_scale gamma (attention(x) projected), x the normalised input; with `g`, errors drawn where the bf16 kernels
    round: qkv, the probabilities for the product with v, ds, attention's result, dz of both products, the sum."""
    r = (lambda t, value=True, grad=True: _Rounds.apply(t, g, value, grad)) if g is not None else (lambda t, value=True, grad=True: t)
    B, N, C = x.shape
    bias = torch.cat((p["q_bias"], torch.zeros_like(p["q_bias"]), p["v_bias"]))
    qkv = r(x @ p["qkv.weight"].t() + bias).view(B, N, 3, heads, C // heads)
    q, k, v = (t.transpose(1, 2) for t in qkv.unbind(2))
    s = r(q @ k.transpose(2, 3) * (C // heads) ** -0.5, value=False).masked_fill(~mask[:, None, None, :], float("-inf"))
    prob = r(torch.softmax(s, 3), grad=False)
    out = r((prob @ v).transpose(1, 2).reshape(B, N, C))
    u = r(out @ p["proj.weight"].t() + p["proj.bias"], value=False)
    return r(residual + row_scale[:, None, None] * p["gamma_1"] * u, grad=False)


def _results(fn, x, residual, p, dout):
    leaves = {"x": x, **p}
    leaves = {n: t.detach().clone().requires_grad_(True) for n, t in leaves.items()}
    y = fn(leaves["x"], {n: t for n, t in leaves.items() if n != "x"})
    grads = torch.autograd.grad(y, list(leaves.values()), dout)
    return {"branch": (y - residual).detach(), **dict(zip(leaves, grads))}


def _misses(got, want, tol):
    return [n for n in want if not float((got[n].detach().cpu().double() - want[n]).norm()) <= tol[n]]


def _case(monkeypatch=None):
    torch.manual_seed(3)
    M, heads, B, N = 128, 4, 5, 40
    lay = MultiwayTransformerEnocderLayer(M, "quick_gelu", heads, 2 * M, (24, 16), 0.4, layer_scale_init_values=1.0)
    with torch.no_grad():
        for n, t in lay.attn.named_parameters():
            torch.nn.init.normal_(t, std=0.1 if t.dim() > 1 else 0.3)
        lay.gamma_1.copy_(torch.randn(M))
    lay = lay.to(BF16).train()
    h, dout = torch.randn(B, N, M).to(BF16), torch.randn(B, N, M).to(BF16)
    mask = torch.arange(N)[None] < torch.tensor([40, 23, 1, 39, 12])[:, None]
    row_scale = torch.tensor([0.0, 1 / 0.6, 1 / 0.6, 1 / 0.6, 1 / 0.6]).to(BF16)
    return lay, heads, h, dout, mask, row_scale


def _expected(lay, heads, x, h, dout, mask, row_scale):
    """-> (value of each result in 64 bits, tolerance of its norm): three times the largest miss of 8 evaluations with drawn errors,
    and half a step of the stored result."""
    p = {n: t.detach().cpu().double() for n, t in lay.attn.named_parameters()}
    p["gamma_1"] = lay.gamma_1.detach().cpu().double()
    x, h, dout, row_scale = (t.detach().cpu().double() for t in (x, h, dout, row_scale))
    want = _results(lambda a, q: _branch64(a, h, q, heads, mask, row_scale), x, h, p, dout)
    tol = {n: 0.0 for n in want}
    for seed in range(8):
        g = torch.Generator().manual_seed(seed)
        drawn = _results(lambda a, q: _branch64(a, h, q, heads, mask, row_scale, g), x, h, p, dout)
        tol = {n: max(t, float((drawn[n] - want[n]).norm())) for n, t in tol.items()}
    return want, {n: 3 * t + U * float(want[n].norm()) for n, t in tol.items()}


def test_the_bound_sees_a_branch_that_is_missing_or_wrong():
    lay, heads, h, dout, mask, row_scale = _case()
    x = torch.nn.functional.layer_norm(h.double(), (h.shape[2],)).to(BF16)
    want, tol = _expected(lay, heads, x, h, dout, mask, row_scale)
    zero = {n: torch.zeros_like(t) for n, t in want.items()}
    assert set(_misses(zero, want, tol)) == set(want)
    for other in (_expected(lay, heads, x, h, dout, torch.ones_like(mask), row_scale)[0], _expected(lay, 2, x, h, dout, mask, row_scale)[0]):
        # (not v_bias: probabilities sum to one, so its gradient is the same whatever they are)
        assert {"branch", "x", "qkv.weight", "q_bias", "proj.weight", "gamma_1"} <= set(_misses(other, want, tol))


@pytest.mark.gpu
@pytest.mark.parametrize("impl", ["fused", "stock"])
def test_bf16_branch_and_its_gradients(impl, monkeypatch):
    lay, heads, h, dout, mask, row_scale = _case()
    lay = lay.to(DEV)
    lay.set_attention(impl)
    x = enc.layer_norm(lay.norm1, h.to(DEV)).detach()
    monkeypatch.setattr(lay, "_drop_path_scale", lambda t: row_scale.to(DEV))
    leaf = x.clone().requires_grad_(True)
    monkeypatch.setattr(enc, "layer_norm", lambda mod, t: leaf)  # the branch behind its normalisation
    y = lay._attention_branch(h.to(DEV), mask.to(DEV), None)
    params = {n: t for n, t in lay.attn.named_parameters()}
    params["gamma_1"] = lay.gamma_1
    grads = torch.autograd.grad(y, [leaf, *params.values()], dout.to(DEV))
    got = {"branch": y.detach().cpu().double() - h.double(), "x": grads[0], **dict(zip(params, grads[1:]))}
    want, tol = _expected(lay, heads, x, h, dout, mask, row_scale)
    ratios = {n: float((got[n].detach().cpu().double() - want[n]).norm()) / tol[n] for n in want}
    if impl == "fused":
        assert not _misses(got, want, tol), ratios
    else:  # the same bound with room for what the stock operations round beside it: u before gamma, its gradient, the biases' sums
        assert all(r <= 2 for r in ratios.values()), ratios


@pytest.mark.gpu
def test_an_encoder_with_a_moe_layer_repeats_itself_in_bf16():
    """Three bf16 layers, the last of them MoE with its noise given, fused attention: finite, every parameter reached by a gradient,
    and a second run gives the same bits."""
    torch.manual_seed(5)
    param = {"num_experts": 4, "topk": 2, "type_route": True}
    e = MultiwayTransformerEncoder(128, "quick_gelu", 4, 256, 3, (20, 12), 0.0, ffn_layers=[2], ffn_param=param).to(DEV).bfloat16()
    for lay in e.layers:
        lay.set_attention("fused")
        assert lay.attn.impl == "fused"
    h = torch.randn(4, 32, 128, device=DEV, dtype=BF16)
    mask = torch.arange(32, device=DEV)[None] < torch.tensor([32, 25, 21, 30], device=DEV)[:, None]
    noise = -torch.log(-torch.log(torch.rand(128, 4, device=DEV).clamp(1e-6, 1 - 1e-6)))
    runs = []
    for _ in range(2):
        e.layers[2].mlp_moe.moe.noise_override = noise  # taken by one call
        e.zero_grad()
        x = h.clone().requires_grad_(True)
        out = e(x, mask)
        (out.float().square().mean() + 0.01 * e.gate_loss()).backward()
        runs.append([out.detach(), x.grad] + [t.grad.clone() for n, t in e.layers[0].attn.named_parameters()])
    assert all(bool(torch.isfinite(t).all()) and float(t.abs().sum()) > 0 for t in runs[0])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
