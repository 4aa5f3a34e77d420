"""eve_amd.fused_linear against its formula in 64 bits, with tolerances derived from the roundings made."""
import pytest
import torch

import eve_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: 2.0 ** -8, F32: 2.0 ** -24}  # half a step of a rounding, relative
W = 2.0 ** -24


def _act64(z, act):
    """act(z), act'(z), max |act''| (bounds what an error of z does to act') in 64 bits."""
    if act == "quick_gelu":
        s = torch.sigmoid(1.702 * z)
        return z * s, s * (1 + 1.702 * z * (1 - s)), 0.86
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5, 0.8
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    return z, torch.ones_like(z), 0.0


def reference(p, act, dout=None):
    """{name: (value, tolerance)}.  With u = half a step of the type, w = 2^-24:
      z      a K-term fp32 sum: K w sum|x||w|, + w |z| for the bias;   act is 1.13-Lipschitz at most (quick_gelu, gelu), and its
             value is evaluated to 16 w (|z| + 1) (fp32 exp, erf and reciprocal, a few steps each), 64 w for the fast forms of bf16;
      y      that, times gamma row_scale, + 4 w of the terms, + u |y| stored;
      slope  from the z that is kept, rounded by u |z|: max|act''| (tol z + u |z|), + 64 w;  relu: exact where z keeps its sign;
      du, dz products of those, dz rounded once more by u;
      dx, dw, dbias, dgamma: sums of such terms, + n w of the terms' sizes for the order, + u of the result stored."""
    u = U[p["x"].dtype]
    t = {k: (None if v is None else v.detach().cpu().double()) for k, v in p.items()}
    N, K = t["w"].shape
    x = t["x"].reshape(-1, K)
    rows = x.shape[0]
    z = x @ t["w"].t()
    t_z = K * W * (x.abs() @ t["w"].abs().t())
    if t["b"] is not None:
        z = z + t["b"]
    t_z = t_z + W * z.abs()
    a, slope, curve = _act64(z, act)
    few = 64 * W * (z.abs() + 1) if act in ("quick_gelu", "gelu") else torch.zeros_like(z)
    t_a = 1.13 * t_z + few
    g = torch.ones(N, dtype=torch.float64) if t["gamma"] is None else t["gamma"]
    rs = torch.ones(rows, 1, dtype=torch.float64)
    if t["row_scale"] is not None:
        rs = t["row_scale"].repeat_interleave(rows // len(t["row_scale"]))[:, None]
    f = g * rs
    y = a * f
    t_y = t_a * f.abs() + 4 * W * y.abs()
    if t["residual"] is not None:
        r = t["residual"].reshape(rows, N)
        y = y + r
        t_y = t_y + 2 * W * r.abs()
    t_y = t_y + u * y.abs()
    out = {"y": (y, t_y)}
    if dout is None:
        return out
    dy = dout.detach().cpu().double().reshape(rows, N)
    keep = t_z + u * z.abs()  # the kept z's error
    t_slope = curve * keep + few
    if act == "relu":
        t_slope = (z.abs() <= t_z).double()
    dz = dy * f * slope
    t_dz = (dy * f).abs() * t_slope + 4 * W * dz.abs() + u * dz.abs()
    out["x"] = (dz @ t["w"], (t_dz + N * W * dz.abs()) @ t["w"].abs())
    out["w"] = (dz.t() @ x, (t_dz + rows * W * dz.abs()).t() @ x.abs())
    out["b"] = (dz.sum(0), (t_dz + rows * W * dz.abs()).sum(0))
    du = dy * rs
    out["gamma"] = ((du * a).sum(0), (du.abs() * (1.13 * keep + few) + (rows + 4) * W * (du * a).abs()).sum(0))
    for n in ("x", "w", "b", "gamma"):
        out[n] = (out[n][0], out[n][1] + u * out[n][0].abs())
    out["residual"] = (dy, torch.zeros_like(dy))
    return out


def assert_within(got, ref, what):
    for n, t in got.items():
        val, tol = ref[n]
        t = t.detach().cpu().double().reshape(val.shape)
        bad = ~((t - val).abs() <= 1.02 * tol + 1e-37)
        if bool(bad.any()):
            i = int(bad.flatten().nonzero()[0])
            raise AssertionError(f"{what}: {n}: {int(bad.sum())} of {bad.numel()} outside the bound; element {i}: "
                                 f"{float(t.flatten()[i]):.9g} for {float(val.flatten()[i]):.9g} +- {float(tol.flatten()[i]):.3g}")


def make(B, T, K, N, dtype, seed, bias=True, gamma=True, scale=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, m=1.0: (torch.randn(*s, generator=g) * m).to(dtype).to(DEV)
    p = {"x": r(B, T, K), "w": r(N, K, m=K ** -0.5), "b": r(N, m=0.3) if bias else None, "gamma": r(N) if gamma else None,
         "row_scale": None, "residual": r(B, T, N) if residual else None}
    if scale:
        p["row_scale"] = ((torch.rand(B, generator=g) < 0.7).float() / 0.7).to(dtype).to(DEV)
    return p, r(B, T, N)


def call(p, act):
    return eve_amd.fused_linear(p["x"], p["w"], p["b"], activation=act, gamma=p["gamma"], row_scale=p["row_scale"], residual=p["residual"])


def step(p, act, dout):
    names = [n for n in ("x", "w", "b", "gamma", "residual") if p[n] is not None]
    q = {n: (t.detach().requires_grad_(True) if n in names else t) for n, t in p.items()}
    y = call(q, act)
    return {"y": y, **dict(zip(names, torch.autograd.grad(y, [q[n] for n in names], dout)))}


SIZES = [(1, 1, 8, 8), (1, 2, 64, 5), (3, 1, 100, 33), (2, 3, 768, 130), (1, 8, 33, 1), (1, 9, 64, 64), (2, 20, 48, 72), (3, 43, 129, 127),
         (2, 128, 128, 128), (4, 65, 200, 257), (5, 60, 1, 3), (2, 300, 264, 136), (16, 300, 40, 24)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["identity", "quick_gelu", "gelu", "relu"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(size, act, dtype):
    p, dout = make(*size, dtype, seed=sum(size))
    ref = reference(p, act, dout)
    with torch.no_grad():
        assert_within({"y": call(p, act)}, ref, "without gradient")
    assert_within(step(p, act, dout), ref, "with gradient")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("parts", range(16))
def test_every_set_of_parts(parts, dtype):
    kw = {n: bool(parts >> i & 1) for i, n in enumerate(("bias", "gamma", "scale", "residual"))}
    for size, act in (((2, 3, 40, 24), "identity"), ((2, 70, 40, 136), "quick_gelu")):
        p, dout = make(*size, dtype, seed=parts, **kw)
        assert_within(step(p, act, dout), reference(p, act, dout), f"{kw}")


def test_large_products_of_the_encoder():
    for K, N, gamma in ((768, 2304, False), (768, 768, True)):
        p, dout = make(8, 237, K, N, BF16, seed=K + N, gamma=gamma, scale=gamma, residual=gamma)
        assert_within(step(p, "identity", dout), reference(p, "identity", dout), f"{K}x{N}")


@pytest.mark.parametrize("wants", [("x",), ("w",), ("b",), ("gamma",), ("residual",), ("w", "gamma"), ("x", "b")])
def test_only_the_gradients_asked_for(wants):
    p, dout = make(2, 40, 64, 72, BF16, seed=3)
    full = step(p, "gelu", dout)
    q = {n: (t.detach().requires_grad_(n in wants) if t is not None else None) for n, t in p.items()}
    y = call(q, "gelu")
    assert torch.equal(y, full["y"])
    for n, g in zip(wants, torch.autograd.grad(y, [q[n] for n in wants], dout)):
        assert torch.equal(g, full[n]), n


def test_strides_and_starts():
    p, dout = make(2, 50, 72, 40, BF16, seed=4)
    want = step(p, "identity", dout)
    q = dict(p)
    q["x"] = p["x"].transpose(0, 1).contiguous().transpose(0, 1)
    q["w"] = p["w"].t().contiguous().t()
    q["residual"] = torch.cat([p["residual"].flatten()[:1], p["residual"].flatten()])[1:].view(p["residual"].shape)  # 2-byte aligned
    q["b"] = torch.cat([p["b"][:1], p["b"]])[1:]
    q["gamma"] = p["gamma"].repeat_interleave(2)[::2]
    got = step(q, "identity", dout.transpose(1, 2).contiguous().transpose(1, 2))
    for n in want:
        assert torch.equal(got[n], want[n]), n
    x2 = p["x"].reshape(100, 72)
    assert torch.equal(eve_amd.fused_linear(x2, p["w"], p["b"]), eve_amd.fused_linear(p["x"], p["w"], p["b"]).reshape(100, 40))
    assert eve_amd.fused_linear(p["x"][0, 0], p["w"]).shape == (40,)


@pytest.mark.parametrize("B,T,K,N", [(0, 3, 8, 8), (2, 3, 0, 8), (2, 3, 8, 0), (2, 0, 8, 8)])
@pytest.mark.parametrize("act", ["identity", "gelu"])
def test_empty_sizes(B, T, K, N, act):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)
    p = {"x": r(B, T, K), "w": r(N, K), "b": r(N), "gamma": r(N), "row_scale": r(B), "residual": r(B, T, N)}
    got = step(p, act, r(B, T, N))
    for n in ("x", "w", "b", "gamma", "residual"):
        assert got[n].shape == p[n].shape
        if n in ("x", "w") or not B * T:
            assert n == "residual" or float(got[n].abs().sum()) == 0.0
    if K == 0:
        z = p["b"].double().cpu()
        a = z if act == "identity" else torch.nn.functional.gelu(z)
        want = p["residual"].double().cpu() + p["row_scale"].double().cpu()[:, None, None] * p["gamma"].double().cpu() * a
        torch.testing.assert_close(got["y"].detach().cpu().double(), want, rtol=1e-5, atol=1e-5)


def test_nan_and_inf_stay_in_their_rows():
    p, _ = make(1, 70, 100, 40, F32, seed=6)
    p["x"][0, 13, 99] = float("nan")
    p["x"][0, 14, 0] = float("inf")
    y = call(p, "identity")
    rows = (~torch.isfinite(y)).any(2)[0].nonzero()[:, 0].tolist()
    assert rows == [13, 14] if float(p["row_scale"][0]) else True


def test_gradient_against_differences():
    p, dout = make(2, 7, 24, 20, F32, seed=7)
    for act in ("quick_gelu", "gelu"):
        got, ref = step(p, act, dout), reference(p, act, dout)
        g = torch.Generator().manual_seed(8)
        for n in ("x", "w", "b", "gamma", "residual"):
            d = torch.randn(p[n].shape, generator=g, dtype=torch.float64)
            e, loss = 1e-5, []
            for sign in (1, -1):
                q = {k: (None if v is None else v.detach().cpu().double()) for k, v in p.items()}
                q[n] = q[n] + sign * e * d
                z = q["x"] @ q["w"].t() + q["b"]
                y = q["residual"] + q["row_scale"][:, None, None] * q["gamma"] * _act64(z, act)[0]
                loss.append(float((y * dout.cpu().double()).sum()))
            diff = (loss[0] - loss[1]) / (2 * e)
            tol = float((ref[n][1].reshape(d.shape) * d.abs()).sum()) + 1e-6  # e^2 third derivatives, and 1e-16 / e of the losses
            assert abs(float((got[n].cpu().double() * d).sum()) - diff) <= tol, (act, n)


def test_other_stream_repeats_and_replays_are_bit_equal():
    p, dout = make(3, 200, 136, 264, BF16, seed=9)
    want = step(p, "quick_gelu", dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(p, "quick_gelu", dout)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[n], got[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(p, "quick_gelu", dout)
    x0 = p["x"].clone()
    for i in range(3):
        p["x"].copy_(x0 * (1 + 0.25 * i))
        graph.replay()
        eager = step(p, "quick_gelu", dout)
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], eager[n]) for n in eager), i


# few tiles and a long contraction (5 to some hundred rows; unaligned rows, tails of the contraction, one column), then problems of
# enough tiles for the streaming kernels, their last rows, columns and contraction steps partly filled
LONG = [(1, 5, 1000, 70), (2, 8, 2056, 24), (2, 20, 2049, 515), (1, 200, 1024, 1000), (3, 70, 301, 333), (1, 6, 31, 1), (2, 400, 2000, 260)]
MANY = [(20, 400, 136, 520), (30, 500, 72, 1096), (9, 999, 200, 776)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", LONG + MANY, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["identity", "quick_gelu"])
def test_long_contractions_and_many_tiles(size, act, dtype):
    p, dout = make(*size, dtype, seed=sum(size) + 1)
    ref = reference(p, act, dout)
    with torch.no_grad():
        assert_within({"y": call(p, act)}, ref, "without gradient")
    assert_within(step(p, act, dout), ref, "with gradient")
