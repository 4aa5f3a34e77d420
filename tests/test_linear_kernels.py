"""Every kernel that csrc/linear.hip may choose for a product, against the formula in 64 bits, and products of more than 2^31
elements."""
import pytest
import torch

import eve_amd
from tests import linear_rules as rules
from tests.test_linear_gpu import BF16, DEV, F32, W, assert_within, call, make, reference, step

# (samples, rows of one, K, N): last tiles and last steps of the contraction partly filled
SIZES = [(20, 275, 776, 200), (9, 900, 200, 648), (9, 1000, 515, 777), (4, 100, 1544, 1608), (1, 260, 3200, 4096), (31, 269, 200, 1288),
         (4, 30, 1529, 1601), (3, 20, 1312, 1448), (33, 151, 1568, 136), (2, 400, 2000, 260), (2, 2, 300, 40)]


@pytest.mark.parametrize("size", [2, 4])
def test_the_sizes_reach_every_kernel(size):
    """By the rules for 256 CUs; the streamed forms of dW with its rows split and whole."""
    fwd = {rules.forward(B * T, K, N, size, 256) for B, T, K, N in SIZES}
    dx, dw = ({rules.backward(B * T, K, N, size, 256)[i] for B, T, K, N in SIZES} for i in range(2))
    assert fwd == {"few", "shared16", "shared32", "tile64", "tile128", "stream128", "stream192"}
    assert dx == {"tile64", "tile128", "stream128", "stream192"}
    assert dw >= {"tile64", "tile128", "tile128 split", "stream128", "stream128 split", "stream256", "stream256 split"}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["identity", "gelu", "relu"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(size, act, dtype):
    p, dout = make(*size, dtype, seed=sum(size) + 2)
    ref = reference(p, act, dout)
    with torch.no_grad():
        assert_within({"y": call(p, act)}, ref, "without gradient")
    assert_within(step(p, act, dout), ref, "with gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bias", [False, True])
def test_plain_products_whose_bias_is_summed_beside_dw(dtype, bias):
    """dz = dy: the streaming dW product sums dbias, over split rows and whole ones."""
    for size in ((9, 900, 200, 648), (4, 100, 1544, 1608)):
        p, dout = make(*size, dtype, seed=sum(size), bias=bias, gamma=False, scale=False, residual=False)
        assert_within(step(p, "identity", dout), reference(p, "identity", dout), f"{size}")


def _rows64(p, rows, act):
    """The formula in 64 bits at some rows of 2-dimensional operands, with the tolerance of tests/test_linear_gpu.py."""
    q = dict(p, x=p["x"][rows][None], residual=None if p["residual"] is None else p["residual"][rows][None])
    return reference(q, act)["y"]


@pytest.mark.gpu
@pytest.mark.parametrize("K,N", [(2056, 16), (8, 2056), (2051, 12), (8, 2051)])
def test_more_than_2_31_elements(K, N):
    """bf16, x or the result (with residual, kept z and gradient) of 1 060 000 rows: forward and dx at rows from the first to the
    last, dW and the column sums as 64-bit products on the GPU, rows in rounds."""
    rows, u = 1_060_000, 2.0 ** -8
    g = torch.Generator(device=DEV).manual_seed(K)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=BF16)
    p = {"x": r(rows, K), "w": r(N, K) * K ** -0.5, "b": r(N), "gamma": r(N), "row_scale": None, "residual": r(rows, N)}
    dout = r(rows, N)
    leaves = [p[n].requires_grad_(True) for n in ("x", "w", "b", "gamma")]
    y = eve_amd.fused_linear(p["x"], p["w"], p["b"], activation="relu", gamma=p["gamma"], residual=p["residual"])
    dx, dw, db, dg = torch.autograd.grad(y, leaves, dout)
    p = {n: None if t is None else t.detach() for n, t in p.items()}
    some = torch.cat([torch.arange(40), torch.arange(rows // 2, rows // 2 + 40), torch.arange(rows - 40, rows)]).to(DEV)
    val, tol = _rows64(p, some, "relu")
    assert bool(((y.detach()[some].cpu().double() - val).abs() <= 1.02 * tol).all())

    def dz_of(part):
        """dz in 64 bits and its error: a slope may be missed where z is within its own error of 0; z is kept in bf16."""
        x, dy = p["x"][part].double(), dout[part].double()
        z = x @ p["w"].double().t() + p["b"].double()
        t_z = K * W * (x.abs() @ p["w"].double().abs().t()) + W * z.abs()
        du = dy * p["gamma"].double()
        dz = du * (z > 0)
        return x, dy, z, dz, du.abs() * (z.abs() <= t_z) + (u + 4 * W) * dz.abs(), t_z

    _, _, _, dz, t_dz, _ = dz_of(some)
    w = p["w"].double()
    want = dz @ w
    tol = (t_dz + N * W * dz.abs()) @ w.abs() + u * want.abs()
    assert bool(((dx[some].double() - want).abs() <= 1.02 * tol).all())
    sums = {n: [0.0, 0.0] for n in ("w", "b", "g")}
    for part in torch.arange(rows, device=DEV).split(53_000):
        x, dy, z, dz, t_dz, t_z = dz_of(part)
        t_dz = t_dz + rows * W * dz.abs()
        a = z.clamp(min=0)
        for n, v, t in (("w", dz.t() @ x, t_dz.t() @ x.abs()), ("b", dz.sum(0), t_dz.sum(0)),
                        ("g", (dy * a).sum(0), (dy.abs() * (t_z + u * z.abs() + rows * W * a)).sum(0))):
            sums[n][0], sums[n][1] = sums[n][0] + v, sums[n][1] + t
    for n, got in (("w", dw), ("b", db), ("g", dg)):
        val, tol = sums[n]
        assert bool(((got.double() - val).abs() <= 1.02 * (tol + u * val.abs())).all()), n
