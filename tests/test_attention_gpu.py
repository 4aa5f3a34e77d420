"""eve_amd.attention / self_attention against attention in 64 bits, with tolerances derived from the roundings made."""
import pytest
import torch

import eve_amd
from tests.attn_reference import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def _make(B, Nq, Nk, H, Hkv, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    shapes = ((B, Nq, H, D), (B, Nk, Hkv, D), (B, Nk, Hkv, D), (B, Nq, H, D))
    return [(torch.randn(*s, generator=g) * (std if i < 2 else 1.0)).to(dtype).to(DEV) for i, s in enumerate(shapes)]


def _mask(kind, B, Nk, seed):
    g = torch.Generator().manual_seed(seed + 1000)
    if kind == "none":
        return None
    if kind == "tail":
        n = torch.randint(0, Nk + 1, (B,), generator=g)
        return (torch.arange(Nk)[None] < n[:, None]).to(DEV)
    if kind == "head":  # the first keys are masked: a tile may begin, or be, without a visible key
        n = torch.randint(0, Nk + 1, (B,), generator=g)
        return (torch.arange(Nk)[None] >= n[:, None]).to(DEV)
    if kind == "holes":
        return (torch.rand(B, Nk, generator=g) > 0.5).to(DEV)
    if kind == "one":
        m = torch.zeros(B, Nk, dtype=torch.bool)
        m[torch.arange(B), torch.randint(0, Nk, (B,), generator=g)] = True
        return m.to(DEV)
    m = torch.rand(B, Nk, generator=g) > 0.3  # "empty": the first sample sees nothing
    m[0] = False
    return m.to(DEV)


CASES = [
    # B, Nq, Nk, H, Hkv, D, mask
    (1, 1, 1, 1, 1, 8, "none"),
    (2, 1, 1, 2, 1, 64, "empty"),
    (2, 31, 33, 3, 3, 64, "none"),
    (1, 32, 64, 2, 2, 64, "holes"),
    (2, 64, 128, 2, 2, 32, "tail"),
    (2, 65, 127, 2, 1, 40, "head"),
    (3, 129, 65, 4, 2, 72, "empty"),
    (2, 237, 237, 3, 3, 64, "tail"),
    (1, 200, 300, 6, 2, 128, "holes"),
    (2, 40, 40, 8, 1, 96, "tail"),
    (1, 7, 130, 6, 2, 120, "one"),
    (2, 3, 1000, 8, 2, 128, "holes"),   # few rows against many keys: split and joined
    (1, 1, 4099, 1, 1, 64, "head"),
    (1, 1, 2500, 5, 1, 16, "none"),
    (9, 129, 31, 8, 8, 24, "empty"),    # 72 heads: blocks dealt by XCD
    (1, 300, 1, 2, 2, 64, "none"),
    (1, 257, 513, 1, 1, 64, "holes"),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_forward_and_gradients(case, dtype):
    *dims, kind = case
    q, k, v, do = _make(*dims, dtype, seed=sum(dims), std=1.5)
    mask = _mask(kind, dims[0], dims[2], sum(dims))
    res = attention64(q, k, v, mask, dout=do)
    with torch.no_grad():
        assert_within({"out": eve_amd.attention(q, k, v, mask)}, res, "without gradient")
    for t in (q, k, v):
        t.requires_grad_(True)
    out = eve_amd.attention(q, k, v, mask)
    grads = torch.autograd.grad(out, (q, k, v), do)
    assert_within(dict(zip(("out", "dq", "dk", "dv"), (out, *grads))), res, "with gradient")


# heads enough, and keys few enough, for the backward that keeps a head in one workgroup
WHOLE = [(44, 33, 129, 3, 3, 64, "holes"), (33, 237, 237, 4, 4, 64, "tail"), (64, 65, 256, 4, 2, 40, "empty"), (32, 1, 140, 8, 4, 64, "none"),
         (130, 200, 250, 1, 1, 16, "head"), (43, 64, 160, 6, 3, 8, "one")]


@pytest.mark.parametrize("case", WHOLE, ids=lambda c: "x".join(map(str, c)))
def test_many_heads_of_few_keys(case):
    test_forward_and_gradients(case, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_product_and_its_gradient(dtype):
    B, N, H, D = 2, 77, 3, 64
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(B, N, 3, H, D, generator=g).to(dtype).to(DEV).requires_grad_(True)
    do = torch.randn(B, N, H, D, generator=g).to(dtype).to(DEV)
    mask = _mask("tail", B, N, 5)
    out = eve_amd.self_attention(qkv, mask)
    (dqkv,) = torch.autograd.grad(out, qkv, do)
    q, k, v = qkv.detach().unbind(2)
    res = attention64(q, k, v, mask, dout=do)
    assert_within(dict(zip(("out", "dq", "dk", "dv"), (out, *dqkv.unbind(2)))), res, "packed")
    # the same bits as from separate tensors: no atomics, one order
    parts = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out2 = eve_amd.attention(*parts, mask)
    assert torch.equal(out2, out)
    for a, b in zip(torch.autograd.grad(out2, parts, do), dqkv.unbind(2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides_offsets_and_expanded_inputs(dtype):
    B, Nq, Nk, H, Hkv, D = 2, 50, 70, 4, 2, 64
    q, k, v, do = _make(B, Nq, Nk, H, Hkv, D, dtype, 9)
    res = attention64(q, k, v, dout=do)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    wide = [torch.cat([t, t * float("nan")], 3)[..., :D] for t in (q, k, v)]
    odd = [torch.cat([t, t[..., :1]], 3)[..., :D] for t in (q, k, v)]               # rows off 16-byte boundaries: copied
    off = [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (q, k, v)]
    strided = [t.repeat_interleave(2, 3)[..., ::2] for t in (q, k, v)]
    for what, parts in (("heads first", heads_first), ("wide rows", wide), ("odd rows", odd), ("odd start", off), ("strided", strided)):
        parts = [t.detach().requires_grad_(True) for t in parts]
        out = eve_amd.attention(*parts)
        grads = torch.autograd.grad(out, parts, do.transpose(1, 2).contiguous().transpose(1, 2))
        assert_within(dict(zip(("out", "dq", "dk", "dv"), (out, *grads))), res, what)
    one = k[:1].expand(B, -1, -1, -1)  # a broadcast input: its gradient is summed over the samples by autograd
    assert_within({"out": eve_amd.attention(q, one, v)}, attention64(q, one, v), "expanded keys")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Nq", [(3, 2), (3, 100), (65, 100)])
def test_what_masked_places_hold_takes_no_part(dtype, B, Nq):
    Nk, H, D = 150, 2, 64
    q, k, v, do = _make(B, Nq, Nk, H, H, D, dtype, 11)
    mask = _mask("empty", B, Nk, 11)
    clean = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*clean, mask)
    grads = torch.autograd.grad(out, clean, do)
    gone = ~mask
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        dirty = [q.clone(), k.clone(), v.clone()]
        dirty[1][gone], dirty[2][gone] = bad, bad
        do2 = do.clone()
        do2[0] = bad  # the sample without a visible key passes no gradient, whatever arrives
        dirty[0][0] = bad
        dirty = [t.requires_grad_(True) for t in dirty]
        out2 = eve_amd.attention(*dirty, mask)
        grads2 = torch.autograd.grad(out2, dirty, do2)
        assert torch.equal(out2, out) and all(torch.equal(a, b) for a, b in zip(grads2, grads)), bad
    assert float(out[0].abs().max()) == 0.0 and float(grads[0][0].abs().max()) == 0.0
    assert float(grads[1][gone].abs().max()) == 0.0 and float(grads[2][gone].abs().max()) == 0.0


def test_large_scores_keep_their_order():
    """Scores far apart and far from zero: the running maximum decides, nothing overflows."""
    q, k, v, do = _make(1, 40, 200, 2, 2, 64, F32, 13, std=6.0)
    res = attention64(q, k, v, dout=do)
    parts = [t.requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*parts)
    assert_within(dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, parts, do)))), res, "large scores")
    same = eve_amd.attention(q.detach() * 0, k.detach(), v.detach())  # all scores equal: the mean of the values
    torch.testing.assert_close(same, v.detach().mean(1, keepdim=True).expand_as(same), rtol=1e-5, atol=1e-6)


def test_a_nan_in_a_visible_place_shows_where_it_belongs():
    q, k, v, _ = _make(2, 5, 70, 2, 2, 64, F32, 15)
    q[0, 1, 0, 3] = float("nan")
    out = eve_amd.attention(q, k, v)
    bad = torch.isnan(out).any(3)
    assert bool(bad[0, 1, 0]) and int(bad.sum()) == 1
    k[1, 69, 1, 0] = float("nan")
    bad = torch.isnan(eve_amd.attention(q, k, v)).any(3)
    assert bool(bad[1, :, 1].all()) and int(bad.sum()) == 6


@pytest.mark.parametrize("B,Nq,Nk", [(0, 4, 4), (2, 0, 4), (2, 4, 0)])
def test_empty_sizes(B, Nq, Nk):
    q, k, v, do = _make(B, Nq, Nk, 2, 2, 64, BF16, 17)
    parts = [t.requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*parts)
    assert out.shape == q.shape and float(out.abs().sum()) == 0.0
    for t, g in zip(parts, torch.autograd.grad(out, parts, do)):
        assert g.shape == t.shape and float(g.abs().sum()) == 0.0


def test_gradient_against_differences():
    """fp32, differences of the 64-bit loss along random directions against the kernels' gradient."""
    q, k, v, do = _make(1, 20, 45, 4, 2, 32, F32, 19)
    mask = _mask("holes", 1, 45, 19)
    parts = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(eve_amd.attention(*parts, mask), parts, do)
    g = torch.Generator().manual_seed(20)
    for i in range(3):
        d = torch.randn(parts[i].shape, generator=g, dtype=torch.float64)
        ts = [t.detach().cpu().double() for t in parts]
        e, loss = 1e-5, []
        for sign in (1, -1):
            moved = list(ts)
            moved[i] = ts[i] + sign * e * d
            loss.append(_loss64(moved, mask, do))
        diff = (loss[0] - loss[1]) / (2 * e)
        got = float((grads[i].double().cpu() * d).sum())
        # the kernel's error is at most its elements' tolerances; the difference's own is e^2 (third derivatives), here < 1e-6
        tol = float((attention64(q, k, v, mask, dout=do)[("dq", "dk", "dv")[i]][1] * d.abs()).sum()) + 1e-5
        assert abs(got - diff) <= tol, (i, got, diff, tol)


def _loss64(ts, mask, do):
    q, k, v = ts
    group = q.shape[2] // k.shape[2]
    s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(group, 2)) * q.shape[3] ** -0.5
    p = torch.softmax(s.masked_fill(~mask.cpu()[:, None, None], float("-inf")), 3)
    return float((torch.einsum("bhij,bjhd->bihd", p, v.repeat_interleave(group, 2)) * do.double().cpu()).sum())


def test_mask_types_and_scale():
    q, k, v, _ = _make(2, 9, 33, 2, 2, 64, BF16, 21)
    mask = _mask("holes", 2, 33, 21)
    want = eve_amd.attention(q, k, v, mask, scale=0.3)
    assert_within({"out": want}, attention64(q, k, v, mask, scale=0.3), "scale")
    for m in (mask.long(), mask.float(), mask.to(torch.uint8), mask.t().contiguous().t()):
        assert torch.equal(eve_amd.attention(q, k, v, m, scale=0.3), want)


def test_other_stream_and_repeated_calls_are_bit_equal():
    q, k, v, do = _make(2, 130, 200, 4, 2, 64, BF16, 23)
    mask = _mask("tail", 2, 200, 23)

    def step():
        parts = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = eve_amd.attention(*parts, mask)
        return (out, *torch.autograd.grad(out, parts, do))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    """Forward and backward in a graph, several replays with new inputs, each against the eager result."""
    for B, Nq, Nk in ((2, 1, 1500), (2, 90, 1500), (64, 100, 200)):
        q, k, v, do = _make(B, Nq, Nk, 4, 2, 64, BF16, 25)
        mask = _mask("holes", B, Nk, 25)
        parts = [t.clone().requires_grad_(True) for t in (q, k, v)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(eve_amd.attention(*parts, mask), parts, do)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = eve_amd.attention(*parts, mask)
            grads = torch.autograd.grad(out, parts, do)
        for i in range(3):
            with torch.no_grad():
                for t, s in zip(parts, (q, k, v)):
                    t.copy_(s * (1 + 0.1 * i))
                mask.logical_xor_(mask.roll(1, 1))
            graph.replay()
            eager = [t.detach().clone().requires_grad_(True) for t in parts]
            out2 = eve_amd.attention(*eager, mask)
            want = (out2, *torch.autograd.grad(out2, eager, do))
            torch.cuda.synchronize()
            for a, b in zip((out, *grads), want):
                assert torch.equal(a, b), (B, Nq, i)


def test_offsets_beyond_32_bits():
    """A key cache whose rows lie 2^26 elements apart: element offsets pass 2^31 and byte offsets 2^32."""
    Nk, step, D = 66, 1 << 26, 64
    store = torch.empty((Nk - 1) * step + 2 * D, dtype=BF16, device=DEV)
    view = torch.as_strided(store, (1, Nk, 2, 1, D), (0, step, D, D, 1))
    q, k, v, do = _make(1, 3, Nk, 2, 1, D, BF16, 27)
    view[:, :, 0], view[:, :, 1] = k, v
    parts = [q.requires_grad_(True), view[:, :, 0].detach().requires_grad_(True), view[:, :, 1].detach().requires_grad_(True)]
    out = eve_amd.attention(*parts)
    grads = torch.autograd.grad(out, parts, do)
    assert_within(dict(zip(("out", "dq", "dk", "dv"), (out, *grads))), attention64(q, k, v, dout=do), "far rows")


@pytest.mark.parametrize("packed", [False, True])
def test_gradient_that_starts_off_a_16_byte_boundary(packed):
    """The gradient of a result that was concatenated behind something else is a contiguous part of a larger tensor, wherever that
    starts; it gives what the same numbers give on a boundary."""
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(2, 19, 3, 2, 16, generator=g).to(torch.bfloat16).to(DEV).requires_grad_(True)
    dout = torch.randn(1 + 2 * 19 * 2 * 16, generator=g).to(torch.bfloat16).to(DEV)

    def out():
        return eve_amd.self_attention(qkv) if packed else eve_amd.attention(*qkv.unbind(2))

    want, = torch.autograd.grad(out(), qkv, dout[1:].clone().view(2, 19, 2, 16))
    joined = torch.cat((torch.zeros(1, dtype=torch.bfloat16, device=DEV), out().flatten()))
    got, = torch.autograd.grad(joined, qkv, dout)
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["tail", "head", "one"])
@pytest.mark.parametrize("Nk", [200, 256])
def test_whole_waves_of_masked_keys_hold_anything(kind, Nk):
    """Enough heads for the one-kernel backward, 32 keys and more masked in a row: NaN there gives the bits that zeros give."""
    B, Nq, H, D = 66, 70, 2, 64
    q, k, v, do = _make(B, Nq, Nk, H, H, D, BF16, 21)
    mask = _mask(kind, B, Nk, 21)
    results = []
    for bad in (0.0, float("nan")):
        parts = [q.clone(), k.masked_fill(~mask[:, :, None, None], bad), v.masked_fill(~mask[:, :, None, None], bad)]
        parts = [t.requires_grad_(True) for t in parts]
        out = eve_amd.attention(*parts, mask)
        results.append((out, *torch.autograd.grad(out, parts, do)))
    for name, a, b in zip(("out", "dq", "dk", "dv"), *results):
        assert torch.isfinite(b).all() and torch.equal(a, b), name
    assert_within(dict(zip(("out", "dq", "dk", "dv"), results[1])), attention64(q, k, v, mask, dout=do), kind)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rise", [0.02, 0.11, 0.3])
def test_scores_that_rise_from_key_to_key(dtype, rise):
    """The maximum moves on in every tile, by less, about and more than what makes a row rescale."""
    B, Nq, Nk, H, D = 1, 70, 700, 2, 64
    q, k, v, do = _make(B, Nq, Nk, H, H, D, dtype, 31, std=0.3)
    along = torch.ones(D, dtype=dtype, device=DEV)
    q = q + along
    k = k + (torch.arange(Nk, device=DEV)[:, None, None] * (rise / 8)).to(dtype) * along  # scale q . k grows by about `rise` a key
    res = attention64(q, k, v, dout=do)
    parts = [t.requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*parts)
    assert_within(dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, parts, do)))), res, f"rise {rise}")


def _few_key_gradients(q, k, v, do, mask, scale):
    """dq and dk in 64 bits and what bf16 may be off: ds rounded once by u = 2^-8, the result once more, and of ds itself, with
    w = 2^-24, 64 w (1 + max |score|) of its terms p |dp| and p |delta| (fp32 products of up to 128 terms, exponential, row sums)."""
    u, w = 2.0 ** -8, 2.0 ** -24
    q, k, v, do = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v, do))
    keep = mask.cpu()[:, None, None, :]
    s = (scale * q @ k.transpose(2, 3)).masked_fill(~keep, float("-inf"))
    p = torch.softmax(s, 3)
    dp = do @ v.transpose(2, 3)
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - delta)
    size = 64 * w * (1 + (scale * (q.abs() @ k.abs().transpose(2, 3)))) * p * (do.abs() @ v.abs().transpose(2, 3) + (p * dp.abs()).sum(3, keepdim=True))
    t_ds = u * ds.abs() + size
    dq, dk = scale * ds @ k, scale * ds.transpose(2, 3) @ q
    t_dq, t_dk = scale * t_ds @ k.abs() + u * dq.abs(), scale * t_ds.transpose(2, 3) @ q.abs() + u * dk.abs()
    return {n: t.transpose(1, 2) for n, t in (("dq", dq), ("dk", dk))}, {n: t.transpose(1, 2) for n, t in (("dq", t_dq), ("dk", t_dk))}


@pytest.mark.parametrize("D", [16, 64, 112])
@pytest.mark.parametrize("Nk", [1, 2, 3, 5, 17, 32])
@pytest.mark.parametrize("low", [False, True])
def test_gradients_of_a_few_keys_keep_their_digits(Nk, D, low):
    """Where keys are few, ds is what is left of nearly equal numbers: the rounding of the stored result must not enter it.  `low`:
    scores far below zero, next to masked keys (whose score would be zero)."""
    B, Nq, H = 3, 40, 2
    q, k, v, do = _make(B, Nq, Nk, H, H, D, BF16, 41 + Nk)
    if low:
        q, k = q - 4.0, k + 4.0
    mask = torch.ones(B, Nk, dtype=torch.bool, device=DEV)
    mask[0, Nk // 2 + 1:] = False
    parts = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = eve_amd.attention(*parts, mask)
    dq, dk, _ = torch.autograd.grad(out, parts, do)
    want, tol = _few_key_gradients(q, k, v, do, mask, D ** -0.5)
    for name, got in (("dq", dq), ("dk", dk)):
        err = (got.detach().cpu().double() - want[name]).abs()
        assert torch.isfinite(got).all() and bool((err <= 1.02 * tol[name] + 1e-30).all()), (name, float((err / (tol[name] + 1e-30)).max()))
