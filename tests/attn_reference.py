"""Attention in 64 bits, one sample and head at a time on the CPU, with what the kernels' roundings can add to each result."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step of a rounding, relative


def attention64(q, k, v, key_mask=None, scale=None, dout=None):
    """-> {name: (value, tolerance)} for out and, with dout, dq, dk, dv; q [B,Nq,H,D], k / v [B,Nk,Hkv,D] of the kernel's type.

    Tolerances, u = half a step of the type, w = 2^-24:
      s      a D-term sum in fp32 of exact products: off by D w sum|q||k| scale, and by 4 w |s| through scale, log2 e and L;
      p      relative 2 max|ds| (its own and the normaliser's) + (Nk + 8) w (a sum of Nk terms, exp2); then u where it enters the
             matrix unit as bf16 (fp32: none, counted as w);
      out    (rel p + u_p + Nk w) sum p|v|, and u |out| when stored;
      delta  from the stored out: sum|do| tol(out), + D w sum|do||out|;      dp: D w sum|do||v|
      ds     p (tol dp + tol delta) + rel p |p (dp - delta)|, and u |ds| at the matrix unit;
      dq, dk, dv: the sums of those, + N w of the terms' sizes, and u of the result when stored."""
    B, Nq, H, D = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    u, w = U[q.dtype], 2.0 ** -24
    G = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)
    res = {"out": (z(B, Nq, H, D), z(B, Nq, H, D))}
    if dout is not None:
        res.update({"dq": (z(B, Nq, H, D), z(B, Nq, H, D)), "dk": (z(B, Nk, Hkv, D), z(B, Nk, Hkv, D)),
                    "dv": (z(B, Nk, Hkv, D), z(B, Nk, Hkv, D))})
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    dout = None if dout is None else dout.detach().cpu().double()
    for b in range(B):
        seen = torch.arange(Nk) if key_mask is None else key_mask[b].detach().cpu().bool().nonzero()[:, 0]
        if not len(seen):
            continue
        for h in range(H):
            qq, kk, vv = q[b, :, h], k[b, seen, h // G], v[b, seen, h // G]
            s = scale * qq @ kk.t()
            p = torch.softmax(s, 1)
            e_s = D * w * scale * (qq.abs() @ kk.abs().t()) + 4 * w * (s.abs() + s.abs().amax(1, keepdim=True))
            rel = 2 * e_s.amax(1, keepdim=True) + (len(seen) + 8) * w
            o = p @ vv
            t_o = ((rel + u + len(seen) * w) * p) @ vv.abs() + u * o.abs()
            res["out"][0][b, :, h], res["out"][1][b, :, h] = o, t_o
            if dout is None:
                continue
            g = dout[b, :, h]
            delta = (g * o).sum(1, keepdim=True)
            t_delta = (g.abs() * t_o).sum(1, keepdim=True) + D * w * (g.abs() * o.abs()).sum(1, keepdim=True)
            dp = g @ vv.t()
            ds = p * (dp - delta)
            t_ds = p * (D * w * (g.abs() @ vv.abs().t()) + t_delta) + (rel + 2 * w) * ds.abs() + u * ds.abs()
            n = len(seen)
            dq = scale * ds @ kk
            res["dq"][0][b, :, h] = dq
            res["dq"][1][b, :, h] = scale * (t_ds + n * w * ds.abs()) @ kk.abs() + u * dq.abs()
            m = Nq * G
            dk, dv = scale * ds.t() @ qq, p.t() @ g
            res["dk"][0][b, seen, h // G] += dk
            res["dk"][1][b, seen, h // G] += scale * (t_ds + m * w * ds.abs()).t() @ qq.abs()
            res["dv"][0][b, seen, h // G] += dv
            res["dv"][1][b, seen, h // G] += ((rel + u + m * w) * p).t() @ g.abs()
    for n in ("dk", "dv"):
        if n in res:
            val, tol = res[n]
            tol += u * val.abs()
    return res


def assert_within(got, res, what):
    """Every element within its tolerance (times 1.02 for the products of the bounds themselves, and the smallest fp32 normal)."""
    for name, t in got.items():
        val, tol = res[name]
        t = t.detach().cpu().double()
        assert t.shape == val.shape, (what, name, tuple(t.shape), tuple(val.shape))
        bad = ~((t - val).abs() <= 1.02 * tol + 1e-37)
        if bool(bad.any()):
            i = int(bad.flatten().nonzero()[0])
            raise AssertionError(f"{what}: {name}: {int(bad.sum())} of {bad.numel()} outside the bound; element {i}: "
                                 f"{float(t.flatten()[i]):.9g} for {float(val.flatten()[i]):.9g} +- {float(tol.flatten()[i]):.3g}")
