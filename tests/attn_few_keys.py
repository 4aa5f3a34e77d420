"""Gradients of attention in 64 bits with what may be off where the rounding of the stored result does not enter delta."""
import torch


def few_key_gradients(q, k, v, do, mask, scale):
    """{name: (value, tolerance)} of dq and dk for equally many heads; mask [B, Nk] or None.  With u = 2^-8 and w = 2^-24: ds is
    rounded once (u |ds|) and is off by 64 w (1 + |score|) of its terms p |dp| and p |delta| (fp32 products of up to 128 terms,
    the exponential, row sums); the result is rounded once more."""
    u, w = 2.0 ** -8, 2.0 ** -24
    q, k, v, do = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v, do))
    s = scale * q @ k.transpose(2, 3)
    if mask is not None:
        s = s.masked_fill(~mask.cpu()[:, None, None, :], float("-inf"))
    p = torch.softmax(s, 3)
    dp = do @ v.transpose(2, 3)
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - delta)
    terms = p * (do.abs() @ v.abs().transpose(2, 3) + (p * dp.abs()).sum(3, keepdim=True))
    t_ds = u * ds.abs() + 64 * w * (1 + scale * (q.abs() @ k.abs().transpose(2, 3))) * terms
    dq, dk = scale * ds @ k, scale * ds.transpose(2, 3) @ q
    t_dq, t_dk = scale * t_ds @ k.abs() + u * dq.abs(), scale * t_ds.transpose(2, 3) @ q.abs() + u * dk.abs()
    return {"dq": (dq.transpose(1, 2), t_dq.transpose(1, 2)), "dk": (dk.transpose(1, 2), t_dk.transpose(1, 2))}
