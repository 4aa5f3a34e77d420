"""Cases that measure the attention block of the encoder layer: attention with its gradient, and the matrix product whose
epilogue adds the bias, applies the activation and adds the scaled result to a residual, with its gradient.

`run` computes them in plain torch operations where `own` is false and through eve_amd's entry points where it is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------------------- cases
def _attend(name, B, Nq, Nk, H, Hkv, D, dtype="bf16", train=False, packed=False, pad=0.0, empty=0):
    return {"name": name, "op": "attend", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hkv": Hkv, "D": D, "dtype": dtype, "train": train,
            "packed": packed, "pad": pad, "empty": empty}


def _linear(name, B, T, K, N, dtype="bf16", train=False, act="identity", bias=True, branch=False, drop=0.0):
    return {"name": name, "op": "linear", "B": B, "T": T, "K": K, "N": N, "dtype": dtype, "train": train, "act": act, "bias": bias,
            "branch": branch, "drop": drop}


def listed():
    return [
        # one text of 40 tokens through the text tower (the smallest call: latency)
        _attend("attend text tower", 1, 40, 40, 12, 12, 64, packed=True),
        # a batch of texts and images of a larger resolution (577 patches + 40 words) in evaluation, padded texts
        _attend("attend rerank batch", 64, 617, 617, 12, 12, 64, packed=True, pad=0.06),
        # one query a sample over a long list of keys whose heads are shared by four query heads each
        _attend("attend one query, long keys", 4, 1, 16384, 16, 4, 128),
        # the training step of the encoder: 64 samples of 197 patches + 40 words, padded texts
        _attend("attend train encoder", 64, 237, 237, 12, 12, 64, train=True, packed=True, pad=0.16),
        # a long sequence (a document, an image of many patches)
        _attend("attend train long", 2, 4096, 4096, 16, 16, 64, train=True),
        # odd length, wide heads shared by four, ragged batch with an item that has no visible key
        _attend("attend train shared heads", 3, 1001, 1001, 16, 4, 128, train=True, pad=0.9, empty=1),
        # other queries than keys, a head width between the tiles, in float32
        _attend("attend train f32", 4, 129, 333, 6, 6, 40, dtype="f32", train=True, pad=0.5),
        # the qkv product for one token
        _linear("linear one token", 1, 1, 768, 2304),
        # a feed-forward product of the larger encoder over a rerank batch: activation, layer scale and residual
        _linear("linear rerank batch", 64, 617, 1024, 4096, act="quick_gelu", branch=True),
        # the qkv product of the training step
        _linear("linear train qkv", 64, 237, 768, 2304, train=True),
        # the output product of the training step: bias, layer scale, DropPath and the residual
        _linear("linear train branch", 64, 237, 768, 768, train=True, branch=True, drop=0.1),
        # odd sizes in float32 with an activation
        _linear("linear train f32 odd", 9, 211, 750, 1001, dtype="f32", train=True, act="gelu", branch=True, drop=0.2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """One more case: lengths and widths over the listed ones' ranges, no larger than the largest of them."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        dtype = "bf16" if rng.random() < 0.75 else "f32"
        train = rng.random() < 0.6
        if rng.random() < 0.5:
            D = 8 * rng.randint(2, 16)
            group = rng.choice([1, 1, 2, 3, 4, 8])
            Hkv = rng.randint(1, 16 // group)
            packed = group == 1 and rng.random() < 0.5
            few = rng.random() < 0.3
            Nk = _log(rng, 1, 30000 if few else 4096)
            Nq = Nk if packed else (rng.randint(1, 4) if few else _log(rng, 1, 4096))
            c = _attend("", _log(rng, 1, 64), Nq, Nk, Hkv * group, Hkv, D, dtype, train, packed, rng.choice([0.0, 0.1, 0.5, 1.0]), 0)
            c["empty"] = 1 if c["B"] > 1 and c["pad"] and rng.random() < 0.3 else 0
            scores = c["B"] * c["H"] * Nq * Nk
            if scores > 2 * 16 * 4096 * 4096:
                continue
        else:
            step = rng.choice([1, 8, 8, 64])
            K, N = (step * max(1, _log(rng, 16, 4096) // step) for _ in range(2))
            branch = rng.random() < 0.5
            c = _linear("", _log(rng, 1, 64), _log(rng, 1, 617), K, N, dtype, train, rng.choice(["identity", "identity", "quick_gelu", "gelu", "relu"]),
                        rng.random() < 0.8, branch, rng.choice([0.0, 0.1]) if branch else 0.0)
        w = work(c)
        if w["flops"] > (most["flops"] if dtype == "bf16" else most["flops"] / 16) or w["bytes"] > most["bytes"]:
            continue
        c.pop("name")
        return c


def work(case):
    c = case
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] == "attend":
        seen = (1.0 - c["empty"] / c["B"]) * (1.0 - c["pad"] / 2)  # the share of the keys that the mask leaves
        q = c["B"] * c["Nq"] * c["H"] * c["D"] * size
        kv = 2 * c["B"] * c["Nk"] * c["Hkv"] * c["D"] * size
        mask = c["B"] * c["Nk"] if c["pad"] or c["empty"] else 0
        product = 2 * c["B"] * c["H"] * c["Nq"] * c["Nk"] * c["D"] * seen
        if not c["train"]:
            return {"bytes": int(2 * q + kv * seen + mask), "flops": int(2 * product)}
        # forward and backward: q, k, v, out's gradient read, out and the three gradients written; seven products
        return {"bytes": int(4 * q + kv * seen + kv + mask), "flops": int(7 * product)}
    rows = c["B"] * c["T"]
    x, y, w = rows * c["K"] * size, rows * c["N"] * size, c["K"] * c["N"] * size
    vectors = (int(c["bias"]) + int(c["branch"])) * c["N"] * size
    product = 2 * rows * c["K"] * c["N"]
    if not c["train"]:
        return {"bytes": x + w + y * (2 if c["branch"] else 1) + vectors, "flops": product}
    # x, the weight, the residual and the output's gradient read; the output and the gradients written
    return {"bytes": 2 * x + 2 * w + 2 * vectors + y * (3 if c["branch"] else 2), "flops": 3 * product}


# ------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    dt = DTYPES[c["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    s = {"case": c}
    if c["op"] == "attend":
        B, Nq, Nk, H, Hkv, D = (c[k] for k in ("B", "Nq", "Nk", "H", "Hkv", "D"))
        if c["packed"]:
            s["qkv"] = normal(B, Nk, 3, H, D)
        else:
            s["q"], s["k"], s["v"] = normal(B, Nq, H, D, std=1.5), normal(B, Nk, Hkv, D), normal(B, Nk, Hkv, D)
        s["mask"] = None
        if c["pad"] or c["empty"]:  # the last keys of each sample are padding
            lengths = Nk - torch.floor(torch.rand(B, generator=g, device="cuda") * c["pad"] * Nk).long()
            lengths[:c["empty"]] = 0
            s["mask"] = torch.arange(Nk, device="cuda")[None, :] < lengths[:, None]
        if c["train"]:
            s["dout"] = normal(B, Nq, H, D)
            for k in ("q", "k", "v", "qkv"):
                if k in s:
                    s[k].requires_grad_(True)
    else:
        B, T, K, N = (c[k] for k in ("B", "T", "K", "N"))
        s["x"], s["w"] = normal(B, T, K), normal(N, K, std=K ** -0.5)
        s["b"] = normal(N, std=0.2) if c["bias"] else None
        s["gamma"] = (normal(N, std=0.05) + 0.1) if c["branch"] else None
        s["residual"] = normal(B, T, N) if c["branch"] else None
        s["row_scale"] = None
        if c["drop"]:
            s["row_scale"] = ((torch.rand(B, generator=g, device="cuda") >= c["drop"]) / (1.0 - c["drop"])).to(dt)
        if c["train"]:
            s["dout"] = normal(B, T, N)
            for k in ("x", "w", "b", "gamma", "residual"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------- a pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _own_attend(s, c) if c["op"] == "attend" else _own_linear(s, c)
    with torch.no_grad():
        return _plain_attend(s, c) if c["op"] == "attend" else _plain_linear(s, c)


def _own_attend(s, c):
    import eve_amd

    with torch.set_grad_enabled(c["train"]):
        if c["packed"]:
            leaves = (s["qkv"],)
            out = eve_amd.self_attention(s["qkv"], key_mask=s["mask"])
        else:
            leaves = (s["q"], s["k"], s["v"])
            out = eve_amd.attention(*leaves, key_mask=s["mask"])
    if not c["train"]:
        return out
    return (out.detach(),) + torch.autograd.grad(out, leaves, s["dout"])


def _own_linear(s, c):
    import eve_amd

    with torch.set_grad_enabled(c["train"]):
        out = eve_amd.fused_linear(s["x"], s["w"], s["b"], activation=c["act"], gamma=s["gamma"], row_scale=s["row_scale"],
                                   residual=s["residual"])
    if not c["train"]:
        return out
    leaves = [s[k] for k in ("x", "w", "b", "gamma", "residual") if s[k] is not None]
    return (out.detach(),) + torch.autograd.grad(out, leaves, s["dout"])


def _heads_first(t, group=1):
    """[B, N, H, D] -> [B, H * group, N, D] in float32, each head `group` times."""
    t = t.detach().float().transpose(1, 2)
    return (t.repeat_interleave(group, 1) if group > 1 else t).contiguous()


def _plain_attend(s, c):
    dt, group, scale = DTYPES[c["dtype"]], c["H"] // c["Hkv"], c["D"] ** -0.5
    q, k, v = s["qkv"].detach().unbind(2) if c["packed"] else (s["q"], s["k"], s["v"])
    q, k, v = _heads_first(q), _heads_first(k, group), _heads_first(v, group)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale)
    if s["mask"] is None:
        p = torch.exp(scores - scores.amax(3, keepdim=True))
    else:
        keep = s["mask"][:, None, None, :]
        scores.masked_fill_(~keep, torch.finfo(torch.float32).min)
        p = torch.exp(scores - scores.amax(3, keepdim=True)) * keep
    del scores
    p /= p.sum(3, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    out = torch.matmul(p, v)
    answer = out.transpose(1, 2).to(dt).contiguous()
    if not c["train"]:
        return answer
    dout = _heads_first(s["dout"])
    ds = torch.matmul(dout, v.transpose(2, 3).contiguous())
    ds -= (dout * out).sum(3, keepdim=True)
    ds *= p
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    B, Nk, Hkv, D = (c[n] for n in ("B", "Nk", "Hkv", "D"))
    dk, dv = (t.reshape(B, Hkv, group, Nk, D).sum(2) for t in (dk, dv))
    grads = [t.transpose(1, 2) for t in (dq, dk, dv)]
    if c["packed"]:
        return answer, torch.stack(grads, 2).to(dt)
    return (answer,) + tuple(t.to(dt).contiguous() for t in grads)


def _activation(z, act):
    """act(z) and its derivative."""
    if act == "quick_gelu":
        g = torch.sigmoid(1.702 * z)
        return z * g, g * (1 + 1.702 * z * (1 - g))
    if act == "gelu":
        half = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * half, half + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    return z, None


def _plain_linear(s, c):
    dt, rows = DTYPES[c["dtype"]], c["B"] * c["T"]
    x, w = s["x"].detach().float().reshape(rows, c["K"]), s["w"].detach().float()
    z = torch.matmul(x, w.t())
    if c["bias"]:
        z += s["b"].float()
    u, slope = _activation(z, c["act"])
    scale = None
    if c["branch"]:
        scale = s["gamma"].detach().float()[None, :]
        rs = None
        if c["drop"]:
            rs = s["row_scale"].float().repeat_interleave(c["T"])[:, None]
            scale = scale * rs
        y = s["residual"].detach().float().reshape(rows, c["N"]) + u * scale
    else:
        y = u
    answer = y.to(dt).reshape(c["B"], c["T"], c["N"])
    if not c["train"]:
        return answer
    dy = s["dout"].float().reshape(rows, c["N"])
    dz = dy if scale is None else dy * scale
    if slope is not None:
        dz = dz * slope
    grads = [torch.matmul(dz, w).to(dt).reshape(c["B"], c["T"], c["K"]), torch.matmul(dz.t(), x).to(dt)]
    if c["bias"]:
        grads.append(dz.sum(0).to(dt))
    if c["branch"]:
        grads.append(((dy if rs is None else dy * rs) * u).sum(0).to(dt))
        grads.append(s["dout"])
    return (answer,) + tuple(grads)


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return _exact_attend(s, case) if case["op"] == "attend" else _exact_linear(s, case)


def _exact_attend(s, c):
    group = c["H"] // c["Hkv"]
    if c["packed"]:
        q, k, v = s["qkv"].detach().unbind(2)
    else:
        q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    outs, grads = [], []
    for b in range(c["B"]):
        seen = torch.arange(c["Nk"], device=q.device) if s["mask"] is None else s["mask"][b].nonzero()[:, 0]
        o, dq, dk, dv = [], [], torch.zeros_like(k[b], dtype=torch.float64), torch.zeros_like(v[b], dtype=torch.float64)
        for h in range(c["H"]):
            leaves = [t.double().requires_grad_(c["train"]) for t in (q[b, :, h], k[b, seen, h // group], v[b, seen, h // group])]
            if len(seen):
                o.append(torch.softmax(leaves[0] @ leaves[1].t() / math.sqrt(c["D"]), 1) @ leaves[2])
            else:
                o.append(leaves[0] * 0)
            if c["train"]:
                d = torch.autograd.grad(o[-1], leaves, s["dout"][b, :, h].double(), allow_unused=True)
                dq.append(d[0])
                if len(seen):
                    dk[seen, h // group] += d[1]
                    dv[seen, h // group] += d[2]
                o[-1] = o[-1].detach()
        outs.append(torch.stack(o, 1))
        if c["train"]:
            grads.append((torch.stack(dq, 1), dk, dv))
    out = torch.stack(outs)
    if not c["train"]:
        return out
    if c["packed"]:
        return out, torch.stack([torch.stack(t, 1) for t in grads])
    return (out,) + tuple(torch.stack(t) for t in zip(*grads))


def _exact_linear(s, c):
    names = [n for n in ("x", "w", "b", "gamma", "residual") if s[n] is not None]
    t = {n: s[n].detach().double().requires_grad_(c["train"]) for n in names}
    z = t["x"] @ t["w"].t()
    if "b" in t:
        z = z + t["b"]
    y = {"identity": lambda a: a, "quick_gelu": lambda a: a * torch.sigmoid(1.702 * a), "gelu": torch.nn.functional.gelu,
         "relu": torch.relu}[c["act"]](z)
    if c["branch"]:
        y = y * t["gamma"]
        if s["row_scale"] is not None:
            y = y * s["row_scale"].double()[:, None, None]
        y = y + t["residual"]
    if not c["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, [t[n] for n in names], s["dout"].double())
