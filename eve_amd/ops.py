"""Tensor-level wrappers over the C ABI (include/eve_moe.h).

Each function checks device / dtype / contiguity, allocates outputs with torch (device
memory and streams are the only things PyTorch is used for here) and enqueues the HIP
kernels on the current stream.  No function here has a CPU implementation.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import wraps
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable as _once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
MODES = {None: _lib.MODE_NONE, "none": _lib.MODE_NONE, "vl": _lib.MODE_VL, "vision": _lib.MODE_VISION,
         "text": _lib.MODE_TEXT}
ACTS = {"quick_gelu": _lib.ACT_QUICK_GELU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU,
        "identity": _lib.ACT_IDENTITY}


def _dt(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"eve_amd: unsupported dtype {t.dtype} (float32 or bfloat16)") from None


def _chk(t: Optional[torch.Tensor], name: str, dtype=None):
    if t is None:
        return
    if not t.is_cuda:
        raise RuntimeError(f"eve_amd: `{name}` must live on a GPU (got {t.device}); there is no CPU path")
    if not t.is_contiguous():
        raise RuntimeError(f"eve_amd: `{name}` must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"eve_amd: `{name}` must be {dtype}, got {t.dtype}")


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream():
    # the current stream's handle; torch.cuda.current_stream() makes a Stream object of it, 2.8 us a call instead of 0.4
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def once_differentiable(backward):
    """torch's decorator of this name, whose wrapping is done only where a graph of the gradient is wanted."""
    wrapped = _once_differentiable(backward)

    @wraps(backward)
    def first(ctx, *grads):
        return (wrapped if torch.is_grad_enabled() else backward)(ctx, *grads)
    return first


def _tracks(*tensors) -> bool:
    """Whether a call on these has to go through autograd (5 us a call on the host, of about 15 of the smallest ones)."""
    if torch.autograd.forward_ad._current_level >= 0:
        return True  # there is no forward-mode rule: autograd refuses such a tensor
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Profile:
    """Optional HIP-event timing of every C-ABI call, recorded on the stream the kernels are
    launched on (bench.py uses it for the per-kernel roofline numbers).  Off by default."""

    def __init__(self):
        self.on = False
        self._ev = []
        self.tagged = {}

    def enable(self):
        self.on, self._ev = True, []

    def disable(self):
        """-> {entry point: (total ms, calls)}; `self.tagged` then holds the same split by the calls' tags
        ({"eve_ffn_fwd[G=2]": ...}: the grouped GEMMs of a 2-group modality split beside those of a 32-expert layer)."""
        self.on = False
        torch.cuda.synchronize()
        out, tagged = {}, {}
        for name, tag, a, b in self._ev:
            dt = a.elapsed_time(b)
            ms, n = out.get(name, (0.0, 0))
            out[name] = (ms + dt, n + 1)
            if tag is not None:
                key = f"{name}[{tag}]"
                ms, n = tagged.get(key, (0.0, 0))
                tagged[key] = (ms + dt, n + 1)
        self._ev = []
        self.tagged = tagged
        return out

    def call(self, name, *args, tag=None):
        if not self.on:
            return _lib.call(name, *args)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        _lib.call(name, *args)
        b.record()
        self._ev.append((name, tag, a, b))


PROFILE = _Profile()


def capacity(S: int, E: int, capacity_factor: float, min_capacity: int) -> int:
    """models/sharded_moe.py:150-160,:177 (host arithmetic inside the library)."""
    return int(_lib.load().eve_capacity(int(S), int(E), float(capacity_factor), int(min_capacity)))


@dataclass
class Routing:
    """Index-form result of top-2 gating (replaces combine_weights / dispatch_mask [S,E,C])."""
    S: int
    E: int
    C: int
    gates: torch.Tensor        # [S,E] f32
    idx: torch.Tensor          # [S,2] i32
    loc: torch.Tensor          # [S,2] i32
    slot: torch.Tensor         # [S,2] i32 (-1 = not dispatched)
    weight: torch.Tensor       # [S,2] f32
    slot_token: torch.Tensor   # [E*C] i32 (-1 = empty)
    slot_weight: torch.Tensor  # [E*C] f32
    exp_counts: torch.Tensor   # [E] i64 (device)
    rows: torch.Tensor         # [E] i32
    l_aux: torch.Tensor        # [1] f32


def gate_logits(h2d: torch.Tensor, vemb, temb, wg: torch.Tensor, T: int, n_vis: int, mode: int) -> torch.Tensor:
    _chk(h2d, "hidden"), _chk(wg, "wg", torch.float32)
    _chk(vemb, "vision_embed", h2d.dtype), _chk(temb, "text_embed", h2d.dtype)
    S, M = h2d.shape
    E = wg.shape[0]
    assert wg.shape[1] == M
    logits = torch.empty(S, E, dtype=torch.float32, device=h2d.device)
    PROFILE.call("eve_gate_logits_fwd", _p(h2d), _p(vemb), _p(temb), _p(wg), _p(logits), S, T, n_vis, mode, M, E,
              _dt(h2d), _stream())
    return logits


def gumbel_from_uniform(u: torch.Tensor) -> torch.Tensor:
    """Gumbel(0,1) variates of standard-uniform draws, torch.distributions.Gumbel's arithmetic in one kernel."""
    _chk(u, "uniform", torch.float32)
    out = torch.empty_like(u)
    PROFILE.call("eve_gumbel_from_uniform", _p(u), _p(out), u.numel(), _stream())
    return out


NOISE_GUMBEL, NOISE_UNIFORM, NOISE_DEVICE_PHILOX = 0, 1, 2  # include/eve_moe.h: values of noise_is_uniform


def noise_code(noise: torch.Tensor, noise_is_uniform, S: int, E: int) -> int:
    """The `noise_is_uniform` argument of the C calls for (noise, flag) -- False / True / NOISE_DEVICE_PHILOX -- after
    checking that `noise` is what that value says: an fp32 [S,E] tensor, or the int64 {seed, offset} generator state
    the gate kernel draws from and advances (`eve_amd.DeviceNoise.state`)."""
    code = int(noise_is_uniform)
    if code == NOISE_DEVICE_PHILOX:
        _chk(noise, "generator state", torch.int64)
        if noise.numel() != 2:
            raise ValueError("eve_amd: the device generator state is an int64 tensor {seed, offset}")
        return code
    if code not in (NOISE_GUMBEL, NOISE_UNIFORM):
        raise ValueError(f"eve_amd: noise_is_uniform={noise_is_uniform!r}")
    _chk(noise, "noise", torch.float32)
    if tuple(noise.shape) != (S, E):
        raise RuntimeError("eve_amd: gate parameter / noise shapes do not match the layer input")
    return code


def gate_top2(logits: torch.Tensor, noise: torch.Tensor, C: int, noise_is_uniform=False) -> Routing:
    """`noise`: Gumbel variates [S,E], or (noise_is_uniform) the torch.rand draws they are made of, or
    (noise_is_uniform == NOISE_DEVICE_PHILOX) the device generator state the kernel draws from itself."""
    _chk(logits, "logits", torch.float32)
    S, E = logits.shape
    code = noise_code(noise, noise_is_uniform, S, E)
    dev = logits.device
    i32 = dict(dtype=torch.int32, device=dev)
    f32 = dict(dtype=torch.float32, device=dev)
    r = Routing(S, E, C, torch.empty(S, E, **f32), torch.empty(S, 2, **i32), torch.empty(S, 2, **i32),
                torch.empty(S, 2, **i32), torch.empty(S, 2, **f32), torch.empty(E * C, **i32),
                torch.empty(E * C, **f32), torch.empty(E, dtype=torch.int64, device=dev), torch.empty(E, **i32),
                torch.empty(1, **f32))
    nbytes = _lib.load().eve_gate_workspace_bytes(S, E)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    PROFILE.call("eve_gate_top2_fwd", _p(logits), _p(noise), code, S, E, C, _p(r.gates), _p(r.idx), _p(r.loc), _p(r.slot),
              _p(r.weight), _p(r.slot_token), _p(r.slot_weight), _p(r.exp_counts), _p(r.rows), _p(r.l_aux), _p(ws),
              nbytes, _stream())
    return r


def gate_top2_bwd_raw(gates, idx, loc, exp_counts, S: int, E: int, C: int, d_weight: Optional[torch.Tensor],
                      d_l_aux: Optional[torch.Tensor]) -> torch.Tensor:
    """dlogits [S,E] from d_weight [S,2] (None = no gradient reached the combine weights) and d_l_aux [1]."""
    if d_weight is not None:
        d_weight = d_weight.contiguous()
    _chk(d_weight, "d_weight", torch.float32), _chk(d_l_aux, "d_l_aux", torch.float32)
    dlogits = torch.empty(S, E, dtype=torch.float32, device=gates.device)
    PROFILE.call("eve_gate_top2_bwd", _p(gates), _p(idx), _p(loc), _p(d_weight), _p(d_l_aux), _p(exp_counts),
              S, E, C, _p(dlogits), _stream())
    return dlogits


def gate_top2_bwd(r: Routing, d_weight: Optional[torch.Tensor], d_l_aux: Optional[torch.Tensor]) -> torch.Tensor:
    return gate_top2_bwd_raw(r.gates, r.idx, r.loc, r.exp_counts, r.S, r.E, r.C, d_weight, d_l_aux)


def gate_wgrad(h2d, vemb, temb, dlogits, T: int, n_vis: int, mode: int) -> torch.Tensor:
    _chk(h2d, "hidden"), _chk(dlogits, "dlogits", torch.float32)
    S, M = h2d.shape
    E = dlogits.shape[1]
    dwg = torch.empty(E, M, dtype=torch.float32, device=h2d.device)
    nbytes = _lib.load().eve_gate_wgrad_workspace_bytes(S, M, E)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h2d.device)
    PROFILE.call("eve_gate_wgrad", _p(h2d), _p(vemb), _p(temb), _p(dlogits), _p(dwg), S, T, n_vis, mode, M, E, _dt(h2d),
              _p(ws), nbytes, _stream())
    return dwg


def dispatch_fwd(h2d, vemb, temb, slot_token: torch.Tensor, T: int, n_vis: int, mode: int,
                 slot: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`slot` [S,2] (the gate's forward map): each token row is then read once for both of its slots."""
    _chk(h2d, "hidden"), _chk(slot_token, "slot_token", torch.int32), _chk(slot, "slot", torch.int32)
    S, M = h2d.shape
    n = slot_token.numel()
    assert slot is None or tuple(slot.shape) == (S, 2)
    xd = torch.empty(n, M, dtype=h2d.dtype, device=h2d.device)
    PROFILE.call("eve_dispatch_fwd", _p(h2d), _p(vemb), _p(temb), _p(slot), _p(slot_token), _p(xd), S, T, n_vis, mode, M, n,
              _dt(h2d), _stream())
    return xd


def dispatch_bwd(dxd: torch.Tensor, slot: torch.Tensor, dlogits, wg, S: int) -> torch.Tensor:
    _chk(dxd, "dxd"), _chk(slot, "slot", torch.int32), _chk(dlogits, "dlogits", torch.float32)
    _chk(wg, "wg", torch.float32)
    M = dxd.shape[-1]
    E = wg.shape[0] if wg is not None else 1
    dh = torch.empty(S, M, dtype=dxd.dtype, device=dxd.device)
    PROFILE.call("eve_dispatch_bwd", _p(dxd), _p(slot), _p(dlogits), _p(wg), _p(dh), S, M, E, _dt(dxd), _stream())
    return dh


def route_bwd(dxd, slot, dlogits, wg, S: int, T: int, n_vis: int, mode: int, want_v: bool, want_t: bool,
              embed_dtype: torch.dtype = torch.float32):
    """dispatch_bwd + embed_grad in one pass: -> (dh [S,M], dvision|None, dtext|None); the embedding
    gradients are stored as `embed_dtype` (fp32, or bf16 for bf16 parameters)."""
    _chk(dxd, "dxd"), _chk(slot, "slot", torch.int32), _chk(dlogits, "dlogits", torch.float32)
    _chk(wg, "wg", torch.float32)
    M = dxd.shape[-1]
    E = wg.shape[0]
    dev = dxd.device
    dh = torch.empty(S, M, dtype=dxd.dtype, device=dev)
    want_v = want_v and mode != _lib.MODE_NONE
    want_t = want_t and mode != _lib.MODE_NONE
    dv = torch.empty(M, dtype=embed_dtype, device=dev) if want_v else None
    dt = torch.empty(M, dtype=embed_dtype, device=dev) if want_t else None
    nbytes = _lib.load().eve_embed_grad_workspace_bytes(S, M) if (want_v or want_t) else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    PROFILE.call("eve_route_bwd", _p(dxd), _p(slot), _p(dlogits), _p(wg), _p(dh), _p(dv), _p(dt), S, T, n_vis, mode, M, E,
                 _dt(dxd), _DTYPES[embed_dtype], _p(ws), nbytes, _stream())
    return dh, dv, dt


def embed_grad(dh: torch.Tensor, T: int, n_vis: int, mode: int, want_v=True, want_t=True):
    _chk(dh, "dh")
    S, M = dh.shape
    dv = torch.empty(M, dtype=torch.float32, device=dh.device) if want_v else None
    dt = torch.empty(M, dtype=torch.float32, device=dh.device) if want_t else None
    nbytes = _lib.load().eve_embed_grad_workspace_bytes(S, M)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dh.device)
    PROFILE.call("eve_embed_grad", _p(dh), _p(dv), _p(dt), S, T, n_vis, mode, M, _dt(dh), _p(ws), nbytes, _stream())
    return dv, dt


def combine_fwd(y: torch.Tensor, slot: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    _chk(y, "expert_output"), _chk(slot, "slot", torch.int32), _chk(weight, "weight", torch.float32)
    S = slot.shape[0]
    M = y.shape[-1]
    out = torch.empty(S, M, dtype=y.dtype, device=y.device)
    PROFILE.call("eve_combine_fwd", _p(y), _p(slot), _p(weight), _p(out), S, M, _dt(y), _stream())
    return out


def combine_bwd(dout: torch.Tensor, y: torch.Tensor, slot, slot_token, slot_weight) -> Tuple[torch.Tensor, torch.Tensor]:
    _chk(dout, "dout", y.dtype), _chk(y, "expert_output")
    S, M = dout.shape
    n = slot_token.numel()
    dy = torch.empty(n, M, dtype=y.dtype, device=y.device)
    dw = torch.empty(S, 2, dtype=torch.float32, device=y.device)
    PROFILE.call("eve_combine_bwd", _p(dout), _p(y), _p(slot), _p(slot_token), _p(slot_weight), _p(dy), _p(dw), S, M, n,
              _dt(y), _stream())
    return dy, dw


def ffn_fwd(x, w1, b1, w2, b2, rows, act: int, save_z: bool = True, shared_gpu: bool = False):
    """x [G,R,M]; w1 [E_l,I,M]; b1 [E_l,I]; w2 [E_l,M,I]; b2 [E_l,M] -> (z|None, a, y).
    `shared_gpu`: other kernels (RCCL exchanges) run beside these launches (EVE_FFN_SHARED_GPU)."""
    for t, n in ((x, "x"), (w1, "w1"), (b1, "b1"), (w2, "w2"), (b2, "b2")):
        _chk(t, n, x.dtype)
    _chk(rows, "rows", torch.int32)
    G, R, M = x.shape
    E_l, I, M2 = w1.shape
    assert M2 == M and w2.shape == (E_l, M, I) and b1.shape == (E_l, I) and b2.shape == (E_l, M) and G % E_l == 0
    z = torch.empty(G, R, I, dtype=x.dtype, device=x.device) if save_z else None
    a = torch.empty(G, R, I, dtype=x.dtype, device=x.device)
    y = torch.empty(G, R, M, dtype=x.dtype, device=x.device)
    PROFILE.call("eve_ffn_fwd", _p(x), _p(w1), _p(b1), _p(w2), _p(b2), _p(z), _p(a), _p(y), _p(rows), G, E_l, R, M, I,
              act, _dt(x), _lib.FFN_SHARED_GPU if shared_gpu else 0, _stream(), tag=f"G={G}")
    return z, a, y


def ffn_bwd(dy, x, z, a, w1, w2, rows, act: int, grads_out=None, shared_gpu: bool = False):
    """-> (dx [G,R,M], dw1, db1, dw2, db2) with the shapes / dtype of the forward operands.
    `grads_out` = (dw1, db1, dw2, db2) to write the parameter gradients into caller-provided tensors."""
    for t, n in ((dy, "dy"), (x, "x"), (z, "z"), (a, "a"), (w1, "w1"), (w2, "w2")):
        _chk(t, n, x.dtype)
    G, R, M = x.shape
    E_l, I, _ = w1.shape
    dev = x.device
    dz = torch.empty(G, R, I, dtype=x.dtype, device=dev)
    dx = torch.empty(G, R, M, dtype=x.dtype, device=dev)  # rows >= rows[g] stay unwritten and are never read
    if grads_out is not None:
        dw1, db1, dw2, db2 = grads_out
        for t, n, shp in ((dw1, "dw1", (E_l, I, M)), (db1, "db1", (E_l, I)), (dw2, "dw2", (E_l, M, I)), (db2, "db2", (E_l, M))):
            _chk(t, n, x.dtype)
            assert tuple(t.shape) == shp, (n, tuple(t.shape), shp)
    else:
        dw1 = torch.empty(E_l, I, M, dtype=x.dtype, device=dev)
        db1 = torch.empty(E_l, I, dtype=x.dtype, device=dev)
        dw2 = torch.empty(E_l, M, I, dtype=x.dtype, device=dev)
        db2 = torch.empty(E_l, M, dtype=x.dtype, device=dev)
    nbytes = _lib.load().eve_ffn_bwd_workspace_bytes(G, E_l, R, M, I, _dt(x))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    PROFILE.call("eve_ffn_bwd", _p(dy), _p(x), _p(z), _p(a), _p(w1), _p(w2), _p(dz), _p(dx), _p(dw1), _p(db1), _p(dw2),
              _p(db2), _p(rows), G, E_l, R, M, I, act, _dt(x), _lib.FFN_SHARED_GPU if shared_gpu else 0, _p(ws), nbytes, _stream(),
              tag=f"G={G}")
    return dx, dw1, db1, dw2, db2


# ------------------------------------------------ hard modality split of the non-MoE layers
def split_ln_fwd(h, gamma_v, beta_v, gamma_t, beta_t, n_vis: int, R: int, eps: float):
    """h [B,T,M] -> (xg [2,R,M], mean [S], rstd [S]); see include/eve_moe.h."""
    _chk(h, "hidden")
    for t, n in ((gamma_v, "gamma_v"), (beta_v, "beta_v"), (gamma_t, "gamma_t"), (beta_t, "beta_t")):
        _chk(t, n, h.dtype)
    B, T, M = h.shape
    xg = torch.empty(2, R, M, dtype=h.dtype, device=h.device)
    mean = torch.empty(B * T, dtype=torch.float32, device=h.device)
    rstd = torch.empty(B * T, dtype=torch.float32, device=h.device)
    PROFILE.call("eve_split_ln_fwd", _p(h), _p(gamma_v), _p(beta_v), _p(gamma_t), _p(beta_t), _p(xg), _p(mean), _p(rstd),
                 B, T, n_vis, R, M, float(eps), _dt(h), _stream())
    return xg, mean, rstd


def split_ln_bwd(dxg, h, mean, rstd, gamma_v, gamma_t, n_vis: int):
    """-> (dh [B,T,M], dparams [4,M] fp32 = dgamma_v, dbeta_v, dgamma_t, dbeta_t)."""
    _chk(dxg, "dxg", h.dtype), _chk(h, "hidden")
    B, T, M = h.shape
    R = dxg.shape[1]
    dh = torch.empty_like(h)
    dparams = torch.empty(4, M, dtype=torch.float32, device=h.device)
    nbytes = _lib.load().eve_split_ln_workspace_bytes(B * T, M)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    PROFILE.call("eve_split_ln_bwd", _p(dxg), _p(h), _p(mean), _p(rstd), _p(gamma_v), _p(gamma_t), _p(dh), _p(dparams),
                 B, T, n_vis, R, M, _dt(h), _p(ws), nbytes, _stream())
    return dh, dparams


def layer_norm_fwd(x2d, gamma, beta, eps: float):
    """Plain LayerNorm over the last dimension of x [S,M] on the split-LayerNorm kernel with a single group (every
    token "vision": row s of the input is row s of the output; the second group does not exist and is never touched).
    -> (y [S,M], mean [S], rstd [S])"""
    _chk(x2d, "x"), _chk(gamma, "weight", x2d.dtype), _chk(beta, "bias", x2d.dtype)
    S, M = x2d.shape
    y = torch.empty_like(x2d)
    mean = torch.empty(S, dtype=torch.float32, device=x2d.device)
    rstd = torch.empty(S, dtype=torch.float32, device=x2d.device)
    PROFILE.call("eve_split_ln_fwd", _p(x2d), _p(gamma), _p(beta), _p(gamma), _p(beta), _p(y), _p(mean), _p(rstd),
                 1, S, S, S, M, float(eps), _dt(x2d), _stream(), tag="plain")
    return y, mean, rstd


def layer_norm_bwd(dy2d, x2d, mean, rstd, gamma):
    """-> (dx [S,M], dgamma [M] fp32, dbeta [M] fp32)."""
    _chk(dy2d, "dy", x2d.dtype), _chk(x2d, "x"), _chk(gamma, "weight", x2d.dtype)
    S, M = x2d.shape
    dx = torch.empty_like(x2d)
    dparams = torch.empty(4, M, dtype=torch.float32, device=x2d.device)
    nbytes = _lib.load().eve_split_ln_workspace_bytes(S, M)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x2d.device)
    PROFILE.call("eve_split_ln_bwd", _p(dy2d), _p(x2d), _p(mean), _p(rstd), _p(gamma), _p(gamma), _p(dx), _p(dparams),
                 1, S, S, S, M, _dt(x2d), _p(ws), nbytes, _stream(), tag="plain")
    return dx, dparams[0], dparams[1]


def split_permute(src, B: int, T: int, n_vis: int, R: int, to_groups: bool):
    _chk(src, "src")
    M = src.shape[-1]
    dst = torch.empty((2, R, M) if to_groups else (B, T, M), dtype=src.dtype, device=src.device)
    PROFILE.call("eve_split_permute", _p(src), _p(dst), B, T, n_vis, R, M, 1 if to_groups else 0, _dt(src), _stream())
    return dst


# ----------------------------------------------------- layer-scale residual branch of the encoder layer
def scale_residual_fwd(x, gamma, row_scale, residual, T: int):
    """residual + (x * gamma) * row_scale[s // T]; x, residual [S,M]; gamma [M] | None; row_scale [S // T] | None."""
    _chk(x, "x"), _chk(residual, "residual", x.dtype), _chk(gamma, "gamma", x.dtype), _chk(row_scale, "row_scale", x.dtype)
    S, M = x.shape
    out = torch.empty_like(x)
    PROFILE.call("eve_scale_residual_fwd", _p(x), _p(gamma), _p(row_scale), _p(residual), _p(out), S, T, M, _dt(x), _stream())
    return out


def scale_residual_bwd(dout, x, gamma, row_scale, T: int):
    """-> (dx [S,M], dgamma [M] fp32 | None)."""
    _chk(dout, "dout"), _chk(x, "x", dout.dtype), _chk(gamma, "gamma", dout.dtype), _chk(row_scale, "row_scale", dout.dtype)
    S, M = dout.shape
    dx = torch.empty_like(dout)
    dgamma = torch.empty(M, dtype=torch.float32, device=dout.device) if gamma is not None else None
    nbytes = _lib.load().eve_scale_residual_workspace_bytes(S, M) if gamma is not None else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dout.device) if nbytes else None
    PROFILE.call("eve_scale_residual_bwd", _p(dout), _p(x), _p(gamma), _p(row_scale), _p(dx), _p(dgamma), S, T, M, _dt(dout),
                 _p(ws), nbytes, _stream())
    return dx, dgamma


# ----------------------------------------------------------------------------------- attention of the encoder layer
ATTN_SCALES = (2.0 ** -100, 2.0 ** 100)  # what eve_attn_* take


def _on_device_of(which: int):
    """Decorates a wrapper: its calls are enqueued on the current stream of the device of argument `which`, whichever device is
    current."""
    def wrap(f):
        @wraps(f)
        def on_device(*args, **kwargs):
            device = args[which].get_device()
            if device < 0:
                raise RuntimeError(f"eve_amd: {f.__name__} must be given GPU tensors; there is no CPU path")
            if device == torch.cuda.current_device():
                return f(*args, **kwargs)
            with torch.cuda.device(device):
                return f(*args, **kwargs)
        return on_device
    return wrap


def _chk_all(like: torch.Tensor, **tensors):
    """_chk of several at once, None among them: contiguous, of one type and on one device with `like`."""
    dtype, device = like.dtype, like.device
    for name, t in tensors.items():
        if t is not None and not (t.dtype == dtype and t.device == device and t.is_contiguous()):
            _chk(t, name, dtype)
            raise RuntimeError(f"eve_amd: `{name}` is on {t.device}, not on {device}")


def _chk_parts(q, k, v):
    if k.device != q.device or v.device != q.device or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("eve_amd: q, k and v must be on one device and of one type")


def _attn_at(t: torch.Tensor):
    """Address and element strides of the first three dimensions of [B,N,H,D]; a dimension of one element has none to speak of."""
    b, n, h, _ = t.shape
    sb, sn, sh, _ = t.stride()
    return t.data_ptr(), 0 if b == 1 else sb, 0 if n == 1 else sn, 0 if h == 1 else sh


def _attn_parts_at(t: torch.Tensor):
    """The same of the three parts of [B,N,3,H,D]."""
    b, n, _, h, _ = t.shape
    sb, sn, step, sh, _ = t.stride()
    at, step = t.data_ptr(), step * t.element_size()
    rest = 0 if b == 1 else sb, 0 if n == 1 else sn, 0 if h == 1 else sh
    return (at, *rest), (at + step, *rest), (at + 2 * step, *rest)


def _attn_reads(at, unit: int) -> bool:
    p, sb, sn, sh = at
    return not (p % 16 or sb % unit or sn % unit or sh % unit or sn > 1 << 22)


def attn_readable(t: torch.Tensor) -> torch.Tensor:
    """`t` [B,N,H,D] (or [B,N,3,H,D], three of them) as the kernels can read it: the last dimension contiguous, rows on 16-byte
    boundaries and at most 2^22 elements apart; else a copy."""
    unit = 16 // t.element_size()
    parts = (_attn_at(t),) if t.dim() == 4 else _attn_parts_at(t)
    if t.stride(-1) == 1 and all(_attn_reads(at, unit) for at in parts):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def attn_dense(t: torch.Tensor) -> torch.Tensor:
    """`t` contiguous and on a 16-byte boundary (a contiguous part of another tensor may lie anywhere); else a copy."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def attn_fwd(q, k, v, key_mask, scale: float, want_lse: bool = True):
    """q [B,Nq,H,D]; k, v [B,Nk,Hkv,D] (attn_readable); key_mask [B,Nk] bool | None -> (out [B,Nq,H,D], lse [B,H,Nq] | None).
    The order inside lse is the kernels' own."""
    _chk_parts(q, k, v)
    return _attn_fwd((*q.shape[:3], *k.shape[1:]), (_attn_at(q), _attn_at(k), _attn_at(v)), q, key_mask, scale, want_lse)


def attn_qkv_fwd(qkv, key_mask, scale: float, want_lse: bool = True):
    """attn_fwd of the three parts of qkv [B,N,3,H,D]."""
    B, N, _, H, D = qkv.shape
    return _attn_fwd((B, N, H, N, H, D), _attn_parts_at(qkv), qkv, key_mask, scale, want_lse)


def attn_bwd(dout, q, k, v, key_mask, out, lse, scale: float, dq, dk, dv) -> None:
    """Writes the gradients into dq, dk, dv, which have q's, k's, v's shapes and lie as attn_readable says."""
    _chk_parts(q, k, v), _chk_parts(out, q, k), _chk_parts(q, dq, dk), _chk_parts(q, dq, dv)
    _attn_bwd((*q.shape[:3], *k.shape[1:]), (_attn_at(q), _attn_at(k), _attn_at(v)), dout, key_mask, out, lse, scale,
              (_attn_at(dq), _attn_at(dk), _attn_at(dv)))


def attn_qkv_bwd(dout, qkv, key_mask, out, lse, scale: float, dqkv) -> None:
    """attn_bwd of the three parts of qkv [B,N,3,H,D] into those of dqkv."""
    B, N, _, H, D = qkv.shape
    _attn_bwd((B, N, H, N, H, D), _attn_parts_at(qkv), dout, key_mask, out, lse, scale, _attn_parts_at(dqkv))


def _attn_shape(dims, dtype, scale):
    B, Nq, H, Nk, Hkv, D = dims
    return _lib.AttnShape(B, Nq, Nk, H, Hkv, D, _DTYPES[dtype], scale)


def _attn_layout(at):
    (_, *a), (_, *b), (_, *c) = at
    return _lib.AttnLayout(*a, *b, *c)


@_on_device_of(2)
def _attn_fwd(dims, at, like, key_mask, scale, want_lse):
    _chk(key_mask, "key_mask", torch.bool)
    B, Nq, H, Nk, _, D = dims
    device = like.device
    shape, layout = _attn_shape(dims, like.dtype, scale), _attn_layout(at)
    out = like.new_empty((B, Nq, H, D))
    lse = torch.empty(B, H, Nq, dtype=torch.float32, device=device) if want_lse else None
    ref = _lib.ctypes.addressof(shape)
    nbytes = _lib.load().eve_attn_fwd_workspace_bytes(ref)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    PROFILE.call("eve_attn_fwd", ref, _lib.ctypes.addressof(layout), at[0][0], at[1][0], at[2][0], _p(key_mask), out.data_ptr(),
                 _p(lse), _p(ws), nbytes, _stream(), tag=PROFILE.on and f"N={Nq}x{Nk}")
    return out, lse


@_on_device_of(2)
def _attn_bwd(dims, at, dout, key_mask, out, lse, scale, grads_at):
    _chk(dout, "dout", out.dtype), _chk(out, "out"), _chk(lse, "lse", torch.float32)
    device = out.device
    shape, layout, grads = _attn_shape(dims, out.dtype, scale), _attn_layout(at), _attn_layout(grads_at)
    ref = _lib.ctypes.addressof(shape)
    nbytes = _lib.load().eve_attn_bwd_workspace_bytes(ref)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    PROFILE.call("eve_attn_bwd", ref, _lib.ctypes.addressof(layout), _lib.ctypes.addressof(grads), at[0][0], at[1][0], at[2][0],
                 _p(key_mask), out.data_ptr(), lse.data_ptr(), dout.data_ptr(), grads_at[0][0], grads_at[1][0], grads_at[2][0],
                 _p(ws), nbytes, _stream(), tag=PROFILE.on and f"N={dims[1]}x{dims[3]}")


# ----------------------------------------------------------------------------- linear layer with its epilogue fused
@_on_device_of(0)
def linear_fwd(x, w, bias, gamma, row_scale, residual, rows_per_scale: int, act: int, save_z: bool = False):
    """x [S,K]; w [N,K]; bias, gamma [N] | None; row_scale [S / rows_per_scale] | None; residual [S,N] | None
    -> (residual + row_scale * gamma * act(x w^T + bias) [S,N], z = x w^T + bias [S,N] | None)."""
    _chk_all(x, x=x, weight=w, bias=bias, gamma=gamma, row_scale=row_scale, residual=residual)
    S, K = x.shape
    N = w.shape[0]
    y = x.new_empty((S, N))
    z = x.new_empty((S, N)) if save_z else None
    PROFILE.call("eve_linear_fwd", _p(x), _p(w), _p(bias), _p(gamma), _p(row_scale), _p(residual), _p(y), _p(z), S,
                 rows_per_scale, K, N, act, _dt(x), _stream(), tag=PROFILE.on and f"{S}x{K}x{N}")
    return y, z


@_on_device_of(0)
def linear_bwd(dy, x, w, z, gamma, row_scale, rows_per_scale: int, act: int, want):
    """-> (dx, dw, dbias, dgamma), None where `want` (four truth values) does not ask for one."""
    _chk_all(x, dy=dy, x=x, weight=w, z=z, gamma=gamma, row_scale=row_scale)
    S, K = x.shape
    N = w.shape[0]
    outs = [x.new_empty(s) if yes else None for s, yes in zip(((S, K), (N, K), (N,), (N,)), want)]
    nbytes = _lib.load().eve_linear_bwd_workspace_bytes(S, K, N, _dt(x))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    PROFILE.call("eve_linear_bwd", _p(dy), _p(x), _p(w), _p(z), _p(gamma), _p(row_scale), *(_p(o) for o in outs), S,
                 rows_per_scale, K, N, act, _dt(x), _p(ws), nbytes, _stream(), tag=PROFILE.on and f"{S}x{K}x{N}")
    return outs
