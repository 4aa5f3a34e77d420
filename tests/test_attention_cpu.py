"""Refusals of eve_amd.attention / self_attention, and of the C entry points beneath, without a GPU."""
import ctypes

import pytest
import torch

import eve_amd
from eve_amd import _lib
from tests.attn_reference import attention64


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("q,k,v,kw,err,text", [
    (_t(2, 4, 64), _t(2, 4, 1, 64), _t(2, 4, 1, 64), {}, ValueError, "must be"),
    (_t(2, 4, 2, 64), _t(2, 4, 2, 64), _t(2, 5, 2, 64), {}, ValueError, "belong"),
    (_t(2, 4, 2, 64), _t(1, 4, 2, 64), _t(1, 4, 2, 64), {}, ValueError, "belong"),
    (_t(2, 4, 3, 64), _t(2, 4, 2, 64), _t(2, 4, 2, 64), {}, ValueError, "share"),
    (_t(2, 4, 2, 12), _t(2, 4, 2, 12), _t(2, 4, 2, 12), {}, ValueError, "width"),
    (_t(2, 4, 2, 136), _t(2, 4, 2, 136), _t(2, 4, 2, 136), {}, ValueError, "width"),
    (_t(2, 4, 2, 64, dtype=torch.float16), _t(2, 4, 2, 64, dtype=torch.float16), _t(2, 4, 2, 64, dtype=torch.float16), {}, TypeError, "float16"),
    (_t(2, 4, 2, 64), _t(2, 4, 2, 64, dtype=torch.bfloat16), _t(2, 4, 2, 64), {}, TypeError, "types"),
    (_t(2, 4, 2, 64), _t(2, 4, 2, 64), _t(2, 4, 2, 64), {"scale": -1.0}, ValueError, "scale"),
    (_t(2, 4, 2, 64), _t(2, 4, 2, 64), _t(2, 4, 2, 64), {"scale": float("nan")}, ValueError, "scale"),
    (_t(2, 4, 2, 64), _t(2, 4, 2, 64), _t(2, 4, 2, 64), {"key_mask": torch.ones(2, 5)}, ValueError, "key_mask"),
    (_t(2, 4, 2, 64), _t(2, 4, 2, 64), _t(2, 4, 2, 64), {}, RuntimeError, "no CPU fallback"),
])
def test_attention_refuses(q, k, v, kw, err, text):
    with pytest.raises(err, match=text):
        eve_amd.attention(q, k, v, **kw)


def test_self_attention_refuses():
    with pytest.raises(ValueError, match="qkv"):
        eve_amd.self_attention(_t(2, 4, 2, 2, 64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        eve_amd.self_attention(_t(2, 4, 3, 2, 64))


def test_c_entry_points_answer_bad_calls_with_codes():
    lib = _lib.load()
    good = dict(B=2, Nq=4, Nk=4, H=2, Hkv=2, D=64, dtype=_lib.F32, scale=0.125)
    lay = _lib.AttnLayout(*[512, 128, 64] * 3)
    p = ctypes.addressof

    def fwd(layout=lay, ptr=16, **kw):
        s = _lib.AttnShape(**{**good, **kw})
        return lib.eve_attn_fwd(p(s), p(layout), ptr, 16, 16, None, 16, None, None, 0, None)

    assert fwd(dtype=7) == -1 and fwd(B=-1) == -1 and fwd(H=3) == -1 and fwd(Hkv=0) == -1 and fwd(scale=0.0) == -1
    assert fwd(D=12) == -4 and fwd(D=256) == -4 and fwd(Nq=0x7fffffff, H=4) == -4
    assert fwd(layout=_lib.AttnLayout(*[510, 126, 63] * 3)) == -1 and b"stride" in lib.eve_moe_last_error()
    assert fwd(ptr=8) == -1 and fwd(ptr=None) == -1
    assert lib.eve_attn_fwd(None, p(lay), 16, 16, 16, None, 16, None, None, 0, None) == -1
    assert fwd(B=0) == 0 and fwd(Nq=0) == 0  # nothing to do, nothing launched
    s = _lib.AttnShape(**good)
    args = [16] * 3 + [None] + [16] * 6
    assert lib.eve_attn_bwd_workspace_bytes(p(s)) >= 2 * 4 * 2 * 4
    assert lib.eve_attn_bwd(p(s), p(lay), p(lay), *args, None, 0, None) == -2
    assert lib.eve_attn_bwd(p(s), p(lay), None, *args, 16, 1 << 20, None) == -1
    long = _lib.AttnShape(**{**good, "Nq": 1, "Nk": 1 << 20})
    assert lib.eve_attn_fwd_workspace_bytes(p(long)) > 0  # few rows against many keys are split
    assert lib.eve_attn_fwd(p(long), p(lay), 16, 16, 16, None, 16, None, None, 0, None) == -2


def test_the_reference_agrees_with_autograd():
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(2, n, h, 16, generator=g) for n, h in ((5, 4), (7, 2), (7, 2), (5, 4)))
    mask = torch.rand(2, 7, generator=g) > 0.4
    mask[1] = False
    ql, kl, vl = (t.double().requires_grad_(True) for t in (q, k, v))
    s = torch.einsum("bihd,bjhd->bhij", ql, kl.repeat_interleave(2, 2)) / 4
    p = torch.nan_to_num(torch.softmax(s.masked_fill(~mask[:, None, None], float("-inf")), 3)) * mask[:, None, None]
    out = torch.einsum("bhij,bjhd->bihd", p, vl.repeat_interleave(2, 2))
    grads = torch.autograd.grad(out[:1], (ql, kl, vl), do[:1].double())
    res = attention64(q, k, v, mask, dout=do)
    for name, want in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        torch.testing.assert_close(res[name][0][:1], want[:1].detach(), rtol=1e-9, atol=1e-12)
        assert float(res[name][0][1].abs().max()) == 0.0
