"""What lies at the ends of what eve_amd.attention and eve_amd.fused_linear take, without a GPU."""
import ctypes

import pytest
import torch

import eve_amd
from eve_amd import _lib, ops


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


BIG = (1 << 32) + 2  # what is left of it in 32 bits is 2


@pytest.mark.parametrize("q,k", [((BIG, 1, 1, 8), (BIG, 1, 1, 8)), ((1, BIG, 1, 8), (1, 3, 1, 8)), ((1, 3, 1, 8), (1, BIG, 1, 8)),
                                 ((1, 3, BIG, 8), (1, 3, 1, 8)), ((1, 1 << 31, 1, 8), (1, 3, 1, 8))])
def test_attention_refuses_sizes_beyond_32_bits(q, k):
    with pytest.raises(ValueError, match="2\\^31"):
        eve_amd.attention(_meta(*q), _meta(*k), _meta(*k))


def test_self_attention_refuses_sizes_beyond_32_bits():
    for shape in ((BIG, 1, 3, 1, 8), (1, BIG, 3, 1, 8), (1, 1, 3, BIG, 8)):
        with pytest.raises(ValueError, match="2\\^31"):
            eve_amd.self_attention(_meta(*shape))


@pytest.mark.parametrize("x,w", [((BIG, 1), (2, 1)), ((1 << 16, 1 << 16, 1), (2, 1)), ((2, BIG), (1, BIG)), ((2, 1), (BIG, 1)),
                                 ((1 << 31, 1), (1, 1))])
def test_fused_linear_refuses_sizes_beyond_32_bits(x, w):
    with pytest.raises(ValueError, match="2\\^31"):
        eve_amd.fused_linear(_meta(*x), _meta(*w))


@pytest.mark.parametrize("make", [lambda: torch.zeros(2, 5, 3, 9)[:, :0, :, :8], lambda: torch.zeros(2, 5, 3, 9)[:0, :, :, 1:],
                                  lambda: torch.zeros(2, 5, 3, 16)[:, :0, :, ::2], lambda: torch.zeros(2, 5, 3, 3, 9)[:, :0, :, :, :8]])
def test_what_is_empty_lies_as_the_kernels_want_it(make):
    """An empty part of a tensor has that tensor's strides, which the entry points check all the same."""
    t = ops.attn_readable(make())
    assert t.shape == make().shape and t.stride(-1) == 1
    assert all(s % 4 == 0 for s in t.stride()[:-1]), t.stride()


def test_more_workgroups_than_a_launch_holds_are_refused():
    """2^32 threads in a dimension: one-wave workgroups for a head of up to 64 rows, four waves else."""
    lib, p = _lib.load(), ctypes.addressof
    lay = _lib.AttnLayout(*[8] * 9)

    def fwd(**kw):
        s = _lib.AttnShape(**{**dict(B=1, Nq=1, Nk=1, H=1, Hkv=1, D=8, dtype=_lib.BF16, scale=1.0), **kw})
        return lib.eve_attn_fwd(p(s), p(lay), 16, 16, 16, None, 16, None, None, 0, None)

    assert fwd(B=1 << 26) == -4 and b"workgroups" in lib.eve_moe_last_error()
    assert fwd(B=1 << 24, Nq=65) == -4 and b"workgroups" in lib.eve_moe_last_error()


@pytest.mark.parametrize("scale", [2.0 ** -101, 1e-38, 2.0 ** 101, 3e38])
def test_scales_whose_reciprocal_leaves_float32_are_refused(scale):
    t = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="scale"):
        eve_amd.attention(t, t, t, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        eve_amd.self_attention(torch.zeros(1, 4, 3, 2, 64), scale=scale)
    s = _lib.AttnShape(1, 4, 4, 2, 2, 64, _lib.F32, scale)
    lay = _lib.AttnLayout(*[512, 128, 64] * 3)
    p = ctypes.addressof
    assert _lib.load().eve_attn_fwd(p(s), p(lay), 16, 16, 16, None, 16, None, None, 0, None) == -1
