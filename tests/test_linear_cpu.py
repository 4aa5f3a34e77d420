"""Refusals of eve_amd.fused_linear, and of the C entry points beneath, without a GPU."""
import pytest
import torch

import eve_amd
from eve_amd import _lib


@pytest.mark.parametrize("kw,err,text", [
    (dict(x=torch.zeros(2, 3, 9)), ValueError, "belong"),
    (dict(weight=torch.zeros(8)), ValueError, "belong"),
    (dict(activation="tanh"), ValueError, "activation"),
    (dict(bias=torch.zeros(7)), ValueError, "bias"),
    (dict(gamma=torch.zeros(1)), ValueError, "gamma"),
    (dict(row_scale=torch.ones(3)), ValueError, "row_scale"),
    (dict(residual=torch.zeros(2, 3, 9)), ValueError, "residual"),
    (dict(residual=torch.zeros(2, 1, 5)), ValueError, "residual"),
    (dict(row_scale=torch.ones(2, requires_grad=True)), ValueError, "no gradient"),
    (dict(x=torch.zeros(8), row_scale=torch.ones(8)), ValueError, "two dimensions"),
    (dict(x=torch.zeros(2, 3, 8, dtype=torch.float16)), TypeError, "float16"),
    (dict(weight=torch.zeros(5, 8, dtype=torch.bfloat16)), TypeError, "weight"),
    (dict(bias=torch.zeros(5, dtype=torch.bfloat16)), TypeError, "bias"),
    (dict(), RuntimeError, "no CPU fallback"),
])
def test_fused_linear_refuses(kw, err, text):
    args = dict(x=torch.zeros(2, 3, 8), weight=torch.zeros(5, 8))
    with pytest.raises(err, match=text):
        eve_amd.fused_linear(**{**args, **kw})


def test_c_entry_points_answer_bad_calls_with_codes():
    lib = _lib.load()

    def fwd(rows=4, T=1, K=8, N=8, act=3, dtype=0, x=16, y=16):
        return lib.eve_linear_fwd(x, 16, None, None, None, None, y, None, rows, T, K, N, act, dtype, None)

    assert fwd(rows=-1) == -1 and fwd(T=0) == -1 and fwd(act=4) == -1 and fwd(dtype=2) == -1 and fwd(x=None) == -1 and fwd(y=None) == -1
    assert fwd(K=1 << 25) == -4
    assert fwd(rows=0) == 0 and fwd(N=0) == 0  # nothing to do, nothing launched

    def bwd(dy=16, z=None, dg=None, act=3, ws=None, n=0):
        return lib.eve_linear_bwd(dy, 16, 16, z, None, None, 16, 16, 16, dg, 4, 1, 8, 8, act, 0, ws, n, None)

    assert lib.eve_linear_bwd_workspace_bytes(4, 8, 8, 0) > 0
    assert bwd() == -2 and bwd(ws=16, n=8) == -2 and bwd(dy=None) == -1
    assert bwd(act=0, ws=16, n=1 << 20) == -1 and bwd(dg=16, ws=16, n=1 << 20) == -1  # both need z


def test_the_wrappers_refuse_cpu_tensors():
    from eve_amd import ops
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.linear_fwd(x, w, None, None, None, None, 1, ops.ACTS["identity"])
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.linear_bwd(torch.zeros(2, 4), x, w, None, None, None, 1, ops.ACTS["identity"], (True, True, False, False))
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.attn_fwd(q, q, q, None, 1.0)
