"""Dense feed-forward operators at the ends of what their inputs may hold: NaN that has
to reach every gradient it belongs to."""
from __future__ import annotations

import pytest
import torch

from elastikernel_b200 import _ops
from oracle import ffn as off

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN = float("nan")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ NaN in a gradient
def _nan_case(T, H, I, dtype, where):
    """Inputs with one NaN, and the h that the forward pass leaves of them."""
    g = _gen(T + H + I)
    x, w1, w2, w3, d = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in
                        ((T, H), (I, H), (H, I), (I, H), (T, H)))
    w1, w2, w3 = w1 * H ** -0.5, w2 * I ** -0.5, w3 * H ** -0.5
    if where == "x":
        x[T // 2, 5] = NAN
    elif where == "w1":
        w1[I // 3, 7] = NAN
    h = off.forward(x, w1, w2, w3, "silu")["h"].to(dtype)  # its planes are products alone: of any gate
    if where == "h1":
        h[0, T - 1, I - 2] = NAN
    elif where == "h3":
        h[1, 0, I // 2] = NAN
    return x, w1, w2, w3, h, d


# (150, 4096, 264): da is cut along K, and the gate's gradient works on summed slices
@pytest.mark.parametrize("T,H,I", [(3, 64, 72), (200, 136, 264), (150, 4096, 264)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("act", list(_ops.GATES))
@pytest.mark.parametrize("where", ["x", "w1", "h1", "h3"])
def test_nan_reaches_every_gradient_it_belongs_to(T, H, I, dtype, act, where, cuda_dev):
    """NaN exactly where the formula in 64 bits has it, and numbers everywhere else."""
    x, w1, w2, w3, h, d = _nan_case(T, H, I, dtype, where)
    ref = off.backward(x, w1, w2, w3, h, d, act)
    got = _ops.gated_ffn_grad(x, w1, w2, w3, h, d, act=act)
    for name, t in zip(("x", "w1", "w2", "w3"), got):
        assert torch.equal(torch.isnan(t), torch.isnan(ref[name])), name
        assert torch.isfinite(t[~torch.isnan(t)]).all(), name
    if where != "h3":  # dh3 takes no part of h3
        assert torch.isnan(got[3]).any()
    assert all(torch.isnan(t).any() for t in got[:3])


@pytest.mark.parametrize("T", [3, 200])
@pytest.mark.parametrize("act", list(_ops.GATES))
@pytest.mark.parametrize("where", ["x", "w1"])
def test_nan_reaches_every_result_it_belongs_to(T, act, where, cuda_dev):
    x, w1, w2, w3, _, _ = _nan_case(T, 144, 272, BF, where)
    ref = off.forward(x, w1, w2, w3, act)
    y, h = _ops.gated_ffn(x, w1, w2, w3, act=act, save=True)
    assert torch.equal(torch.isnan(y), torch.isnan(ref["y"])) and torch.isnan(y).any()
    assert torch.equal(torch.isnan(h), torch.isnan(ref["h"]))
    if where == "x":  # the quantisation of a weight has no NaN
        q = _ops.gated_ffn_fp8(x, _ops.quant_ffn_weights_fp8(w1, w2, w3), act=act)
        assert torch.equal(torch.isnan(q), torch.isnan(ref["y"]))
