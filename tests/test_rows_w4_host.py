"""Host-only checks (no GPU) of the row dispatch / combine / gradient entry
points and the 4-bit-weight entry points: the oracles' gradients against
differences, the quantisation's error bound, and every refusal of the C ABI,
which returns before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from elastikernel_b200 import _lib, _ops
from elastikernel_b200._lib import lib
from oracle import rows as orows
from oracle import w4 as ow4


def _p(v: int = 256) -> ctypes.c_void_p:
    return ctypes.c_void_p(v)


# ------------------------------------------------------------------ oracles
def test_order_oracle_is_stable_and_drops():
    ids = np.array([[1, 0], [-1, 1], [0, 2]], np.int32)
    slots, rows, counts = orows.order(ids, 4)
    assert slots.tolist() == [1, 4, 0, 3, 5, 6]
    assert rows.tolist() == [2, 0, -1, 3, 1, 4]
    assert counts.tolist() == [2, 2, 1, 0]


def test_combine_gradient_against_differences():
    rng = np.random.default_rng(0)
    T, k, E, H = 5, 3, 4, 6
    ids = rng.integers(-1, E, (T, k)).astype(np.int32)
    _, sr, _ = orows.order(ids, E)
    y, w, d = rng.normal(size=(T * k, H)), rng.normal(size=(T, k)), rng.normal(size=(T, H))
    d_y, d_w = orows.combine_grad(y, sr, w, d)
    h = 1e-5

    def loss(y, w):
        return (orows.combine(y, sr, w) * d).sum()

    for i in np.ndindex(*y.shape):
        a, b = y.copy(), y.copy()
        a[i] += h
        b[i] -= h
        assert abs((loss(a, w) - loss(b, w)) / (2 * h) - d_y[i]) < 1e-8
    for i in np.ndindex(*w.shape):
        a, b = w.copy(), w.copy()
        a[i] += h
        b[i] -= h
        assert abs((loss(y, a) - loss(y, b)) / (2 * h) - d_w[i]) < 1e-8


def test_route_gradient_against_differences():
    rng = np.random.default_rng(1)
    T, E, k = 4, 7, 3
    z = rng.normal(size=(T, E))
    ids = np.argsort(-z, axis=1)[:, :k].astype(np.int32)
    d = rng.normal(size=(T, k))
    g = orows.route_grad(ids, orows.route_weights(z, ids), d, E)
    h = 1e-6
    for i in np.ndindex(T, E):
        a, b = z.copy(), z.copy()
        a[i] += h
        b[i] -= h
        num = ((orows.route_weights(a, ids) - orows.route_weights(b, ids)) * d).sum() / (2 * h)
        assert abs(num - g[i]) < 1e-8


def test_route_gradient_with_dropped_choices_against_differences():
    """softmax over the chosen logits -> some choices dropped -> weighted combine:
    the logits' gradient takes the routed ids, not those with -1 for the dropped."""
    rng = np.random.default_rng(2)
    T, E, k, H = 5, 6, 3, 4
    z, d = rng.normal(size=(T, E)), rng.normal(size=(T, H))
    ids = np.argsort(-z, axis=1)[:, :k].astype(np.int32)
    kept = ids.copy()
    kept[[0, 1, 1, 3], [1, 0, 2, 2]] = -1
    _, sr, _ = orows.order(kept, E)
    y = rng.normal(size=(T * k, H))

    def loss(z):
        return (orows.combine(y, sr, orows.route_weights(z, ids)) * d).sum()

    w = orows.route_weights(z, ids)
    d_w = orows.combine_grad(y, sr, w, d)[1]
    g, masked = orows.route_grad(ids, w, d_w, E), orows.route_grad(kept, w, d_w, E)
    h = 1e-6
    for i in np.ndindex(T, E):
        a, b = z.copy(), z.copy()
        a[i] += h
        b[i] -= h
        assert abs((loss(a) - loss(b)) / (2 * h) - g[i]) < 1e-8
    assert np.abs(g.sum(axis=1)).max() < 1e-12  # a softmax's gradient
    assert np.abs(masked[[0, 1, 3]].sum(axis=1)).min() > 1e-3  # which the masked ids lose


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("K,group", [(128, 32), (200, 64), (257, 128), (1, 32)])
def test_quantisation_error_is_half_a_step(symmetric, K, group):
    """|w - value| <= s / 2 plus the clamp's excess: rounding s down by half an ulp
    of bf16 (2^-8) leaves up to 15 * 2^-8 of a step past the last code, and the
    rounded minimum up to 2^-8 |min| below the first."""
    g = torch.Generator().manual_seed(K)
    w = torch.randn((9, K), generator=g)
    codes, s, m = ow4.quantise(w, group, symmetric, torch.bfloat16)
    v = ow4.values(codes, s, m, K, group)
    step = s.double().numpy()[:, np.arange(K) // group]
    slack = 0 if m is None else np.abs(m.double().numpy()[:, np.arange(K) // group]) * 2.0 ** -8
    assert (np.abs(v - w.double().numpy()) <= step * (0.5 + 15 * 2.0 ** -8) + slack + 1e-6).all()


# ------------------------------------------------------------------ refusals
def _bad(rc: int, text: str) -> None:
    assert rc == _lib.EK_ERR_INVALID
    assert text in _lib.last_error()


def test_dispatch_refusals():
    f = lib().ek_moe_dispatch
    n = None
    _bad(f(_p(), 4, 2, 0, n, 0, 0, _p(), _p(), _p(), _p(), n, _p(), n), "1 <= E")
    _bad(f(_p(), 4, 2, 1025, n, 0, 0, _p(), _p(), _p(), _p(), n, _p(), n), "1 <= E")
    _bad(f(_p(), -1, 2, 8, n, 0, 0, _p(), _p(), _p(), _p(), n, _p(), n), "bad sizes")
    _bad(f(_p(), 4, 0, 8, n, 0, 0, _p(), _p(), _p(), _p(), n, _p(), n), "bad sizes")
    _bad(f(_p(), 4, 2, 8, _p(), 0, 0, _p(), _p(), _p(), _p(), _p(), _p(), n), "bad sizes")
    _bad(f(_p(), 4, 2, 8, _p(), 16, 2, _p(), _p(), _p(), _p(), _p(), _p(), n), "bad sizes or type")
    _bad(f(_p(), 1 << 28, 8, 8, n, 0, 0, _p(), _p(), _p(), _p(), n, _p(), n), "too many slots")
    _bad(f(n, 4, 2, 8, n, 0, 0, _p(), _p(), _p(), _p(), n, _p(), n), "null pointer")
    _bad(f(_p(), 4, 2, 8, n, 0, 0, _p(), n, _p(), _p(), n, _p(), n), "null pointer")
    _bad(f(_p(), 4, 2, 8, _p(), 16, 0, _p(), _p(), _p(), _p(), n, _p(), n), "null pointer")
    _bad(f(_p(), 4, 2, 8, _p(257), 16, 0, _p(), _p(), _p(), _p(), _p(), _p(), n), "aligned")


def test_row_gradient_refusals():
    L = lib()
    n = None
    _bad(L.ek_moe_dispatch_grad(_p(), _p(), 4, 2, 8, 0, 0, _p(), n), "bad sizes")
    _bad(L.ek_moe_dispatch_grad(_p(), n, 4, 2, 8, 16, 0, _p(), n), "null pointer")
    _bad(L.ek_moe_dispatch_grad(_p(258), _p(), 4, 2, 8, 16, 3, _p(), n), "aligned")
    _bad(L.ek_moe_combine_weighted(_p(), _p(), _p(), 4, 2, -1, 16, 0, _p(), n), "bad sizes")
    _bad(L.ek_moe_combine_weighted(_p(), _p(), n, 4, 2, 8, 16, 0, _p(), n), "null pointer")
    _bad(L.ek_moe_combine_weighted(_p(), _p(), _p(), 4, 2, 8, 16, 7, _p(), n), "type")
    _bad(L.ek_moe_combine_weighted_grad(_p(), _p(), _p(), _p(), n, 4, 2, 8, 16, 0, _p(), _p(), n), "null pointer")
    _bad(L.ek_moe_combine_weighted_grad(_p(), _p(), _p(), _p(), _p(), 4, 2, 8, 16, 0, _p(), n, n), "null pointer")
    _bad(L.ek_moe_route_grad(_p(), _p(), _p(), 4, 0, 2, _p(), n), "bad sizes")
    _bad(L.ek_moe_route_grad(_p(), _p(), n, 4, 8, 2, _p(), n), "null pointer")
    # an empty batch is nothing to do
    assert L.ek_moe_dispatch_grad(n, n, 0, 2, 0, 16, 0, n, n) == _lib.EK_OK
    assert L.ek_moe_combine_weighted(n, n, n, 0, 2, 0, 16, 0, n, n) == _lib.EK_OK
    assert L.ek_moe_route_grad(n, n, n, 0, 8, 2, n, n) == _lib.EK_OK


def test_w4_refusals():
    L = lib()
    n = None
    _bad(L.ek_quant_w4(_p(), 0, 8, 64, 48, 1, 0, _p(), _p(), n, n), "group")
    _bad(L.ek_quant_w4(_p(), 2, 8, 64, 32, 1, 0, _p(), _p(), n, n), "types")
    _bad(L.ek_quant_w4(_p(), 0, 8, 64, 32, 1, 3, _p(), _p(), n, n), "types")
    _bad(L.ek_quant_w4(_p(), 0, 8, 64, 32, 0, 0, _p(), _p(), n, n), "null pointer")
    _bad(L.ek_quant_w4(_p(), 0, 8, 0, 32, 1, 0, _p(), _p(), n, n), "K >= 1")
    _bad(L.ek_dequant_w4(_p(264), _p(), n, 8, 64, 32, 0, _p(), n), "16-byte aligned")
    _bad(L.ek_dequant_w4(_p(), _p(), n, 8, 64, 32, 0, n, n), "null pointer")
    def gemm(A=_p(), codes=_p(), scales=_p(), C=_p(), M=1, N=8, K=64, group=32, dtype=0, ws=_p(), size=1 << 40):
        return L.ek_gemm_w4(A, codes, scales, n, C, M, N, K, group, dtype, 148, ws, size, n)

    _bad(gemm(group=16), "group")
    _bad(gemm(M=-1), "bad sizes")
    _bad(gemm(dtype=3), "type")
    _bad(gemm(A=n), "null pointer")
    _bad(gemm(ws=n), "null pointer")
    _bad(gemm(codes=_p(264)), "16-byte aligned")
    _bad(gemm(scales=_p(257)), "misaligned")
    _bad(gemm(C=_p(257)), "aligned")
    _bad(gemm(size=L.ek_gemm_w4_workspace_bytes(1, 8, 64, 148) - 1), "workspace")
    _bad(gemm(ws=_p(264)), "workspace")
    _bad(gemm(K=(1 << 28) + 1), "2^28")
    _bad(gemm(N=1 << 24, K=1 << 13), "2^32 scales")
    assert L.ek_gemm_w4_workspace_bytes(1, 8, (1 << 31) - 1, 148) == _ops._SIZE_MAX
    assert gemm(M=0, A=n) == _lib.EK_OK
    assert L.ek_gemm_w4_workspace_bytes(0, 8, 64, 148) == 0
    assert L.ek_gemm_w4_workspace_bytes(1, 8, 0, 148) == L.ek_gemm_w4_workspace_bytes(1, 8, 64, 0) == _ops._SIZE_MAX


def test_moe_w4_refusals():
    L = lib()
    n = None
    big = 1 << 40

    def gate_up(x=_p(), x_rows=8, slots=n, topk=1, c1=_p(), m1=n, c3=_p(), counts=_p(), act=_p(), dt=0, rows=8, E=4,
                H=64, I=32, group=32, ws=_p(), size=big):
        return L.ek_moe_gate_up_w4(x, x_rows, slots, topk, c1, _p(), m1, c3, _p(), n, counts, act, dt, rows, E, H, I,
                                   group, 148, ws, size, n)

    _bad(gate_up(E=0), "bad sizes")
    _bad(gate_up(E=1025), "bad sizes")
    _bad(gate_up(H=(1 << 28) + 1, E=1), "bad sizes")
    _bad(gate_up(E=1024, I=1 << 20, H=1 << 17), "2^32 scales")
    _bad(gate_up(x_rows=4), "do not match")
    _bad(gate_up(slots=_p(), topk=0), "do not match")
    _bad(gate_up(slots=_p(), topk=2), "do not match")
    _bad(gate_up(dt=1), "bf16 or fp32")
    _bad(gate_up(group=100), "group")
    _bad(gate_up(m1=_p()), "null pointer")
    _bad(gate_up(counts=n), "null pointer")
    _bad(gate_up(ws=n), "null pointer")
    _bad(gate_up(c3=_p(264)), "16-byte aligned")
    _bad(gate_up(act=_p(258), dt=3), "aligned")
    _bad(gate_up(size=16), "workspace")
    assert gate_up(rows=0, x_rows=0) == _lib.EK_OK

    def down(act=_p(), adt=0, codes=_p(), counts=_p(), y=_p(), ydt=3, rows=8, E=4, H=64, size=big):
        return L.ek_moe_down_w4(act, adt, codes, _p(), n, counts, y, ydt, rows, E, H, 32, 32, 148, _p(), size, n)

    _bad(down(counts=n), "null pointer")
    _bad(down(H=0), "bad sizes")
    _bad(down(adt=2), "bf16 or fp32")
    _bad(down(ydt=1), "bf16 or fp32")
    _bad(down(y=_p(258)), "aligned")
    _bad(down(size=0), "workspace")
    assert down(rows=0) == _lib.EK_OK

    def experts(x=_p(), T=4, topk=2, ids=_p(), slots=_p(), rows=_p(), counts=_p(), c2=_p(), m3=n, out=_p(), E=4,
                group=32, size=big):
        return L.ek_moe_experts_w4(x, T, topk, ids, _p(), slots, rows, counts, _p(), _p(), n, _p(), _p(), m3, c2, _p(),
                                   n, out, E, 64, 32, group, 148, _p(), size, n)

    _bad(experts(topk=0), "bad sizes")
    _bad(experts(T=-1), "bad sizes")
    _bad(experts(T=1 << 24), "too many rows")
    _bad(experts(ids=n), "null pointer")
    _bad(experts(rows=n), "null pointer")
    _bad(experts(counts=n), "null pointer")
    _bad(experts(m3=_p()), "null pointer")
    _bad(experts(c2=_p(8)), "16-byte aligned")
    _bad(experts(out=_p(257)), "aligned")
    _bad(experts(size=8), "workspace")
    assert experts(T=0) == _lib.EK_OK
    assert L.ek_moe_w4_workspace_bytes(4, 8, 4, 64, 32, 0) == _ops._SIZE_MAX

    def fused(x=_p(), logits=_p(), T=4, topk=2, c1=_p(), m2=n, out=_p(), E=4, group=32, ws=_p(), size=big):
        return L.ek_fused_moe_w4(x, logits, T, topk, c1, _p(), n, _p(), _p(), n, _p(), _p(), m2, out, E, 64, 32, group,
                                 148, ws, size, n)

    _bad(fused(E=257), "1 <= E <= 256")
    _bad(fused(topk=5), "1 <= k")
    _bad(fused(topk=9, E=16), "1 <= k")
    _bad(fused(T=-1), "bad sizes")
    _bad(fused(T=1 << 24), "too many rows")
    _bad(fused(logits=n), "null pointer")
    _bad(fused(ws=n), "null pointer")
    _bad(fused(logits=_p(258)), "aligned")
    _bad(fused(c1=_p(8)), "16-byte aligned")
    _bad(fused(group=8), "group")
    _bad(fused(size=L.ek_fused_moe_w4_workspace_bytes(4, 2, 4, 64, 32, 148) - 1), "workspace")
    assert fused(T=0) == _lib.EK_OK
    assert L.ek_fused_moe_w4_workspace_bytes(4, 9, 16, 64, 32, 148) == _ops._SIZE_MAX


def test_front_end_refuses_cpu_tensors():
    ids = torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.moe_dispatch(torch.zeros((2, 8)), ids, 4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.quant_w4(torch.zeros((2, 64)))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.moe_route_grad(ids, torch.zeros((2, 2)), torch.zeros((2, 2)), 4)


def test_front_end_refuses_a_permutation_without_slot_rows():
    perm = {"sorted_slots": None, "T": 2, "topk": 2}
    with pytest.raises(RuntimeError, match="moe_dispatch"):
        _ops.moe_dispatch_grad(perm, torch.zeros((4, 8)))


@pytest.mark.parametrize("change,text", [
    (dict(group=16), "group"), (dict(K=65), "codes"), (dict(codes=torch.zeros((4, 32), dtype=torch.int8)), "codes"),
    (dict(scales=torch.zeros((4, 2))), "scales"), (dict(scales=torch.zeros((4, 3), dtype=torch.bfloat16)), "scales"),
    (dict(scales=torch.zeros((4, 2), dtype=torch.float16)), "must be torch.bfloat16"),
    (dict(mins=torch.zeros((4, 1), dtype=torch.bfloat16)), "mins"),
    (dict(codes=torch.zeros((32, 4), dtype=torch.uint8).t()), "contiguous")])
def test_front_end_checks_the_weight(change, text):
    qw = dict(codes=torch.zeros((4, 32), dtype=torch.uint8), scales=torch.zeros((4, 2), dtype=torch.bfloat16),
              mins=None, K=64, group=32)
    qw.update(change)
    with pytest.raises(RuntimeError, match=text):
        _ops.gemm_w4(torch.zeros((1, 64), dtype=torch.bfloat16), qw)


def test_route_gradient_refuses_more_experts_than_its_counters_hold():
    f = lib().ek_moe_route_grad
    _bad(f(_p(), _p(), _p(), 4, (1 << 30) + 1, 2, _p(), None), "2^30")
    _bad(f(_p(), _p(), _p(), 4, (1 << 31) - 1, 40, _p(), None), "2^30")
    assert f(None, None, None, 0, 1 << 30, 2, None, None) == _lib.EK_OK


@pytest.mark.parametrize("H", [(1 << 30) + 1, (1 << 31) - 1])
@pytest.mark.parametrize("dtype", [_lib.EK_DTYPE_BF16, _lib.EK_DTYPE_FP32])
def test_rows_longer_than_their_counters_are_refused(H, dtype):
    L = lib()
    n = None
    _bad(L.ek_moe_dispatch(_p(), 1, 1, 8, _p(), H, dtype, _p(), _p(), _p(), _p(), _p(), _p(), n), "2^30 elements")
    _bad(L.ek_moe_dispatch_grad(_p(), _p(), 1, 1, 1, H, dtype, _p(), n), "2^30 elements")
    _bad(L.ek_moe_combine_weighted(_p(), _p(), _p(), 1, 1, 1, H, dtype, _p(), n), "2^30 elements")
    _bad(L.ek_moe_combine_weighted_grad(_p(), _p(), _p(), _p(), _p(), 1, 1, 1, H, dtype, _p(), _p(), n), "2^30 elements")


def test_front_end_refuses_sizes_past_32_bits(monkeypatch):
    """They would wrap to small ones on their way into the library (2^32 + 8 to 8).
    Shapes alone: expanded tensors of one element."""
    monkeypatch.setattr(_ops, "_require_cuda", lambda *t: torch.device("cuda", 0))
    one, big = torch.zeros(1, dtype=torch.bfloat16), (1 << 32) + 8
    for shape in ((1, big), (big, 1), (1, (1 << 30) + 1)):
        with pytest.raises(RuntimeError, match="2.30 elements"):
            _ops._check_rows("x", one.expand(shape))
    ids = torch.zeros(1, dtype=torch.int32)
    for shape in ((big, 1), (1, big), (1 << 20, 1 << 11)):
        monkeypatch.setattr(_ops, "_contig", lambda *a: None)
        with pytest.raises(RuntimeError, match="too many slots"):
            _ops.moe_dispatch(None, ids.expand(shape), 4)
    for E in (big, 4 - (1 << 32)):
        with pytest.raises(RuntimeError, match="1 <= E <= 1024"):
            _ops.moe_dispatch(None, ids.view(1, 1), E)
    w = torch.zeros((1, 1))
    with pytest.raises(RuntimeError, match="2.30"):
        _ops.moe_route_grad(ids.view(1, 1), w, w, big)
    with pytest.raises(RuntimeError, match="2.28"):
        _ops.quant_w4(one.expand(1, big))
    qw = dict(codes=torch.zeros((4, 32), dtype=torch.uint8), scales=torch.zeros((4, 1), dtype=torch.bfloat16), mins=None,
              K=64, group=64)
    with pytest.raises(RuntimeError, match="2.28"):
        _ops._check_w4("w", dict(qw, K=big))
    with pytest.raises(RuntimeError, match="2.31 rows"):
        _ops.gemm_w4(one.expand(big, 64), qw)
