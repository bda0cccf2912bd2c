"""Host-only checks (no GPU) of the dense feed-forward operators: the oracle's gradient
against differences and against autograd, its quantisation, and every refusal of the
C ABI and of the front end, which return before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from elastikernel_b200 import _lib, _ops
from elastikernel_b200._lib import lib
from oracle import ffn as off
from oracle import fp8 as ofp8

BIG = 1 << 40


def _p(v: int = 256) -> ctypes.c_void_p:
    return ctypes.c_void_p(v)


def _bad(rc: int, text: str) -> None:
    assert rc == _lib.EK_ERR_INVALID and text in _lib.last_error(), _lib.last_error()


def _case(T=5, H=6, I=7, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g, dtype=torch.float64) for s in ((T, H), (I, H), (H, I), (I, H), (T, H))]


# ------------------------------------------------------------------ oracle
@pytest.mark.parametrize("act", list(_ops.GATES))
def test_gradient_against_differences(act):
    *ts, d = _case()
    h = off.forward(*ts, act)["h"]
    grads = off.backward(*ts, h, d, act)
    step = 1e-5
    for i, name in enumerate(("x", "w1", "w2", "w3")):
        for at in np.ndindex(*ts[i].shape):
            up, dn = [t.clone() for t in ts], [t.clone() for t in ts]
            up[i][at] += step
            dn[i][at] -= step
            diff = ((off.forward(*up, act)["y"] - off.forward(*dn, act)["y"]) * d).sum() / (2 * step)
            assert abs(diff - grads[name][at]) < 1e-6


@pytest.mark.parametrize("act", list(_ops.GATES))
def test_gradient_against_autograd(act):
    *ts, d = _case(seed=1)
    leaves = [t.clone().requires_grad_() for t in ts]
    h1, h3 = leaves[0] @ leaves[1].T, leaves[0] @ leaves[3].T
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[act]
    ((f(h1) * h3) @ leaves[2].T).backward(d)
    grads = off.backward(*ts, torch.stack([h1, h3]).detach(), d, act)
    for name, leaf in zip(("x", "w1", "w2", "w3"), leaves):
        assert torch.allclose(grads[name], leaf.grad, rtol=1e-10, atol=1e-12)


def test_quantisation_is_the_library_s():
    """The oracle's rounding in 64 bits against the codes and scales of the fp8 oracle."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn((7, 300), generator=g).to(torch.bfloat16).float()
    x[2] = 0
    x[3, :128] *= 2.0 ** -20
    q, s = ofp8.quant_blocks(x, 1, 128)
    assert np.array_equal(ofp8.dequant_blocks(q, s, 1, 128).astype(np.float32),
                          off.e4m3_groups(x.double()).numpy().astype(np.float32))


# ------------------------------------------------------------------ the C ABI's refusals
def test_block_product_refusals():
    L = lib()

    def gemm(A=_p(), W=_p(), sa=_p(), sw=_p(), C=_p(), M=4, N=8, K=32, out=0, sms=148, ws=_p(), size=BIG):
        return L.ek_gemm_fp8_block(A, W, sa, sw, C, M, N, K, out, sms, ws, size, None)

    _bad(gemm(K=24), "multiple of 16")
    _bad(gemm(K=0), "multiple of 16")
    _bad(gemm(M=-1), "multiple of 16")
    _bad(gemm(out=2), "bf16, fp16 or fp32")
    for name in ("A", "W", "sa", "sw", "C"):
        _bad(gemm(**{name: None}), "null operand")
    _bad(gemm(A=_p(264)), "16-byte aligned")
    _bad(gemm(W=_p(264)), "16-byte aligned")
    _bad(gemm(ws=_p(264)), "16-byte aligned")
    _bad(gemm(sms=5000), "num_sms")
    _bad(gemm(size=64), "workspace")
    _bad(gemm(ws=None), "workspace")
    assert gemm(M=0, A=None) == gemm(N=0, W=None) == _lib.EK_OK
    f = L.ek_gemm_fp8_block_workspace_bytes
    assert f(1, 8, 24, 148) == f(-1, 8, 32, 148) == f(1, 8, 32, 0) == _ops._SIZE_MAX
    assert f(0, 8, 32, 148) == 0


def test_gated_ffn_refusals():
    L = lib()

    def ffn(x=_p(), w1=_p(), w2=_p(), w3=_p(), y=_p(), h=None, T=4, H=16, I=24, dtype=0, gate=0, sms=148, ws=_p(),
            size=BIG):
        return L.ek_gated_ffn(x, w1, w2, w3, y, h, T, H, I, dtype, gate, sms, ws, size, None)

    def grad(x=_p(), w1=_p(), w2=_p(), w3=_p(), h=_p(), d=_p(), dx=_p(), dw=_p(), dw2=_p(), T=4, H=16, I=24, dtype=0,
             gate=0, sms=148, ws=_p(), size=BIG):
        return L.ek_gated_ffn_grad(x, w1, w2, w3, h, d, dx, dw, dw2, T, H, I, dtype, gate, sms, ws, size, None)

    for f in (ffn, grad):
        _bad(f(H=12), "multiples of 8")
        _bad(f(I=0), "multiples of 8")
        _bad(f(T=-1), "multiples of 8")
        _bad(f(H=(1 << 28) + 8), "2^28")
        _bad(f(gate=3), "gate function")
        _bad(f(dtype=3), "bf16 or fp16")
        _bad(f(sms=5000), "num_sms")
        _bad(f(size=64), "workspace")
        for name in ("x", "w1", "w2", "w3", "ws"):
            _bad(f(**{name: None}), "null operand")
            _bad(f(**{name: _p(264)}), "16-byte aligned")
    _bad(ffn(y=None), "null operand")
    _bad(ffn(h=_p(264)), "16-byte aligned")
    for name in ("h", "d", "dx", "dw", "dw2"):
        _bad(grad(**{name: None}), "null operand")
        _bad(grad(**{name: _p(264)}), "16-byte aligned")
    assert ffn(T=0, x=None) == _lib.EK_OK
    for f in (L.ek_gated_ffn_workspace_bytes, L.ek_gated_ffn_grad_workspace_bytes):
        assert f(4, 12, 24, 148) == f(-1, 16, 24, 148) == f(4, 16, 24, 0) == _ops._SIZE_MAX
        assert f(0, 16, 24, 148) == 0
        assert f(1000, 1024, 2048, 148) >= 1000 * 2048 * 2


def test_gated_ffn_fp8_refusals():
    L = lib()

    def ffn(x=_p(), w1=_p(), w2=_p(), w3=_p(), s1=_p(), s2=_p(), s3=_p(), y=_p(), T=4, H=16, I=32, gate=0, sms=148,
            ws=_p(), size=BIG):
        return L.ek_gated_ffn_fp8(x, w1, w2, w3, s1, s2, s3, y, T, H, I, gate, sms, ws, size, None)

    _bad(ffn(H=24), "multiples of 16")
    _bad(ffn(gate=-1), "gate function")
    _bad(ffn(sms=5000), "num_sms")
    _bad(ffn(size=64), "workspace")
    for name in ("x", "w1", "w2", "w3", "s1", "s2", "s3", "y", "ws"):
        _bad(ffn(**{name: None}), "null operand")
    for name in ("x", "w1", "w2", "w3", "y", "ws"):
        _bad(ffn(**{name: _p(264)}), "16-byte aligned")
    assert ffn(T=0, x=None) == _lib.EK_OK
    f = L.ek_gated_ffn_fp8_workspace_bytes
    assert f(4, 24, 32, 148) == f(4, 16, 32, 2000) == _ops._SIZE_MAX and f(0, 16, 32, 148) == 0


def test_sizes_whose_last_tile_passes_an_int_are_refused():
    L, top = lib(), (1 << 31) - 1
    for n in (top - 254, top):
        _bad(L.ek_gemm_fp8_block(_p(), _p(), _p(), _p(), _p(), n, 16, 16, 0, 148, _p(), BIG, None), "2^31")
        _bad(L.ek_gemm_fp8_block(_p(), _p(), _p(), _p(), _p(), 16, n, 16, 0, 148, _p(), BIG, None), "2^31")
        _bad(L.ek_gated_ffn(*[_p()] * 6, n, 16, 16, 0, 0, 148, _p(), BIG, None), "2^31")
        _bad(L.ek_gated_ffn_grad(*[_p()] * 9, n, 16, 16, 0, 0, 148, _p(), BIG, None), "2^31")
        _bad(L.ek_gated_ffn_fp8(*[_p()] * 8, n, 16, 16, 0, 148, _p(), BIG, None), "2^31")
        assert L.ek_gated_ffn_workspace_bytes(n, 16, 16, 148) == _ops._SIZE_MAX
    _bad(L.ek_gemm_fp8_block(_p(), _p(), _p(), _p(), _p(), 16, 16, top - 15, 0, 148, _p(), BIG, None), "2^28")
    assert L.ek_gated_ffn_workspace_bytes(top - 255, 16, 16, 148) < _ops._SIZE_MAX


@pytest.mark.parametrize("T,H,I", [(1, 8, 8), (64, 4096, 14336), (128, 256, 384), (129, 4096, 264), (4096, 4096, 14336)])
def test_workspaces_hold_any_smaller_partition(T, H, I):
    """A call sized for the whole device may run in a partition of it, for which the
    library plans anew: few tokens' segments then need no more, and tiles are cut into as
    many slices as the workspace holds, so its least part is what lies between the
    products."""
    L = lib()
    for f in (L.ek_gated_ffn_workspace_bytes, L.ek_gated_ffn_grad_workspace_bytes, L.ek_gated_ffn_fp8_workspace_bytes):
        most = f(T, H, I, 148)
        if f is L.ek_gated_ffn_fp8_workspace_bytes and (H % 16 or I % 16):
            assert most == _ops._SIZE_MAX
            continue
        assert T * I <= most < _ops._SIZE_MAX
        if T <= 64 and f is not L.ek_gated_ffn_grad_workspace_bytes:
            assert all(f(T, H, I, n) <= most for n in range(1, 148))


# ------------------------------------------------------------------ the front end's refusals
def _any_device(monkeypatch):
    monkeypatch.setattr(_ops, "_require_cuda", lambda *t: torch.device("cuda", 0))


F8, BF = torch.float8_e4m3fn, torch.bfloat16


def test_front_end_refuses_cpu_tensors():
    x = torch.zeros((2, 16), dtype=BF)
    w = torch.zeros((16, 16), dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.gated_ffn(x, w, w, w)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.gated_ffn_grad(x, w, w, w, torch.zeros((2, 2, 16), dtype=BF), x)
    q = w.to(F8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.gemm_fp8_block(x.to(F8), q, torch.ones((2, 1)), torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _ops.gated_ffn_fp8(x, dict(H=16, I=16, w1q=q, w2q=q, w3q=q, w1s=None, w2s=None, w3s=None))


@pytest.mark.parametrize("change,text", [
    (dict(a_q=torch.zeros((2, 32))), "a_q must be"), (dict(w_q=torch.zeros((8, 48), dtype=F8)), "w_q must be"),
    (dict(a_q=torch.zeros((2, 24), dtype=F8)), "multiple of 16"), (dict(a_q=torch.zeros((2, 0), dtype=F8)), "multiple of 16"),
    (dict(a_q=torch.zeros(32, dtype=F8)), "2-D"), (dict(a_scale=torch.ones((2, 2))), "a_scale must be"),
    (dict(a_scale=torch.ones((2, 1), dtype=BF)), "a_scale must be"), (dict(w_scale=torch.ones((2, 1))), "w_scale must be"),
    (dict(w_q=torch.zeros((32, 8), dtype=F8).t()), "contiguous"), (dict(dtype=torch.float64), "bf16, fp16 or fp32"),
    (dict(out=torch.zeros((2, 9))), "out must be"), (dict(out=torch.zeros((8, 2)).t()), "out must be")])
def test_front_end_checks_the_block_product(change, text, monkeypatch):
    _any_device(monkeypatch)
    args = dict(a_q=torch.zeros((2, 32), dtype=F8), w_q=torch.zeros((8, 32), dtype=F8), a_scale=torch.ones((2, 1)),
                w_scale=torch.ones((1, 1)))
    args.update(change)
    with pytest.raises(RuntimeError, match=text):
        _ops.gemm_fp8_block(**args)


@pytest.mark.parametrize("change,text", [
    (dict(x=torch.zeros((2, 16))), "bf16 or fp16"), (dict(x=torch.zeros((2, 12), dtype=BF)), "multiples of 8"),
    (dict(w1=torch.zeros((24, 16), dtype=torch.float16)), "w1 must be"), (dict(w2=torch.zeros((24, 16), dtype=BF)), "w2 must be"),
    (dict(w3=torch.zeros((16, 24), dtype=BF).t()), "contiguous"), (dict(act="relu"), "act must be"),
    (dict(x=torch.zeros(16, dtype=BF)), "must be")])
def test_front_end_checks_the_block(change, text, monkeypatch):
    _any_device(monkeypatch)
    args = dict(x=torch.zeros((2, 16), dtype=BF), w1=torch.zeros((24, 16), dtype=BF), w2=torch.zeros((16, 24), dtype=BF),
                w3=torch.zeros((24, 16), dtype=BF))
    args.update(change)
    with pytest.raises(RuntimeError, match=text):
        _ops.gated_ffn(**args)
    h, d = torch.zeros((2, 2, 24), dtype=BF), torch.zeros((2, 16), dtype=BF)
    with pytest.raises(RuntimeError, match=text):
        _ops.gated_ffn_grad(**args, h=h, d_out=d)


def test_front_end_checks_the_gradients_and_out(monkeypatch):
    _any_device(monkeypatch)
    x, w1, w2 = torch.zeros((2, 16), dtype=BF), torch.zeros((24, 16), dtype=BF), torch.zeros((16, 24), dtype=BF)
    h = torch.zeros((2, 2, 24), dtype=BF)
    with pytest.raises(RuntimeError, match="h must be"):
        _ops.gated_ffn_grad(x, w1, w2, w1, h[:1], x)
    with pytest.raises(RuntimeError, match="d_out must be"):
        _ops.gated_ffn_grad(x, w1, w2, w1, h, x.float())
    with pytest.raises(RuntimeError, match="out must be"):
        _ops.gated_ffn(x, w1, w2, w1, out=x.float())
    with pytest.raises(RuntimeError, match="out must be"):
        _ops.gated_ffn(x, w1, w2, w1, out=torch.zeros((16, 2), dtype=BF).t())
    with pytest.raises(RuntimeError, match="w1 and w3"):
        _ops.quant_ffn_weights_fp8(w1, w2, w1[:8])
    q = {n: torch.zeros(s, dtype=F8) for n, s in (("w1q", (32, 16)), ("w2q", (16, 32)), ("w3q", (32, 16)))}
    qw = dict(q, H=16, I=32, w1s=torch.ones((1, 1)), w2s=torch.ones((1, 1)), w3s=torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="bfloat16"):
        _ops.gated_ffn_fp8(x.half(), qw)
    with pytest.raises(RuntimeError, match="w2s must be"):
        _ops.gated_ffn_fp8(x, dict(qw, w2s=torch.ones((2, 1))))
    with pytest.raises(RuntimeError, match="the dict says"):
        _ops.gated_ffn_fp8(x, dict(qw, I=48))
    with pytest.raises(RuntimeError, match="out must be"):
        _ops.gated_ffn_fp8(x, qw, out=x[:1])


def test_front_end_refuses_sizes_past_32_bits(monkeypatch):
    """They would wrap to small ones on their way into the library."""
    _any_device(monkeypatch)
    one, big = torch.zeros(1, dtype=BF), (1 << 32) + 16
    w = torch.zeros((16, 16), dtype=BF)
    with pytest.raises(RuntimeError, match="2.31"):
        _ops.gated_ffn(one.expand(big, 16), w, w, w)
    with pytest.raises(RuntimeError, match="2.28"):
        _ops.gated_ffn(one.expand(1, big), w, w, w)
    q = one.to(F8)
    with pytest.raises(RuntimeError, match="2.28"):
        _ops.gemm_fp8_block(q.expand(1, big), w.to(F8), torch.ones((1, 1)), torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="2.31"):
        _ops.gemm_fp8_block(q.expand(big, 16), w.to(F8), torch.ones((1, 1)), torch.ones((1, 1)))
