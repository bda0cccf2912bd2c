"""Dense feed-forward operators on the GPU against the float64 oracle (oracle/ffn.py).

Tolerances (derived, not fitted). u = eps / 2 of a type bounds one rounding
relative to the value, `tiny` (half the smallest step) below its normal range.

* A sum of K products in fp32, in any order and with the tensor cores adding 16 (32
  in 8 bits) at a time and dropping bits below the largest of them, is off by at
  most (K/16 + 16) 2^-22 of S, the sum of the products' magnitudes; block scales
  add three roundings of 2^-24 per block, within the same bound. The result is
  rounded once: u |ref|.
* Values rounded between two products (activations a, gradients of the
  pre-activations) are off by at most u |a| + tiny each, independently and with
  either sign. What that leaves in a sum of a_i w_i has the scale
  R = sqrt(sum ((u |a_i| + tiny) w_i)^2), and by Hoeffding's inequality it passes 7.5 R
  with a probability of 2 exp(-28) = 1e-12 per element.
* A result past its type's range is infinite, as the rounding of the exact one is.
* The gate functions and their fp32 inputs add a relative 2^-14 of u's size at most
  to a rounded value, covered by taking 8 R for 7.5 R. For fp16 (u = 2^-11) the
  pre-activations' own bound, 2^-22 (K/16 + 16) S, is added through the weights.
* The 8-bit block: a code flips where an activation lies within its fp32 error of a
  border, which moves it by one step, at most 2^-3 of its value. Such borders are met
  with a probability below 2^-9 per code, so its root mean square error stays within
  u / sqrt 3 of the final rounding plus 2^-9: below u (2^-8) in all; per element three
  flips of the largest activation are allowed.
"""
from __future__ import annotations

import pytest
import torch

from elastikernel_b200 import _lib, _ops
from elastikernel_b200.green_ctx import create_sm_partition
from elastikernel_b200.sm_aware_matmul import call_sm_aware_fp8_block
from oracle import ffn as off

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
F8 = torch.float8_e4m3fn


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _acc(K):
    return (K / 16 + 16) * 2.0 ** -22


def _within(name, got, ref, bound):
    g = got.double()
    assert g.shape == ref.shape
    bound = bound + _u(got.dtype) * ref.abs() * (1 + 2.0 ** -6) + _tiny(got.dtype)
    # a value past the type's largest rounds to infinity of its sign; within the bound of
    # that border either side is right
    top = torch.finfo(got.dtype).max
    past, near = ref.abs() - bound > top, ref.abs() + bound > top
    assert (g[past] == torch.inf * ref[past].sign()).all(), f"{name}: overflow"
    assert torch.isfinite(g[~near]).all(), f"{name}: not finite"
    err = torch.where(near & ~torch.isfinite(g), torch.zeros_like(g), (g - ref).abs())
    over = (err - bound).max().item()
    assert over <= 0, f"{name}: {over:.3e} over its bound (largest error {err.max().item():.3e})"


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(g, R, K):
    """e4m3 values over the type's whole range, zeros and subnormals among them."""
    v = torch.randn((R, K), generator=g, device="cuda") * torch.exp2(
        torch.randint(-6, 6, (R, K), generator=g, device="cuda").float())
    return v.clamp(-448, 448).to(F8)


def _scales(g, *shape):
    return torch.exp(torch.randn(shape, generator=g, device="cuda"))


# ------------------------------------------------------------------ block-scaled product
def _block_case(M, N, K, seed=0):
    g = _gen(seed + M + 7 * N + 13 * K)
    a, w = _codes(g, M, K), _codes(g, N, K)
    return a, w, _scales(g, M, -(-K // 128)), _scales(g, -(-N // 128), -(-K // 128))


def _block_check(out, a, w, sa, sw):
    va, vw = off.expand(a, sa, 1), off.expand(w, sw, 128)
    _within("C", out, va @ vw.T, _acc(a.shape[1]) * (va.abs() @ vw.abs().T))


@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 128, 129, 256, 257, 400])
@pytest.mark.parametrize("N,K,dtype", [(1, 16, F32), (77, 144, BF), (128, 128, FP), (130, 1040, F32), (520, 2064, BF),
                                       (1000, 512, BF)])
def test_block_product(M, N, K, dtype, cuda_dev):
    a, w, sa, sw = _block_case(M, N, K)
    _block_check(_ops.gemm_fp8_block(a, w, sa, sw, dtype=dtype), a, w, sa, sw)


@pytest.mark.parametrize("M,N,K", [(3, 40000, 128), (128, 24, 16384), (300, 24, 16384), (2500, 300, 96), (1500, 2600, 640)])
def test_block_product_long_axes(M, N, K, cuda_dev):
    a, w, sa, sw = _block_case(M, N, K)
    _block_check(_ops.gemm_fp8_block(a, w, sa, sw, dtype=F32), a, w, sa, sw)


@pytest.mark.parametrize("M", [5, 200])
def test_block_product_is_exact_on_integers(M, cuda_dev):
    """Small integers under power-of-two scales: every partial sum is exact."""
    g = _gen(M)
    N, K = 270, 400
    a = torch.randint(-8, 9, (M, K), generator=g, device="cuda").float().to(F8)
    w = torch.randint(-8, 9, (N, K), generator=g, device="cuda").float().to(F8)
    sa = torch.exp2(torch.randint(-2, 3, (M, 4), generator=g, device="cuda").float())
    sw = torch.exp2(torch.randint(-2, 3, (3, 4), generator=g, device="cuda").float())
    ref = off.expand(a, sa, 1) @ off.expand(w, sw, 128).T
    assert torch.equal(_ops.gemm_fp8_block(a, w, sa, sw, dtype=F32).double(), ref)
    for t in (BF, FP):
        assert torch.equal(_ops.gemm_fp8_block(a, w, sa, sw, dtype=t), ref.to(t))


@pytest.mark.parametrize("M", [7, 300])
def test_block_product_quantised_inputs(M, cuda_dev):
    g = _gen(3)
    x = torch.randn((M, 1500 // 16 * 16), generator=g, device="cuda").to(BF)
    wt = torch.randn((333, x.shape[1]), generator=g, device="cuda").to(BF)
    a, sa = _ops.quant_e4m3(x, block=(1, 128))
    w, sw = _ops.quant_e4m3(wt, block=(128, 128))
    _block_check(_ops.gemm_fp8_block(a, w, sa, sw), a, w, sa, sw)


@pytest.mark.parametrize("M", [4, 260])
def test_block_product_rows_do_not_mix(M, cuda_dev):
    a, w, sa, sw = _block_case(M, 300, 272)
    ref = _ops.gemm_fp8_block(a, w, sa, sw, dtype=F32)
    bad = a.float()
    bad[1, 5] = float("nan")
    sb, sv = sa.clone(), sw.clone()
    sb[2, 1] = float("inf")
    sv[1, 0] = float("nan")
    got = _ops.gemm_fp8_block(bad.to(F8), w, sb, sv, dtype=F32)
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(got[keep][:, :128], ref[keep][:, :128])
    assert torch.equal(got[keep][:, 256:], ref[keep][:, 256:])
    assert torch.isnan(got[1]).all() and torch.isnan(got[:, 128:256]).all()
    assert not torch.isfinite(got[2]).any()
    zero = _ops.gemm_fp8_block(a, w, torch.zeros_like(sa), sw, dtype=F32)
    assert (zero == 0).all()


@pytest.mark.parametrize("M", [20, 300])
@pytest.mark.parametrize("N", [256, 301])
def test_block_product_misaligned_views_and_guards(M, N, cuda_dev):
    a, w, sa, sw = _block_case(M, N, 160)
    ref = _ops.gemm_fp8_block(a, w, sa, sw)
    mis = []
    for t in (a, w):
        flat = torch.empty(t.numel() + 1, dtype=torch.uint8, device="cuda")
        flat[1:] = t.view(torch.uint8).reshape(-1)
        mis.append(flat[1:].view(F8).view(t.shape))
    for t in (sa, sw):
        flat = torch.empty(t.numel() + 1, device="cuda")
        flat[1:] = t.reshape(-1)
        mis.append(flat[1:].view(t.shape))
    guard = torch.full((M * N + 9,), 7.0, dtype=BF, device="cuda")
    out = guard[1:1 + M * N].view(M, N)
    assert _ops.gemm_fp8_block(*mis, out=out) is out
    assert torch.equal(out, ref) and guard[0] == 7 and (guard[1 + M * N:] == 7).all()


@pytest.mark.parametrize("num_sms", [1, 2, 3, 16, 50, 148, 300])
@pytest.mark.parametrize("M,N,K", [(9, 600, 784), (100, 2100, 1040), (300, 700, 2064)])
def test_block_product_planned_for_any_size(M, N, K, num_sms, cuda_dev):
    """Other runs, tiles and slices of K: the same product."""
    a, w, sa, sw = _block_case(M, N, K)
    _block_check(_ops.gemm_fp8_block(a, w, sa, sw, dtype=F32, num_sms=num_sms), a, w, sa, sw)


def test_block_product_empty(cuda_dev):
    a, w, sa, sw = _block_case(4, 5, 32)
    assert _ops.gemm_fp8_block(a[:0], w, sa[:0], sw).shape == (0, 5)
    assert _ops.gemm_fp8_block(a, w[:0], sa, sw[:0]).shape == (4, 0)


# ------------------------------------------------------------------ gated block
def _ffn_case(T, H, I, dtype, seed=0, scale=1.0):
    g = _gen(seed + T + 3 * H + 5 * I)

    def r(*s, by=1.0):
        return (torch.randn(s, generator=g, device="cuda") * by).to(dtype)

    return (r(T, H, by=scale), r(I, H, by=2.0 * H ** -0.5), r(H, I, by=I ** -0.5), r(I, H, by=H ** -0.5))


def _rounded(a, w, dtype):
    """8 R of rounded values a [.., K] through w [K, ..]."""
    return 8 * ((_u(dtype) * a.abs() + _tiny(dtype)).square() @ w.square()).sqrt()


def _forward_bound(x, w1, w2, w3, r, act):
    """(bound of h, bound of y)"""
    X, W1, W2, W3 = (t.double() for t in (x, w1, w2, w3))
    H, I = X.shape[1], W1.shape[0]
    s1, s3 = X.abs() @ W1.abs().T, X.abs() @ W3.abs().T
    da = _acc(H) * (s1 * (off.slope(r["h"][0], act) * r["h"][1]).abs() + s3 * off.gate(r["h"][0], act).abs())
    da = da + 2.0 ** -20 * r["h"].abs().prod(dim=0)  # the gate function's own fp32 error
    return (_acc(H) * torch.stack([s1, s3]),
            _rounded(r["a"], W2.T, x.dtype) + (da + _acc(I) * r["a"].abs()) @ W2.abs().T)


def _check_grads(x, w1, w2, w3, h, act, num_sms=None, d_out=None, got=None):
    (T, H), I, dtype = x.shape, w1.shape[0], x.dtype
    if d_out is None:
        d_out = (torch.randn((T, H), generator=_gen(5), device="cuda") * 0.5).to(dtype)
    r = off.backward(x, w1, w2, w3, h, d_out, act)
    X, W1, W2, W3, D = (t.double() for t in (x, w1, w2, w3, d_out))
    hd = h.double()
    f, df = off.gate(hd[0], act), off.slope(hd[0], act)
    e_da = _acc(H) * (D.abs() @ W2.abs())  # error of da
    eps = 2.0 ** -19                        # of the gate function and the products beside it
    e1 = e_da * (hd[1] * df).abs() + eps * (r["da"] * hd[1]).abs()
    e3 = e_da * f.abs() + eps * (r["da"] * hd[0]).abs()
    ea = eps * (hd[0] * hd[1]).abs()
    if got is None:
        got = _ops.gated_ffn_grad(x, w1, w2, w3, h, d_out, act=act, num_sms=num_sms)
    bx = torch.sqrt(_rounded(r["d1"], W1, dtype) ** 2 + _rounded(r["d3"], W3, dtype) ** 2)
    _within("d_x", got[0], r["x"], bx + (e1 + _acc(2 * I) * r["d1"].abs()) @ W1.abs() +
            (e3 + _acc(2 * I) * r["d3"].abs()) @ W3.abs())
    for name, at, d, e in (("w1", 1, r["d1"], e1), ("w3", 3, r["d3"], e3)):
        _within("d_" + name, got[at], r[name], _rounded(d.T, X, dtype) + (e + _acc(T) * d.abs()).T @ X.abs())
    _within("d_w2", got[2], r["w2"], _rounded(r["a"].T, D, dtype).T + D.abs().T @ (ea + _acc(T) * r["a"].abs()))


def _check_fp8(x, w1, w2, w3, act, y=None):
    I = w1.shape[0]
    qw = _ops.quant_ffn_weights_fp8(w1, w2, w3)
    W = {n: off.expand(qw[n + "q"], qw[n + "s"], 128) for n in ("w1", "w2", "w3")}
    r = off.forward_fp8(x, W["w1"], W["w2"], W["w3"], act)
    y = _ops.gated_ffn_fp8(x, qw, act=act) if y is None else y
    flips = 3 * 2.0 ** -3 * r["a"].abs().amax(dim=1, keepdim=True) * W["w2"].abs().amax(dim=1)
    _within("y", y, r["y"], flips + _acc(I) * (r["aq"].abs() @ W["w2"].abs().T))
    rms = (y.double() - r["y"]).square().mean().sqrt() / r["y"].square().mean().sqrt().clamp(min=1e-30)
    assert rms <= _u(BF)
    return y


SIZES = [(1, 8, 8), (2, 136, 72), (16, 64, 256), (17, 1032, 520), (33, 256, 128), (64, 72, 1000), (65, 520, 264),
         (128, 256, 384), (129, 256, 384), (200, 8, 1016), (256, 1032, 136), (257, 136, 72), (600, 320, 712)]


@pytest.mark.parametrize("T,H,I", SIZES)
@pytest.mark.parametrize("dtype,act", [(BF, "silu"), (FP, "gelu"), (FP, "gelu_tanh"), (BF, "gelu"), (FP, "silu")])
def test_gated_ffn(T, H, I, dtype, act, cuda_dev):
    x, w1, w2, w3 = _ffn_case(T, H, I, dtype)
    r = off.forward(x, w1, w2, w3, act)
    bh, by = _forward_bound(x, w1, w2, w3, r, act)
    y = _ops.gated_ffn(x, w1, w2, w3, act=act)
    _within("y", y, r["y"], by)
    y2, h = _ops.gated_ffn(x, w1, w2, w3, act=act, save=True)
    assert torch.equal(y, y2)
    _within("h", h, r["h"], bh)


@pytest.mark.parametrize("T,H,I", SIZES + [(2000, 64, 40), (300, 2048, 4104)])
@pytest.mark.parametrize("dtype,act", [(BF, "silu"), (FP, "gelu"), (BF, "gelu_tanh")])
def test_gated_ffn_grad(T, H, I, dtype, act, cuda_dev):
    x, w1, w2, w3 = _ffn_case(T, H, I, dtype)
    _check_grads(x, w1, w2, w3, off.forward(x, w1, w2, w3, act)["h"].to(dtype), act)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradient_against_differences(act, cuda_dev):
    """The kernels' gradient of sum(y * d) against central differences of the kernels'
    own forward pass: a step of 1/8 in one weight moves the sum by grad / 4, in
    integers and powers of two that 16 bits hold, so what is left is the rounding of
    a and y (relative 2 u) and the third derivative's step^2."""
    T, H, I = 40, 64, 96
    x, w1, w2, w3 = _ffn_case(T, H, I, FP)
    d = torch.randn((T, H), generator=_gen(9), device="cuda").to(FP)
    _, h = _ops.gated_ffn(x, w1, w2, w3, act=act, save=True)
    grads = _ops.gated_ffn_grad(x, w1, w2, w3, h, d, act=act)
    ts = [x, w1, w2, w3]
    for i, at in ((0, (3, 5)), (1, (7, 11)), (2, (13, 17)), (3, (19, 23))):
        step = 1 / 64

        def loss(sign):
            moved = [t.clone() for t in ts]
            moved[i][at] += sign * step
            moved = [m.double() for m in moved]
            real = (moved[i][at] - ts[i][at].double()).item()
            return (off.forward(*moved, act)["y"] * d.double()).sum().item(), real

        (up, su), (dn, sd) = loss(1), loss(-1)
        diff = (up - dn) / (su - sd)
        scale = grads[i].double().square().mean().sqrt().item()
        # rounding of h, dh, a: each relative u of terms whose sum has this scale; the
        # difference's own error: step^2 / 6 of a third derivative of the same scale
        assert abs(grads[i][at].item() - diff) <= 16 * _u(FP) * scale + 4 * step ** 2 * scale


@pytest.mark.parametrize("T,H,I", [(150, 4096, 264), (200, 2056, 136), (140, 1544, 72)])
@pytest.mark.parametrize("dtype,act", [(BF, "gelu"), (FP, "silu"), (BF, "gelu_tanh")])
def test_gate_cut_along_k(T, H, I, dtype, act, cuda_dev):
    """Few tiles over a long axis: the gate functions and their gradient work on summed
    slices (in 8 bits with the quantisation)."""
    x, w1, w2, w3 = _ffn_case(T, H, I, dtype)
    r = off.forward(x, w1, w2, w3, act)
    bh, by = _forward_bound(x, w1, w2, w3, r, act)
    y, h = _ops.gated_ffn(x, w1, w2, w3, act=act, save=True)
    _within("y", y, r["y"], by)
    _within("h", h, r["h"], bh)
    _check_grads(x, w1, w2, w3, r["h"].to(dtype), act)
    if dtype == BF:
        I16 = I // 16 * 16
        H16 = H // 16 * 16
        _check_fp8(*(t.contiguous() for t in (x[:, :H16], w1[:I16, :H16], w2[:H16, :I16], w3[:I16, :H16])), act)


@pytest.mark.parametrize("num_sms", [1, 2, 6, 16, 50, 148, 300])
@pytest.mark.parametrize("T,H,I", [(520, 776, 1288), (70, 264, 2504)])
def test_gated_ffn_planned_for_any_size(T, H, I, num_sms, cuda_dev):
    """Other numbers of pairs deal the gradients' units out otherwise, none left out."""
    x, w1, w2, w3 = _ffn_case(T, H, I, BF)
    r = off.forward(x, w1, w2, w3, "silu")
    _within("y", _ops.gated_ffn(x, w1, w2, w3, num_sms=num_sms), r["y"], _forward_bound(x, w1, w2, w3, r, "silu")[1])
    _check_grads(x, w1, w2, w3, r["h"].to(BF), "silu", num_sms)


def test_extreme_activations(cuda_dev):
    """Pre-activations far past where the gate saturates: no NaN from inf * 0."""
    for T in (3, 140):
        x = torch.ones((T, 8), device="cuda", dtype=BF)
        w1 = torch.zeros((16, 8), device="cuda", dtype=BF)
        w1[:, 0] = torch.tensor([0., -1e30, 1e30, -3e4, 3e4, -100, 100, -20, 20, -1e-30, 1e-30, 5, -5, 30, -30, 1.0])
        w3 = torch.zeros_like(w1)
        w3[:, 1] = 0.5
        w2 = torch.ones((8, 16), device="cuda", dtype=BF)
        for act in _ops.GATES:
            r = off.forward(x, w1, w2, w3, act)
            y, h = _ops.gated_ffn(x, w1, w2, w3, act=act, save=True)
            assert torch.isfinite(y).all() and torch.isfinite(h).all()
            g = _ops.gated_ffn_grad(x, w1, w2, w3, h, torch.ones_like(x), act=act)
            b = off.backward(x, w1, w2, w3, h, torch.ones_like(x), act)
            # the terms of a column are few: absolute sums bound everything
            for got, name in ((g[1], "w1"), (g[2], "w2"), (g[3], "w3")):
                ref = b[name]
                if act == "gelu_tanh":  # 64 bits overflow at z^3 = 1e90, times 0 there
                    ref = torch.nan_to_num(ref, nan=0.0) if name == "w1" else ref
                assert torch.isfinite(got).all()
                assert ((got.double() - ref).abs() <= 2.0 ** -6 * ref.abs() + 2.0 ** -14 * T).all(), (act, name)
            big = r["y"].abs().max()
            assert ((y.double() - r["y"]).abs() <= 2.0 ** -6 * big).all()


@pytest.mark.parametrize("T", [4, 260])
def test_infinite_tokens_stay_in_their_rows(T, cuda_dev):
    x, w1, w2, w3 = _ffn_case(T, 136, 200, BF)
    d = torch.randn_like(x)
    y, h = _ops.gated_ffn(x, w1, w2, w3, save=True)
    dx = _ops.gated_ffn_grad(x, w1, w2, w3, h, d)[0]
    bad = x.clone()
    bad[1, 3], bad[2, 0] = float("inf"), float("nan")
    yb, hb = _ops.gated_ffn(bad, w1, w2, w3, save=True)
    keep = [i for i in range(T) if i not in (1, 2)]
    assert torch.equal(yb[keep], y[keep]) and torch.equal(hb[:, keep], h[:, keep])
    assert not torch.isfinite(yb[1]).any() and torch.isnan(yb[2]).all()
    dxb = _ops.gated_ffn_grad(bad, w1, w2, w3, hb, d)[0]
    assert torch.equal(dxb[keep], dx[keep])


def test_planes_do_not_mix(cuda_dev):
    """A gradient with NaN in one plane leaves the other plane's gradients alone (the
    tails of a plane's rows and columns are not read as the next plane's)."""
    T, H, I = 70, 136, 72
    x, w1, w2, w3 = _ffn_case(T, H, I, BF)
    _, h = _ops.gated_ffn(x, w1, w2, w3, save=True)
    d = torch.randn_like(x)
    _, g1, g2, g3 = _ops.gated_ffn_grad(x, w1, w2, w3, h, d)
    hb = h.clone()
    hb[1, 0, 0] = float("inf")  # h3: dh1 and a of (0, 0) turn infinite, dh3 does not
    _, b1, b2, b3 = _ops.gated_ffn_grad(x, w1, w2, w3, hb, d)
    assert torch.equal(b3, g3)
    assert torch.equal(b1[1:], g1[1:]) and torch.equal(b2[:, 1:], g2[:, 1:])
    assert not torch.isfinite(b1[0]).all() and not torch.isfinite(b2[:, 0]).all()


def test_gated_ffn_empty_misaligned_and_in_place(cuda_dev):
    x, w1, w2, w3 = _ffn_case(5, 64, 40, BF)
    y, h = _ops.gated_ffn(x[:0], w1, w2, w3, save=True)
    assert y.shape == (0, 64) and h.shape == (2, 0, 40)
    dx, d1, d2, d3 = _ops.gated_ffn_grad(x[:0], w1, w2, w3, h, y)
    assert dx.shape == (0, 64)
    for d, w in ((d1, w1), (d2, w2), (d3, w3)):
        assert d.shape == w.shape and (d == 0).all()
    for T in (5, 150):
        x, w1, w2, w3 = _ffn_case(T, 64, 40, BF)
        ref, h = _ops.gated_ffn(x, w1, w2, w3, save=True)
        d = torch.randn_like(x)
        grads = _ops.gated_ffn_grad(x, w1, w2, w3, h, d)

        def shift(t):
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            flat[1:] = t.reshape(-1)
            return flat[1:].view(t.shape)

        out = shift(torch.zeros_like(x))
        assert _ops.gated_ffn(shift(x), shift(w1), shift(w2), shift(w3), out=out) is out
        assert torch.equal(out, ref)
        for a, b in zip(grads, _ops.gated_ffn_grad(*map(shift, (x, w1, w2, w3, h, d)))):
            assert torch.equal(a, b)
        own = x.clone()
        assert _ops.gated_ffn(own, w1, w2, w3, out=own) is own
        assert torch.equal(own, ref)


# ------------------------------------------------------------------ 8-bit block
@pytest.mark.parametrize("T,H,I", [(1, 16, 16), (3, 144, 272), (16, 512, 256), (40, 1040, 400), (100, 256, 640),
                                   (128, 384, 128), (129, 384, 128), (300, 1040, 400), (513, 256, 1552)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_ffn_fp8(T, H, I, act, cuda_dev):
    x, w1, w2, w3 = _ffn_case(T, H, I, BF)
    x[0] = 0
    y = _check_fp8(x, w1, w2, w3, act)
    assert (y[0] == 0).all()
    out = torch.empty_like(x)
    qw = _ops.quant_ffn_weights_fp8(w1, w2, w3)
    assert _ops.gated_ffn_fp8(x, qw, act=act, out=out) is out
    assert torch.equal(out, y)


def test_gated_ffn_fp8_many_groups(cuda_dev):
    """So many groups that the quantisation takes several a turn, the last of a row short,
    the rows' end inside a turn."""
    _check_fp8(*_ffn_case(38011, 528, 144, BF), "silu")


@pytest.mark.parametrize("T", [3, 40, 200, 700])
@pytest.mark.parametrize("by,back", [(2.0 ** -62, 2.0 ** 118), (2.0 ** -74, 1.0)])
def test_gated_ffn_fp8_of_vanishing_activations(T, by, back, cuda_dev):
    """Activations whose scale has no reciprocal in fp32, or is none itself, with exact
    zeros among them.

    A code is off by at most 2^-4 of a value, or half a step of the least code, 2^-10, of a
    scale that is at most largest / 448 + 2^-126; 2^-3 more of either for the quotient's
    rounding; a itself by the sums' errors and half an fp32 denormal step, 2^-150, twice."""
    H, I = 528, 400
    x, w1, w2, w3 = _ffn_case(T, H, I, BF)
    w3[::5] = 0
    qw = _ops.quant_ffn_weights_fp8(w1, w2, w3)
    qw["w1s"], qw["w3s"], qw["w2s"] = qw["w1s"] * by, qw["w3s"] * by, qw["w2s"] * back
    W1, W2, W3 = (off.expand(qw[n + "q"], qw[n + "s"], 128) for n in ("w1", "w2", "w3"))
    X = off.e4m3_groups(x.double())
    h1, h3 = X @ W1.T, X @ W3.T
    a = off.gate(h1, "silu") * h3
    da = _acc(H) * ((X.abs() @ W1.abs().T) * (off.slope(h1, "silu") * h3).abs() +
                    (X.abs() @ W3.abs().T) * off.gate(h1, "silu").abs()) + 2.0 ** -20 * (h1 * h3).abs() + 2.0 ** -149
    top = (a.abs() + da).amax(dim=1, keepdim=True)
    code = (1 + 2.0 ** -3) * (2.0 ** -4 * (a.abs() + da) + 2.0 ** -10 * (top / 448 + 2.0 ** -126))
    _within("y", _ops.gated_ffn_fp8(x, qw), a @ W2.T, (da + code + _acc(I) * (a.abs() + da + code)) @ W2.abs().T)


def test_gated_ffn_fp8_is_its_stages(cuda_dev):
    """The block's second product is gemm_fp8_block over quantised activations: with
    weights that make every pre-activation exact, the stages agree bit for bit."""
    for T in (9, 200):
        g = _gen(T)
        H = I = 256
        x = torch.randint(-4, 5, (T, H), generator=g, device="cuda").to(BF)
        x[:, 0], x[:, 128] = 7.0, 7.0  # the group's largest: scale 7 / 448 = 2^-6
        eye = torch.eye(H, device="cuda").to(F8)
        one = torch.ones((2, 2), device="cuda")
        w2 = torch.randint(-4, 5, (H, I), generator=g, device="cuda").float().to(F8)
        qw = {"H": H, "I": I, "w1q": eye, "w1s": one, "w3q": eye, "w3s": one, "w2q": w2, "w2s": one}
        y = _ops.gated_ffn_fp8(x, qw, act="gelu")
        xd = x.float()
        a = (off.gate(xd.double(), "gelu") * xd.double()).float()  # fp32 activations, one rounding away
        aq, sa = _ops.quant_e4m3(a, block=(1, 128))
        ref = _ops.gemm_fp8_block(aq, w2, sa, one)
        # a border may be met by the fp32 error of gelu: a flipped code is one step of 2^-3
        same = (y == ref).all(dim=1)
        assert same.float().mean() >= 0.9


def test_gated_ffn_fp8_empty(cuda_dev):
    x, w1, w2, w3 = _ffn_case(4, 32, 48, BF)
    qw = _ops.quant_ffn_weights_fp8(w1, w2, w3)
    assert _ops.gated_ffn_fp8(x[:0], qw).shape == (0, 32)


# ------------------------------------------------------------------ past 32 bits
def _picked(n, m=40):
    """Some of n indices, the first and the last ones among them."""
    g = torch.Generator().manual_seed(n)
    i = torch.cat([torch.arange(3), torch.randint(0, n, (m,), generator=g), torch.arange(n - 3, n)])
    return i.unique().cuda()


def test_block_product_past_2_31_elements(cuda_dev):
    M, N, K = 70001, 32768, 32
    a, w, sa, sw = _block_case(M, N, K)
    out = _ops.gemm_fp8_block(a, w, sa, sw)
    r = _picked(M)
    va, vw = off.expand(a[r], sa[r], 1), off.expand(w, sw, 128)
    _within("C", out[r], va @ vw.T, _acc(K) * (va.abs() @ vw.abs().T))


def test_gated_ffn_past_2_31_elements(cuda_dev):
    """150,000 tokens of 16,384 activations: planes of 2.46e9 elements."""
    T, H, I = 150001, 64, 16384
    x, w1, w2, w3 = _ffn_case(T, H, I, BF)
    y, h = _ops.gated_ffn(x, w1, w2, w3, save=True)
    d = torch.zeros_like(x)
    r = _picked(T)
    d[r] = torch.randn((r.numel(), H), generator=_gen(3), device="cuda").to(BF)
    f = off.forward(x[r], w1, w2, w3, "silu")
    bh, by = _forward_bound(x[r], w1, w2, w3, f, "silu")
    _within("y", y[r], f["y"], by)
    _within("h", h[:, r], f["h"], bh)
    got = _ops.gated_ffn_grad(x, w1, w2, w3, h, d)
    assert (got[0][[i for i in range(7, 4000) if i not in set(r.tolist())]] == 0).all()
    # the other tokens' gradients are zero: the sums are those of the picked ones alone
    _check_grads(x[r], w1, w2, w3, h[:, r].contiguous(), "silu", d_out=d[r], got=(got[0][r], *got[1:]))
    del h, got
    qw = _ops.quant_ffn_weights_fp8(w1, w2, w3)
    q = _ops.gated_ffn_fp8(x, qw)
    _check_fp8(x[r], w1, w2, w3, "silu", y=q[r])


# ------------------------------------------------------------------ as they are used
def _all_calls(T, dev="cuda"):
    """One call of each operator over T tokens: a list of (function, inputs)."""
    x, w1, w2, w3 = _ffn_case(T, 264, 520, BF)
    d = torch.randn((T, 264), generator=_gen(1), device="cuda").to(BF)
    h = torch.randn((2, T, 520), generator=_gen(2), device="cuda").to(BF)
    a, w, sa, sw = _block_case(T, 600, 784)
    fx, f1, f2, f3 = _ffn_case(T, 272, 528, BF)
    qw = _ops.quant_ffn_weights_fp8(f1, f2, f3)
    return [lambda: _ops.gated_ffn(x, w1, w2, w3, save=True), lambda: _ops.gated_ffn_grad(x, w1, w2, w3, h, d),
            lambda: (_ops.gemm_fp8_block(a, w, sa, sw),), lambda: (_ops.gated_ffn_fp8(fx, qw),)]


@pytest.mark.parametrize("T", [1, 50, 300])
def test_calls_repeat_bit_for_bit(T, cuda_dev):
    for f in _all_calls(T):
        ref = f()
        for _ in range(3):
            for a, b in zip(ref, f()):
                assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 50, 300])
def test_in_a_graph(T, cuda_dev):
    """Two captured graphs of the operators, replayed one after the other and at once
    on two streams, over inputs that change: each has its own workspace."""
    calls = _all_calls(T)
    refs = [f() for f in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            with torch.cuda.graph(g, stream=s):
                outs.append([f() for f in calls])
        graphs.append(g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        for o in outs:
            for ts in o:
                for t in ts:
                    t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        for o in outs:
            for ts, rs in zip(o, refs):
                for t, r in zip(ts, rs):
                    assert torch.equal(t, r)


@pytest.mark.parametrize("T", [2, 300])
def test_in_a_graph_behind_copies_and_joined_streams(T, cuda_dev):
    """A captured call whose predecessors are a copy, a launch of another stream that was
    joined, and a fill of the inputs themselves."""
    x, w1, w2, w3 = _ffn_case(T, 272, 528, BF)
    qw = _ops.quant_ffn_weights_fp8(w1, w2, w3)
    refs = [_ops.gated_ffn(x, w1, w2, w3), _ops.gated_ffn_fp8(x, qw), _ops.gated_ffn(x * 2, w1, w2, w3)]
    src, at, weight = x.clone(), torch.zeros_like(x), torch.zeros_like(w2)
    side, s = torch.cuda.Stream(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            at.copy_(src)
            first = _ops.gated_ffn(at, w1, w2, w3)
            side.wait_stream(s)
            with torch.cuda.stream(side):
                weight.copy_(w2)
                second = _ops.gated_ffn_fp8(at, qw)
            s.wait_stream(side)
            at.mul_(2)
            third = _ops.gated_ffn(at, w1, weight, w3)
    for _ in range(3):
        weight.zero_()
        for o in (first, second, third):
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        for o, r in zip((first, second, third), refs):
            assert torch.equal(o, r)


@pytest.mark.parametrize("T", [2, 300])
def test_weights_written_right_before_the_call(T, cuda_dev):
    """The weights' last writer is the launch before the call: no launch of the call may
    fetch them earlier."""
    x, w1, w2, w3 = _ffn_case(T, 1032, 2056, BF)
    ref = _ops.gated_ffn(x, w1, w2, w3)
    h = _ops.gated_ffn(x, w1, w2, w3, save=True)[1]
    grads = _ops.gated_ffn_grad(x, w1, w2, w3, h, x)
    live = [torch.empty_like(w) for w in (w1, w2, w3)]
    for _ in range(20):
        for t in live:
            t.fill_(float("nan"))
        for t, w in zip(live, (w1, w2, w3)):
            t.copy_(w)
        assert torch.equal(_ops.gated_ffn(x, *live), ref)
        for t in live:
            t.fill_(float("nan"))
        for t, w in zip(live, (w1, w2, w3)):
            torch.mul(w, 1, out=t)
        for a, b in zip(_ops.gated_ffn_grad(x, *live, h, x), grads):
            assert torch.equal(a, b)


def test_two_streams_at_once(cuda_dev):
    calls = [_all_calls(T) for T in (30, 300)]
    refs = [[f() for f in c] for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append([f() for f in calls[i]])
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            for ts, rs in zip(run, refs[i]):
                for t, r in zip(ts, rs):
                    assert torch.equal(t, r)


@pytest.mark.parametrize("T", [20, 400])
def test_on_a_partition(T, cuda_dev):
    """A partition of 16 SMs: fewer and longer runs, other splits of K."""
    calls = _all_calls(T)
    refs = [f() for f in calls]
    stream, sms = create_sm_partition(cuda_dev, 16)
    torch.cuda.synchronize()
    a, w, sa, sw = _block_case(T, 333, 400)
    with torch.cuda.stream(stream):
        got = [f() for f in calls]
        c = call_sm_aware_fp8_block(a, w, sa, sw)
    torch.cuda.synchronize()
    _block_check(c, a, w, sa, sw)
    for ts, rs in zip(got, refs):
        for t, r in zip(ts, rs):
            # the sums' order differs: a code or a rounding may fall on the other side
            scale = r.double().square().mean().sqrt()
            assert ((t.double() - r.double()).abs() <= 2.0 ** -6 * r.double().abs() + 2.0 ** -3 * scale).all()
            assert (t.double() - r.double()).square().mean().sqrt() <= 2.0 ** -7 * scale
    x, w1, w2, w3 = _ffn_case(T, 264, 520, BF)
    y1 = _ops.gated_ffn(x, w1, w2, w3, num_sms=1)  # a planned size below one pair
    r = off.forward(x, w1, w2, w3, "silu")
    _within("y", y1, r["y"], _forward_bound(x, w1, w2, w3, r, "silu")[1])


def test_training_step_beside_routed_experts(cuda_dev):
    """A shared expert beside the routed ones, as a layer uses them: the shared block's
    forward pass and gradients, and the routed layer's output added, against autograd
    in 64 bits over the same weights."""
    T, H, I, E, k = 96, 256, 384, 8, 2
    x, w1, w2, w3 = _ffn_case(T, H, I, BF)
    g = _gen(11)
    e1, e3 = ((torch.randn((E, I, H), generator=g, device="cuda") * H ** -0.5).to(BF) for _ in range(2))
    e2 = (torch.randn((E, H, I), generator=g, device="cuda") * I ** -0.5).to(BF)
    logits = torch.randn((T, E), generator=g, device="cuda")
    routed = _ops.fused_moe(x, logits, e1, e2, e3, k)
    y, h = _ops.gated_ffn(x, w1, w2, w3, save=True)
    d_out = (y + routed).mul(2.0 / T)  # of mean over tokens of |y + routed|^2, routed held fixed
    grads = _ops.gated_ffn_grad(x, w1, w2, w3, h, d_out)
    leaves = [t.double().requires_grad_() for t in (x, w1, w2, w3)]
    X, W1, W2, W3 = leaves
    h1 = X @ W1.T
    out = (h1 * torch.sigmoid(h1) * (X @ W3.T)) @ W2.T + routed.double()
    (out.square().sum() / T).backward()
    for got, leaf in zip(grads, leaves):
        scale = leaf.grad.square().mean().sqrt()
        # h, dh, a, y and d_out are rounded to 8 bits of mantissa on the way: five independent
        # roundings of relative u / sqrt 3 at most each, and the result's own
        assert (got.double() - leaf.grad).square().mean().sqrt() <= _u(BF) * (6 / 3) ** 0.5 * 1.5 * scale
    w = w2 - (0.01 * grads[2].float()).to(BF)  # a step: the weights the next pass takes
    assert torch.isfinite(_ops.gated_ffn(x, w1, w, w3)).all()


def test_eight_bit_block_after_training(cuda_dev):
    """Weights trained in 16 bits, quantised and served in 8: the two blocks differ by
    the quantisation alone."""
    for T in (8, 256):
        x, w1, w2, w3 = _ffn_case(T, 512, 768, BF)
        y = _ops.gated_ffn(x, w1, w2, w3)
        q = _ops.gated_ffn_fp8(x, _ops.quant_ffn_weights_fp8(w1, w2, w3))
        rel = (q.double() - y.double()).square().mean().sqrt() / y.double().square().mean().sqrt()
        # five quantised operands (x, w1, w3, a, w2), each off by a relative 2^-4 / sqrt 3 at
        # most, x twice through both factors of a: sqrt(6) * 2^-4 / sqrt 3
        assert rel <= 6 ** 0.5 * 2.0 ** -4 / 3 ** 0.5


def test_other_device_and_status(cuda_dev):
    """The status word stays clean, and inputs are used on their own device."""
    x, w1, w2, w3 = _ffn_case(4, 64, 64, BF)
    y = _ops.gated_ffn(x, w1, w2, w3)
    assert y.device == x.device
    assert _lib.device_status(0) == 0
