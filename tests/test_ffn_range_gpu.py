"""Dense feed-forward operators at the ends of what their inputs may hold: NaN that has
to reach every gradient it belongs to, scales of any value, quotients on a border between
two codes."""
from __future__ import annotations

import pytest
import torch

from elastikernel_b200 import _ops
from oracle import ffn as off

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn
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


# ------------------------------------------------------------------ scales of any value
def _sums_bound(va, vw, K):
    """Of a product of fp32 sums (test_ffn_gpu's first rule) of K blocks, each of which, and
    each sum so far, may end below fp32's normal numbers: half a denormal step apiece."""
    return (K / 16 + 16) * 2.0 ** -22 * (va.abs() @ vw.abs().T) + 2 * (K // 128 + 1) * 2.0 ** -150


def _fits(got, ref, bound):
    """got is ref within the bound and one rounding of its type; past the type's largest
    number, infinite with ref's sign."""
    g, info = got.double(), torch.finfo(got.dtype)
    past = ref.abs() > info.max * (1 + 2.0 ** -10)
    assert (ref[~past].abs() < info.max * (1 - 2.0 ** -10)).all()  # no case is at the border
    assert torch.equal(g[past], torch.inf * ref[past].sign())
    assert torch.isfinite(g[~past]).all()
    bound = bound + info.eps / 2 * ref.abs() * (1 + 2.0 ** -6) + info.smallest_normal * info.eps / 2
    over = ((g - ref).abs() - bound)[~past]
    assert over.numel() == 0 or over.max() <= 0, f"{over.max():.3e} over its bound"


def _far_scales(g, exponent, *shape):
    """fp32 of magnitude 2^exponent to 2^(exponent + 1), some negative"""
    s = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64) + 1
    s = torch.where(torch.rand(shape, generator=g, device="cuda") < 0.2, -s, s)
    return (s * 2.0 ** exponent).float()


# few tokens; the kernel of tiles, whole and cut along K, its scales read one by one (3
# blocks of K) and four at a time; a device's and a small partition's plans
@pytest.mark.parametrize("M,N,K,num_sms", [(1, 300, 512, None), (15, 200, 384, 8), (40, 130, 272, None), (64, 300, 512, 4),
                                           (120, 520, 512, 2), (128, 300, 272, None), (200, 300, 512, 4),
                                           (300, 130, 400, 2), (200, 300, 4096, None), (260, 77, 2000, None)])
@pytest.mark.parametrize("ea,ew", [(-70, -70), (-75, -74), (-21, -121), (-126, -11), (-2, -148), (-148, -2), (-60, -66),
                                   (-126, 126), (126, -126), (-148, 120), (120, -148), (104, -104), (-104, 104)])
def test_block_product_of_far_scales(M, N, K, num_sms, ea, ew, cuda_dev):
    """Scales whose product fp32 holds badly or not at all, the results of which it does; and
    scales far apart whose product is ordinary."""
    g = _gen(M + N + K)
    a, w = (torch.randn((r, K), generator=g, device="cuda").mul(60).clamp(-448, 448).to(F8) for r in (M, N))
    sa, sw = _far_scales(g, ea, M, -(-K // 128)), _far_scales(g, ew, -(-N // 128), -(-K // 128))
    va, vw = off.expand(a, sa, 1), off.expand(w, sw, 128)
    _fits(_ops.gemm_fp8_block(a, w, sa, sw, dtype=torch.float32, num_sms=num_sms), va @ vw.T, _sums_bound(va, vw, K))


@pytest.mark.parametrize("M,N,K,num_sms", [(1, 300, 512, None), (40, 130, 272, None), (64, 300, 512, 4), (128, 300, 400, 2),
                                           (200, 300, 512, 4), (300, 130, 272, 2), (200, 300, 4096, None)])
@pytest.mark.parametrize("ea,ew", [(70, 66), (66, 70), (127, 10), (10, 127), (120, 120)])
def test_block_product_of_huge_scales(M, N, K, num_sms, ea, ew, cuda_dev):
    """Products of scales past fp32's largest number: what the codes leave at zero is zero,
    what they make large is infinite, and least codes (2^-18 together) bring the first
    two's product back into range."""
    g = _gen(M * N + K)
    a = torch.rand((M, K), generator=g, device="cuda").add(0.5).to(F8)
    w = torch.rand((N, K), generator=g, device="cuda").add(0.5).to(F8)
    a[::3] = 0          # rows of zeros
    w[1::4] = 0         # columns of zeros
    w[:, :128] = 0      # and a block of K that is zero for all
    w[2::4, 128:] = 0
    a[:, 160] = 0
    a[1::3, 160], w[2::4, 160] = 2.0 ** -9, 2.0 ** -9  # a single product of 2^-18
    sa, sw = _far_scales(g, ea, M, -(-K // 128)).abs(), _far_scales(g, ew, -(-N // 128), -(-K // 128)).abs()
    va, vw = off.expand(a, sa, 1), off.expand(w, sw, 128)
    ref = va @ vw.T
    got = _ops.gemm_fp8_block(a, w, sa, sw, dtype=torch.float32, num_sms=num_sms)
    _fits(got, ref, _sums_bound(va, vw, K))
    assert (got[::3] == 0).all() and (got[:, 1::4] == 0).all()


@pytest.mark.parametrize("M,N,K,num_sms", [(1, 300, 512, None), (40, 130, 272, None), (128, 300, 400, 2), (200, 300, 512, 4),
                                           (300, 130, 272, 2), (200, 300, 4096, None)])
@pytest.mark.parametrize("which", ["a", "w", "both"])
def test_block_product_of_zero_scales_beside_huge_ones(M, N, K, num_sms, which, cuda_dev):
    """A scale of zero makes its block zero, whatever the sum and the other scale."""
    g = _gen(M + K)
    a, w = (torch.full((r, K), 448.0, device="cuda").to(F8) for r in (M, N))
    sa, sw = _far_scales(g, 126, M, -(-K // 128)), _far_scales(g, 126, -(-N // 128), -(-K // 128))
    if which != "w":
        sa.zero_()
    if which != "a":
        sw.zero_()
    assert (_ops.gemm_fp8_block(a, w, sa, sw, dtype=torch.float32, num_sms=num_sms) == 0).all()


@pytest.mark.parametrize("T,num_sms", [(3, None), (40, None), (100, None), (300, None), (300, 4)])
def test_gated_ffn_fp8_of_zero_blocks_under_huge_scales(T, num_sms, cuda_dev):
    """Blocks of zero codes under any finite scale add nothing: not NaN."""
    H, I = 512, 384
    g = _gen(T)
    x, w1, w2, w3 = (torch.randn(s, generator=g, device="cuda").to(BF) for s in ((T, H), (I, H), (H, I), (I, H)))
    qw = _ops.quant_ffn_weights_fp8(w1 * H ** -0.5, w2 * I ** -0.5, w3 * H ** -0.5)
    for n in ("w1", "w3", "w2"):
        qw[n + "q"][:, 128:256] = 0
    plain = _ops.gated_ffn_fp8(x, qw, num_sms=num_sms)
    x[:, 128:256] *= 2.0 ** 70  # tokens' scales of about 2^63
    far = dict(qw)
    for n in ("w1", "w3", "w2"):
        far[n + "s"] = qw[n + "s"].clone()
        far[n + "s"][:, 1] = 2.0 ** 127
    assert torch.isfinite(plain).all() and (plain != 0).any()
    assert torch.equal(_ops.gated_ffn_fp8(x, far, num_sms=num_sms), plain)


@pytest.mark.parametrize("T,num_sms", [(3, None), (40, None), (100, None), (300, None), (300, 4)])
def test_gated_ffn_fp8_of_vanishing_products_of_scales(T, num_sms, cuda_dev):
    """Tokens and W3 of 2^-69 each, products of scales of one bit or none; W1 and W2 bring
    the result back.

    A code is off by at most 2^-4 of a value or 2^-10 of its scale, 2^-3 more of either for
    the quotient's rounding, as in ordinary ranges; h3 by the sums' errors and, around its
    blocks and their sums, half a denormal step each."""
    H, I = 528, 400
    g = _gen(T + 1)
    x, w1, w2, w3 = (torch.randn(s, generator=g, device="cuda").to(BF) for s in ((T, H), (I, H), (H, I), (I, H)))
    qw = _ops.quant_ffn_weights_fp8(w1 * H ** -0.5, w2 * I ** -0.5, w3 * H ** -0.5)
    x = x * 2.0 ** -69
    qw["w1s"], qw["w3s"], qw["w2s"] = qw["w1s"] * 2.0 ** 120, qw["w3s"] * 2.0 ** -69, qw["w2s"] * 2.0 ** 90
    W1, W2, W3 = (off.expand(qw[n + "q"], qw[n + "s"], 128) for n in ("w1", "w2", "w3"))
    X = off.e4m3_groups(x.double())
    acc = (H / 16 + 16) * 2.0 ** -22
    h1, h3 = X @ W1.T, X @ W3.T
    a = off.gate(h1, "silu") * h3
    da = (acc * (X.abs() @ W1.abs().T) * (off.slope(h1, "silu") * h3).abs() +
          (acc * (X.abs() @ W3.abs().T) + 12 * 2.0 ** -150) * off.gate(h1, "silu").abs() + 2.0 ** -20 * a.abs())
    top = (a.abs() + da).amax(dim=1, keepdim=True)
    code = (1 + 2.0 ** -3) * (2.0 ** -4 * (a.abs() + da) + 2.0 ** -10 * top / 448)
    bound = (da + code + (I / 16 + 16) * 2.0 ** -22 * (a.abs() + da + code)) @ W2.abs().T
    got = _ops.gated_ffn_fp8(x, qw, num_sms=num_sms)
    ref = a @ W2.T
    _fits(got, ref, bound)
    assert (got.double() - ref).square().mean().sqrt() <= 2.0 ** -4 * ref.square().mean().sqrt()


# ------------------------------------------------------------------ codes on a border
@pytest.mark.parametrize("T,num_sms", [(20, None), (100, None), (128, 2), (300, None), (300, 2), (600, 8), (1300, None)])
@pytest.mark.parametrize("by", [0, 100, -105])
def test_gated_ffn_fp8_codes_are_ieee_quotients(T, num_sms, by, cuda_dev):
    """Activations that fp32 holds exactly as the formula has them, many of them halfway
    between two codes but for the rounding of their scale; the second weight the identity, so
    that every code shows: bit for bit quant_e4m3's, by whichever kernel.

    Token t has one nonzero value, 448, in block b = t % 16 of K (scale 1, code 448). W1 is 1
    there, so f(h1) = 448 exactly (silu's exp(-448) is zero); h3 = 448 c s with one rounding,
    a = 448 h3 with another. Of a code c of 12 x 2^j under a largest of 8 x 2^j the quotient is 84
    2^j, a tie, within an ulp. W3's scales of about 2^by bring the activations' scales to where
    a quotient's residues would leave fp32's range."""
    H = I = 2048
    g = _gen(7)
    B = H // 128
    x = torch.zeros((T, H), device="cuda", dtype=BF)
    b = torch.arange(T, device="cuda") % B
    x[torch.arange(T, device="cuda"), 128 * b] = 448.0
    w1 = torch.zeros((I, H), device="cuda")
    w3 = torch.zeros((I, H), device="cuda")
    w1[:, ::128] = 1.0
    c = 12.0 * torch.exp2(torch.randint(-9, -1, (I, B), generator=g, device="cuda").float())
    c = torch.where(torch.rand((I, B), generator=g, device="cuda") < 0.5, c, c * 13 / 12)
    c[::128] = 8.0      # the largest of each group
    w3[:, ::128] = c * torch.where(torch.rand((I, B), generator=g, device="cuda") < 0.5, 1.0, -1.0)
    one = torch.ones((B, B), device="cuda")
    s3 = (torch.rand((B, B), generator=g, device="cuda") + 1) * 2.0 ** by
    eye = torch.eye(H, device="cuda")
    qw = {"H": H, "I": I, "w1q": w1.to(F8), "w1s": one, "w3q": w3.to(F8), "w3s": s3, "w2q": eye.to(F8), "w2s": one}
    a = 448.0 * ((448.0 * w3[:, ::128]) * s3.repeat_interleave(128, dim=0))  # [I, B]: feature, block of the token
    q, s = _ops.quant_e4m3(a.t().contiguous(), block=(1, 128))
    want = (q.float() * s.repeat_interleave(128, dim=1)).to(BF)[b]
    # the border is met: some codes are not those of products with the scale's reciprocal
    rough = (a.t() * (1.0 / s).repeat_interleave(128, dim=1)).to(F8)
    assert not torch.equal(rough.float(), q.float())
    assert torch.equal(_ops.gated_ffn_fp8(x, qw, num_sms=num_sms), want)


# ------------------------------------------------------------------ the kernels against themselves
@pytest.mark.parametrize("T", [24, 160])
@pytest.mark.parametrize("act", list(_ops.GATES))
def test_gradient_against_the_forward_kernels_own_differences(T, act, cuda_dev):
    """The kernels' gradient of sum(y * d) against central differences of the forward
    kernels, at the largest element of each gradient.

    The tolerance is the sum of what 64 bits say of this difference (its distance from the
    derivative), what they say of taking the derivative at the rounded h, and roundings.
    In the difference: u |y| d of every y that moves, in both passes, and u |a| through w2
    and d of every a that moves; in the gradient u of each product's rounded factor and of the
    result. Independent and of either sign, they leave 7.5 root mean squares with a probability of
    1e-12 (Hoeffding); 8 for the fp32 sums beside them. At most a fourth of the gradient is left
    to them: an error of sign, factor or index does not pass."""
    H, I, u = 64, 96, torch.finfo(FP).eps / 2
    g = _gen(T)
    x, w1, w2, w3, d = (torch.randn(s, generator=g, device="cuda").mul(by).to(FP) for s, by in
                        (((T, H), 1.0), ((I, H), 2 * H ** -0.5), ((H, I), I ** -0.5), ((I, H), H ** -0.5), ((T, H), 1.0)))
    ts = [x, w1, w2, w3]
    _, h = _ops.gated_ffn(*ts, act=act, save=True)
    got = _ops.gated_ffn_grad(*ts, h, d, act=act)
    f = off.forward(*ts, act)
    at_h, exact = off.backward(*ts, h, d, act), off.backward(*ts, f["h"], d, act)
    X, W1, W2, W3, D = (t.double() for t in (*ts, d))
    through = (D @ W2).abs()  # what an error of a costs
    for i, name in enumerate(("x", "w1", "w2", "w3")):
        r, c = divmod(exact[name].abs().argmax().item(), exact[name].shape[1])
        step = 2.0 ** (-2 if name == "x" else -3)
        sums, sums64, reals = [], [], []
        for sign in (1, -1):
            moved = [t.clone() for t in ts]
            moved[i][r, c] += sign * step
            reals.append(moved[i][r, c].item())
            sums.append((_ops.gated_ffn(*moved, act=act).double() * D).sum().item())
            sums64.append((off.forward(*moved, act)["y"] * D).sum().item())
        width = reals[0] - reals[1]
        diff, diff64 = (sums[0] - sums[1]) / width, (sums64[0] - sums64[1]) / width
        ya = 2 * u * (f["y"] * D).abs()      # both passes' roundings of y
        aa = 2 * u * f["a"].abs() * through  # and of a
        if name == "x":
            ya, aa = ya[r], aa[r]
            terms = torch.cat([exact["d1"][r] * W1[:, c], exact["d3"][r] * W3[:, c]])
        elif name == "w2":
            ya, aa, terms = ya[:, r], aa[:0], D[:, r] * f["a"][:, c]
        else:
            aa, terms = aa[:, r], exact["d1" if name == "w1" else "d3"][:, r] * X[:, c]
        ref = exact[name][r, c].item()
        rounding = 8 * ((ya.square().sum() + aa.square().sum()).sqrt().item() / width + u * terms.square().sum().sqrt().item())
        assert rounding <= abs(ref) / 4, name
        tol = rounding + u * abs(ref) + abs(diff64 - ref) + abs(at_h[name][r, c].item() - ref)
        assert abs(got[i][r, c].item() - diff) <= tol, (name, got[i][r, c].item(), diff, ref, tol)


@pytest.mark.parametrize("T", [3, 140])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("act", list(_ops.GATES))
def test_each_extreme_activation_by_itself(T, dtype, act, cuda_dev):
    """Pre-activations far past where the gate saturates, the second weight the identity: each
    activation is a column of the result.

    h1 and h3 are exact (one product each, in the type); a is off by its rounding, half a
    step below the type's normal numbers, and 2^-13 of |z| for the gate's exponential, whose
    argument has 2^-24 of up to 100 in it and an error of 2 + |z| ulp; y by one more rounding
    of the same value, which changes nothing."""
    z = [0.0, -3e4, 3e4, -100, 100, -20, 20, -1e-3, 1e-3, 5, -5, 30, -30, 1.0, -1.0, 0.5]
    z += [-1e30, 1e30, -1e-30, 1e-30, -87.0, -88.5, 88.5, -10] if dtype == BF else [-87.0, -88.5, 88.5, -10, 11, -12, 2, -2]
    n = len(z)
    x = torch.zeros((T, n), device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = 1.0, 0.5
    w1 = torch.zeros((n, n), device="cuda", dtype=dtype)
    w1[:, 0] = torch.tensor(z)
    w3 = torch.zeros((n, n), device="cuda", dtype=dtype)
    w3[:, 1] = 1.0
    w2 = torch.eye(n, device="cuda", dtype=dtype)
    r = off.forward(x, w1, w2, w3, act)
    y, h = _ops.gated_ffn(x, w1, w2, w3, act=act, save=True)
    assert torch.equal(h.double(), r["h"])
    info = torch.finfo(dtype)
    ref = r["a"]
    bound = info.eps / 2 * ref.abs() + info.smallest_normal * info.eps / 2 + 2.0 ** -13 * ref.abs()
    # under exp(-87) the logistic function's reciprocal is zero in fp32: |z| 2^-126 at most
    bound = bound + r["h"][0].abs().clamp(max=100) * 2.0 ** -126
    over = (y.double() - ref).abs() - bound
    assert (over <= 0).all(), (act, torch.tensor(z)[(over > 0).any(dim=0).cpu()])
