"""4-bit-weight products on the GPU against the float64 oracle (oracle/w4.py).

Tolerances (derived, not fitted). A product of K terms summed in fp32 in any
order, scaled per group, costs at most K/4 + 32 effective roundings of 2^-24
of S, the sum of the terms' magnitudes (groups of at least 16 terms are added
at once by the tensor cores, which may drop the bits below the largest one:
two units of 2^-24 per 16 terms and one per group); the result is then
rounded once (eps/2). Small integers with power-of-two scales are exact and
compared bit for bit after the one rounding.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from elastikernel_b200 import _lib, _ops
from elastikernel_b200.sm_aware_matmul import call_sm_aware_w4
from oracle import w4 as ow4
from oracle.moe import route_ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _np(t):
    return t.double().cpu().numpy()


def _integer_weight(N, K, group, mins, dtype, seed, dev, lead=()):
    """Random codes with power-of-two scales (and small integer minima)."""
    g = torch.Generator().manual_seed(seed)
    shape = lead + (N,)
    G = -(-K // group)
    codes = torch.randint(0, 256, shape + (-(-K // 32) * 16,), generator=g, dtype=torch.uint8)  # padding codes too
    scales = (2.0 ** torch.randint(-2, 2, shape + (G,), generator=g)).to(dtype)
    m = torch.randint(-3, 4, shape + (G,), generator=g).to(dtype) if mins else None
    return {"codes": codes.to(dev), "scales": scales.to(dev), "mins": None if m is None else m.to(dev), "K": K,
            "group": group}


def _values(qw):
    return ow4.values(qw["codes"], qw["scales"], qw["mins"], qw["K"], qw["group"])


def _bound(qw):
    return ow4.abs_bound(qw["codes"], qw["scales"], qw["mins"], qw["K"], qw["group"])


def _close(got, exact, S, K, extra=0.0):
    eps = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    err = np.abs(_np(got) - exact)
    bound = eps * np.abs(exact) * (1 + 2.0 ** -8) + (K / 4 + 32) * 2.0 ** -24 * S + extra + tiny
    assert np.isfinite(_np(got)).all()
    assert (err <= bound).all(), f"worst {np.max(err - bound):.3e} over its bound"


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("N,K,group,src,dtype", [
    (1, 1, 32, torch.float32, BF), (7, 31, 32, BF, BF), (16, 128, 128, FP, FP), (33, 200, 64, torch.float32, FP),
    (5, 4096, 128, BF, BF), (300, 257, 128, torch.float32, BF), (3, 160, 32, FP, BF)])
def test_quantise_is_bit_exact(N, K, group, symmetric, src, dtype, cuda_dev):
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn((N, K), generator=g) * 0.02).to(src)
    w[0] = 0
    if N > 2:
        w[1] = 0.5      # a constant row: no range
        w[2] *= 1e-9    # scales that fp16 cannot hold
    qw = _ops.quant_w4(w.to(cuda_dev), group, symmetric, dtype)
    codes, s, m = ow4.quantise(w, group, symmetric, dtype)
    assert torch.equal(qw["codes"].cpu(), codes)
    assert torch.equal(qw["scales"].cpu(), s)
    assert (qw["mins"] is None) if symmetric else torch.equal(qw["mins"].cpu(), m)
    v = torch.from_numpy(ow4.values(codes, s, m, K, group))
    # the fp32 value s * q + m is rounded once more to dtype
    d = _ops.dequant_w4(qw).double().cpu()
    assert ((d - v).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * v.abs() + 2.0 ** -25).all()


def test_quantise_extremes(cuda_dev):
    w = torch.tensor([[3e38, -3e38] + [0.0] * 30], device=cuda_dev)
    for sym in (True, False):
        qw = _ops.quant_w4(w, 32, sym, FP)
        assert qw["scales"].isfinite().all() and _ops.dequant_w4(qw).isfinite().sum() >= 30
    qw = _ops.quant_w4(torch.empty((0, 64), device=cuda_dev), 32)
    assert qw["codes"].shape == (0, 32) and _ops.dequant_w4(qw).shape == (0, 64)


# ------------------------------------------------------------------ dense products
GEMM = [  # M, N, K, group
    (1, 1, 1, 32), (1, 16, 128, 128), (1, 4096, 4096, 128), (2, 33, 96, 32), (3, 100, 257, 64), (5, 17, 1000, 128),
    (8, 130, 4096, 128), (9, 48, 2048, 64), (16, 2304, 512, 32), (17, 65, 7168, 128), (33, 129, 640, 64),
    (64, 256, 1024, 128), (65, 40, 130, 32), (100, 24, 512, 128), (1, 28672, 256, 128), (7, 64, 14336, 128),
    (200, 136, 384, 64),
]


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("M,N,K,group", GEMM)
def test_gemm_integers_exact(M, N, K, group, dtype, mins, cuda_dev):
    qw = _integer_weight(N, K, group, mins, dtype, M + N + K, cuda_dev)
    g = torch.Generator().manual_seed(K)
    x = torch.randint(-2, 3, (M, K), generator=g).to(dtype)
    got = _ops.gemm_w4(x.to(cuda_dev), qw)
    exact = torch.from_numpy(_np(x) @ _values(qw).T)  # multiples of 1/4 below 2^20: exact in fp32
    assert torch.equal(got.cpu(), exact.to(dtype))


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("M,N,K,group", GEMM)
def test_gemm_random(M, N, K, group, dtype, symmetric, cuda_dev):
    g = torch.Generator().manual_seed(M * 7 + K)
    w = torch.randn((N, K), generator=g) / K ** 0.5
    x = (torch.randn((M, K), generator=g) + 0.5).to(dtype)
    qw = _ops.quant_w4(w.to(cuda_dev), group, symmetric, dtype)
    got = _ops.gemm_w4(x.to(cuda_dev), qw)
    _close(got, _np(x) @ _values(qw).T, np.abs(_np(x)) @ _bound(qw).T, K)
    out = torch.full((M, N), 9.0, dtype=dtype, device=cuda_dev)
    assert _ops.gemm_w4(x.to(cuda_dev), qw, out=out) is out and torch.equal(out, got)


def test_gemm_rows_do_not_mix(cuda_dev):
    """A non-finite token spoils its own output row alone; infinite and NaN
    values beyond K or M are never read."""
    M, N, K = 5, 70, 200
    qw = _ops.quant_w4(torch.randn((N, K), device=cuda_dev), 64)
    buf = torch.full((M * K + 64,), float("nan"), dtype=BF, device=cuda_dev)
    x = buf[8:8 + M * K].view(M, K)
    x.copy_(torch.randn((M, K), device=cuda_dev))
    clean = _ops.gemm_w4(x.clone(), qw)
    assert torch.equal(_ops.gemm_w4(x, qw), clean)
    x[3, 7] = float("inf")
    got = _ops.gemm_w4(x, qw)
    keep = [0, 1, 2, 4]
    assert torch.equal(got[keep], clean[keep]) and not got[3].isfinite().any()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_gemm_misaligned_views(dtype, cuda_dev):
    for M, N, K in ((1, 64, 256), (4, 50, 257), (20, 33, 130)):
        qw = _integer_weight(N, K, 32, True, dtype, 1, cuda_dev)
        x = torch.randint(-2, 3, (M * K + 1,), device=cuda_dev).to(dtype)[1:].view(M, K)
        out = torch.empty((M * N + 1,), dtype=dtype, device=cuda_dev)[1:].view(M, N)
        _ops.gemm_w4(x, qw, out=out)
        assert torch.equal(out, _ops.gemm_w4(x.clone(), qw))
        assert torch.equal(out.cpu(), torch.from_numpy(_np(x) @ _values(qw).T).to(dtype))


def test_gemm_large_values_and_scales(cuda_dev):
    """fp16 tokens near the type's limit against tiny scales: no overflow on the way."""
    K = 512
    x = torch.full((2, K), 6e4, dtype=FP, device=cuda_dev)
    qw = _integer_weight(24, K, 64, False, FP, 4, cuda_dev)
    qw["scales"] = torch.full_like(qw["scales"], 2.0 ** -20)
    _close(_ops.gemm_w4(x, qw), _np(x) @ _values(qw).T, np.abs(_np(x)) @ _bound(qw).T, K)


def test_gemm_past_2_31_weights(cuda_dev):
    N, K = 270000, 8192  # 2.2e9 weights, 1.1 GB of codes
    qw = {"codes": torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=cuda_dev),
          "scales": torch.ones((N, K // 128), dtype=BF, device=cuda_dev), "mins": None, "K": K, "group": 128}
    x = torch.zeros((1, K), dtype=BF, device=cuda_dev)
    x[0, 5], x[0, K - 1] = 1.0, 2.0
    got = _ops.gemm_w4(x, qw)
    want = ((qw["codes"][:, 2] >> 4).float() - 8) + 2 * ((qw["codes"][:, -1] >> 4).float() - 8)
    assert torch.equal(got[0], want.to(BF))


def test_gemm_on_a_partition_and_in_a_graph(cuda_dev):
    from elastikernel_b200.green_ctx import create_sm_partition

    qw = _integer_weight(520, 1024, 128, True, BF, 2, cuda_dev)
    x = torch.randint(-2, 3, (6, 1024), device=cuda_dev).to(BF)
    want = torch.from_numpy(_np(x) @ _values(qw).T).to(BF)
    stream, _ = create_sm_partition(cuda_dev, 32)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        part = call_sm_aware_w4(x, qw)
    stream.synchronize()
    assert torch.equal(part.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _ops.gemm_w4(x, qw)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held.cpu(), -want)


def test_gemm_empty_and_refusals(cuda_dev):
    qw = _integer_weight(16, 64, 32, False, BF, 3, cuda_dev)
    x = torch.zeros((2, 64), dtype=BF, device=cuda_dev)
    assert _ops.gemm_w4(x[:0], qw).shape == (0, 16)
    for call, text in [(lambda: _ops.gemm_w4(x.half(), qw), "scales must be"),
                       (lambda: _ops.gemm_w4(x[:, :32].contiguous(), qw), r"a \[M, 64\]"),
                       (lambda: _ops.gemm_w4(x.t().contiguous().t(), qw), "contiguous"),
                       (lambda: _ops.gemm_w4(x, qw, out=x), "out must be"),
                       (lambda: _ops.quant_w4(x, 100), "group"),
                       (lambda: _ops.quant_w4(x.double()), "bf16, fp16 or fp32"),
                       (lambda: _ops.quant_w4(x, 32, dtype=torch.float32), "dtype")]:
        with pytest.raises(RuntimeError, match=text):
            call()


# ------------------------------------------------------------------ experts
MOE = [  # T, k, E, H, I, group, mins
    (1, 1, 1, 32, 32, 32, False), (1, 2, 8, 4096, 512, 128, False), (3, 2, 4, 200, 136, 64, True),
    (17, 8, 60, 512, 260, 32, False), (64, 8, 32, 1024, 256, 128, False), (40, 3, 5, 257, 65, 64, True),
    (300, 2, 4, 256, 384, 128, False), (33, 1, 300, 64, 96, 32, False), (700, 2, 6, 128, 192, 64, True),
    (128, 8, 16, 136, 72, 32, False), (1, 8, 8, 64, 14336, 128, False), (4, 2, 3, 14336, 40, 64, True),
]


def _moe_setup(case, dev):
    T, k, E, H, I, group, mins = case
    g = torch.Generator().manual_seed(T + E + H)
    ws = [torch.randn(s, generator=g) / s[-1] ** 0.5 for s in ((E, I, H), (E, H, I), (E, I, H))]
    qw = _ops.quant_moe_weights_w4(*(w.to(dev) for w in ws), group=group, symmetric=not mins)
    x = torch.randn((T, H), generator=g).to(BF).to(dev)
    ids = torch.topk(torch.randn((T, E), generator=g), k, dim=1).indices.int().to(dev)
    return x, ids, qw


@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("case", MOE, ids=lambda c: f"T{c[0]}k{c[1]}E{c[2]}H{c[3]}I{c[4]}")
def test_expert_products(case, drop, cuda_dev):
    """gate/up and down, each against the oracle on its own inputs."""
    T, k, E, H, I, group, mins = case
    x, ids, qw = _moe_setup(case, cuda_dev)
    if drop:
        ids[::2, 0] = -1
    p = _ops.moe_dispatch(x, ids, E)
    kept = int(p["num_rows_padded"])
    act = _ops.moe_gate_up_w4(p, qw)
    assert torch.equal(act[:kept], _ops.moe_gate_up_w4(p, qw, x=x)[:kept])  # fetched through the permutation
    wide = _ops.moe_gate_up_w4(p, qw, dtype=torch.float32)
    assert torch.equal(wide[:kept].to(BF), act[:kept])
    y = _ops.moe_down_w4(p, act, qw)
    assert torch.equal(_ops.moe_down_w4(p, act, qw, dtype=torch.float32)[:kept].to(BF), y[:kept])
    counts = p["expert_counts"].tolist()
    v = {n: _values(qw[n]) for n in ("w1", "w3", "w2")}
    b = {n: _bound(qw[n]) for n in ("w1", "w3", "w2")}
    xp, r = _np(p["x_perm"]), 0
    for e, c in enumerate(counts):
        if c:
            rows = slice(r, r + c)
            h, u = xp[rows] @ v["w1"][e].T, xp[rows] @ v["w3"][e].T
            n = (H / 4 + 32) * 2.0 ** -24
            dh, du = n * (np.abs(xp[rows]) @ b["w1"][e].T), n * (np.abs(xp[rows]) @ b["w3"][e].T)
            silu = h / (1 + np.exp(-h))
            # |silu'| <= 1.1; exp, the quotient and the product: 8 roundings of 2^-24
            extra = 1.1 * dh * (np.abs(u) + du) + np.abs(silu) * du + 8 * 2.0 ** -24 * np.abs(silu * u)
            _close(act[rows], silu * u, 0.0, 0, extra)
            a = _np(act[rows])
            _close(y[rows], a @ v["w2"][e].T, np.abs(a) @ b["w2"][e].T, I)
        r += c
    assert r == kept


@pytest.mark.parametrize("case", MOE, ids=lambda c: f"T{c[0]}k{c[1]}E{c[2]}H{c[3]}I{c[4]}")
def test_fused_layer(case, cuda_dev):
    """The layer against the oracle: act has 11 significant bits (2^-11 of each
    term), the experts' rows are fp32, the output is rounded once (2^-8)."""
    T, k, E, H, I, group, mins = case
    if E > 256:
        pytest.skip("moe_route takes up to 256 experts")
    x, _, qw = _moe_setup(case, cuda_dev)
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(T)).to(cuda_dev)
    got = _ops.fused_moe_w4(x, logits, qw, k)
    ids, w = route_ref(logits.cpu().numpy(), k)
    v = {n: _values(qw[n]) for n in ("w1", "w3", "w2")}
    exact, spread = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        xt = _np(x[t])
        for j in range(k):
            e = int(ids[t, j])
            h = v["w1"][e] @ xt
            a = h / (1 + np.exp(-h)) * (v["w3"][e] @ xt)
            y = v["w2"][e] @ a
            exact[t] += w[t, j] * y
            spread[t] += w[t, j] * (np.abs(y) + np.abs(v["w2"][e]) @ np.abs(a))
    # the fp32 sums inside are 2^-24-sized; 1 % on top of the roundings covers them
    bound = 2.0 ** -8 * np.abs(exact) * 1.01 + 2.0 ** -11 * 1.01 * spread + 1e-30
    assert (np.abs(_np(got) - exact) <= bound).all()
    # the same from its parts, bit for bit
    rids, rw = _ops.moe_route(logits, k)
    assert torch.equal(_ops.moe_experts_w4(_ops.moe_dispatch(None, rids, E), x, rids, rw, qw), got)
    # stage by stage with bf16 activations and rows: their roundings on top (2^-8 of each term, twice)
    p = _ops.moe_dispatch(None, torch.from_numpy(np.asarray(ids, np.int32)).to(cuda_dev), E)
    y = _ops.moe_down_w4(p, _ops.moe_gate_up_w4(p, qw, x=x), qw)
    staged = _ops.moe_combine_weighted(p, y, _ops.moe_route(logits, k)[1])
    assert (np.abs(_np(staged) - exact) <= 2.0 ** -8 * (1.01 * np.abs(exact) + 1.01 * spread) + 1e-30).all()
    out = torch.empty_like(x)
    assert _ops.fused_moe_w4(x, logits, qw, k, out=out) is out and torch.equal(out, got)


def test_experts_with_dropped_slots(cuda_dev):
    """Dropped slots weigh nothing; a token without any gets zero."""
    T, k, E, H, I = 21, 3, 6, 96, 160
    x, ids, qw = _moe_setup((T, k, E, H, I, 32, True), cuda_dev)
    ids[5] = -1
    ids[::4, 1] = -1
    w = torch.rand((T, k), device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, E)
    got = _ops.moe_experts_w4(p, x, ids, w, qw)
    y = _ops.moe_down_w4(p, _ops.moe_gate_up_w4(p, qw, dtype=torch.float32), qw, dtype=torch.float32)
    kept = int(p["num_rows_padded"])
    want = _ops.moe_combine_weighted(p, torch.where(torch.arange(T * k, device=cuda_dev)[:, None] < kept, y, 0.0), w)
    assert torch.equal(want.to(BF), got) and not got[5].any()
    none = torch.full_like(ids, -1)
    assert not _ops.moe_experts_w4(_ops.moe_dispatch(None, none, E), x, none, w, qw).any()


def test_token_of_nan_logits_is_reported_and_dropped(cuda_dev):
    x, _, qw = _moe_setup((5, 2, 8, 64, 96, 32, False), cuda_dev)
    logits = torch.randn((5, 8), device=cuda_dev)
    clean = _ops.fused_moe_w4(x, logits, qw, 2)
    logits[3] = float("nan")
    got = _ops.fused_moe_w4(x, logits, qw, 2)
    assert _lib.device_status(0) == _lib.EK_STATUS_BAD_INDEX
    keep = [0, 1, 2, 4]
    assert torch.equal(got[keep], clean[keep]) and not got[3].any()


def test_layer_forward_and_router_backward(cuda_dev):
    """The operators together, as a router is trained over frozen 4-bit experts:
    the logits' gradient against differences of the oracle's layer."""
    T, k, E, H, I = 6, 2, 5, 64, 96
    x, _, qw = _moe_setup((T, k, E, H, I, 32, False), cuda_dev)
    g = torch.Generator().manual_seed(11)
    logits, d_out = torch.randn((T, E), generator=g), torch.randn((T, H), generator=g).to(BF)
    ids, w = _ops.moe_route(logits.to(cuda_dev), k)
    p = _ops.moe_dispatch(x, ids, E)
    y = _ops.moe_down_w4(p, _ops.moe_gate_up_w4(p, qw), qw)
    d_y, d_w = _ops.moe_combine_weighted_grad(p, y, w, d_out.to(cuda_dev))
    d_logits = _np(_ops.moe_route_grad(ids, w, d_w, E))
    rows = _np(y)[p["slot_rows"].cpu().numpy()].reshape(T, k, H)
    chosen = ids.cpu().numpy().astype(np.int64)

    def loss(z):
        c = np.take_along_axis(z, chosen, axis=1)
        c = np.exp(c - c.max(axis=1, keepdims=True))
        c /= c.sum(axis=1, keepdims=True)
        return ((c[:, :, None] * rows).sum(axis=1) * _np(d_out)).sum()

    z = logits.double().numpy()
    for i in np.ndindex(T, E):
        a, b = z.copy(), z.copy()
        a[i] += 1e-5
        b[i] -= 1e-5
        num = (loss(a) - loss(b)) / 2e-5
        # differences: h^2 |f'''| ~ 1e-10 |f| and rounding 1e-16 |f| / h; fp32 sums: (H + k) 2^-24 |f|
        scale = np.abs(rows[i[0]] * _np(d_out)[i[0]]).sum()
        assert abs(num - d_logits[i]) <= ((H + 16) * 2.0 ** -24 + 1e-9) * scale
    # and the tokens' gradient of the way in, for rows' gradients that come back from the experts
    d_x = _ops.moe_dispatch_grad(p, d_y)
    wts = _np(w)
    want = (wts.sum(axis=1, keepdims=True) * _np(d_out))
    # two bf16 roundings: each row's and the sum's
    assert (np.abs(_np(d_x) - want) <= 2.0 ** -7 * 1.01 * np.abs(want) + 1e-6).all()


def test_layer_in_a_graph(cuda_dev):
    x, _, qw = _moe_setup((9, 2, 8, 256, 128, 64, True), cuda_dev)
    logits = torch.randn((9, 8), device=cuda_dev)
    _ops.fused_moe_w4(x, logits, qw, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _ops.fused_moe_w4(x, logits, qw, 2)
    for _ in range(2):
        logits.normal_()
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, _ops.fused_moe_w4(x, logits, qw, 2))


def test_experts_with_many_choices(cuda_dev):
    """More choices than a warp has lanes, each of many parts: the combine's list in pieces."""
    T, k, E, H, I = 3, 40, 48, 64, 4096
    x, ids, qw = _moe_setup((T, k, E, H, I, 128, False), cuda_dev)
    ids[1, 3] = -1
    w = torch.rand((T, k), device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, E)
    got = _ops.moe_experts_w4(p, x, ids, w, qw)
    y = _ops.moe_down_w4(p, _ops.moe_gate_up_w4(p, qw, dtype=torch.float32), qw, dtype=torch.float32)
    kept = int(p["num_rows_padded"])
    want = _ops.moe_combine_weighted(p, torch.where(torch.arange(T * k, device=cuda_dev)[:, None] < kept, y, 0.0), w)
    assert torch.equal(want.to(BF), got)


def test_results_written_over_their_inputs(cuda_dev):
    """out may be the tokens themselves: they are read before it is written."""
    qw = _integer_weight(256, 256, 64, True, BF, 6, cuda_dev)
    for M in (1, 3, 16, 40):
        x = torch.randint(-2, 3, (M, 256), device=cuda_dev).to(BF)
        want = _ops.gemm_w4(x, qw)
        assert _ops.gemm_w4(x, qw, out=x) is x and torch.equal(x, want)
    x, _, qw = _moe_setup((40, 2, 8, 256, 128, 64, False), cuda_dev)
    logits = torch.randn((40, 8), device=cuda_dev)
    want = _ops.fused_moe_w4(x, logits, qw, 2)
    assert torch.equal(_ops.fused_moe_w4(x, logits, qw, 2, out=x), want)


def test_two_streams_at_once(cuda_dev):
    """Calls in flight on two streams: each has its own workspace."""
    qw = _integer_weight(2048, 1024, 64, True, BF, 7, cuda_dev)
    xs = [torch.randint(-2, 3, (m, 1024), device=cuda_dev).to(BF) for m in (1, 16)]
    layer = _moe_setup((24, 2, 8, 512, 256, 64, False), cuda_dev)
    logits = torch.randn((24, 8), device=cuda_dev)
    want = [_ops.gemm_w4(x, qw) for x in xs] + [_ops.fused_moe_w4(layer[0], logits, layer[2], 2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for s, out in zip(streams, got):
            with torch.cuda.stream(s):
                out.append([_ops.gemm_w4(x, qw) for x in xs] + [_ops.fused_moe_w4(layer[0], logits, layer[2], 2)])
    torch.cuda.synchronize()
    for out in got[0] + got[1]:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_layer_empty_and_refusals(cuda_dev):
    x, ids, qw = _moe_setup((4, 2, 4, 64, 32, 32, False), cuda_dev)
    assert _ops.fused_moe_w4(x[:0], torch.empty((0, 4), device=cuda_dev), qw, 2).shape == (0, 64)
    p = _ops.moe_dispatch(None, ids, 4)
    for call, text in [(lambda: _ops.moe_gate_up_w4(p, qw), "no rows"),
                       (lambda: _ops.moe_gate_up_w4(p, qw, x=x[:3]), "shape"),
                       (lambda: _ops.moe_gate_up_w4(p, qw, x=x.half()), "bfloat16"),
                       (lambda: _ops.moe_down_w4(p, x, qw), "shape"),
                       (lambda: _ops.moe_gate_up_w4(_ops.moe_permute(ids, 4, x=x), qw), "shape"),
                       (lambda: _ops.fused_moe_w4(x, torch.empty((4, 3), device=cuda_dev), qw, 2), "gate_logits"),
                       (lambda: _ops.quant_moe_weights_w4(*[torch.zeros((2, 8, 32), device=cuda_dev)] * 3), "w2")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    assert _lib.device_status(0) == 0


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("stage", ["gate_up", "down", "experts"])
def test_nothing_is_written_after_an_empty_product(stage, captured, cuda_dev, monkeypatch):
    """Every slot dropped: what follows on the stream still comes after the launch
    that writes the tokens, so the workspace may be used again at once."""
    T, k, E, H, I = 4096, 2, 4, 2048, 2048
    w = torch.randn((E, I, H), device=cuda_dev, dtype=BF) * 0.02
    qw = _ops.quant_moe_weights_w4(w, w, w, group=128)
    x = torch.randn((T, H), device=cuda_dev).to(BF)
    act = torch.randn((T * k, I), device=cuda_dev).to(BF)
    ids = torch.full((T, k), -1, dtype=torch.int32, device=cuda_dev)
    wts = torch.rand((T, k), device=cuda_dev)
    perm = _ops.moe_dispatch(None, ids, E)
    buf = torch.empty(256 << 20, dtype=torch.uint8, device=cuda_dev)
    monkeypatch.setattr(_ops, "_scratch", lambda nbytes, codes: buf[:nbytes])
    bad = torch.zeros(20, dtype=torch.int64, device=cuda_dev)

    def once(i):
        if stage == "gate_up":
            _ops.moe_gate_up_w4(perm, qw, x=x)
        elif stage == "down":
            _ops.moe_down_w4(perm, act, qw)
        else:
            assert _ops.moe_experts_w4(perm, x, ids, wts, qw).shape == (T, H)
        buf.fill_(0x5A)
        bad[i] = (buf != 0x5A).sum()

    once(0)
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for i in range(20):
                once(i)
        graph.replay()
    else:
        for i in range(20):
            once(i)
    torch.cuda.synchronize()
    assert not bad.any()


def _by_definition(x, qw):
    """sum_k w x term by term, so that infinities meet the weights themselves."""
    with np.errstate(invalid="ignore"):
        return (_np(x)[:, None, :] * _values(qw)[None]).sum(axis=2)


def _same_kind(got, exact, rows):
    """Infinities of one sign, NaN and finite values where the definition has them."""
    a, b = _np(got)[rows], exact[rows]
    assert np.array_equal(np.isnan(a), np.isnan(b))
    assert np.array_equal(np.isposinf(a), np.isposinf(b)) and np.array_equal(np.isneginf(a), np.isneginf(b))


@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("M,N,K,group", [(1, 300, 257, 32), (2, 64, 4096, 128), (4, 40, 96, 64), (20, 70, 1030, 64),
                                         (40, 515, 700, 128)])
def test_gemm_infinite_tokens(M, N, K, group, dtype, mins, cuda_dev):
    """An infinite token element gives what (s q + m) x gives, weight by weight:
    an infinity of the product's sign, NaN where the weight is zero or two
    infinities oppose each other."""
    qw = _integer_weight(N, K, group, mins, dtype, M + N + K, cuda_dev)
    g = torch.Generator().manual_seed(K)
    x = torch.randint(-2, 3, (M, K), generator=g).to(dtype)
    clean = _ops.gemm_w4(x.to(cuda_dev), qw)
    bad = sorted({0, M // 2, M - 1})
    x[0, K - 1] = float("inf")
    if M > 1:
        x[M // 2, 3], x[M // 2, K // 2] = float("-inf"), float("inf")  # two of them, in two groups for most K
    if M > 2:
        x[M - 1, 7] = float("-inf")
        x[M - 1, 8] = float("-inf")
    got = _ops.gemm_w4(x.to(cuda_dev), qw)
    _same_kind(got, _by_definition(x, qw), bad)
    rest = [i for i in range(M) if i not in bad]
    assert torch.equal(got[rest], clean[rest])
    x[0, 0] = float("nan")
    assert _ops.gemm_w4(x.to(cuda_dev), qw)[0].isnan().all()


@pytest.mark.parametrize("M", [1, 3, 40])
def test_infinite_tokens_written_over(M, cuda_dev):
    """In place: the rows are looked at again while their outputs are written."""
    qw = _integer_weight(256, 256, 64, True, BF, 8, cuda_dev)
    x = torch.randint(-2, 3, (M, 256), generator=torch.Generator().manual_seed(M)).to(BF)
    x[0, 9] = float("inf")
    x[M - 1, 250] = float("-inf")
    exact, x = _by_definition(x, qw), x.to(cuda_dev)
    want = _ops.gemm_w4(x, qw)
    _same_kind(want, exact, [0, M - 1])
    assert _ops.gemm_w4(x, qw, out=x) is x and torch.equal(x.nan_to_num(7.0), want.nan_to_num(7.0))


def test_gemm_overflow_is_not_an_infinite_token(cuda_dev):
    """Finite tokens whose sum passes the type's range: an infinity of the sum's sign."""
    for mins in (False, True):
        qw = _integer_weight(48, 512, 64, mins, FP, 5, cuda_dev)
        x = torch.full((3, 512), 6e4, dtype=FP)
        exact = torch.from_numpy(_by_definition(x, qw)).to(FP)
        got = _ops.gemm_w4(x.to(cuda_dev), qw).cpu()
        assert exact.isinf().any() and torch.equal(got.isinf(), exact.isinf())
        assert torch.equal(got[got.isinf()], exact[exact.isinf()])


@pytest.mark.parametrize("T", [3, 90])
@pytest.mark.parametrize("mins", [False, True])
def test_expert_products_of_infinite_tokens(T, mins, cuda_dev):
    """gate/up, down and the layer: the kinds of the outputs follow the definition
    from the products' own inputs."""
    k, E, H, I = 2, 4, 264, 150
    x, ids, qw = _moe_setup((T, k, E, H, I, 32, mins), cuda_dev)
    x[1, 5] = float("inf")
    x[2, 200] = float("-inf")
    w = torch.full((T, k), 0.5, device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, E)
    act = _ops.moe_gate_up_w4(p, qw, dtype=torch.float32)
    y = _ops.moe_down_w4(p, act, qw, dtype=torch.float32)
    xp, a, r = _np(p["x_perm"]), _np(act), 0
    v = {n: _values(qw[n]) for n in ("w1", "w3", "w2")}
    exact_y = np.zeros((T * k, H))
    with np.errstate(invalid="ignore", over="ignore"):
        for e, c in enumerate(p["expert_counts"].tolist()):
            for i in range(r, r + c):
                h, u = (xp[i] * v["w1"][e]).sum(1), (xp[i] * v["w3"][e]).sum(1)
                _same_kind(act[i:i + 1], (h / (1 + np.exp(-h)) * u)[None], [0])
                exact_y[i] = (a[i] * v["w2"][e]).sum(1)
                _same_kind(y[i:i + 1], exact_y[i:i + 1], [0])
            r += c
        sr = p["slot_rows"].cpu().numpy().reshape(T, k)
        _same_kind(_ops.moe_experts_w4(p, x, ids, w, qw), (exact_y[sr] * 0.5).sum(axis=1), np.arange(T))


def test_router_backward_with_dropped_choices(cuda_dev):
    """Choices dropped for capacity were in the softmax: the logits' gradient, from
    the routed ids, against differences of softmax, drop and combine."""
    T, k, E, H, I = 7, 3, 6, 64, 96
    x, _, qw = _moe_setup((T, k, E, H, I, 32, True), cuda_dev)
    g = torch.Generator().manual_seed(12)
    logits, d_out = torch.randn((T, E), generator=g), torch.randn((T, H), generator=g).to(BF)
    ids, w = _ops.moe_route(logits.to(cuda_dev), k)
    over_capacity = torch.zeros((T, k), dtype=torch.bool, device=cuda_dev)
    over_capacity[0, 0] = over_capacity[2, 1] = over_capacity[2, 2] = over_capacity[5] = True
    p = _ops.moe_dispatch(x, ids.masked_fill(over_capacity, -1), E)
    y = _ops.moe_down_w4(p, _ops.moe_gate_up_w4(p, qw), qw)
    _, d_w = _ops.moe_combine_weighted_grad(p, y, w, d_out.to(cuda_dev))
    d_logits = _np(_ops.moe_route_grad(ids, w, d_w, E))
    sr = p["slot_rows"].cpu().numpy()
    rows = np.where((sr >= 0)[:, None], _np(y)[np.maximum(sr, 0)], 0.0).reshape(T, k, H)
    chosen = ids.cpu().numpy().astype(np.int64)

    def loss(z):
        c = np.exp(np.take_along_axis(z, chosen, axis=1))
        c /= c.sum(axis=1, keepdims=True)
        return ((c[:, :, None] * rows).sum(axis=1) * _np(d_out)).sum()

    z = logits.double().numpy()
    for i in np.ndindex(T, E):
        a, b = z.copy(), z.copy()
        a[i] += 1e-5
        b[i] -= 1e-5
        # differences: h^2 times the third derivative (1e-10 of the row), 2^-53 |f| / h of
        # the whole loss (below 100: 6e-10); fp32 sums: (H + 16) 2^-24 of the row
        scale = np.abs(rows[i[0]] * _np(d_out)[i[0]]).sum()
        assert abs((loss(a) - loss(b)) / 2e-5 - d_logits[i]) <= ((H + 16) * 2.0 ** -24 + 1e-9) * scale + 1e-9
    assert not d_logits[5].any()
    lost = _np(_ops.moe_route_grad(ids.masked_fill(over_capacity, -1), w, d_w, E))
    assert np.abs(lost - d_logits)[[0, 2]].max(axis=1).min() > 1e-3


@pytest.mark.parametrize("T", [2, 100])
def test_layer_on_a_partition(T, cuda_dev):
    """The 4-bit layer and its stages on a partition of 32 SMs: other cuts of the
    same sums, which are exact in the stages (small integers, power-of-two scales)."""
    from elastikernel_b200.green_ctx import create_sm_partition

    k, E, H, I = 2, 6, 320, 512
    g = torch.Generator().manual_seed(T)
    qw = {"E": E, "H": H, "I": I, "w1": _integer_weight(I, H, 64, True, BF, 1, cuda_dev, (E,)),
          "w3": _integer_weight(I, H, 64, True, BF, 2, cuda_dev, (E,)),
          "w2": _integer_weight(H, I, 64, True, BF, 3, cuda_dev, (E,))}
    x = torch.randint(-2, 3, (T, H), generator=g).to(BF).to(cuda_dev)
    act = torch.randint(-2, 3, (T * k, I), generator=g).to(BF).to(cuda_dev)
    logits = torch.randn((T, E), generator=g).to(cuda_dev)
    ids, w = _ops.moe_route(logits, k)
    p = _ops.moe_dispatch(x, ids, E)

    def once():
        return (_ops.moe_gate_up_w4(p, qw), _ops.moe_down_w4(p, act, qw, dtype=torch.float32),
                _ops.fused_moe_w4(x, logits, qw, k))

    want = once()
    stream, _ = create_sm_partition(cuda_dev, 32)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = once()
    stream.synchronize()
    # the gate and up sums are exact, so the activations are the same; so is the down product of integers
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # The layer's down product adds the same rounded activations in other cuts, each sum within
    # (I / 4 + 32) 2^-24 of S, its terms' magnitudes (1 + 2^-11 for their rounding); then one
    # rounding to bf16 each (2^-8).
    a, b, S = _np(_ops.moe_gate_up_w4(p, qw, dtype=torch.float32)), _bound(qw["w2"]), np.zeros((T, H))
    rows, experts = p["slot_rows"].cpu().numpy().reshape(T, k), ids.cpu().numpy()
    for t, j in np.ndindex(T, k):
        S[t] += float(w[t, j]) * (b[experts[t, j]] @ np.abs(a[rows[t, j]])) * (1 + 2.0 ** -11)
    one, other = _np(got[2]), _np(want[2])
    n = (I / 4 + 32) * 2.0 ** -24
    assert (np.abs(one - other) <= 2.0 ** -8 * (np.abs(one) + np.abs(other)) * (1 + 2.0 ** -7) + 2 * n * S).all()
