"""Row dispatch, weighted combine, their gradients and the routing gradient on
the GPU against the float64 oracle (oracle/rows.py).

Tolerances (derived, not fitted). A value computed in fp32 and rounded once
to T is off by at most eps(T)/2 of itself, plus the fp32 sum's own error: n
terms cost at most n roundings of 2^-24 of the sum of the terms' magnitudes S.
Each test passes n = the terms of the sum + 2 (the product and the last
rounding). Sums of small integers are exact in fp32 and compared for equality.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from elastikernel_b200 import _lib, _ops
from oracle import rows as orows

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CASES = [  # T, k, E, H, dtype, drop
    (1, 1, 1, 1, "bf16", "none"),
    (1, 8, 256, 7168, "bf16", "none"),
    (5, 3, 7, 33, "fp16", "some"),
    (48, 2, 8, 4096, "bf16", "none"),
    (64, 8, 256, 512, "bf16", "tail"),
    (127, 2, 8, 1111, "fp32", "some"),
    (257, 8, 300, 264, "fp32", "some"),
    (300, 5, 16, 130, "bf16", "all"),
    (513, 9, 40, 72, "fp16", "some"),
    (1030, 8, 16, 65, "bf16", "tail"),
    (1025, 1, 1024, 20, "fp32", "none"),
    (4100, 2, 3, 40, "fp16", "some"),
    (9000, 8, 64, 96, "bf16", "some"),
    (1500, 3, 12, 200, "fp32", "some"),
    (1200, 8, 9, 1024, "bf16", "some"),
    (200, 33, 64, 48, "fp16", "some"),
    (2, 17, 5, 2050, "bf16", "some"),
]
ID = [f"T{c[0]}k{c[1]}E{c[2]}H{c[3]}-{c[4]}-{c[5]}" for c in CASES]


def _ids(T, k, E, drop, rng):
    ids = rng.integers(0, E, (T, k)).astype(np.int32)  # an expert may be taken twice by a token, or by none
    if drop == "some":
        ids[rng.random((T, k)) < 0.3] = -1
    elif drop == "tail":
        ids[T - T // 3:] = -5
    elif drop == "all":
        ids[:] = -1
    return ids


def _setup(case, integers=False):
    T, k, E, H, dtype, drop = case
    rng = np.random.default_rng(T * 31 + k)
    ids = _ids(T, k, E, drop, rng)

    def rows(n):
        v = rng.integers(-2, 3, (n, H)) if integers else rng.normal(size=(n, H))
        return torch.from_numpy(v.astype(np.float32)).to(DTYPES[dtype])

    w = 2.0 ** rng.integers(-2, 2, (T, k)) if integers else rng.random((T, k))
    return ids, rows, torch.from_numpy(w.astype(np.float32))


def _np(t):
    return t.double().cpu().numpy()


def _close(got, exact, S, n, dtype):
    eps = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a subnormal step and more
    err = np.abs(_np(got) - exact)
    bound = eps * np.abs(exact) * (1 + 2.0 ** -10) + n * 2.0 ** -24 * S * (1 + eps) + tiny
    assert (err <= bound).all(), f"worst {np.max(err - bound):.3e} over its bound"


@pytest.mark.parametrize("case", CASES, ids=ID)
def test_dispatch(case, cuda_dev):
    T, k, E, H, dtype, _ = case
    ids, rows, _ = _setup(case)
    x = rows(T)
    p = _ops.moe_dispatch(x.to(cuda_dev), torch.from_numpy(ids).to(cuda_dev), E)
    slots, slot_rows, counts = orows.order(ids, E)
    assert np.array_equal(p["sorted_slots"].cpu().numpy(), slots)
    assert np.array_equal(p["slot_rows"].cpu().numpy(), slot_rows)
    assert np.array_equal(p["expert_counts"].cpu().numpy(), counts)
    assert int(p["num_rows_padded"]) == counts.sum()
    assert np.array_equal(_np(p["x_perm"]), orows.dispatch(_np(x), ids, E))


def test_dispatch_agrees_with_permute(cuda_dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((700, 128), generator=g).to(torch.bfloat16).to(cuda_dev)
    ids = torch.randint(0, 32, (700, 4), generator=g, dtype=torch.int32).to(cuda_dev)
    a, b = _ops.moe_dispatch(x, ids, 32), _ops.moe_permute(ids, 32, x=x, block_m=1)
    for key in ("sorted_slots", "expert_counts", "num_rows_padded", "x_perm"):
        assert torch.equal(a[key], b[key]), key


@pytest.mark.parametrize("integers", [True, False])
@pytest.mark.parametrize("case", CASES, ids=ID)
def test_dispatch_grad(case, integers, cuda_dev):
    T, k, E, H, dtype, _ = case
    ids, rows, _ = _setup(case, integers)
    d = rows(T * k)
    p = _ops.moe_dispatch(None, torch.from_numpy(ids).to(cuda_dev), E)
    got = _ops.moe_dispatch_grad(p, d.to(cuda_dev))
    v = orows.slot_values(_np(d), orows.order(ids, E)[1], T, k)
    if integers:
        assert np.array_equal(_np(got), v.sum(axis=1))  # |sum| <= 2 k < 256: exact in every type
    else:
        _close(got, v.sum(axis=1), np.abs(v).sum(axis=1), k + 2, DTYPES[dtype])


@pytest.mark.parametrize("case", CASES, ids=ID)
def test_combine_weighted(case, cuda_dev):
    T, k, E, H, dtype, _ = case
    ids, rows, w = _setup(case)
    y = rows(T * k)
    p = _ops.moe_dispatch(None, torch.from_numpy(ids).to(cuda_dev), E)
    sr = orows.order(ids, E)[1]
    # rows past the last kept one must not be read
    kept = int((sr >= 0).sum())
    yd = y.to(cuda_dev)
    yd[kept:] = float("nan")
    got = _ops.moe_combine_weighted(p, yd, w.to(cuda_dev))
    _close(got, orows.combine(_np(y), sr, w.numpy()), orows.combine(np.abs(_np(y)), sr, w.numpy()), k + 2,
           DTYPES[dtype])
    out = torch.full((T, H), 7.0, dtype=DTYPES[dtype], device=cuda_dev)
    assert _ops.moe_combine_weighted(p, yd, w.to(cuda_dev), out=out) is out
    assert torch.equal(out, got)


@pytest.mark.parametrize("integers", [True, False])
@pytest.mark.parametrize("case", CASES, ids=ID)
def test_combine_weighted_grad(case, integers, cuda_dev):
    T, k, E, H, dtype, _ = case
    ids, rows, w = _setup(case, integers)
    y, d = rows(T * k), rows(T)
    sr = orows.order(ids, E)[1]
    p = _ops.moe_dispatch(None, torch.from_numpy(ids).to(cuda_dev), E)
    yd = y.to(cuda_dev)
    yd[int((sr >= 0).sum()):] = float("nan")
    d_y, d_w = _ops.moe_combine_weighted_grad(p, yd, w.to(cuda_dev), d.to(cuda_dev))
    e_y, e_w = orows.combine_grad(_np(y), sr, w.numpy(), _np(d))
    if integers:  # products of {-2..2} and powers of two; sums below 4 H < 2^24
        assert np.array_equal(_np(d_y), e_y) and np.array_equal(_np(d_w), e_w)
    else:
        _close(d_y, e_y, np.abs(e_y), 2, DTYPES[dtype])
        S = (np.abs(orows.slot_values(_np(y), sr, T, k)) * np.abs(_np(d))[:, None, :]).sum(axis=2)
        _close(d_w, e_w, S, H + 2, torch.float32)


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 256, 8), (3, 5, 5), (333, 8, 2), (1000, 60, 6), (77, 1000, 8),
                                   (50, 33, 12), (5000, 256, 8), (9, 4, 1)])
def test_route_grad(T, E, k, cuda_dev):
    rng = np.random.default_rng(T + E)
    z = torch.from_numpy(rng.normal(size=(T, E)).astype(np.float32))
    if E <= 256 and k <= 8:
        ids, w = _ops.moe_route(z.to(cuda_dev), k)
    else:
        top = torch.topk(z, k, dim=1)
        ids, w = top.indices.int().to(cuda_dev), torch.softmax(top.values, 1).to(cuda_dev)
    d = torch.from_numpy(rng.normal(size=(T, k)).astype(np.float32))
    got = _ops.moe_route_grad(ids, w, d.to(cuda_dev), E)
    e = orows.route_grad(ids.cpu().numpy(), w.cpu().numpy(), d.numpy(), E)
    # |dw_j| + sum |w_i dw_i| bounds what cancels; k + 4 roundings
    S = np.zeros_like(e)
    m = np.abs(w.cpu().numpy() * d.numpy()).sum(axis=1, keepdims=True)
    np.put_along_axis(S, ids.cpu().numpy().astype(np.int64), w.cpu().numpy() * (np.abs(d.numpy()) + m), 1)
    _close(got, e, S, k + 4, torch.float32)
    assert (_np(got)[e == 0] == 0).all()


def test_route_grad_repeated_and_foreign_ids(cuda_dev):
    ids = np.array([[2, 2, 0], [-1, 9, 1]], np.int32)
    w = np.array([[0.25, 0.25, 0.5], [0.5, 0.25, 0.25]], np.float32)
    d = np.array([[1, 2, 4], [8, 4, 2]], np.float32)
    got = _ops.moe_route_grad(*(torch.from_numpy(a).to(cuda_dev) for a in (ids, w, d)), 4)
    assert np.array_equal(_np(got), orows.route_grad(ids, w, d, 4))  # dyadic values: exact


def test_misaligned_views(cuda_dev):
    """Contiguous views that start one element into their storage."""
    T, k, E, H = 37, 3, 6, 96
    ids = torch.from_numpy(_ids(T, k, E, "some", np.random.default_rng(5))).to(cuda_dev)
    g = torch.Generator().manual_seed(5)

    def off(n, dtype):
        return torch.randn((n * H + 1,), generator=g).to(dtype).to(cuda_dev)[1:].view(n, H)

    for dtype in DTYPES.values():
        x, y, d = off(T, dtype), off(T * k, dtype), off(T, dtype)
        w = torch.rand((T, k), generator=g).to(cuda_dev)
        p, pa = _ops.moe_dispatch(x, ids, E), _ops.moe_dispatch(x.clone(), ids, E)
        assert torch.equal(p["x_perm"], pa["x_perm"])
        assert torch.equal(_ops.moe_dispatch_grad(p, y), _ops.moe_dispatch_grad(p, y.clone()))
        assert torch.equal(_ops.moe_combine_weighted(p, y, w), _ops.moe_combine_weighted(p, y.clone(), w))
        a, b = _ops.moe_combine_weighted_grad(p, y, w, d), _ops.moe_combine_weighted_grad(p, y.clone(), w, d.clone())
        assert torch.equal(a[0], b[0])
        # another vector width sums in another order: both within H + 2 roundings of the exact value
        S = (y.double().abs() @ d.double().abs().t()).max()
        assert (a[1] - b[1]).abs().max() <= 2 * (H + 2) * 2.0 ** -24 * S


def test_out_of_range_id_is_reported_and_dropped(cuda_dev):
    ids = torch.tensor([[0, 4], [1, 2]], dtype=torch.int32, device=cuda_dev)
    x = torch.ones((2, 16), device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, 4)
    assert _lib.device_status(0) == _lib.EK_STATUS_BAD_INDEX
    assert p["slot_rows"].tolist() == [0, -1, 1, 2]
    assert p["x_perm"][3].abs().sum() == 0


def test_empty_batch(cuda_dev):
    ids = torch.empty((0, 2), dtype=torch.int32, device=cuda_dev)
    x = torch.empty((0, 64), device=cuda_dev)
    w = torch.empty((0, 2), device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, 4)
    assert p["expert_counts"].tolist() == [0, 0, 0, 0] and int(p["num_rows_padded"]) == 0
    assert _ops.moe_dispatch_grad(p, x).shape == (0, 64)
    assert _ops.moe_combine_weighted(p, x, w).shape == (0, 64)
    d_y, d_w = _ops.moe_combine_weighted_grad(p, x, w, x)
    assert d_y.shape == (0, 64) and d_w.shape == (0, 2)
    assert _ops.moe_route_grad(ids, w, w, 4).shape == (0, 4)


def test_infinite_and_nan_rows_stay_with_their_tokens(cuda_dev):
    """A non-finite row touches its own token alone."""
    ids = torch.tensor([[0, 1], [1, 2], [-1, 0]], dtype=torch.int32, device=cuda_dev)
    p = _ops.moe_dispatch(None, ids, 3)
    y = torch.ones((6, 40), dtype=torch.bfloat16, device=cuda_dev)
    y[int(p["slot_rows"][0])] = float("inf")
    y[int(p["slot_rows"][3])] = float("nan")
    w = torch.full((3, 2), 0.5, device=cuda_dev)
    out = _ops.moe_combine_weighted(p, y, w)
    assert out[0].isinf().all() and out[1].isnan().all() and (out[2] == 0.5).all()
    _, d_w = _ops.moe_combine_weighted_grad(p, y, w, torch.ones((3, 40), dtype=torch.bfloat16, device=cuda_dev))
    assert d_w[0, 0].isinf() and d_w[0, 1] == 40 and d_w[1, 1].isnan() and d_w[2, 0] == 0 and d_w[2, 1] == 40


def test_rows_past_2_31_elements(cuda_dev):
    T, k, E, H = 140000, 8, 4, 2056  # 1.12 M rows, 2.3e9 elements
    x = torch.empty((T, H), dtype=torch.bfloat16, device=cuda_dev).random_(-8, 9)
    ids = torch.randint(0, E, (T, k), device=cuda_dev, dtype=torch.int32)
    w = torch.full((T, k), 0.125, device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, E)
    assert torch.equal(_ops.moe_combine_weighted(p, p["x_perm"], w), x)
    d_x = _ops.moe_dispatch_grad(p, p["x_perm"])
    assert torch.equal(d_x, x * 8)
    d_y, d_w = _ops.moe_combine_weighted_grad(p, p["x_perm"], w, x)
    sr = p["slot_rows"].view(T, k)
    for t in (0, 1, T // 2, T - 1):
        assert torch.equal(d_y[sr[t].long()], (x[t] / 8).expand(k, H))
    assert torch.equal(d_w, (x.float() * x.float()).sum(1, keepdim=True).expand(T, k))  # integers < 2^24


def test_other_stream_and_graph_replay(cuda_dev):
    """The whole round on a side stream, then captured and replayed on new contents."""
    T, k, E, H = 200, 4, 16, 256
    g = torch.Generator().manual_seed(9)
    x = torch.empty((T, H), dtype=torch.bfloat16, device=cuda_dev)
    ids = torch.empty((T, k), dtype=torch.int32, device=cuda_dev)
    w = torch.empty((T, k), device=cuda_dev)

    def fill(seed):
        g.manual_seed(seed)
        x.copy_(torch.randn((T, H), generator=g))
        ids.copy_(torch.randint(-1, E, (T, k), generator=g))
        w.copy_(torch.rand((T, k), generator=g))

    def once():
        p = _ops.moe_dispatch(x, ids, E)
        out = _ops.moe_combine_weighted(p, p["x_perm"], w)
        d_y, d_w = _ops.moe_combine_weighted_grad(p, p["x_perm"], w, x)
        return p["sorted_slots"], out, d_y, d_w, _ops.moe_dispatch_grad(p, d_y), _ops.moe_route_grad(
            ids.clamp(min=0), w, d_w, E)

    s = torch.cuda.Stream()
    fill(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        side = once()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, once()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for seed in (2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, once()))


def test_front_end_refusals(cuda_dev):
    ids = torch.zeros((4, 2), dtype=torch.int32, device=cuda_dev)
    x = torch.zeros((4, 16), dtype=torch.bfloat16, device=cuda_dev)
    w = torch.zeros((4, 2), device=cuda_dev)
    p = _ops.moe_dispatch(x, ids, 2)
    y = p["x_perm"]
    for call, text in [
            (lambda: _ops.moe_dispatch(x, ids.long(), 2), "int32"),
            (lambda: _ops.moe_dispatch(x, ids.t(), 2), "contiguous"),
            (lambda: _ops.moe_dispatch(x[:3], ids, 2), "4 rows"),
            (lambda: _ops.moe_dispatch(x.double(), ids, 2), "bf16, fp16 or fp32"),
            (lambda: _ops.moe_dispatch(torch.zeros((16, 4), device=cuda_dev).t(), ids, 2), "contiguous"),
            (lambda: _ops.moe_dispatch(x, ids, 0), "1 <= E"),
            (lambda: _ops.moe_combine_weighted(p, y, w.double()), "topk_weights"),
            (lambda: _ops.moe_combine_weighted(p, y, w[:3]), "topk_weights"),
            (lambda: _ops.moe_combine_weighted(p, y, w, out=x.float()), "out must be"),
            (lambda: _ops.moe_combine_weighted(p, y, w, out=y[2:6]), "overlap"),
            (lambda: _ops.moe_combine_weighted_grad(p, y, w, x.float()), "d_out"),
            (lambda: _ops.moe_combine_weighted_grad(p, y, w, x[:3]), "d_out"),
            (lambda: _ops.moe_route_grad(ids, w, w, 0), "positive"),
            (lambda: _ops.moe_route_grad(ids, w, w[:3], 4), "d_weights"),
            (lambda: _ops.moe_dispatch_grad(_ops.moe_permute(ids, 2, block_m=1), y), "slot_rows")]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_route_grad_of_a_warp_past_2_31_logits(cuda_dev):
    """A warp's 16 tokens have more than 2^31 logits (9 GB in all)."""
    T, E = 17, (1 << 27) + 1
    ids = torch.tensor([[E - 1, 3]], dtype=torch.int32, device=cuda_dev).expand(T, 2).contiguous()
    w = torch.full((T, 2), 0.5, device=cuda_dev)
    d = torch.tensor([[1.0, 3.0]], device=cuda_dev).expand(T, 2).contiguous()
    got = _ops.moe_route_grad(ids, w, d, E)
    assert (got[:, E - 1] == -0.5).all() and (got[:, 3] == 0.5).all()
    assert int(torch.count_nonzero(got)) == 2 * T


def _poisoned_empty(monkeypatch):
    """torch.empty gives memory full of NaN, so that what nobody writes is seen."""
    plain = torch.empty

    def empty(*size, **kw):
        t = plain(*size, **kw)
        return t.view(torch.uint8).fill_(0xFF).view(t.dtype) if t.is_cuda and t.numel() and t.dtype != torch.int32 else t

    monkeypatch.setattr(torch, "empty", empty)


def _order_with_drops(T, k, E, drop, dev):
    """Distinct experts per token: all ids, and the same with dropped slots at -1."""
    g = torch.Generator().manual_seed(T + k)
    ids = torch.topk(torch.randn((T, E), generator=g), k, dim=1).indices.int()
    kept = ids.clone()
    kept[torch.from_numpy(_ids(T, k, E, drop, np.random.default_rng(T)) < 0)] = -1
    if drop == "some":
        kept[0, 0] = -1
    return ids.to(dev), kept.to(dev), torch.rand((T, k), generator=g).to(dev)


@pytest.mark.parametrize("drop", ["none", "some", "tail", "all"])
@pytest.mark.parametrize("T,H,I", [(1, 2048, 1024), (2, 2048, 1024), (4, 2048, 1024), (16, 2048, 1024), (300, 256, 640)])
def test_dropped_slots_through_the_bf16_experts(T, H, I, drop, cuda_dev, monkeypatch):
    """The layer over an order with dropped slots is the layer over the whole order
    with their weights at zero, bit for bit (each output sums the same K blocks in
    the same order); a K split sums in another order, so neither side splits."""
    E, k = 8, 2
    ids, kept, w = _order_with_drops(T, k, E, drop, cuda_dev)
    g = torch.Generator().manual_seed(H + T)
    x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(cuda_dev)
    w1, w3 = (torch.randn((E, I, H), generator=g).mul_(H ** -0.5).to(torch.bfloat16).to(cuda_dev) for _ in range(2))
    w2 = torch.randn((E, H, I), generator=g).mul_(I ** -0.5).to(torch.bfloat16).to(cuda_dev)
    _poisoned_empty(monkeypatch)
    full = _ops.moe_permute(ids, E, x=x, block_m=1)
    masked = torch.where(kept >= 0, w, 0.0)
    want = _ops.moe_down_packed(full, _ops.moe_gate_up_packed(full, w1, w3, ksplit=False), w2, masked, ksplit=False)
    p = _ops.moe_dispatch(x, kept, E)
    act = _ops.moe_gate_up_packed(p, w1, w3, ksplit=False)
    y = _ops.moe_down_packed(p, act, w2, w, ksplit=False)
    assert torch.equal(y, want)
    assert torch.equal(_ops.moe_combine(y, T, k), _ops.moe_combine(want, T, k))
    if bool((kept < 0).any()):  # left to itself the product does not split an order that is not whole
        assert torch.equal(_ops.moe_down_packed(p, act, w2, w), want)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("drop", ["some", "tail", "all"])
@pytest.mark.parametrize("T", [5, 300])
def test_dropped_slots_through_the_e4m3_experts(T, drop, pow2, cuda_dev, monkeypatch):
    H, I, E, k = 256, 512, 8, 2
    ids, kept, w = _order_with_drops(T, k, E, drop, cuda_dev)
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(cuda_dev)
    w1, w3 = (torch.randn((E, I, H), generator=g).mul_(H ** -0.5).to(torch.bfloat16).to(cuda_dev) for _ in range(2))
    w2 = torch.randn((E, H, I), generator=g).mul_(I ** -0.5).to(torch.bfloat16).to(cuda_dev)
    qw = _ops.quant_moe_weights_fp8(w1, w2, w3, pow2=pow2)
    _poisoned_empty(monkeypatch)

    def layer(p, weights):
        xq, xs = _ops.quant_e4m3_kmajor(p["x_perm"], pow2=pow2)
        act = _ops.moe_gate_up_fp8bs(p, xq, xs, qw)
        aq, as_ = _ops.quant_e4m3_kmajor(act, pow2=pow2)
        return _ops.moe_combine(_ops.moe_down_fp8bs(p, aq, as_, qw, weights), T, k)

    want = layer(_ops.moe_permute(ids, E, x=x, block_m=1), torch.where(kept >= 0, w, 0.0))
    assert torch.equal(layer(_ops.moe_dispatch(x, kept, E), w), want)


def test_padded_products_refuse_a_dispatch_order(cuda_dev):
    p = _ops.moe_dispatch(torch.zeros((4, 64), dtype=torch.bfloat16, device=cuda_dev),
                          torch.zeros((4, 2), dtype=torch.int32, device=cuda_dev), 2)
    w1, w2 = (torch.zeros(s, dtype=torch.bfloat16, device=cuda_dev) for s in ((2, 32, 64), (2, 64, 32)))
    act = torch.zeros((8, 32), dtype=torch.bfloat16, device=cuda_dev)
    for call in (lambda: _ops.moe_gate_up(p, w1, w1),
                 lambda: _ops.moe_down(p, act, w2, torch.ones((4, 2), device=cuda_dev))):
        with pytest.raises(RuntimeError, match="moe_permute"):
            call()


@pytest.mark.parametrize("H,dtype", [((1 << 29) + 12, "fp32"), ((1 << 30) - 3, "bf16"), (1 << 30, "bf16")])
def test_rows_past_2_31_bytes(H, dtype, cuda_dev):
    """Single rows whose bytes do not fit 31 bits, through each operator on rows."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.empty((1, H), dtype=DTYPES[dtype], device=cuda_dev).random_(-8, 9)
    p = _ops.moe_dispatch(x, torch.zeros((1, 1), dtype=torch.int32, device=cuda_dev), 2)
    assert torch.equal(p["x_perm"], x)
    w = torch.full((1, 1), 2.0, device=cuda_dev)
    out = torch.full_like(x, -77)
    assert torch.equal(_ops.moe_combine_weighted(p, x, w, out=out), x * 2)
    assert torch.equal(_ops.moe_dispatch_grad(p, x), x)
    one = torch.zeros_like(x)
    one[0, 5], one[0, H - 1] = 1, 2  # the dot product meets two elements alone: exact
    d_y, d_w = _ops.moe_combine_weighted_grad(p, x, w, one)
    assert torch.equal(d_y, one * 2)
    assert d_w.item() == x[0, 5].item() + 2 * x[0, H - 1].item()


@pytest.mark.parametrize("E", [3, 64, 1000])
@pytest.mark.parametrize("k", [16, 17, 20, 31, 32, 33, 40, 100])
def test_route_grad_of_many_choices(k, E, cuda_dev):
    """Up to 32 choices a token's lanes hold them, past that every logit looks
    through them; repeated ids (more choices than experts among them) and ids outside
    [0, E) in each. |w (dw - mean)| bounds a term, an entry sums up to k of them
    and the mean k products: 2 k + 4 roundings."""
    T = 37
    rng = np.random.default_rng(k * E)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[rng.random((T, k)) < 0.1] = -1
    ids[rng.random((T, k)) < 0.05] = E + 3
    ids[5] = 2  # one expert for all choices
    w = rng.random((T, k)).astype(np.float32)
    w /= w.sum(axis=1, keepdims=True)
    d = rng.normal(size=(T, k)).astype(np.float32)
    got = _ops.moe_route_grad(*(torch.from_numpy(a).to(cuda_dev) for a in (ids, w, d)), E)
    S = np.zeros((T, E))
    m = np.abs(w * d).sum(axis=1, keepdims=True)
    t, j = np.nonzero((ids >= 0) & (ids < E))
    np.add.at(S, (t, ids[t, j]), (w * (np.abs(d) + m))[t, j])
    _close(got, orows.route_grad(ids, w, d, E), S, 2 * k + 4, torch.float32)
    assert (_np(got)[S == 0] == 0).all()


@pytest.mark.parametrize("integers", [True, False])
@pytest.mark.parametrize("T,k,H,dtype", [(1300, 9, 64, "bf16"), (1300, 9, 64, "fp32"), (1200, 17, 33, "fp16"),
                                         (1184, 12, 1024, "bf16"), (2500, 33, 7, "bf16")])
def test_combine_grad_of_short_rows_in_several_turns(T, k, H, dtype, integers, cuda_dev):
    """A warp per token (many short rows) with more choices than one turn takes."""
    case = (T, k, 24, H, dtype, "some")
    ids, rows, w = _setup(case, integers)
    y, d = rows(T * k), rows(T)
    sr = orows.order(ids, 24)[1]
    p = _ops.moe_dispatch(None, torch.from_numpy(ids).to(cuda_dev), 24)
    d_y, d_w = _ops.moe_combine_weighted_grad(p, y.to(cuda_dev), w.to(cuda_dev), d.to(cuda_dev))
    e_y, e_w = orows.combine_grad(_np(y), sr, w.numpy(), _np(d))
    if integers:
        assert np.array_equal(_np(d_y), e_y) and np.array_equal(_np(d_w), e_w)
    else:
        _close(d_y, e_y, np.abs(e_y), 2, DTYPES[dtype])
        S = (np.abs(orows.slot_values(_np(y), sr, T, k)) * np.abs(_np(d))[:, None, :]).sum(axis=2)
        _close(d_w, e_w, S, H + 2, torch.float32)


@pytest.mark.parametrize("T", [24, 600])
def test_rows_on_a_partition(T, cuda_dev):
    """The row operators on a partition of 32 SMs: as on the whole device."""
    from elastikernel_b200.green_ctx import create_sm_partition

    k, E, H = 4, 16, 264
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(cuda_dev)
    ids = torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32).to(cuda_dev)
    w = torch.rand((T, k), generator=g).to(cuda_dev)

    def once():
        p = _ops.moe_dispatch(x, ids, E)
        out = _ops.moe_combine_weighted(p, p["x_perm"], w)
        d_y, d_w = _ops.moe_combine_weighted_grad(p, p["x_perm"], w, x)
        return p["sorted_slots"], p["x_perm"], out, d_y, d_w, _ops.moe_dispatch_grad(p, d_y), _ops.moe_route_grad(
            ids.clamp(min=0), w, d_w, E)

    want = once()
    stream, _ = create_sm_partition(cuda_dev, 32)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = once()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
