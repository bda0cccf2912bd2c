"""Operators around the fused-MoE layer and the small-batch GEMM, with their plain forms.

* dispatch: tokens sorted by expert (rows copied into expert-major order), and its
  gradient (the rows' gradients summed back per token);
* combine: the experts' rows back to the tokens with the routing weights applied,
  and its gradient (rows and weights);
* route_grad: the gradient of the renormalised top-k routing weights with respect
  to the gate logits;
* gemm_w4: products of a few token rows with a 4-bit weight matrix with group scales;
* moe_w4: the whole MoE layer over 4-bit experts, for small batches.

``listed()`` names the measured cases, ``draw(rng)`` makes further ones of the
same ranges, ``prepare(case, seed)`` makes the inputs on the GPU, ``run(state)``
is one pass (plain torch, or the package's operators when ``own`` is set) and
``exact(case, seed)`` the same outputs in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_W4_PAD = 32  # a row of codes is padded to a whole number of 32 elements (16 bytes)


# ------------------------------------------------------------------------ cases
def _rows_case(op, T, k, E, H, dtype, drop=0.0, **extra):
    return dict(op=op, T=T, k=k, E=E, H=H, dtype=dtype, drop=drop, **extra)


def _gemm_case(M, N, K, dtype, group, mins):
    return dict(op="gemm_w4", M=M, N=N, K=K, dtype=dtype, group=group, mins=mins)


def _moe_case(T, k, E, H, I, group, mins):
    return dict(op="moe_w4", T=T, k=k, E=E, H=H, I=I, group=group, mins=mins)


def listed():
    return [
        # a decode batch over the DeepSeek-V3 shape: 512 short rows, launch latency counts
        dict(name="dispatch-decode", **_rows_case("dispatch", 64, 8, 256, 7168, "bf16")),
        # a training or prompt batch of the same shape, a tenth of the slots over capacity or padding
        dict(name="dispatch-long", **_rows_case("dispatch", 8192, 8, 256, 7168, "bf16", drop=0.1)),
        # backward of the dispatch at the Mixtral shape, every slot kept
        dict(name="dispatch-grad", **_rows_case("dispatch_grad", 8192, 2, 8, 4096, "bf16")),
        # the way back for a decode batch at the Mixtral shape
        dict(name="combine-decode", **_rows_case("combine", 48, 2, 8, 4096, "bf16")),
        # backward of the way back over a long batch
        dict(name="combine-grad-long", **_rows_case("combine_grad", 4096, 8, 256, 7168, "bf16", drop=0.1)),
        # odd sizes in fp32: rows that no wide load fits, a batch with padding
        dict(name="combine-grad-ragged", **_rows_case("combine_grad", 1001, 3, 60, 1111, "fp32", drop=0.2)),
        # router training: a short batch over few experts, a long one over many
        dict(name="route-grad-short", op="route_grad", T=333, k=2, E=8),
        dict(name="route-grad-long", op="route_grad", T=32768, k=8, E=256),
        # one token through a square projection: latency of the smallest weight
        dict(name="gemm-w4-token", **_gemm_case(1, 4096, 4096, "bf16", 128, False)),
        # a decode batch through a wide projection, small groups with minima
        dict(name="gemm-w4-batch", **_gemm_case(16, 14336, 4096, "fp16", 64, True)),
        # one token through a Mixtral-shaped layer
        dict(name="moe-w4-token", **_moe_case(1, 2, 8, 4096, 14336, 128, False)),
        # a decode batch on one expert-parallel rank of the DeepSeek-V3 shape
        dict(name="moe-w4-batch", **_moe_case(64, 8, 32, 7168, 2048, 128, False)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dispatch", "dispatch_grad", "combine", "combine_grad", "route_grad", "gemm_w4", "moe_w4"])
    if op == "route_grad":
        E = _log_int(rng, 2, 256)
        return dict(op=op, T=_log_int(rng, 1, 32768), k=rng.randint(1, min(8, E)), E=E)
    if op == "gemm_w4":
        while True:
            M, N, K = _log_int(rng, 1, 64), _log_int(rng, 64, 28672), _log_int(rng, 128, 14336)
            if rng.random() < 0.6:
                K = max(128, K // 128 * 128)
            if N * K <= 14336 * 4096:
                break
        return _gemm_case(M, N, K, rng.choice(["bf16", "fp16"]), rng.choice([32, 64, 128]), rng.random() < 0.4)
    if op == "moe_w4":
        while True:
            E = _log_int(rng, 2, 64)
            H, I = 8 * _log_int(rng, 32, 896), 8 * _log_int(rng, 32, 1792)
            if E * H * I <= 8 * 4096 * 14336:
                break
        return _moe_case(_log_int(rng, 1, 64), rng.randint(1, min(8, E)), E, H, I, rng.choice([32, 64, 128]),
                         rng.random() < 0.4)
    while True:
        T, H = _log_int(rng, 1, 16384), _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            H = max(64, H // 64 * 64)
        E = _log_int(rng, 2, 512)
        k = rng.randint(1, min(8, E))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = _rows_case(op, T, k, E, H, dtype, drop=rng.choice([0.0, 0.0, 0.1, 0.5]))
        if work(c)["bytes"] <= 900e6:
            return c


def _padded(K):
    return -(-K // _W4_PAD) * _W4_PAD


def _w4_bytes(rows, K, group, mins):
    """Codes (two per byte) and the 16-bit scales and minima of `rows` weight rows."""
    return rows * (K / 2 + -(-K // group) * 2 * (2 if mins else 1))


def work(case):
    op = case["op"]
    if op == "route_grad":
        T, k, E = case["T"], case["k"], case["E"]
        return {"bytes": T * k * 12 + T * E * 4, "flops": 4 * T * k}
    if op == "gemm_w4":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": _w4_bytes(N, K, case["group"], case["mins"]) + 2 * M * (N + K), "flops": 2 * M * N * K}
    if op == "moe_w4":
        T, k, E, H, I = (case[n] for n in ("T", "k", "E", "H", "I"))
        hit = E * (1.0 - (1.0 - k / E) ** T)  # experts that at least one token takes, uniform routing
        w = 2 * _w4_bytes(I, H, case["group"], case["mins"]) + _w4_bytes(H, I, case["group"], case["mins"])
        return {"bytes": hit * w + T * (2 * H * 2 + 4 * E), "flops": 6 * T * k * H * I}
    T, k, E, H = (case[n] for n in ("T", "k", "E", "H"))
    row, n = H * _BYTES[case["dtype"]], T * k
    kept = n * (1.0 - case["drop"])
    if op == "dispatch":  # ids in; rows, both maps and the counts out
        return {"bytes": T * row + n * row + n * 12 + 4 * E, "flops": 0}
    if op == "dispatch_grad":
        return {"bytes": kept * row + T * row + 4 * n, "flops": n * H}
    if op == "combine":
        return {"bytes": kept * row + T * row + 8 * n, "flops": 2 * n * H}
    return {"bytes": kept * row + T * row + n * row + 12 * n, "flops": 3 * n * H}


# ------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _routing(case, g):
    """Distinct experts per token, some experts more popular, as a trained router gives;
    `drop` of the slots are -1: half of them the tokens of a padded tail, half over capacity."""
    T, k, E = case["T"], case["k"], case["E"]
    logits = torch.randn((T, E), generator=g, device="cuda") + 0.7 * torch.randn((1, E), generator=g, device="cuda")
    ids = torch.topk(logits, k, dim=1).indices.to(torch.int32)
    drop = case.get("drop", 0.0)
    if drop > 0:
        ids[T - int(T * drop / 2):] = -1
        over = torch.rand((T, k), generator=g, device="cuda") < drop / 2
        ids = torch.where(over, torch.full_like(ids, -1), ids)
    return ids.contiguous()


def _weights_of(case, g):
    p = torch.randn((case["T"], case["k"]), generator=g, device="cuda").exp()
    return (p / p.sum(dim=1, keepdim=True)).contiguous()


def _quantise(w, group, mins, dtype):
    """4-bit codes (low nibble first, rows padded to 32 elements), scales and minima of w [N, K] fp32."""
    N, K = w.shape
    G = -(-K // group)
    wp = torch.zeros((N, G * group), device=w.device)
    wp[:, :K] = w
    v = wp.view(N, G, group)
    if mins:
        lo = v.amin(dim=2).to(dtype)
        s = ((v.amax(dim=2) - lo.float()) / 15.0).to(dtype)
    else:
        lo = None
        s = (v.abs().amax(dim=2) / 7.0).to(dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (v - lo.float()[:, :, None]) / s.float()[:, :, None] if mins else v / s.float()[:, :, None] + 8.0
    q = q.round_().clamp_(0, 15).to(torch.uint8).view(N, G * group)[:, :_padded(K)]
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), s, lo


def _quantised_stack(E, N, K, case, dtype, g):
    parts = [_quantise(torch.randn((N, K), generator=g, device="cuda") / math.sqrt(K), case["group"], case["mins"],
                       dtype) for _ in range(E)]
    codes = torch.stack([p[0] for p in parts])
    return codes, torch.stack([p[1] for p in parts]), torch.stack([p[2] for p in parts]) if case["mins"] else None


def _as_qw(codes, scales, mins, K, group):
    """The 4-bit weight a program holds: the same tensors plain or own."""
    return {"codes": codes, "scales": scales, "mins": mins, "K": K, "group": group}


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"case": case, "op": op}
    if op == "route_grad":
        logits = torch.randn((case["T"], case["E"]), generator=g, device="cuda")
        top = torch.topk(logits, case["k"], dim=1)
        st["ids"] = top.indices.to(torch.int32).contiguous()
        st["weights"] = torch.softmax(top.values, dim=1).contiguous()
        st["d_weights"] = torch.randn((case["T"], case["k"]), generator=g, device="cuda")
        return st
    if op == "gemm_w4":
        dt = _DTYPES[case["dtype"]]
        st["x"] = torch.randn((case["M"], case["K"]), generator=g, device="cuda").to(dt)
        w = torch.randn((case["N"], case["K"]), generator=g, device="cuda") / math.sqrt(case["K"])
        st["qw"] = _as_qw(*_quantise(w, case["group"], case["mins"], dt), case["K"], case["group"])
        return st
    if op == "moe_w4":
        T, E, H, I = (case[n] for n in ("T", "E", "H", "I"))
        st["x"] = torch.randn((T, H), generator=g, device="cuda").to(torch.bfloat16)
        st["logits"] = torch.randn((T, E), generator=g, device="cuda")
        st["qw"] = {"E": E, "H": H, "I": I}
        for name, n, kk in (("w1", I, H), ("w3", I, H), ("w2", H, I)):
            st["qw"][name] = _as_qw(*_quantised_stack(E, n, kk, case, torch.bfloat16, g), kk, case["group"])
        return st
    dt = _DTYPES[case["dtype"]]
    T, k, E, H = (case[n] for n in ("T", "k", "E", "H"))
    st["ids"] = _routing(case, g)
    if op == "dispatch":
        st["x"] = torch.randn((T, H), generator=g, device="cuda").to(dt)
        return st
    if own:
        from elastikernel_b200 import _ops

        st["perm"] = _ops.moe_dispatch(None, st["ids"], E)
    else:
        st["perm"] = _plain_maps(st["ids"], E)
    st["rows"] = torch.randn((T * k, H), generator=g, device="cuda").to(dt)
    if op != "dispatch_grad":
        st["weights"] = _weights_of(case, g)
    if op == "combine_grad":
        st["d_out"] = torch.randn((T, H), generator=g, device="cuda").to(dt)
    return st


# ------------------------------------------------------------------------ plain forms
def _plain_maps(ids, E):
    T, k = ids.shape
    n = T * k
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, torch.full_like(flat, E), flat)
    order = torch.sort(key, stable=True).indices
    rank = torch.empty_like(order)
    rank[order] = torch.arange(n, device=ids.device)
    kept = key < E
    total = kept.sum()
    pos = torch.arange(n, device=ids.device)
    counts = (key[:, None] == torch.arange(E, device=ids.device)).sum(dim=0) if n * E <= 1 << 24 else \
        torch.zeros(E + 1, dtype=torch.long, device=ids.device).index_add_(0, key, torch.ones_like(key))[:E]
    return {"sorted_slots": torch.where(pos < total, order, torch.full_like(order, n)).to(torch.int32),
            "slot_rows": torch.where(kept, rank, torch.full_like(rank, -1)).to(torch.int32),
            "expert_counts": counts.to(torch.int32), "T": T, "topk": k}


def _plain_dispatch(x, ids, E):
    m = _plain_maps(ids, E)
    slots = m["sorted_slots"].long()
    live = slots < ids.numel()
    rows = torch.where(live[:, None], x[torch.where(live, slots, torch.zeros_like(slots)) // ids.shape[1]],
                       torch.zeros((), dtype=x.dtype, device=x.device))
    return rows, m["sorted_slots"], m["slot_rows"], m["expert_counts"]


def _slot_values(rows, perm):
    """Each slot's row in fp32, [T, k, H]; zero for a dropped slot."""
    r = perm["slot_rows"].long()
    v = torch.where((r >= 0)[:, None], rows[r.clamp(min=0)].float(), torch.zeros((), device=rows.device))
    return v.view(perm["T"], perm["topk"], rows.shape[1])


def _plain_combine_grad(rows, perm, weights, d_out):
    v = _slot_values(rows, perm)
    d_w = (v * d_out.float()[:, None, :]).sum(dim=2)
    slots = perm["sorted_slots"].long()
    live = slots < weights.numel()
    s = torch.where(live, slots, torch.zeros_like(slots))
    d_rows = weights.reshape(-1)[s][:, None] * d_out[s // perm["topk"]].float()
    d_rows = torch.where(live[:, None], d_rows, torch.zeros((), device=rows.device))
    return d_rows.to(rows.dtype), d_w


def _plain_route_grad(ids, w, d_w, E):
    g = w * (d_w - (w * d_w).sum(dim=1, keepdim=True))
    out = torch.zeros((ids.shape[0], E), device=w.device)
    return out.scatter_add_(1, ids.long(), g)


def _plain_weight(codes, scales, mins, K, group):
    """The fp32 weight matrix [..., N, K] that packed codes stand for."""
    q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)[..., :K].float()
    at = torch.arange(K, device=codes.device) // group
    s = scales.float()[..., at]
    return q * s + mins.float()[..., at] if mins is not None else (q - 8.0) * s


def _expert_weight(qw, e):
    """Expert e's fp32 weight; e is a one-element index tensor on the device."""
    c, s, m = (None if t is None else t.index_select(0, e)[0] for t in (qw["codes"], qw["scales"], qw["mins"]))
    return _plain_weight(c, s, m, qw["K"], qw["group"])


def _plain_moe(x, logits, qw, k):
    T, E = logits.shape
    p = (logits - logits.amax(dim=1, keepdim=True)).exp()
    p = p / p.sum(dim=1, keepdim=True)
    top, ids = torch.sort(p, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    gate = torch.zeros((T, E), device=x.device).scatter_(1, ids, top / top.sum(dim=1, keepdim=True))
    xf = x.float()
    out = torch.zeros_like(xf)
    if T * k < E:  # few slots: fetch each slot's expert
        todo = [(ids[t, j:j + 1], slice(t, t + 1), gate[t:t + 1].gather(1, ids[t:t + 1, j:j + 1]))
                for t in range(T) for j in range(k)]
    else:          # many: every expert over the whole batch, weight 0 where it was not chosen
        every = torch.arange(E, device=x.device)
        todo = [(every[e:e + 1], slice(0, T), gate[:, e:e + 1]) for e in range(E)]
    for e, rows, wt in todo:
        h1 = xf[rows] @ _expert_weight(qw["w1"], e).t()
        h3 = xf[rows] @ _expert_weight(qw["w3"], e).t()
        act = h1 / (1.0 + (-h1).exp()) * h3
        out[rows] += wt * (act @ _expert_weight(qw["w2"], e).t())
    return out.to(x.dtype)


def _run_plain(st):
    op = st["op"]
    if op == "dispatch":
        return _plain_dispatch(st["x"], st["ids"], st["case"]["E"])
    if op == "dispatch_grad":
        return _slot_values(st["rows"], st["perm"]).sum(dim=1).to(st["rows"].dtype)
    if op == "combine":
        v = _slot_values(st["rows"], st["perm"])
        return (v * st["weights"][:, :, None]).sum(dim=1).to(st["rows"].dtype)
    if op == "combine_grad":
        return _plain_combine_grad(st["rows"], st["perm"], st["weights"], st["d_out"])
    if op == "route_grad":
        return _plain_route_grad(st["ids"], st["weights"], st["d_weights"], st["case"]["E"])
    if op == "gemm_w4":
        qw = st["qw"]
        w = _plain_weight(qw["codes"], qw["scales"], qw["mins"], qw["K"], qw["group"])
        return (st["x"].float() @ w.t()).to(st["x"].dtype)
    return _plain_moe(st["x"], st["logits"], st["qw"], st["case"]["k"])


# ------------------------------------------------------------------------ the package's operators
def _run_own(st):
    from elastikernel_b200 import _ops

    op = st["op"]
    if op == "dispatch":
        p = _ops.moe_dispatch(st["x"], st["ids"], st["case"]["E"])
        return p["x_perm"], p["sorted_slots"], p["slot_rows"], p["expert_counts"]
    if op == "dispatch_grad":
        return _ops.moe_dispatch_grad(st["perm"], st["rows"])
    if op == "combine":
        return _ops.moe_combine_weighted(st["perm"], st["rows"], st["weights"])
    if op == "combine_grad":
        return _ops.moe_combine_weighted_grad(st["perm"], st["rows"], st["weights"], st["d_out"])
    if op == "route_grad":
        return _ops.moe_route_grad(st["ids"], st["weights"], st["d_weights"], st["case"]["E"])
    if op == "gemm_w4":
        return _ops.gemm_w4(st["x"], st["qw"])
    return _ops.fused_moe_w4(st["x"], st["logits"], st["qw"], st["case"]["k"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------ 64-bit values
def _exact_maps(ids, E):
    """Expert-major order by counting, on the host."""
    flat = ids.cpu().numpy().reshape(-1)
    n = flat.size
    by_expert = [np.flatnonzero(flat == e) for e in range(E)]
    order = np.concatenate(by_expert) if by_expert else np.zeros(0, np.int64)
    slots = np.full(n, n, np.int32)
    slots[:order.size] = order
    rows = np.full(n, -1, np.int32)
    rows[order] = np.arange(order.size, dtype=np.int32)
    return slots, rows, np.array([b.size for b in by_expert], np.int32)


def _to_dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _exact_w4(codes, scales, mins, K, group):
    N = codes.shape[0]
    q = torch.empty((N, codes.shape[1] * 2), dtype=torch.float64, device=codes.device)
    q[:, 0::2] = (codes % 16).double()
    q[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    w = q[:, :K]
    for gi in range(-(-K // group)):
        part = w[:, gi * group:(gi + 1) * group]
        if mins is None:
            part.sub_(8.0).mul_(scales[:, gi:gi + 1].double())
        else:
            part.mul_(scales[:, gi:gi + 1].double()).add_(mins[:, gi:gi + 1].double())
    return w


def _exact_moe(st):
    x, qw, k = st["x"].double(), st["qw"], st["case"]["k"]
    lg = st["logits"].double().cpu().numpy()
    order = np.argsort(-lg, axis=1, kind="stable")[:, :k]
    z = np.take_along_axis(lg, order, axis=1)
    z = np.exp(z - z.max(axis=1, keepdims=True))
    z /= z.sum(axis=1, keepdims=True)
    out = torch.zeros_like(x)
    for e in np.unique(order):
        t, j = np.nonzero(order == e)
        tt = _to_dev(t)

        def w(name):
            q = qw[name]
            return _exact_w4(q["codes"][e], q["scales"][e], None if q["mins"] is None else q["mins"][e], q["K"],
                             q["group"])

        a, b = x[tt] @ w("w1").T, x[tt] @ w("w3").T
        out.index_add_(0, tt, _to_dev(z[t, j])[:, None] * ((a * torch.sigmoid(a) * b) @ w("w2").T))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "gemm_w4":
        q = st["qw"]
        return st["x"].double() @ _exact_w4(q["codes"], q["scales"], q["mins"], q["K"], q["group"]).T
    if op == "moe_w4":
        return _exact_moe(st)
    if op == "route_grad":
        w, d = st["weights"].double(), st["d_weights"].double()
        k = case["k"]
        jac = torch.diag_embed(w) - w[:, :, None] * w[:, None, :]
        out = torch.zeros((case["T"], case["E"]), dtype=torch.float64, device="cuda")
        t = torch.arange(case["T"], device="cuda")
        for j in range(k):
            out[t, st["ids"][:, j].long()] += (jac[:, j, :] * d).sum(dim=1)
        return out
    T, k, E, H = (case[n] for n in ("T", "k", "E", "H"))
    slots, rowof, counts = _exact_maps(st["ids"], E)
    if op == "dispatch":
        kept = int(counts.sum())
        rows = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
        rows[:kept] = st["x"].double()[_to_dev(slots[:kept] // k).long()]
        return rows, _to_dev(slots), _to_dev(rowof), _to_dev(counts)
    y = st["rows"].double()
    out = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    d_w = torch.zeros((T, k), dtype=torch.float64, device="cuda")
    d_rows = torch.zeros_like(y)
    for j in range(k):
        r = rowof[j::k]
        t = _to_dev(np.flatnonzero(r >= 0))
        rr = _to_dev(r[r >= 0]).long()
        if op == "dispatch_grad":
            out[t] += y[rr]
            continue
        w = st["weights"][t, j].double()[:, None]
        if op == "combine":
            out[t] += w * y[rr]
            continue
        d = st["d_out"][t].double()
        d_w[t, j] = (d * y[rr]).sum(dim=1)
        d_rows[rr] = w * d
    return (d_rows, d_w) if op == "combine_grad" else out
